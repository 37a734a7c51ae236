// attn_shared.cu -- attention of groups of sequences whose first tokens are the same pages: what has to
// be known of the groups before the attention's kernels run.
//
// A group's rows see its prefix whole, so that the prefix is one more sequence, of all the group's new
// tokens and not causal: its keys are read once for the group, and its rows fill the tensor cores' tiles.  The
// kernels of the paged attention run twice: over the groups' prefixes, where results and log 2 of the weights'
// sums stay in 32 bits (AttnArgs::base), and over what every sequence has behind its prefix (AttnArgs::first), where
//     out = (l_own 2^m_own out_own + 2^lse_pre out_pre) / (l_own 2^m_own + 2^lse_pre)
// is formed as a row is written.
#include "kv_launch.h"

namespace hc {

namespace {

// A warp per group: how many tokens its sequences share for this step.  All new tokens have to see them all, so that
// they are at most the tokens that every sequence had before; a group of one sequence shares nothing.
__global__ void __launch_bounds__(1024) attn_groups_kernel(KvBatchDev b, KvSharedDev g, int cap) {
    for (int s = threadIdx.x; s < b.n_seq; s += 1024) g.first[s] = 0;
    __syncthreads();
    const int ln = lane_id();
    for (int i = threadIdx.x >> 5; i < g.n; i += 32) {
        const int a0 = __ldg(g.seq_start + i), a1 = __ldg(g.seq_start + i + 1), given = __ldg(g.length + i);
        const int s0 = min(max(a0, 0), b.n_seq), s1 = min(max(a1, s0), b.n_seq);
        int most = min(max(given, 0), cap), rows = 0;
        if (s0 != a0 || s1 != a1 || most != given)
            if (ln == 0) atomicOr(b.err, kErrKvRange);
        for (int s = s0 + ln; s < s1; s += 32) {
            const KvSeq q = kv_seq(b, cap, s);
            if (q.q1 == q.q0) continue;
            ++rows;
            most = min(most, q.len - (q.q1 - q.q0));
        }
        most = max(__reduce_min_sync(0xffffffffu, most), 0);
        if (__reduce_add_sync(0xffffffffu, rows) < 2) most = 0;
        for (int s = s0 + ln; s < s1; s += 32) g.first[s] = most;
        if (ln == 0) {
            // offsets of the groups' new tokens: those of their first sequences (cut as kv_seq cuts them)
            g.q_start[i] = s0 < b.n_seq ? __ldg(b.q_start + s0) : __ldg(b.q_start + b.n_seq);
            if (i == g.n - 1) g.q_start[g.n] = __ldg(b.q_start + s1);
            g.len[i] = most;
            g.row[i] = min(s0, b.n_seq - 1);
        }
    }
}

}  // namespace

cudaError_t launch_attn_groups(const KvBatchDev& b, const KvSharedDev& g, int cap, cudaStream_t s) {
    attn_groups_kernel<<<1, 1024, 0, s>>>(b, g, cap);
    return cudaGetLastError();
}

}  // namespace hc
