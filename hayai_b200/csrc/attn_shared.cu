// attn_shared.cu -- attention of groups of sequences whose first tokens are the same pages: what has to
// be known of the groups before the attention's kernels run, and the joining after them.
//
// A group's rows see its prefix whole, so that the prefix is one more sequence, of all the group's new tokens and
// not causal: its keys are read once for the group, and its rows fill the tensor cores' tiles.  One call is
//     attn_groups    what every group shares for this step, and its tiles
//     attn_prefix    prefixes of more than a few rows per kv head (attn_prefix.cu), in pieces
//     attn_few       prefixes of few rows, one result each
//     attn_many/few  what every sequence has behind its prefix (AttnArgs::first)
//     attn_join      out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over a row's parts
#include "attn_rows.cuh"
#include "block_scan.cuh"

namespace hc {

namespace {

constexpr int kTileRows = 256, kUnit = 128, kOver = 2;

// A warp per group: how many tokens its sequences share for this step.  All new tokens have to see them all, so that
// they are at most the tokens that every sequence had before; a group of one sequence shares nothing.  Then the
// groups' tiles, in a line whose places the blocks of attn_prefix.cu share equally.
__global__ void __launch_bounds__(1024) attn_groups_kernel(KvBatchDev b, KvSharedDev g, int cap) {
    __shared__ long long scratch[33];
    __shared__ int len_s[HC_KV_SEQS], tok_s[HC_KV_SEQS], tile_s[HC_KV_SEQS + 1], place_s[HC_KV_SEQS];
    const int tid = threadIdx.x, ln = lane_id(), group = g.heads / g.kv_heads;
    let_next_start();
    int *const from_s = tile_s, *const to_s = place_s;  // the groups' sequences, until their tiles are counted
    __shared__ unsigned long long saved_s;
    if (tid == 0) saved_s = 0;
    for (int s = tid; s < b.n_seq; s += 1024) g.first[s] = 0;
    __syncthreads();
    for (int i = tid >> 5; i < g.n; i += 32) {
        const int a0 = __ldg(g.seq_start + i), a1 = __ldg(g.seq_start + i + 1), given = __ldg(g.length + i);
        const int s0 = min(max(a0, 0), b.n_seq), s1 = min(max(a1, s0), b.n_seq);
        int most = min(max(given, 0), cap), seqs = 0;
        if (s0 != a0 || s1 != a1 || most != given)
            if (ln == 0) atomicOr(b.err, kErrKvRange);
        for (int s = s0 + ln; s < s1; s += 32) {
            const KvSeq q = kv_seq(b, cap, s);
            if (q.q1 == q.q0) continue;
            ++seqs;
            most = min(most, q.len - (q.q1 - q.q0));
        }
        most = max(__reduce_min_sync(0xffffffffu, most), 0);
        seqs = __reduce_add_sync(0xffffffffu, seqs);
        if (seqs < 2) most = 0;
        if (ln == 0) {
            len_s[i] = most;
            from_s[i] = s0;
            to_s[i] = s1;
            atomicAdd(&saved_s, (unsigned long long)most * max(seqs - 1, 0));
        }
    }
    __syncthreads();
    const bool worth = saved_s >= (unsigned long long)g.least;
    for (int i = tid >> 5; i < g.n; i += 32) {
        const int s0 = from_s[i], s1 = to_s[i], most = worth ? len_s[i] : 0;
        for (int s = s0 + ln; s < s1; s += 32) g.first[s] = most;
        __syncwarp();
        if (ln == 0) {
            // its new tokens' rows, cut as kv_seq cuts them
            const int q0 = min(max(__ldg(b.q_start + s0), 0), b.n_tok), q1 = min(max(__ldg(b.q_start + s1), q0), b.n_tok);
            const int tok = most ? q1 - q0 : 0;
            len_s[i] = most;
            tok_s[i] = tok;
            const bool few = (long long)tok * group <= g.few_rows;
            g.q_start[i] = q0;
            if (i == g.n - 1) g.q_start[g.n] = q1;
            g.len[i] = few ? most : 0;
            g.row[i] = min(s0, b.n_seq - 1);
        }
    }
    __syncthreads();
    // ---- tiles and places of every group
    auto units_of = [&](int i) { return (len_s[i] + kUnit - 1) / kUnit; };
    long long tiles[2] = {0, 0}, places[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        if (i >= g.n || tok_s[i] == 0) continue;
        const long long r = (long long)tok_s[i] * group, n = (r + kTileRows - 1) / kTileRows;
        tiles[e] = n * g.kv_heads;
        const bool narrow = r - (n - 1) * kTileRows <= kTileRows / 2;
        if (r > g.few_rows) places[e] = (n * (2ll * units_of(i) + kOver) - (narrow ? units_of(i) : 0)) * g.kv_heads;
    }
    long long all_tiles, U;
    long long at = block_scan(tiles[0] + tiles[1], scratch, all_tiles);
    long long pl = block_scan(places[0] + places[1], scratch, U);
    const bool fits = all_tiles <= g.max_tiles && U < 0x7fffffff;
    if (!fits && tid == 0) atomicOr(b.err, kErrKvRange);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int i = 2 * tid + e;
        if (i < g.n && fits) tile_s[i] = (int)at, place_s[i] = (int)pl;
        at += tiles[e];
        pl += places[e];
    }
    const int n_tiles = fits ? (int)all_tiles : 0;
    const int G = fits ? max(1, min(g.blocks, (int)U / 4)) : 1;  // shares of four places and more: every one has a unit
    __syncthreads();
    const AttnShares share(max((int)(fits ? U : 0), 1), G);
    long long rows_before = 0;
    for (int t0 = 0; t0 < n_tiles; t0 += 1024) {
        const int t = t0 + tid;
        PrefixTile x{};
        long long rows = 0;
        if (t < n_tiles) {
            int lo = 0, hi = g.n - 1;  // the last group whose tiles start at or before t, of those at one place the last
            while (lo < hi) {
                const int m = (lo + hi + 1) >> 1;
                if (tile_s[m] <= t) lo = m;
                else hi = m - 1;
            }
            const int r = tok_s[lo] * group, per = (r + kTileRows - 1) / kTileRows, local = t - tile_s[lo];
            const int units = units_of(lo), rest = r - (per - 1) * kTileRows;
            const bool few = r <= g.few_rows, narrow = rest <= kTileRows / 2;
            x.hk = local / per;
            const int k = local - x.hk * per;
            x.r0 = k * kTileRows;
            x.nr = k == per - 1 ? rest : kTileRows;
            x.q0 = g.q_start[lo];
            x.len = len_s[lo];
            x.row = g.row[lo];
            x.cost = k == per - 1 && narrow ? 1 : 2;
            x.place = place_s[lo];
            if (!few) {
                x.units = units;
                x.place += x.hk * (per * (2 * units + kOver) - (narrow ? units : 0)) + k * (2 * units + kOver);
                x.c0 = share.owner(x.place);
                x.pieces = (share.owner(x.place + x.cost * (units - 1)) - x.c0 + 1) * (x.cost == 1 ? 2 : 1);
                rows = (long long)x.pieces * x.nr;
                const int end = x.place + x.cost * units + kOver;
                for (int c = x.place ? share.owner(x.place - 1) + 1 : 0; c < G && share.begin(c) < end; ++c) g.first_tile[c] = t;
            }
        }
        long long total;
        x.piece = (int)(rows_before + block_scan(rows, scratch, total));
        rows_before += total;
        if (t < n_tiles) g.tiles[t] = x;
    }
    // groups that overlap (offsets that do not ascend) may want more room than any others: nothing is made of them
    const bool room = rows_before <= g.max_pieces;
    if (tid == 0) {
        if (!room) atomicOr(b.err, kErrKvRange);
        g.line[kLineTiles] = room ? n_tiles : 0;
        g.line[kLinePlaces] = fits && room ? (int)U : 0;
        g.line[kLineBlocks] = G;
    }
}

// A warp per row of a tile, eight rows of one at a time.  Bound by memory and its latency: a row's parts are asked for
// together, before the weights that they count with are there.
template <class T, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnArgs a, PrefixArgs p) {
    constexpr int RUNS = kTileRows / 8, U = 8;
    after_previous();
    const int n_tiles = __ldcg(p.line + kLineTiles), ln = lane_id();
    const bool mine = ln < D / 4;
    for (int w = blockIdx.x; w < n_tiles * RUNS; w += gridDim.x) {
        const int4* const xt = reinterpret_cast<const int4*>(p.tiles + w / RUNS);
        PrefixTile x;
        reinterpret_cast<int4*>(&x)[0] = __ldcg(xt);
        reinterpret_cast<int4*>(&x)[1] = __ldcg(xt + 1);
        reinterpret_cast<int4*>(&x)[2] = __ldcg(xt + 2);
        const int r = w % RUNS * 8 + (threadIdx.x >> 5);
        if (r >= x.nr) continue;
        const int row = x.r0 + r, t = a.by_group(row);
        const long long at = (long long)(x.q0 + t) * a.heads + x.hk * a.group + row - t * a.group;
        // the parts: what is behind the prefix (divided by its sum), then the prefix's pieces, or its one result
        const int n = x.pieces;
        const size_t step = n ? x.nr : 0;
        const float4* const o = reinterpret_cast<const float4*>(n ? p.part + ((size_t)x.piece + r) * D : p.few + at * D) + ln;
        const float2* const ml = reinterpret_cast<const float2*>(p.part_ml) + x.piece + r;
        float4 y0 = make_float4(0.f, 0.f, 0.f, 0.f), y[U];
        if (mine) y0 = __ldcg(reinterpret_cast<const float4*>(a.base + at * D) + ln);
        const float own = __ldcg(a.base_lse + at);
        float2 v = make_float2(-INFINITY, 0.f);
        if (n) {
            if (ln < n) v = __ldcg(ml + ln * step);
        } else if (ln == 0) {
            const float e = __ldcg(p.few_lse + at);
            v = make_float2(e, e == -INFINITY ? 0.f : 1.f);
        }
        const int parts = max(n, 1);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (mine && k < parts) y[k] = __ldcg(o + k * step * (D / 4));
        }
        AttnJoin j;
        auto ml_of = [&](int i) { return i < 32 ? v : __ldcg(ml + i * step); };  // a lane asks for its own part of a run of 32
        auto o_of = [&](int i) {
            if (i >= U) return __ldcg(o + i * step * (D / 4));
            float4 z = y[0];
#pragma unroll
            for (int k = 1; k < U; ++k)
                if (i == k) z = y[k];
            return z;
        };
        j.join(1, mine, [&](int) { return make_float2(own, own == -INFINITY ? 0.f : 1.f); }, [&](int) { return y0; });
        j.join(parts, mine, ml_of, o_of);
        if (mine) attn_store<T>(a, x.q0, x.hk, row, D, 4 * ln, j.y, j.l, false);
        if (ln == 0) attn_store_lse(a, x.q0, x.hk, row, j.m, j.l, false);
    }
}

template <class T>
cudaError_t join(int head_dim, const AttnArgs& a, const PrefixArgs& p, int sms, cudaStream_t s) {
    return launch_early(head_dim == 64 ? attn_join_kernel<T, 64> : attn_join_kernel<T, 128>, sms * 8, 256, 0, s, a, p);
}

}  // namespace

cudaError_t launch_attn_groups(const KvBatchDev& b, const KvSharedDev& g, int cap, cudaStream_t s) {
    attn_groups_kernel<<<1, 1024, 0, s>>>(b, g, cap);
    return cudaGetLastError();
}

cudaError_t launch_attn_join(int dtype, int head_dim, const AttnArgs& a, const PrefixArgs& p, int sms, cudaStream_t s) {
    if (dtype == T_F32) return join<float>(head_dim, a, p, sms, s);
    if (dtype == T_F16) return join<__half>(head_dim, a, p, sms, s);
    return join<__nv_bfloat16>(head_dim, a, p, sms, s);
}

}  // namespace hc
