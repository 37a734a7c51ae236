// attn_paged.cu -- attention of a batch's new tokens over the paged key/value cache.
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
// over the positions j that token i sees, m_i the largest score; lse_i = m_i + log sum_j p_ij.
// One block per (token, query head): a pass over the visible positions in tiles of 128 with the
// running maximum and sum.
#include <math.h>

#include "kv_launch.h"

namespace hc {

template <class T, class C, int D>
__global__ void __launch_bounds__(128) attn_simple_kernel(AttnArgs a) {
    __shared__ float q[D], p[128], red[4];
    __shared__ long long row[128];
    const int t = blockIdx.x, h = blockIdx.y, hk = h / a.group, tid = threadIdx.x;
    const int s = kv_find_seq<32>(a.b, t);
    if (s < 0) return;
    const KvSeq sq = kv_seq(a.b, a.b.max_pages * a.c.page_size, s);
    const int pos = sq.len - sq.q1 + t;
    if (tid < D / 8) {
        float x[8];
        Elem<T>::load8((const T*)a.q + t * a.ldq + h * D + tid * 8, x);
        for (int i = 0; i < 8; ++i) q[tid * 8 + i] = x[i];
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    const int end = a.causal ? min(sq.len, pos + 1) : sq.len;
    for (int j0 = 0; j0 < end; j0 += 128) {
        const int j = j0 + tid;
        bool see = j < end && (!a.window || pos - j < a.window || j < a.sink);
        float sc = -INFINITY, vs = 1.f;
        long long at = 0;
        if (see) {
            const int pg = j / a.c.page_size, r = j - pg * a.c.page_size;
            const int page = __ldg(a.b.table + s * a.b.table_stride + pg);
            if ((unsigned)page >= (unsigned)a.c.n_pages) {
                atomicOr(a.b.err, kErrKvRange);
                see = false;
            } else {
                at = 64ll * ((long long)page * a.c.page + (long long)r * a.c.row + (long long)hk * a.c.head);
                const C* k = (const C*)(a.c.k + at);
                float d = 0.f;
                for (int i = 0; i < D; i += 8) {
                    float x[8];
                    Elem<C>::load8(k + i, x);
                    for (int e = 0; e < 8; ++e) d += q[i + e] * x[e];
                }
                if (sizeof(C) == 1) {
                    const long long sat = page * a.c.spage + (long long)hk * a.c.page_size + r;
                    d *= a.c.ks[sat];
                    vs = a.c.vs[sat];
                }
                sc = d * a.scale;
            }
        }
        row[tid] = see ? at : -1;
        float mx = sc;
        for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, w));
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = mx;
        __syncthreads();
        const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float e = see ? expf(sc - base) : 0.f;
        p[tid] = e * vs;
        float sum = e;
        for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(~0u, sum, w);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = sum;
        __syncthreads();
        const float f = expf(m - base);
        l = l * f + red[0] + red[1] + red[2] + red[3];
        o *= f;
        m = mn;
        if (tid < D)
            for (int k = 0; k < 128; ++k)
                if (row[k] >= 0) {
                    const C x = ((const C*)(a.c.v + row[k]))[tid];
                    o += p[k] * (float)x;
                }
        __syncthreads();
    }
    if (tid < D) ((T*)a.out)[t * a.ldo + h * D + tid] = (T)(l == 0.f ? 0.f : o / l);
    if (tid == 0 && a.lse) a.lse[(long long)t * a.heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

namespace {

template <class T, class C>
cudaError_t launch(int D, const AttnArgs& a, cudaStream_t s) {
    const dim3 grid(a.b.n_tok, a.heads);
    if (D == 64)
        attn_simple_kernel<T, C, 64><<<grid, 128, 0, s>>>(a);
    else
        attn_simple_kernel<T, C, 128><<<grid, 128, 0, s>>>(a);
    return cudaGetLastError();
}

template <class T>
cudaError_t by_cache(int ct, int D, const AttnArgs& a, cudaStream_t s) {
    if (ct == T_F16) return launch<T, __half>(D, a, s);
    if (ct == T_BF16) return launch<T, __nv_bfloat16>(D, a, s);
    return launch<T, int8_t>(D, a, s);
}

}  // namespace

cudaError_t launch_attn_paged(int ct, int dt, int D, const AttnArgs& a, cudaStream_t s) {
    if (dt == T_F32) return by_cache<float>(ct, D, a, s);
    if (dt == T_F16) return by_cache<__half>(ct, D, a, s);
    return by_cache<__nv_bfloat16>(ct, D, a, s);
}

}  // namespace hc
