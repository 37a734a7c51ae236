// kv_cache.cu -- writing the step's key and value rows into the paged cache, and reading rows of
// it back.
//
// One row is one token's head_dim values of one head.  An 8-bit cache holds
//     scale = max|x| * r, r = f32(1/127),   code = x / scale rounded to nearest (ties to even)
// with the product and the quotient rounded to f32 as IEEE rounds them and codes held to [-127,
// 127], so that they do not depend on the kernel; a row of zeros has scale 0 and codes 0, and a row that
// is not finite has scale NaN, so that it reads back as NaN and is not hidden.  The scale stays in f32: 4 bytes beside 64 to 128.
// Reading back gives code * scale, rounded once to the type of the rows.
//
// Measured: 30080 tokens of 8 heads of 128 from bf16 into 8-bit pages 43 us in a graph (4.3 TB/s), 31720
// back into bf16 36 us (5.4 TB/s, 84 % of the copy rate); one token 1.8 us in a graph.
#include "kv_rows.cuh"

namespace hc {

// One group of D / 8 lanes per (token, U heads): each lane holds 8 values of each row, k and v.
// Bound by memory: every value is read once and written once.
template <class T, class C, int D, int U>
__global__ void __launch_bounds__(256) kv_append_kernel(KvDev c, KvBatchDev b, KvRows r, FastDiv by_page) {
    constexpr int GL = D / 8;
    if (kv_check_block(c, b)) return;
    const int chunks = (c.n_heads + U - 1) / U;
    const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) / GL;
    const int l = threadIdx.x & (GL - 1);
    const int t = (int)min(g / chunks, (long long)b.n_tok - 1), h0 = (int)(g % chunks) * U;
    const bool real = g < (long long)b.n_tok * chunks;
    const T* src[2] = {(const T*)r.k + t * r.ldk + l * 8, (const T*)r.v + t * r.ldv + l * 8};
    typename Elem<T>::Raw raw[2][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) raw[w][u] = Elem<T>::load8(src[w] + min(h0 + u, c.n_heads - 1) * D);
    uint32_t at = 0;
    long long sat = 0;
    int pos;
    const bool has = kv_slot<GL>(c, b, by_page, t, at, sat, pos) && real;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = h0 + u;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float x[8];
            Elem<T>::values(raw[w][u], x);
            C* dst = kv_elem<C>(w ? c.v : c.k, at + (uint32_t)h * c.head) + l * 8;
            if constexpr (sizeof(C) == 1) {
                uint32_t top = Elem<T>::top(raw[w][u]);
#pragma unroll
                for (int o = GL / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float m = __uint_as_float(top);
                const float scale = top < 0x7f800000u ? m * (1.f / 127.f) : __int_as_float(0x7fffffff);
                uint32_t q[2];
                kv_codes(x, m, scale, q);
                if (has && h < c.n_heads) {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(q[0], q[1]);
                    if (l == 0) (w ? c.vs : c.ks)[sat + (long long)h * c.page_size] = scale;
                }
            } else {
                if (has && h < c.n_heads) Elem<C>::store8(dst, x);
            }
        }
    }
}

template <class T, class C, int D, int U>
__global__ void __launch_bounds__(256) kv_read_kernel(KvDev c, KvBatchDev b, KvRows r, FastDiv by_page) {
    constexpr int GL = D / 8;
    if (kv_check_block(c, b)) return;
    const int chunks = (c.n_heads + U - 1) / U;
    const long long g = ((long long)blockIdx.x * 256 + threadIdx.x) / GL;
    const int l = threadIdx.x & (GL - 1);
    const int t = (int)min(g / chunks, (long long)b.n_tok - 1), h0 = (int)(g % chunks) * U;
    uint32_t at = 0;
    long long sat = 0;
    int pos;
    if (!kv_slot<GL>(c, b, by_page, t, at, sat, pos) || g >= (long long)b.n_tok * chunks) return;
    typename Elem<C>::Raw raw[2][U];
    float sc[2][U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int h = min(h0 + u, c.n_heads - 1);
            raw[w][u] = Elem<C>::load8(kv_elem<C>(w ? c.v : c.k, at + (uint32_t)h * c.head) + l * 8);
            if constexpr (sizeof(C) == 1) sc[w][u] = __ldg((w ? c.vs : c.ks) + sat + (long long)h * c.page_size);
        }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if (h0 + u >= c.n_heads) continue;
            float x[8];
            Elem<C>::values(raw[w][u], x);
            if constexpr (sizeof(C) == 1)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= sc[w][u];
            Elem<T>::store8((T*)(w ? r.v : r.k) + t * (w ? r.ldv : r.ldk) + (h0 + u) * D + l * 8, x);
        }
}

namespace {

template <class T, class C, int D, int U>
cudaError_t start(bool write, const KvDev& c, const KvBatchDev& b, const KvRows& r, cudaStream_t s) {
    const long long groups = (long long)b.n_tok * ((c.n_heads + U - 1) / U);
    const unsigned grid = (unsigned)((groups * (D / 8) + 255) / 256) + 1;  // and kv_check_block's
    const FastDiv by_page((uint32_t)c.page_size);
    if (write)
        kv_append_kernel<T, C, D, U><<<grid, 256, 0, s>>>(c, b, r, by_page);
    else
        kv_read_kernel<T, C, D, U><<<grid, 256, 0, s>>>(c, b, r, by_page);
    return cudaGetLastError();
}

// A thread's rows: one where all rows fit the GPU's threads at once (the call's time is its chain of
// loads), two (f32) or four where they do not (the chain is paid once for more bytes on their way).
template <class T, class C, int D>
cudaError_t launch(bool write, const KvDev& c, const KvBatchDev& b, const KvRows& r, cudaStream_t s) {
    if ((long long)b.n_tok * c.n_heads * (D / 8) <= 148 * 2048) return start<T, C, D, 1>(write, c, b, r, s);
    return start<T, C, D, sizeof(T) == 4 ? 2 : 4>(write, c, b, r, s);
}

template <class T, int D>
cudaError_t by_cache(bool write, int ct, const KvDev& c, const KvBatchDev& b, const KvRows& r, cudaStream_t s) {
    if (ct == T_F16) return launch<T, __half, D>(write, c, b, r, s);
    if (ct == T_BF16) return launch<T, __nv_bfloat16, D>(write, c, b, r, s);
    return launch<T, int8_t, D>(write, c, b, r, s);
}

template <int D>
cudaError_t by_type(bool write, int ct, int dt, const KvDev& c, const KvBatchDev& b, const KvRows& r, cudaStream_t s) {
    if (dt == T_F32) return by_cache<float, D>(write, ct, c, b, r, s);
    if (dt == T_F16) return by_cache<__half, D>(write, ct, c, b, r, s);
    return by_cache<__nv_bfloat16, D>(write, ct, c, b, r, s);
}

}  // namespace

cudaError_t launch_kv_append(int ct, int dt, int head_dim, const KvDev& c, const KvBatchDev& b, const KvRows& r,
                             cudaStream_t s) {
    return head_dim == 64 ? by_type<64>(true, ct, dt, c, b, r, s) : by_type<128>(true, ct, dt, c, b, r, s);
}
cudaError_t launch_kv_read(int ct, int dt, int head_dim, const KvDev& c, const KvBatchDev& b, const KvRows& r,
                           cudaStream_t s) {
    return head_dim == 64 ? by_type<64>(false, ct, dt, c, b, r, s) : by_type<128>(false, ct, dt, c, b, r, s);
}

}  // namespace hc
