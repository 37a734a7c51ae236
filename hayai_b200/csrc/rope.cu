// rope.cu -- rotary positions: rows of queries or keys turned by their tokens' positions, alone
// (hc_rope_dev) or together with the step's rows going into the paged cache (hc_kv_append_rope_dev).
//
//     (a, b) -> (a c - b s, a s + b c),   c + i s = amplitude * exp(i pos t_j)
// for the pairs j of a head's first rot values: (j, j + rot/2), or (2 j, 2 j + 1).
//
// Angles.  A position times a frequency in f32 is off by whole radians far out (2^20 * 2^-24).  The
// frequencies are kept in turns as 64-bit fixed point fractions instead, whose product with a whole
// position wraps at whole turns by itself: three integer instructions leave the angle to 2^-32 of a
// turn for every position of 32 bits, and sincospi takes it from there, rounded to 24 bits: off by 2^-25 of
// half a turn at most, as much as cos and sin are rounded by themselves.  A position's angles are made once
// per block and token, and serve all heads.
//
// Bound by memory: a row is read once and written once.  A lane holds two chunks of 8 values, in the half layout
// the two partners, so that nothing is exchanged between lanes but an 8-bit row's largest value.
//
// Measured: 9000 tokens of 32 bf16 heads of 128 26 us (5.6 TB/s, 86 % of the copy rate); 15947 tokens of prompts, 32
// query heads turned and 8 kv heads turned and stored in 8 bits, 82 us (4.4 TB/s), one token 3.6 us in a graph.
// The same prompts into bf16 pages 72 us (5.5 TB/s), f32 rows into f16 pages 119 (6.0); 64 and 256 single tokens 4.0 and 4.4
// us, into 8-bit pages 4.3 and 4.8.  Rows at odd addresses, and heads turned in part that is no whole number of chunks, go a
// value at a time (rope_any_kernel): 9000 tokens of 32 bf16 heads of 128 61 us, of 80 with 20 turned 51, one token 3.9.
// In blocks of one round, each of which finds its tokens' places for itself, the prompts took 139 us; in 8 rounds 82, in 32
// 92.  Queries, keys and values in loops of their own (a row's quantising for queries as well: 151 us).
#include <type_traits>

#include "kv_rows.cuh"

namespace hc {

namespace {

constexpr int kThreads = 256, kRounds = 8;

// cos and sin of pair j at a position, times the amplitude.
__device__ __forceinline__ float2 rope_angle(const RopeDev& r, int j, int pos) {
    const uint64_t turn = r.turns[j] * (uint64_t)(int64_t)pos;
    float s, c;
    sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
    return make_float2(c * r.amplitude, s * r.amplitude);
}

// A lane's two chunks of a row of D values (lane l of D / 16) and how they turn.
struct RopeLane {
    int c0, c1;    // first values of the chunks
    bool t0, t1;   // the chunk is turned
    int j0, j1;    // the pair of the chunk's first angle (half layout: both chunks have the same eight)
    __device__ __forceinline__ RopeLane(const RopeDev& r, int l) {
        if (r.pairs) {
            c0 = 16 * l, c1 = 16 * l + 8;
            t0 = c0 < r.rot, t1 = c1 < r.rot;
            j0 = c0 / 2, j1 = c1 / 2;
        } else {
            t0 = t1 = 16 * l < r.rot;
            c0 = t0 ? 8 * l : 16 * l;
            c1 = t0 ? r.rot / 2 + 8 * l : 16 * l + 8;
            j0 = 8 * l, j1 = 8 * l + 4;
        }
    }
    // The lane's 8 angles, of a position's rot / 2 in shared memory.
    __device__ __forceinline__ void angles(const float2* at, float2 (&cs)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t0) cs[i] = at[j0 + i];
            if (t1) cs[4 + i] = at[j1 + i];
        }
    }
    __device__ __forceinline__ void turn(bool pairs, const float2 (&cs)[8], float (&a)[8], float (&b)[8]) const {
        auto one = [](const float2& c, float& x, float& y) {
            const float u = x, v = y;
            x = fmaf(u, c.x, -(v * c.y));
            y = fmaf(u, c.y, v * c.x);
        };
        if (pairs) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (t0) one(cs[i], a[2 * i], a[2 * i + 1]);
                if (t1) one(cs[4 + i], b[2 * i], b[2 * i + 1]);
            }
        } else if (t0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) one(cs[i], a[i], b[i]);
        }
    }
};

// Rows by given positions: a block takes `tokens` of them, a lane the same two chunks of U heads.
template <class T, int U>
__global__ void __launch_bounds__(kThreads) rope_rows_kernel(const __grid_constant__ RopeDev r, const int* __restrict__ pos,
                                                             const T* x, long long ldx, T* out, long long ldo, int n_tok,
                                                             int heads, int tokens) {
    extern __shared__ float2 cs_s[];
    const int half = r.rot / 2, lanes = r.dim / 16, hc = (heads + U - 1) / U, t0 = blockIdx.x * tokens;
    const int n = min(tokens, n_tok - t0);
    for (int i = threadIdx.x; i < n * half; i += kThreads) {
        const int t = i / half, j = i - t * half;
        cs_s[i] = rope_angle(r, j, __ldg(pos + t0 + t));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * hc * lanes; i += kThreads) {
        const int g = i / lanes, t = g / hc, h0 = (g - t * hc) * U;
        const RopeLane ln(r, i - g * lanes);
        const T* const src = x + (t0 + t) * ldx + (long long)h0 * r.dim;
        T* const dst = out + (t0 + t) * ldo + (long long)h0 * r.dim;
        typename Elem<T>::Raw raw[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long o = (long long)min(u, heads - 1 - h0) * r.dim;
            raw[u][0] = Elem<T>::load8_own(src + o + ln.c0);
            raw[u][1] = Elem<T>::load8_own(src + o + ln.c1);
        }
        float2 cs[8];
        ln.angles(cs_s + t * half, cs);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h0 + u >= heads) break;
            float a[8], b[8];
            Elem<T>::values(raw[u][0], a);
            Elem<T>::values(raw[u][1], b);
            ln.turn(r.pairs, cs, a, b);
            Elem<T>::store8(dst + u * r.dim + ln.c0, a);
            Elem<T>::store8(dst + u * r.dim + ln.c1, b);
        }
    }
}

template <class T>
__device__ __forceinline__ float rope_value(T x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same_v<T, __half>)
        return __half2float(x);
    else
        return __bfloat162float(x);
}
template <class T>
__device__ __forceinline__ T rope_rounded(float x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same_v<T, __half>)
        return __float2half_rn(x);
    else
        return __float2bfloat16_rn(x);
}

// The same for sizes, strides or addresses that do not come in 16 bytes: a thread per pair, or per value
// that is not turned, over up to 8 heads.
template <class T>
__global__ void __launch_bounds__(kThreads) rope_any_kernel(const __grid_constant__ RopeDev r, const int* __restrict__ pos,
                                                            const T* x, long long ldx, T* out, long long ldo, int n_tok,
                                                            int heads) {
    constexpr int U = 8;
    const int half = r.rot / 2, places = r.dim - half, hc = (heads + U - 1) / U;
    const long long i = (long long)blockIdx.x * kThreads + threadIdx.x;
    const long long t = i / ((long long)places * hc);
    if (t >= n_tok) return;
    const int rest = (int)(i - t * places * hc), h0 = rest / places * U, p = rest % places;
    const bool turned = p < half;
    const int ia = !turned ? p + half : r.pairs ? 2 * p : p, ib = !turned ? ia : r.pairs ? 2 * p + 1 : p + half;
    const float2 cs = turned ? rope_angle(r, p, __ldg(pos + t)) : make_float2(1.f, 0.f);
    for (int h = h0; h < min(h0 + U, heads); ++h) {
        const T* const src = x + t * ldx + (long long)h * r.dim;
        T* const dst = out + t * ldo + (long long)h * r.dim;
        if (turned) {
            const float a = rope_value<T>(src[ia]), b = rope_value<T>(src[ib]);
            dst[ia] = rope_rounded<T>(fmaf(a, cs.x, -(b * cs.y)));
            dst[ib] = rope_rounded<T>(fmaf(a, cs.y, b * cs.x));
        } else {
            dst[ia] = src[ia];
        }
    }
}

// A step's rows by their positions in the cache: a group of D / 16 lanes per (token, U rows), the rows being U of the
// token's query heads, of its key heads or of its value heads.
template <class T, class C, int D, int U>
__global__ void __launch_bounds__(kThreads) kv_append_rope_kernel(const __grid_constant__ RopeDev r, KvDev c, KvBatchDev b,
                                                                  RopeAppend a, FastDiv by_page, int tokens) {
    constexpr int GL = D / 16, GROUPS = kThreads / GL;
    using Raw = typename Elem<T>::Raw;
    extern __shared__ float2 cs_s[];
    __shared__ uint32_t at_s[32];
    __shared__ long long sat_s[32];
    __shared__ int pos_s[32], has_s[32];
    if (kv_check_block(c, b)) return;
    const int half = r.rot / 2, nq = (a.heads + U - 1) / U, nk = (c.n_heads + U - 1) / U, hc = nq + 2 * nk;
    const int t0 = blockIdx.x * tokens, n = min(tokens, b.n_tok - t0), l = threadIdx.x & (GL - 1), group = threadIdx.x / GL;
    const RopeLane ln(r, l);
    // An item's rows: what they are (0 queries, 1 keys, 2 values), the first head, and how many there are.
    struct Item {
        int t, what, h0, rows;
    };
    auto item_of = [&](int i) {
        Item x;
        x.t = i / hc;
        const int k = i - x.t * hc;
        x.what = (k >= nq) + (k >= nq + nk);
        x.h0 = (k - (x.what == 0 ? 0 : x.what == 1 ? nq : nq + nk)) * U;
        x.rows = min(U, (x.what ? c.n_heads : a.heads) - x.h0);
        return x;
    };
    auto load = [&](const Item& x, Raw (&raw)[U][2]) {
        const T* const src = (x.what == 0   ? (const T*)a.q + (t0 + x.t) * a.ldq
                              : x.what == 1 ? (const T*)a.k + (t0 + x.t) * a.ldk
                                            : (const T*)a.v + (t0 + x.t) * a.ldv) + (long long)x.h0 * D;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int o = min(u, x.rows - 1) * D;
            raw[u][0] = Elem<T>::load8_own(src + o + ln.c0);
            raw[u][1] = Elem<T>::load8_own(src + o + ln.c1);
        }
    };
    Raw raw[U][2];
    Item x = item_of(min(group, n * hc - 1));
    load(x, raw);  // on their way while the tokens' places and angles are found
    {
        // eight lanes to a token, whatever D is: at most 32 tokens
        const int t = threadIdx.x >> 3;
        uint32_t at = 0;
        long long sat = 0;
        int pos = -1;
        const bool has = kv_slot<8>(c, b, by_page, t0 + min(t, n - 1), at, sat, pos);
        if (t < n && (threadIdx.x & 7) == 0) at_s[t] = at, sat_s[t] = sat, pos_s[t] = pos, has_s[t] = has;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * half; i += kThreads) {
        const int t = i / half;
        cs_s[i] = rope_angle(r, i - t * half, pos_s[t]);
    }
    __syncthreads();
    const uint32_t lanes = ((1u << GL) - 1) << (threadIdx.x & 31 & ~(GL - 1));  // the group's, which exchange below
#pragma unroll 1
    for (int i = group; i < n * hc; i += GROUPS) {
        if (i >= GROUPS) {
            x = item_of(i);
            load(x, raw);
        }
        if (x.what == 0) {
            if (pos_s[x.t] < 0) continue;
            float2 cs[8];
            ln.angles(cs_s + x.t * half, cs);
            T* const dst = (T*)a.q_out + (t0 + x.t) * a.ldqo + (long long)x.h0 * D;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u >= x.rows) break;
                float p[8], q[8];
                Elem<T>::values(raw[u][0], p);
                Elem<T>::values(raw[u][1], q);
                ln.turn(r.pairs, cs, p, q);
                Elem<T>::store8(dst + u * D + ln.c0, p);
                Elem<T>::store8(dst + u * D + ln.c1, q);
            }
            continue;
        }
        if (!has_s[x.t]) continue;
        const bool v = x.what == 2;
        uint8_t* const pool = v ? c.v : c.k;
        const uint32_t at = at_s[x.t] + (uint32_t)x.h0 * c.head;
        float2 cs[8];
        if (!v) ln.angles(cs_s + x.t * half, cs);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= x.rows) break;
            float p[8], q[8];
            Elem<T>::values(raw[u][0], p);
            Elem<T>::values(raw[u][1], q);
            if (!v) ln.turn(r.pairs, cs, p, q);
            C* const dst = kv_elem<C>(pool, at + (uint32_t)u * c.head);
            if constexpr (sizeof(C) == 1) {
                // as bits, whose order is that of the sizes, infinity and NaN above all
                uint32_t top = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    top = max(top, max(__float_as_uint(p[k]) & 0x7fffffffu, __float_as_uint(q[k]) & 0x7fffffffu));
#pragma unroll
                for (int o = GL / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(lanes, top, o));
                const float m = __uint_as_float(top);
                const float scale = top < 0x7f800000u ? m * (1.f / 127.f) : __int_as_float(0x7fffffff);
                uint32_t e[2], f[2];
                kv_codes(p, m, scale, e);
                kv_codes(q, m, scale, f);
                *reinterpret_cast<uint2*>(dst + ln.c0) = make_uint2(e[0], e[1]);
                *reinterpret_cast<uint2*>(dst + ln.c1) = make_uint2(f[0], f[1]);
                if (l == 0) (v ? c.vs : c.ks)[sat_s[x.t] + (long long)(x.h0 + u) * c.page_size] = scale;
            } else {
                Elem<C>::store8(dst + ln.c0, p);
                Elem<C>::store8(dst + ln.c1, q);
            }
        }
    }
}

template <class T, int U>
cudaError_t rows(const RopeDev& r, const RopeRows& a, cudaStream_t s) {
    const int per = (a.heads + U - 1) / U * (r.dim / 16);  // threads of a token
    const int tokens = max(1, kThreads / per);
    rope_rows_kernel<T, U><<<(unsigned)((a.n_tok + tokens - 1) / tokens), kThreads, (size_t)tokens * r.rot * 4, s>>>(
        r, a.pos, (const T*)a.x, a.ldx, (T*)a.out, a.ldo, a.n_tok, a.heads, tokens);
    return cudaGetLastError();
}

template <class T>
cudaError_t rows_by_size(const RopeDev& r, const RopeRows& a, bool wide, int sms, cudaStream_t s) {
    if (!wide) {
        const long long n = (long long)a.n_tok * ((a.heads + 7) / 8) * (r.dim - r.rot / 2);
        rope_any_kernel<T><<<(unsigned)((n + kThreads - 1) / kThreads), kThreads, 0, s>>>(r, a.pos, (const T*)a.x, a.ldx,
                                                                                          (T*)a.out, a.ldo, a.n_tok, a.heads);
        return cudaGetLastError();
    }
    // one row a lane where all fit the GPU's threads at once, else more rows on their way and angles read once for them
    if ((long long)a.n_tok * a.heads * (r.dim / 16) <= sms * 2048) return rows<T, 1>(r, a, s);
    return rows<T, sizeof(T) == 4 ? 2 : 4>(r, a, s);
}

template <class T, class C, int D, int U>
cudaError_t append(const RopeDev& r, const KvDev& c, const KvBatchDev& b, const RopeAppend& a, int sms, cudaStream_t s) {
    const int per = ((a.heads + U - 1) / U + 2 * ((c.n_heads + U - 1) / U)) * (D / 16);
    // of many tokens a block takes several rounds: finding their places is a chain of loads that all of them share
    const int tokens = min(32, max(max(1, kThreads / per), min(kRounds, b.n_tok / (sms * 4))));
    kv_append_rope_kernel<T, C, D, U><<<(unsigned)((b.n_tok + tokens - 1) / tokens + 1), kThreads, (size_t)tokens * r.rot * 4,
                                        s>>>(r, c, b, a, FastDiv((uint32_t)c.page_size), tokens);
    return cudaGetLastError();
}

template <class T, class C>
cudaError_t append_by_size(int dim, const RopeDev& r, const KvDev& c, const KvBatchDev& b, const RopeAppend& a,
                           int sms, cudaStream_t s) {
    const bool few = (long long)b.n_tok * (a.heads + 2 * c.n_heads) * (dim / 16) <= sms * 2048;
    constexpr int U = sizeof(T) == 4 ? 2 : 4;
    if (dim == 64) return few ? append<T, C, 64, 1>(r, c, b, a, sms, s) : append<T, C, 64, U>(r, c, b, a, sms, s);
    return few ? append<T, C, 128, 1>(r, c, b, a, sms, s) : append<T, C, 128, U>(r, c, b, a, sms, s);
}

template <class T>
cudaError_t append_by_cache(int ct, int dim, const RopeDev& r, const KvDev& c, const KvBatchDev& b, const RopeAppend& a,
                            int sms, cudaStream_t s) {
    if (ct == T_F16) return append_by_size<T, __half>(dim, r, c, b, a, sms, s);
    if (ct == T_BF16) return append_by_size<T, __nv_bfloat16>(dim, r, c, b, a, sms, s);
    return append_by_size<T, int8_t>(dim, r, c, b, a, sms, s);
}

}  // namespace

cudaError_t launch_rope(int dtype, const RopeDev& r, const RopeRows& a, bool wide, int sms, cudaStream_t s) {
    if (dtype == T_F32) return rows_by_size<float>(r, a, wide, sms, s);
    if (dtype == T_F16) return rows_by_size<__half>(r, a, wide, sms, s);
    return rows_by_size<__nv_bfloat16>(r, a, wide, sms, s);
}

cudaError_t launch_kv_append_rope(int cache_type, int dtype, int head_dim, const RopeDev& r, const KvDev& c,
                                  const KvBatchDev& b, const RopeAppend& a, int sms, cudaStream_t s) {
    if (dtype == T_F32) return append_by_cache<float>(cache_type, head_dim, r, c, b, a, sms, s);
    if (dtype == T_F16) return append_by_cache<__half>(cache_type, head_dim, r, c, b, a, sms, s);
    return append_by_cache<__nv_bfloat16>(cache_type, head_dim, r, c, b, a, sms, s);
}

}  // namespace hc
