// attn_rows.cuh -- the shape of attention work that its kernels share: row tiles of a sequence,
// the positions that a tile sees, and the flat order in which blocks divide the work.
//
// The query rows of one kv head are the (token, head of the group) pairs of a sequence, token
// major: row r is token r / group, head r % group, so the heads of a group share every key and
// value that is loaded.  A tile of `tile` rows sees the positions of its rows together: with a
// window the first n1 = min(sink, lo) and then [lo, end).  They are counted through as v = 0 ..
// nvis - 1, position j = v < n1 ? v : v - n1 + lo, and cut into units of `unit` of them.
//
// All units of a call, in the order (sequence, kv head, tile, unit), are one line; after a tile's
// units come `over` places that stand for what starting and finishing a tile costs.  Of the U
// places the workers take equal shares, whatever the lengths are.  A tile whose units fall to several workers is joined from their partial results,
// in the workers' order (the same bits every time).
#pragma once

#include <math.h>

#include "kv_launch.h"

namespace hc {

struct AttnTile {
    int r0, nr;        // first row and number of rows
    int p_lo, p_hi;    // positions of the first and last row
    int lo, n1, nvis;  // visible positions (see above)
    int units, span;   // span: units + a.over
};

__device__ __forceinline__ AttnTile attn_tile(const AttnArgs& a, const KvSeq& q, int tile, int rows, int unit) {
    AttnTile t;
    const int n = q.q1 - q.q0;
    t.r0 = tile * rows;
    t.nr = min(rows, n * a.group - t.r0);
    t.p_lo = q.len - n + a.by_group(t.r0);
    t.p_hi = q.len - n + a.by_group(t.r0 + t.nr - 1);
    const int end = a.causal ? max(min(q.len, t.p_hi + 1), 0) : q.len;
    t.lo = a.window ? min(max(t.p_lo - a.window + 1, 0), end) : 0;
    t.n1 = min(a.sink, t.lo);
    t.nvis = t.n1 + end - t.lo;
    t.units = max(1, (t.nvis + unit - 1) / unit);  // a tile that sees nothing still has to write zeros
    t.span = t.units + a.over;
    return t;
}

__device__ __forceinline__ int attn_tiles(const AttnArgs& a, const KvSeq& q, int rows) {
    const int r = (q.q1 - q.q0) * a.group;
    return r >= a.row_min && r <= a.row_max ? (r + rows - 1) / rows : 0;
}

// Places of every sequence, as an inclusive prefix sum in `pre` (n_seq ints of shared memory);
// returns U, or -1 (and the error flag) if they do not fit 31 bits.  The whole block calls it, with 32
// words of shared memory as scratch; word 18 then holds the number of items (of 2^16 and more: at
// least that).
template <int THREADS>
__device__ __forceinline__ int attn_schedule(const AttnArgs& a, int rows, int unit, int* pre, int* scratch) {
    static_assert(THREADS <= 32 * 16, "scratch");
    long long& carry_s = *reinterpret_cast<long long*>(scratch);
    int* const wsum = scratch + 2;
    int* const items = scratch + 18;  // the number of items, at most 2^16 counted
    if (threadIdx.x == 0) *items = 0;
    __syncthreads();
    const int cap = a.b.max_pages * a.c.page_size, tid = threadIdx.x, wid = tid >> 5, ln = tid & 31;
    const bool by_warp = a.max_rows > 8 * rows;  // many tiles in a sequence: its tiles over a warp's lanes
    if (by_warp) {
        for (int s = wid; s < a.b.n_seq; s += THREADS / 32) {
            const KvSeq q = kv_seq(a.b, cap, s);
            const int n = attn_tiles(a, q, rows);
            long long w = 0;
            for (int t = ln; t < n; t += 32) w += attn_tile(a, q, t, rows, unit).span;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
            if (ln == 0) {
                pre[s] = (int)min(w * a.c.n_heads, 0x7fffffffll);
                if (n && *(volatile int*)items < 1 << 16) atomicAdd(items, min(n * a.c.n_heads, 1 << 16));
            }
        }
    } else {
        for (int s = tid; s < a.b.n_seq; s += THREADS) {
            const KvSeq q = kv_seq(a.b, cap, s);
            const int n = attn_tiles(a, q, rows);
            long long w = 0;
            for (int t = 0; t < n; ++t) w += attn_tile(a, q, t, rows, unit).span;
            pre[s] = (int)min(w * a.c.n_heads, 0x7fffffffll);
            if (n && *(volatile int*)items < 1 << 16) atomicAdd(items, min(n * a.c.n_heads, 1 << 16));
        }
    }
    if (tid == 0) carry_s = 0;
    __syncthreads();
    for (int s0 = 0; s0 < a.b.n_seq; s0 += THREADS) {
        const int s = s0 + tid;
        const int own = s < a.b.n_seq ? pre[s] : 0;
        long long x = own;  // sums may pass 31 bits: checked below, before any index is taken from them
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (ln >= o) x += y;
        }
        if (ln == 31) wsum[wid] = (int)min(x, 0x7fffffffll);
        __syncthreads();
        long long base = carry_s;
        for (int w = 0; w < wid; ++w) base += wsum[w];
        if (s < a.b.n_seq) pre[s] = (int)min(base + x, 0x7fffffffll);
        __syncthreads();
        if (tid == 0)
            for (int w = 0; w < THREADS / 32; ++w) carry_s += wsum[w];
        __syncthreads();
    }
    if (carry_s >= 0x7fffffffll) {
        if (tid == 0) atomicOr(a.b.err, kErrKvRange);
        return -1;
    }
    return (int)carry_s;
}

// The same for at most 32 sequences of few tiles, by every warp for itself and without a barrier:
// lane s gets its sequence, and the places up to its end.
struct AttnLanes {
    KvSeq q;
    int pre;
};
__device__ __forceinline__ int attn_schedule_lanes(const AttnArgs& a, int rows, int unit, AttnLanes& v) {
    const int ln = lane_id();
    v.q = {0, 0, 0};
    unsigned long long x = 0;
    if (ln < a.b.n_seq) {
        v.q = kv_seq(a.b, a.b.max_pages * a.c.page_size, ln);
        const int n = attn_tiles(a, v.q, rows);
        for (int t = 0; t < n; ++t) x += attn_tile(a, v.q, t, rows, unit).span;
    }
    x = min(x * a.c.n_heads, 0x7fffffffull);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (ln >= o) x += y;
    }
    v.pre = (int)min(x, 0x7fffffffull);
    const int U = __shfl_sync(0xffffffffu, v.pre, 31);
    if (U == 0x7fffffff) {
        if (ln == 0) atomicOr(a.b.err, kErrKvRange);
        return -1;
    }
    return U;
}

// A tile that several workers share, for the joining.
struct AttnShared {
    int valid, q0, hk, r0, nr, u_item, units;
};

// An item of the line, (sequence, kv head, tile), and its first place.
struct AttnIter {
    int s, hk, tile, n_tiles, u_item;
    KvSeq q;
    AttnTile t;

    __device__ __forceinline__ void seq(const AttnArgs& a, int rows) {
        q = kv_seq(a.b, a.b.max_pages * a.c.page_size, s);
        n_tiles = attn_tiles(a, q, rows);
        hk = tile = 0;
    }
    // The item that holds place u (0 <= u < U).
    __device__ __forceinline__ void seek(const AttnArgs& a, const int* pre, int u, int rows, int unit) {
        int lo = 0, hi = a.b.n_seq - 1;  // first sequence whose prefix is past u
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if (pre[m] > u) hi = m;
            else lo = m + 1;
        }
        s = lo;
        seq(a, rows);
        enter(a, s ? pre[s - 1] : 0, pre[s], u, rows, unit);
    }
    __device__ __forceinline__ void seek(const AttnArgs& a, const AttnLanes& v, int u, int rows, int unit) {
        s = __popc(__ballot_sync(0xffffffffu, v.pre <= u));
        q = {__shfl_sync(0xffffffffu, v.q.q0, s), __shfl_sync(0xffffffffu, v.q.q1, s), __shfl_sync(0xffffffffu, v.q.len, s)};
        n_tiles = attn_tiles(a, q, rows);
        tile = 0;
        const int before = __shfl_sync(0xffffffffu, v.pre, s ? s - 1 : 0);
        enter(a, s ? before : 0, __shfl_sync(0xffffffffu, v.pre, s), u, rows, unit);
    }
    // The item of sequence s, whose places are [before, end), that holds place u.
    __device__ __forceinline__ void enter(const AttnArgs& a, int before, int end, int u, int rows, int unit) {
        const int w = (end - before) / a.c.n_heads;
        hk = (u - before) / w;
        u_item = before + hk * w;
        t = attn_tile(a, q, 0, rows, unit);
        while (u_item + t.span <= u) {
            u_item += t.span;
            t = attn_tile(a, q, ++tile, rows, unit);
        }
    }
    // The next item (there has to be one).
    __device__ __forceinline__ void next(const AttnArgs& a, int rows, int unit) {
        u_item += t.span;
        if (++tile == n_tiles) {
            tile = 0;
            if (++hk == a.c.n_heads) {
                do {
                    ++s;
                    seq(a, rows);
                } while (n_tiles == 0);
            }
        }
        t = attn_tile(a, q, tile, rows, unit);
    }
};

// The workers' shares of U places: U / G each, and one more for the first U % G.
struct AttnShares {
    int q, rem;
    __device__ __forceinline__ AttnShares(int U, int G) : q(U / G), rem(U - q * G) {}
    __device__ __forceinline__ int begin(int c) const { return c * q + min(c, rem); }
    // The worker whose share holds place u.
    __device__ __forceinline__ int owner(int u) const {
        const int big = rem * (q + 1);
        return u < big ? u / (q + 1) : rem + (u - big) / q;
    }
};

// The power of two that brings a query row whose largest |x| has the bits m to [2^14, 2^15), and its reciprocal:
// in f16 the other elements then have the most room below.  Rows that are not finite stay as they are.
struct RowSize {
    float by = 1.f, back = 1.f;
    __device__ __forceinline__ explicit RowSize(uint32_t m) {
        const uint32_t e = max(m >> 23, 15u);  // of rows under 2^-112 the power alone stays a normal number
        if (e < 255) {
            by = __uint_as_float((268 - e) << 23);
            back = __uint_as_float((e - 14) << 23);
        }
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Copy 16 bytes (or with ok false: 16 zero bytes) to shared memory.
__device__ __forceinline__ void cp16_or_zero(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// Four adjacent values of the weighted sum of row `row` of an item's kv head, over l.
template <class T>
__device__ __forceinline__ void attn_store(const AttnArgs& a, int q0, int hk, int row, int D, int d, const float (&y)[4],
                                           float l) {
    const bool none = l == 0.f;  // saw nothing (a sum that is not a number is kept)
    const float k = none ? 0.f : 1.f / l;
    const int t = a.by_group(row);
    T* out = (T*)a.out + (long long)(q0 + t) * a.ldo + (hk * a.group + row - t * a.group) * D + d;
    float z[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = none ? 0.f : y[i] * k;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(out) = make_float4(z[0], z[1], z[2], z[3]);
    else if constexpr (__is_same(T, __half))
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_h2(z[0], z[1]), pack_h2(z[2], z[3]));
    else
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_b2(z[0], z[1]), pack_b2(z[2], z[3]));
}
__device__ __forceinline__ void attn_store_lse(const AttnArgs& a, int q0, int hk, int row, float m, float l) {
    const int t = a.by_group(row);
    if (a.lse)
        a.lse[(long long)(q0 + t) * a.heads + hk * a.group + row - t * a.group] =
            l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147181f;
}

// One row of n partial results joined by a warp: ml(i) gives piece i's (m, l), (-inf, 0) if it has
// none, and y(i) the lane's 4 of its D values.  All (m, l) are loaded together and the values eight
// pieces at a time: with one piece after the other the trips to L2 took 8 to 15 us of a call.
struct AttnJoin {
    float m = -INFINITY, l = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
    template <class ML, class Y>
    __device__ __forceinline__ void join(int n, bool mine, ML ml, Y at) {
        const int ln = lane_id();
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int cnt = min(32, n - i0);
            float2 v = make_float2(-INFINITY, 0.f);
            if (ln < cnt) v = ml(i0 + ln);
            float top = v.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, m);
            // a piece that saw nothing has m = -inf and l = 0; one of scores that are not numbers has m = -inf only
            const float f = v.x == -INFINITY ? (v.y == 0.f ? 0.f : 1.f) : ex2(v.x - top);
            const float old = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - top);
            l = l * old + warp_sum(v.y * f);
            m = top;
#pragma unroll
            for (int k = 0; k < 4; ++k) y[k] = old == 0.f ? 0.f : y[k] * old;
#pragma unroll 1
            for (int i = 0; i < cnt; i += 8) {
                float4 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (mine && i + k < cnt) x[k] = at(i0 + i + k);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float g = __shfl_sync(0xffffffffu, f, (i + k) & 31);
                    if (i + k >= cnt || g == 0.f) continue;
                    y[0] = fmaf(x[k].x, g, y[0]), y[1] = fmaf(x[k].y, g, y[1]);
                    y[2] = fmaf(x[k].z, g, y[2]), y[3] = fmaf(x[k].w, g, y[3]);
                }
            }
        }
    }
};

}  // namespace hc
