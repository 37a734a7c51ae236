// attn_rows.cuh -- the shape of attention work that its kernels share: row tiles of a sequence,
// the positions that a tile sees, and the flat order in which blocks divide the work.
//
// The query rows of one kv head are the (token, head of the group) pairs of a sequence, token
// major: row r is token r / group, head r % group, so the heads of a group share every key and
// value that is loaded.  A tile of `tile` rows sees the positions of its rows together: with a
// window the first n1 = min(sink, lo) and then [lo, end).  They are counted through as v = 0 ..
// nvis - 1, position j = v < n1 ? v : v - n1 + lo, and cut into units of `unit` of them.
//
// All units of a call, in the order (sequence, kv head, tile, unit), are one line of U units; block
// c of G works on [c U / G, (c + 1) U / G), so that blocks differ by one unit at most whatever the
// lengths are.  A tile whose units fall to several blocks is joined from their partial results by
// the block that finishes last, in block order (the same bits every time).
#pragma once

#include <math.h>

#include "kv_launch.h"

namespace hc {

struct AttnTile {
    int r0, nr;        // first row and number of rows
    int p_lo, p_hi;    // positions of the first and last row
    int lo, n1, nvis;  // visible positions (see above)
    int units;
};

__device__ __forceinline__ AttnTile attn_tile(const AttnArgs& a, const KvSeq& q, int tile, int rows, int unit) {
    AttnTile t;
    const int n = q.q1 - q.q0;
    t.r0 = tile * rows;
    t.nr = min(rows, n * a.group - t.r0);
    t.p_lo = q.len - n + t.r0 / a.group;
    t.p_hi = q.len - n + (t.r0 + t.nr - 1) / a.group;
    const int end = a.causal ? max(min(q.len, t.p_hi + 1), 0) : q.len;
    t.lo = a.window ? min(max(t.p_lo - a.window + 1, 0), end) : 0;
    t.n1 = min(a.sink, t.lo);
    t.nvis = t.n1 + end - t.lo;
    t.units = max(1, (t.nvis + unit - 1) / unit);  // a tile that sees nothing still has to write zeros
    return t;
}

__device__ __forceinline__ int attn_tiles(const AttnArgs& a, const KvSeq& q, int rows) {
    const int r = (q.q1 - q.q0) * a.group;
    return r >= a.row_min && r <= a.row_max ? (r + rows - 1) / rows : 0;
}

// Units of every sequence, as an inclusive prefix sum in `pre` (n_seq ints of shared memory);
// returns U, or -1 (and the error flag) if they do not fit 31 bits.  The whole block calls it.
template <int THREADS>
__device__ __forceinline__ int attn_schedule(const AttnArgs& a, int rows, int unit, int* pre) {
    __shared__ long long carry_s;
    __shared__ int wsum[THREADS / 32];
    const int cap = a.b.max_pages * a.c.page_size, tid = threadIdx.x, wid = tid >> 5, ln = tid & 31;
    const bool by_warp = a.max_rows > 8 * rows;  // many tiles in a sequence: its tiles over a warp's lanes
    if (by_warp) {
        for (int s = wid; s < a.b.n_seq; s += THREADS / 32) {
            const KvSeq q = kv_seq(a.b, cap, s);
            const int n = attn_tiles(a, q, rows);
            long long w = 0;
            for (int t = ln; t < n; t += 32) w += attn_tile(a, q, t, rows, unit).units;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
            if (ln == 0) pre[s] = (int)min(w * a.c.n_heads, 0x7fffffffll);
        }
    } else {
        for (int s = tid; s < a.b.n_seq; s += THREADS) {
            const KvSeq q = kv_seq(a.b, cap, s);
            const int n = attn_tiles(a, q, rows);
            long long w = 0;
            for (int t = 0; t < n; ++t) w += attn_tile(a, q, t, rows, unit).units;
            pre[s] = (int)min(w * a.c.n_heads, 0x7fffffffll);
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

// A place in the line of units: the item (sequence, kv head, tile) and its first unit.
struct AttnIter {
    int s, hk, tile, n_tiles, u_item;
    KvSeq q;
    AttnTile t;

    __device__ __forceinline__ void seq(const AttnArgs& a, int rows) {
        q = kv_seq(a.b, a.b.max_pages * a.c.page_size, s);
        n_tiles = attn_tiles(a, q, rows);
        hk = tile = 0;
    }
    // The item that holds unit u (0 <= u < U).
    __device__ __forceinline__ void seek(const AttnArgs& a, const int* pre, int u, int rows, int unit) {
        int lo = 0, hi = a.b.n_seq - 1;  // first sequence whose prefix is past u
        while (lo < hi) {
            const int m = (lo + hi) >> 1;
            if (pre[m] > u) hi = m;
            else lo = m + 1;
        }
        s = lo;
        seq(a, rows);
        const int before = s ? pre[s - 1] : 0, w = (pre[s] - before) / a.c.n_heads;
        hk = (u - before) / w;
        u_item = before + hk * w;
        t = attn_tile(a, q, 0, rows, unit);
        while (u_item + t.units <= u) {
            u_item += t.units;
            t = attn_tile(a, q, ++tile, rows, unit);
        }
    }
    // The next item (there has to be one).
    __device__ __forceinline__ void next(const AttnArgs& a, int rows, int unit) {
        u_item += t.units;
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

__device__ __forceinline__ int attn_begin(int c, int U, int G) { return (int)((long long)c * U / G); }
// The block of G whose range holds unit u.
__device__ __forceinline__ int attn_owner(int u, int U, int G) { return (int)(((long long)(u + 1) * G - 1) / U); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four values (y, the weighted sum) of row r of the item's tile, and at d = 0 its lse.
template <class T, int D>
__device__ __forceinline__ void attn_store(const AttnArgs& a, const AttnIter& it, int r, int d, float4 y, float m, float l) {
    const int row = it.t.r0 + r, h = it.hk * a.group + row % a.group;
    const long long tok = it.q.q0 + row / a.group;
    const bool none = l == 0.f;  // saw nothing (a sum that is not a number is kept)
    const float k = none ? 0.f : 1.f / l;
    if (none) y = make_float4(0.f, 0.f, 0.f, 0.f);
    T* out = (T*)a.out + tok * a.ldo + h * D + d;
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(out) = make_float4(y.x * k, y.y * k, y.z * k, y.w * k);
    else if constexpr (__is_same(T, __half))
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_h2(y.x * k, y.y * k), pack_h2(y.z * k, y.w * k));
    else
        *reinterpret_cast<uint2*>(out) = make_uint2(pack_b2(y.x * k, y.y * k), pack_b2(y.z * k, y.w * k));
    if (d == 0 && a.lse) a.lse[tok * a.heads + h] = none ? -INFINITY : (m + log2f(l)) * 0.693147181f;
}

}  // namespace hc
