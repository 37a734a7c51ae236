// kv.cuh -- what the paged key/value cache's kernels share: the cache and batch as the kernels
// get them, the sequence and slot of a token, and loads and stores of the element types.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "err_flags.h"

namespace hc {

// hc_kv_cache with strides in 64-byte units of the element arrays (a row of 64 int8 codes, the
// smallest, is one unit): 32 bits of them reach 256 GB, more than the GPU has.
struct KvDev {
    uint8_t *k, *v;
    float *ks, *vs;       // scales of an 8-bit cache: [page][head][row]
    uint32_t page, head, row;  // strides of k and v, 64-byte units
    long long spage;           // page stride of the scales, floats
    int n_pages, page_size, n_heads;
};

struct KvBatchDev {
    const int* table;  // [n_seq][table_stride] page numbers
    long long table_stride;
    const int *q_start, *kv_len;
    int n_seq, n_tok, max_pages;
    int* err;
};

// A sequence's new tokens [q0, q1) of the batch and its length, with offsets and lengths that do
// not fit the batch cut to it (and the error flag set).
struct KvSeq {
    int q0, q1, len;
    int first;  // attention over what comes behind a shared prefix: its first position
};
__device__ __forceinline__ KvSeq kv_seq(const KvBatchDev& b, int cap, int s) {
    KvSeq r{};
    const int a = __ldg(b.q_start + s), e = __ldg(b.q_start + s + 1), n = __ldg(b.kv_len + s);
    r.q0 = min(max(a, 0), b.n_tok);
    r.q1 = min(max(e, r.q0), b.n_tok);
    r.len = min(max(n, 0), cap);
    if (r.q0 != a || r.q1 != e || r.len != n) atomicOr(b.err, kErrKvRange);
    return r;
}

// The sequence whose new tokens include t (or -1), with q_start of the next and its length, found by
// GL lanes together.  A step of single tokens has s = t, so that place is looked at first, while the
// first of the search's steps is on its way: the largest s with q_start[s] <= t (of empty sequences
// at the same offset the last, which is the one that is not empty), GL candidates per step.  All
// lanes of the group call it with the same t.
struct KvPlace {
    int s, next, len;
};
template <int GL>
__device__ __forceinline__ KvPlace kv_find_seq(const KvBatchDev& b, int t) {
    const int l = lane_id() & (GL - 1), g0 = lane_id() & ~(GL - 1);
    const uint32_t mask = GL == 32 ? 0xffffffffu : ((1u << GL) - 1u) << g0;
    KvPlace p;
    p.s = min(t, b.n_seq - 1);
    const int at = __ldg(b.q_start + p.s);
    p.next = __ldg(b.q_start + p.s + 1);
    p.len = __ldg(b.kv_len + p.s);
    int lo = 0, n = b.n_seq, step = (n + GL - 1) / GL;
    bool le = l * step < n && __ldg(b.q_start + l * step) <= t;
    if (at <= t && t < p.next) return p;
    for (;;) {
        const int c = __popc(__ballot_sync(mask, le) & mask);
        if (c == 0) break;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        if (n <= 1) break;
        step = (n + GL - 1) / GL;
        le = l * step < n && __ldg(b.q_start + lo + l * step) <= t;
    }
    const int first = __ldg(b.q_start + lo);
    p.next = __ldg(b.q_start + lo + 1);
    p.len = __ldg(b.kv_len + lo);
    p.s = first <= t && t < p.next ? lo : -1;
    return p;
}

// ---------------------------------------------------------------- 8 elements of a row
// (raw as loaded, so that many rows wait in few registers; as values.  load8 is for what no thread of the kernel writes,
// load8_own for rows that it may write over, in place)
template <class T>
struct Elem;
template <>
struct Elem<float> {
    struct Raw {
        float4 a, b;
    };
    static __device__ __forceinline__ Raw load8(const float* p) {
        return {__ldg(reinterpret_cast<const float4*>(p)), __ldg(reinterpret_cast<const float4*>(p) + 1)};
    }
    static __device__ __forceinline__ Raw load8_own(const float* p) {
        return {reinterpret_cast<const float4*>(p)[0], reinterpret_cast<const float4*>(p)[1]};
    }
    static __device__ __forceinline__ void values(const Raw& r, float (&x)[8]) {
        x[0] = r.a.x, x[1] = r.a.y, x[2] = r.a.z, x[3] = r.a.w, x[4] = r.b.x, x[5] = r.b.y, x[6] = r.b.z, x[7] = r.b.w;
    }
    // The largest |x| as f32 bits, whose order is that of the values, infinity and NaN above all.
    static __device__ __forceinline__ uint32_t top(const Raw& r) {
        auto bits = [](float x) { return __float_as_uint(x) & 0x7fffffffu; };
        return max(max(max(bits(r.a.x), bits(r.a.y)), max(bits(r.a.z), bits(r.a.w))),
                   max(max(bits(r.b.x), bits(r.b.y)), max(bits(r.b.z), bits(r.b.w))));
    }
    static __device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
};
// The larger of the 16-bit magnitudes of 8 packed values.
__device__ __forceinline__ uint32_t top16(const uint4& r) {
    const uint32_t m = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
    return max(m & 0xffffu, m >> 16);
}
template <>
struct Elem<__half> {
    using Raw = uint4;
    static __device__ __forceinline__ Raw load8(const __half* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
    static __device__ __forceinline__ Raw load8_own(const __half* p) { return *reinterpret_cast<const uint4*>(p); }
    static __device__ __forceinline__ void values(const Raw& r, float (&x)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(u32_as_h2(w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint32_t top(const Raw& r) { return __float_as_uint(h2f((uint16_t)top16(r))); }
    static __device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
    }
};
__device__ __forceinline__ uint32_t pack_b2(float lo, float hi) {
    __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&b);
}
template <>
struct Elem<__nv_bfloat16> {
    using Raw = uint4;
    static __device__ __forceinline__ Raw load8(const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
    static __device__ __forceinline__ Raw load8_own(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }
    static __device__ __forceinline__ void values(const Raw& r, float (&x)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint32_t top(const Raw& r) { return top16(r) << 16; }
    static __device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
        *reinterpret_cast<uint4*>(p) =
            make_uint4(pack_b2(x[0], x[1]), pack_b2(x[2], x[3]), pack_b2(x[4], x[5]), pack_b2(x[6], x[7]));
    }
};
template <>
struct Elem<int8_t> {  // codes as they are
    using Raw = uint2;
    static __device__ __forceinline__ Raw load8(const int8_t* p) { return __ldg(reinterpret_cast<const uint2*>(p)); }
    static __device__ __forceinline__ void values(const Raw& r, float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = s8_to_f32_flipped((i < 4 ? r.x : r.y) ^ 0x80808080u, i & 3);
    }
};

}  // namespace hc
