// kv_rows.cuh -- what the kernels that write rows into the paged cache, or read rows of it, share: a token's
// place in the pages, the batch's check, and the codes of 8-bit rows.
#pragma once

#include "kv_launch.h"

namespace hc {

// Where the batch's token t lives: its page's and row's offset in the cache (64-byte units, of
// head 0) and in the scales, and its position; false where it has no place (a position below zero: no
// sequence has it, or it lies before its sequence's first).
template <int GL>
__device__ __forceinline__ bool kv_slot(const KvDev& c, const KvBatchDev& b, const FastDiv& by_page, int t, uint32_t& at,
                                        long long& sat, int& pos) {
    const KvPlace k = kv_find_seq<GL>(b, t);
    pos = k.s < 0 ? -1 : k.len - k.next + t;
    if (pos < 0) return false;
    const int p = by_page(pos), r = pos - p * c.page_size;
    const int page = p < b.max_pages ? __ldg(b.table + k.s * b.table_stride + p) : -1;
    if ((unsigned)page >= (unsigned)c.n_pages) {
        atomicOr(b.err, kErrKvRange);
        return false;
    }
    at = (uint32_t)page * c.page + (uint32_t)r * c.row;
    sat = page * c.spage + r;
    return true;
}

// The grid's last block looks the batch's offsets and lengths over (the others read no more of them than their
// tokens' places take) and sets the error flag where attention would cut them.
__device__ __forceinline__ bool kv_check_block(const KvDev& c, const KvBatchDev& b) {
    if (blockIdx.x != gridDim.x - 1) return false;
    for (int s = threadIdx.x; s < b.n_seq; s += blockDim.x) kv_seq(b, b.max_pages * c.page_size, s);
    return true;
}

template <class C>
__device__ __forceinline__ C* kv_elem(uint8_t* base, uint32_t units) {
    return reinterpret_cast<C*>(base + (unsigned long long)units * 64);
}

// Codes of 8 values of a row with largest |x| m and scale s, four to a word.  The quotient rounded as
// IEEE division rounds it takes three instructions a value where the row shares the divisor, by
// Markstein's theorem (IBM J. Res. Dev. 34, 1990): with r the reciprocal of s rounded to nearest and
// q = x r, fma(fma(-q, s, x), r, q) is x / s rounded to nearest, unless s has a significand of all
// ones.  That, and rows whose scale or remainders are not normal numbers, are divided.  (An estimate
// with a division where it lies near a half is slower: ratios of 8-bit significands meet halves in
// two of three warps.)  1.5 * 2^23 added rounds to whole numbers, ties to even, and leaves them in the
// low bits in two's complement.
__device__ __forceinline__ void kv_codes(const float (&x)[8], float m, float s, uint32_t (&q)[2]) {
    constexpr float kMagic = 12582912.f;
    float f[8];
    if (m >= 1e-30f && m <= 1e30f && (__float_as_uint(s) & 0x7fffffu) != 0x7fffffu) {
        const float r = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = x[i] * r;
            f[i] = fmaf(fmaf(-y, s, x[i]), r, y) + kMagic;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            f[i] = (s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -127.f), 127.f) : 0.f) + kMagic;
    }
#pragma unroll
    for (int w = 0; w < 2; ++w)
        q[w] = prmt(prmt(__float_as_uint(f[4 * w]), __float_as_uint(f[4 * w + 1]), 0x0040u),
                    prmt(__float_as_uint(f[4 * w + 2]), __float_as_uint(f[4 * w + 3]), 0x0040u), 0x5410u);
}

}  // namespace hc
