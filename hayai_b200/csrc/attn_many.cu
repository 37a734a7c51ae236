// attn_many.cu -- attention over the paged cache for sequences with many rows per kv head (prompts,
// chunks of prompts), on the 5th-generation tensor cores.
//
// The mathematics is attn_few.cu's: one pass with a running maximum m and sum per row, m moved only
// when a score passes it by 8 (in log 2).  Work comes in tiles of 256 rows (attn_rows.cuh), two
// halves of 128 with their own accumulators, and units of 128 positions; one block of 16 warps per SM
// takes an equal share of the line of units.
//
//   warps 0-3, 4-7   one thread per row of half 0 and 1: S from TMEM, weights P (below) back into
//                    the same TMEM columns in 16 bits, m and the sum in registers; the row's O in TMEM
//                    is rescaled by its thread in the rare units where m moves;
//   warps 8-11       bring keys and values in: 16-byte asynchronous copies (8-bit pages: by way of a
//                    staging ring, from which each thread converts what it copied itself) into
//                    128-byte-swizzled operand tiles, a ring of 3 (8-bit) or 5 of 32 KB;
//   warp 12          issues S = Q K^T and O += P V (P from TMEM, V as it lies: its tile is read with
//                    the transposed, d-major view), one half's products while the other half's
//                    weights are made;
//   warp 13          walks the block's tiles and hands them to the others as segments (ring of 4);
//   warps 14-15      bring the queries in, the next segment's while the last unit's weights are made.
//
// Per unit and half the tensor cores take 2 x 512 cycles (D = 128) and the 16384 exponentials 1024 of
// the special function unit: the two pipes are equally loaded, and the rest of the softmax has to fit
// under them.
//
// Measured: 10.9k prompt tokens in 4 sequences (32 heads on 8 of 128, bf16) 397 us, 636 TFLOP/s of the
// visible pairs (38 % of cuBLAS's rate); 2048 tokens over 30k cached 8-bit ones 410 us, 600 TFLOP/s.  A unit
// of both halves takes about 4400 cycles (8-bit: 6000): the softmax's trips through TMEM and its chain
// are not all under the products.
//
// Formats: products of f16 (f16 and 8-bit caches) or bf16; P = 2^(s - m) is rounded to that type, of the
// order of the 16-bit results' own rounding, and summed in f32.  f16 weights are taken 2^7 times as large,
// with the lag of m up to 2^15: they keep their 11 bits down to 2^-21 of the row's maximum, and below it are
// off by up to 2^-32 of it (O stands in TMEM for the whole tile, so a unit cannot have a factor of its own as
// in attn_few.cu).  8-bit codes are exact in f16; a K scale multiplies its column of S, a V scale its column
// of P, and m follows the largest score + log2 of its V scale, so that P times scale stays under 2^15
// whatever the scales are.  Where a unit's scales lie within 2^6 of each other the largest stands for all,
// which may take that much of the room; elsewhere each position counts with its own, as a large one may have
// no weight or be masked.  Scales under 2^-80, zero above all, count as 2^-80, so that the weights' own sum
// stays in f32's range.  Rows of bf16 on f16 products are scaled by a power of two to have their largest
// element in [2^14, 2^15), and are exact to 2^-39 of it.
#include <math.h>

#include <type_traits>

#include "attn_phases.h"
#include "attn_rows.cuh"
#include "tc5.cuh"

namespace hc {

constexpr int kManyRows = 256, kManyUnit = 128, kManyThreads = 512, kManyRegs = 192, kManyRegsLow = 64;

template <class C, int D>
struct ManyCfg {
    static constexpr int ES = sizeof(C);
    static constexpr bool I8 = ES == 1, BF = ES == 2 && !__is_same(C, __half);
    static constexpr int TILE = 128 * D * 2;                 // an operand tile: 128 rows of D 16-bit values
    static constexpr int NB = many_ring(I8, D);              // ring of key and value tiles
    static constexpr int CPR = D * ES / 16;                  // 16-byte chunks of a cache row
    static constexpr int STG = I8 ? 128 * D : 0, NSTG = I8 ? 3 : 0;  // staging ring of tiles of codes
    static constexpr int oQ = 0, oKV = 2 * TILE, oSTG = oKV + NB * TILE, oSC = oSTG + NSTG * STG;
    static constexpr int oRS = oSC + (I8 ? 4 * 1024 : 0);    // scales: ring of 4 units, K then V
    static constexpr int oBAR = oRS + 2048;                  // the rows' score factors, of two segments
    static constexpr int oSEG = oBAR + 256, oMISC = oSEG + 256, BYTES = oMISC + 512;
};

// One thread's wait with a limit; false once any wait of the thread has run out.
__device__ __forceinline__ bool many_wait(uint32_t bar, uint32_t parity, bool& ok) {
    if (ok && !mbar_wait(bar, parity)) ok = false;
    return ok;
}

// V tile as B operand, N = d: 64 values of d to a 128-byte row, rows = positions (K of the product),
// halves of d one tile half apart (leading byte offset), 8 positions 1024 bytes apart (stride).
__device__ __forceinline__ uint64_t many_v_desc(uint32_t saddr, uint32_t half_bytes) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(half_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}

// The products' instructions as a whole warp issues them, by the lane that elect picks: control and
// operands are then uniform for the compiler, which halves what an issue costs (70 against 55 cycles
// and less per product of 128 x 64 x 16; one of 128 x 128 x 16 runs 64).
__device__ __forceinline__ void many_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void many_mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void many_commit(uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar)
        : "memory");
}

__device__ __forceinline__ void tc_ld32(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// The wait for loads still in flight, tied to their registers so that no use moves before it.
__device__ __forceinline__ void tc_wait_ld32(float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ uint32_t tc_ld1(uint32_t taddr) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r)
                 : "r"(taddr)
                 : "memory");
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const float* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
        "fma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n.reg .b64 x, y, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 w, x, y;\nmov.b64 {%0, %1}, w;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// A run of one tile's units, as the block's roles get it.
struct ManySeg {
    int lo, hi;               // units [lo, hi); lo = hi: there are no more
    int nr, r0;               // rows of the tile, its first
    int q0, q1, len, s, hk;   // the sequence and kv head
    int vlo, n1, nvis;        // its visible positions (AttnTile)
    int whole, slot;          // the whole tile; else the block's slot of partial results
    int pad[2];
};

// 32 bytes to global memory: in one store where they lie on 32 bytes (a thread per row stores to as
// many lines as it has lanes, and each line once instead of twice).
__device__ __forceinline__ void many_store32(void* p, const uint32_t (&y)[8], bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]),
                     "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                     : "memory");
    } else {
        reinterpret_cast<uint4*>(p)[0] = make_uint4(y[0], y[1], y[2], y[3]);
        reinterpret_cast<uint4*>(p)[1] = make_uint4(y[4], y[5], y[6], y[7]);
    }
}

// The range of a row's visible positions in the tile's count v: v < c and (v >= b or v < a).
struct ManyRow {
    int a, b, c;
};
__device__ __forceinline__ ManyRow many_row(const AttnArgs& ar, const KvSeq& q, const AttnTile& t, int row, bool real) {
    ManyRow r;
    const int pos = q.len - (q.q1 - q.q0) + ar.by_group(row);
    const int lim = ar.causal ? min(pos + 1, q.len) : q.len;  // positions j < lim
    r.c = lim <= t.n1 ? lim : lim < t.lo ? t.n1 : lim - t.lo + t.n1;
    if (!real) r.c = 0;
    r.b = ar.window ? max(pos - ar.window + 1, t.lo) - t.lo + t.n1 : 0;
    r.a = ar.sink <= t.lo ? t.n1 : ar.sink - t.lo + t.n1;
    return r;
}

// O += P V of one unit by the rows' threads, leaving out weights of zero.
template <bool BF, int D>
__device__ __noinline__ void many_product(uint32_t tO, uint32_t tP, const uint8_t* v, bool fresh) {
#pragma unroll 1
    for (int k = 0; k < D / 32; ++k) {
        float o[32];
        tc_ld32(tO + 32 * k, o);
        tc_wait_ld32(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = fresh ? 0.f : o[i];
#pragma unroll 1
        for (int t = 0; t < 128; ++t) {
            const uint32_t two = tc_ld1(tP + (t >> 1)), w = t & 1 ? two >> 16 : two & 0xffffu;
            const float p = BF ? __uint_as_float(w << 16) : h2f((uint16_t)w);
            if (p != 0.f) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int d = 32 * k + i;
                    const uint16_t x = *reinterpret_cast<const uint16_t*>(v + (d >> 6) * (128 * 128) + t * 128 +
                                                                         ((((d & 63) >> 3) ^ (t & 7)) << 4) + (d & 7) * 2);
                    o[i] += p * (BF ? __uint_as_float((uint32_t)x << 16) : h2f(x));
                }
            }
            __syncwarp();
        }
        tc_st32(tO + 32 * k, o);
    }
    tc_wait_st();
}

template <class T, class C, int D>
__global__ void __launch_bounds__(kManyThreads, 1) attn_many_kernel(const __grid_constant__ AttnArgs a) {
    using F = ManyCfg<C, D>;
    constexpr bool I8 = F::I8, BF = F::BF;
    constexpr int ROWS = kManyRows, UNIT = kManyUnit, NB = F::NB, TILE = F::TILE, HALF = 128 * 128;
    constexpr int PS = ROWS * (D + 2);
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sb = smem_addr(smem), bars = sb + F::oBAR;
    // barriers: key and value tiles full and empty; S ready, P ready, O ready, queries in, queries free
    // (of each half); segments full and empty; a unit checked (of each half)
    const uint32_t b_full = bars, b_empty = bars + 8 * NB, b_s = bars + 16 * NB, b_p = b_s + 16, b_o = b_s + 32,
                   b_q = b_s + 48, b_qf = b_s + 64, b_seg = b_s + 80, b_sege = b_seg + 32, b_chk = b_sege + 32;
    float* const rsc = reinterpret_cast<float*>(smem + F::oRS);
    ManySeg* const segs = reinterpret_cast<ManySeg*>(smem + F::oSEG);
    int* const misc = reinterpret_cast<int*>(smem + F::oMISC);  // TMEM base, last, [2..3] a product done by hand, [4..9] checks; [16..] scratch
    AttnShared* const shared_s = reinterpret_cast<AttnShared*>(misc + 64);  // the block's first and last tile, where shared
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), ln = lane_id(), c = blockIdx.x;

    // the schedule's prefix sums lie in the last key and value tile until warp 13 has its place
    int* const pre_s = reinterpret_cast<int*>(smem + F::oKV + (NB - 1) * TILE);
    const int U = attn_schedule<kManyThreads>(a, ROWS, UNIT, pre_s, misc + 16);
    // blocks: enough of the line for each, and a tile not in so many pieces that joining them takes longer
    const int G = max(1, min(min((int)gridDim.x, U / 4), 16 * misc[16 + 18]));
    if (U <= 0 || c >= G) return;
    const AttnShares share(U, G);
    if (threadIdx.x == 0) {
        for (int i = 0; i < NB; ++i) {
            mbar_init(b_full + 8 * i, 4);
            mbar_init(b_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_s + 8 * i, 1);
            mbar_init(b_p + 8 * i, 4);
            mbar_init(b_o + 8 * i, 1);
            mbar_init(b_q + 8 * i, 2);
            mbar_init(b_qf + 8 * i, 1);
            mbar_init(b_chk + 8 * i, 4);
            misc[4 + 3 * i] = misc[5 + 3 * i] = misc[6 + 3 * i] = 0;
            shared_s[i] = {0, 0, 0, 0, 0, 0, 1};
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(b_seg + 8 * i, 1);
            mbar_init(b_sege + 8 * i, 15);  // 8 softmax, 4 copying and 2 query warps, and the products' thread
        }
        mbar_fence_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(misc)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *(volatile uint32_t*)misc, 0);
    bool ok = true;
    // The n-th segment, once it is there; a role's warp gives it back when it needs it no more.
    auto segment = [&](int n) {
        many_wait(b_seg + 8 * (n & 3), (n >> 2) & 1, ok);
        return segs + (n & 3);
    };
    auto give_back = [&](int n) {
        __syncwarp();
        if (ln == 0) mbar_arrive(b_sege + 8 * (n & 3));
    };

    if (warp < 8) {
        // ================================================================ softmax, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegs));
        const int half = warp >> 2, rt = threadIdx.x & 127;  // half of the tile, row of the half
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tS = tmem + lanes + half * 128, tO = tmem + lanes + 256 + half * 128;
        uint32_t ph_s = 0, ph_o = 0;
        int checks = 0;  // units checked for values that are not finite
        int unit = 0;   // units of the block so far, for the scales' ring
        for (int n = 0;; ++n) {
            const ManySeg* const sg = segment(n);
            const int lo = sg->lo, hi = sg->hi, nr = sg->nr;
            if (!ok || lo == hi) break;
            const int kvt = 2 * unit;  // key and value tiles before this segment's
            unit += hi - lo;
            const KvSeq q{sg->q0, sg->q1, sg->len};
            const int r0 = sg->r0, hk = sg->hk, whole = sg->whole, slot = sg->slot;
            AttnTile tl;
            tl.lo = sg->vlo, tl.n1 = sg->n1;
            give_back(n);  // here: an arrival after the results' stores would wait for them
            if (half * 128 < nr) {
                const int r = half * 128 + rt, row = r0 + r;
                const bool real = r < nr;
                const ManyRow vis = many_row(a, q, tl, row, real);
                // a unit is whole for this half's rows if it ends before every row's limit and starts past
                // every row's window (or lies in the first tokens that all see)
                const ManyRow first = many_row(a, q, tl, r0 + half * 128, true),
                              lastr = many_row(a, q, tl, r0 + min(half * 128 + 127, nr - 1), true);
                const int cmin = min(first.c, lastr.c), bmax = lastr.b, amin = first.a;

                constexpr float kLift = BF ? 0.f : 7.f;  // log2 of the weights' common factor
                float rs = 0.f;
                float m = -INFINITY;
                float2 l2 = make_float2(0.f, 0.f);
                for (int st = lo; st < hi; ++st) {
                    const int v0 = st * UNIT;
                    const bool full = v0 + UNIT <= cmin && (v0 >= bmax || v0 + UNIT <= amin);
                    uint32_t odd = 0;
                    const uint8_t* vtile = nullptr;
                    if constexpr (!I8) {
                        // A value that is not finite, in a unit that some row does not see whole: 0 * infinity must not
                        // reach a masked row, so that the unit's product is then done by the rows' threads (rare).  The
                        // look at V comes before the wait for the scores where that is sound (attn_phases.h); elsewhere
                        // the scores are waited for here, and found there again below: this half has to give its weights
                        // before their barrier goes on.
                        if (!full) {
                            if (!many_early_look(st, lo) && !many_wait(b_s + 8 * half, ph_s, ok)) break;
                            const int vt = kvt + 2 * (st - lo) + 1;
                            if (!many_wait(b_full + 8 * (vt % NB), (vt / NB) & 1, ok)) break;
                            vtile = smem + F::oKV + (vt % NB) * TILE;
                            constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                            if (v0 + rt >= cmin || bmax > v0) {  // a position that all rows see is no matter
#pragma unroll 4
                                for (int i = 0; i < D / 8; ++i) {
                                    const uint4 x = *reinterpret_cast<const uint4*>(vtile + (i >> 3) * HALF + rt * 128 +
                                                                                    (((i + rt) & 7) << 4));
                                    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                    for (int k = 0; k < 4; ++k) odd |= (y[k] & E) == E || ((y[k] >> 16) & E) == E;
                                }
                            }
                            // the half's four warps decide together: three flags in turn, each cleared a check ahead
                            int* const flag = misc + 4 + 3 * half;
                            if (__any_sync(0xffffffffu, odd != 0) && ln == 0) flag[checks % 3] = 1;
                            if (rt == 0) flag[(checks + 1) % 3] = 0;
                            __syncwarp();
                            if (ln == 0) mbar_arrive(b_chk + 8 * half);
                            if (!many_wait(b_chk + 8 * half, checks & 1, ok)) break;
                            odd = *(volatile int*)&flag[checks % 3];
                            ++checks;
                        }
                    }
                    if (!many_wait(b_s + 8 * half, ph_s, ok)) break;
                    // read by the products' warp after the arrivals; it has read the last unit's before it issued this S
                    if (!I8 && rt == 0) misc[2 + half] = (int)odd;
                    ph_s ^= 1;
                    tc_fence_after();
                    // the queries and their factors came before this unit's products; their own barrier may be two
                    // segments further by now, so it cannot be waited for here
                    if (st == lo) rs = rsc[(n & 1) * 256 + r];
                    auto size = [](float x) { return fabsf(x) <= 3.4e38f ? fabsf(x) : 0.f; };  // what is not finite has none
                    // log2 of a power of two over a size (its bits), but near zero no less than -80: a weight is then up to
                    // 2^95, and the sum of 2^30 of them finite
                    auto size_log2 = [](uint32_t bits) { return max((int)(bits >> 23) - 126, -80); };
                    float ev = 0.f;
                    bool mixed = false;
                    const float4 *ksc = nullptr, *vsc = nullptr;
                    if constexpr (I8) {
                        // V's tile is not given back before this unit's weights, so its barrier is at its phase (K's
                        // may be one further); K's scales were written before it by the same threads
                        const int vt = kvt + 2 * (st - lo) + 1;
                        if (!many_wait(b_full + 8 * (vt % NB), (vt / NB) & 1, ok)) break;
                        const uint8_t* sc = smem + F::oSC + ((kvt / 2 + st - lo) & 3) * 1024;
                        ksc = reinterpret_cast<const float4*>(sc);
                        vsc = reinterpret_cast<const float4*>(sc + 512);
                        const float4 v = vsc[ln];
                        const float vs[4] = {v.x, v.y, v.z, v.w};
                        uint32_t most = 0, least = 0x7f7fffffu;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (v0 + 4 * ln + i >= lastr.c) continue;  // no row of this half sees it
                            const uint32_t b = __float_as_uint(size(vs[i]));
                            most = max(most, b);
                            least = min(least, b);
                        }
                        const int top = size_log2(__reduce_max_sync(0xffffffffu, most));
                        ev = (float)top;
                        mixed = size_log2(__reduce_min_sync(0xffffffffu, least)) < top - 6;
                    }
                    const int vc = vis.c - v0, vb = vis.b - v0, va = vis.a - v0;
                    // 32 scores from TMEM: times their K scales, masked
                    auto scores = [&](int k, float* s) {
                        if constexpr (I8) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float4 f = ksc[8 * k + i];
                                const float2 x = mul2(make_float2(s[4 * i], s[4 * i + 1]), make_float2(f.x, f.y));
                                const float2 y = mul2(make_float2(s[4 * i + 2], s[4 * i + 3]), make_float2(f.z, f.w));
                                s[4 * i] = x.x, s[4 * i + 1] = x.y, s[4 * i + 2] = y.x, s[4 * i + 3] = y.y;
                            }
                        }
                        if (!full) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const int v = 32 * k + i;
                                if (!(v < vc && (v >= vb || v < va))) s[i] = -INFINITY;
                            }
                        }
                    };
                    // 16-bit caches hold S in registers; with scales to multiply by that is more than a thread has, and S
                    // is read twice, 32 columns at a time with the next 32 on their way
                    float sa[I8 ? 2 : 4][32];
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if constexpr (I8) {
                        tc_ld32(tS, sa[0]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float* s = sa[k & 1];
                            tc_wait_ld32(s);
                            tc_ld32(tS + (k < 3 ? 32 * (k + 1) : 0), sa[(k + 1) & 1]);  // last: the second pass's first
                            scores(k, s);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], s[i], s[i + 1]);
                        }
                        tc_wait_ld32(sa[0]);  // before other loads and waits
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) tc_ld32(tS + 32 * k, sa[k]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) tc_wait_ld32(sa[k]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            float* s = sa[k];
                            scores(k, s);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], s[i], s[i + 1]);
                        }
                    }
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    float cand = top == -INFINITY ? top : top * rs + ev;
                    if constexpr (I8) {
                        if (mixed) {  // rare: the largest score + log2 of its own scale
                            cand = -INFINITY;
#pragma unroll 1
                            for (int k = 0; k < 4; ++k) {
                                float* s = sa[1];
                                tc_ld32(tS + 32 * k, s);
                                tc_wait_ld32(s);
                                scores(k, s);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    const float x = reinterpret_cast<const float*>(vsc)[32 * k + i];
                                    const int e = size_log2(__float_as_uint(size(x)));
                                    cand = fmaxf(cand, s[i] == -INFINITY ? s[i] : fmaf(s[i], rs, (float)e));
                                }
                            }
                        }
                    }
                    if (__any_sync(0xffffffffu, cand > m + 8.f)) {
                        const float mn = fmaxf(m, cand), f = mn == -INFINITY ? 1.f : ex2(m - mn);
                        m = mn;
                        l2.x *= f;
                        l2.y *= f;
                        if (st != lo) {  // the unit's S came after the last P V: O is complete
#pragma unroll 1
                            for (int k = 0; k < D / 32; ++k) {
                                float o[32];
                                tc_ld32(tO + 32 * k, o);
                                tc_wait_ld32(o);
#pragma unroll
                                for (int i = 0; i < 32; ++i) o[i] *= f;
                                tc_st32(tO + 32 * k, o);
                            }
                        }
                    }
                    const float mm = m == -INFINITY ? 0.f : m;
                    const float2 rs2 = make_float2(rs, rs), nm2 = make_float2(kLift - mm, kLift - mm);
                    auto weights = [&](auto masked) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float* s = sa[I8 ? k & 1 : k];
                        if constexpr (I8) {
                            if (k > 0) tc_wait_ld32(s);
                            if (k < 3) tc_ld32(tS + 32 * (k + 1), sa[(k + 1) & 1]);
                            scores(k, s);
                        }
                        uint32_t pk[16];
                        float4 vs4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int e = 2 * i;
                            const float2 x = fma2(make_float2(s[e], s[e + 1]), rs2, nm2);
                            float2 p = make_float2(ex2(x.x), ex2(x.y));
                            l2 = add2(l2, p);
                            if constexpr (I8) {
                                if ((i & 1) == 0) vs4 = vsc[8 * k + (i >> 1)];
                                p = mul2(p, i & 1 ? make_float2(vs4.z, vs4.w) : make_float2(vs4.x, vs4.y));
                                if constexpr (decltype(masked)::value) {  // whatever a masked position's scale is
                                    if (s[e] == -INFINITY) p.x = 0.f;
                                    if (s[e + 1] == -INFINITY) p.y = 0.f;
                                }
                            }
                            pk[i] = BF ? pack_b2(p.x, p.y) : pack_h2(p.x, p.y);
                        }
                        tc_st16(tS + 16 * k, pk);
                    }
                    };
                    if (I8 && !full)
                        weights(std::true_type());
                    else
                        weights(std::false_type());
                    tc_wait_st();
                    if constexpr (!I8)
                        if (odd) many_product<BF, D>(tO, tS, vtile, st == lo);
                    tc_fence_before();
                    __syncwarp();
                    if (ln == 0) mbar_arrive(b_p + 8 * half);
                }
                // ---- the tile's end: O out
                many_wait(b_o + 8 * half, ph_o, ok);
                ph_o ^= 1;
                tc_fence_after();
                const float l = l2.x + l2.y;
                m -= kLift;  // the sums are of 2^(s - m)
                const float k1 = l == 0.f ? 0.f : 1.f / l;
                const bool wide = (((uintptr_t)a.out | (uintptr_t)(a.ldo * 2)) & 31) == 0;  // rows start on 32 bytes
                const int tr = a.by_group(row);
                T* const out = (T*)a.out + (long long)(q.q0 + tr) * a.ldo + (hk * a.group + row - tr * a.group) * D;
                float* const part = a.part + (size_t)(2 * c + slot) * PS;
#pragma unroll 1
                for (int k = 0; k < D / 32; ++k) {
                    float o[32];
                    tc_ld32(tO + 32 * k, o);
                    tc_wait_ld32(o);
                    if (!real || !ok) continue;
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            uint32_t y[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const float u = l == 0.f ? 0.f : o[16 * i + 2 * e] * k1, v = l == 0.f ? 0.f : o[16 * i + 2 * e + 1] * k1;
                                y[e] = __is_same(T, __half) ? pack_h2(u, v) : pack_b2(u, v);
                            }
                            many_store32(out + 32 * k + 16 * i, y, wide);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<float4*>(part + r * D + 32 * k + 4 * i) =
                                make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
                tc_fence_before();
                if (real && ok) {
                    if (whole)
                        attn_store_lse(a, q.q0, hk, row, m, l);
                    else
                        *reinterpret_cast<float2*>(part + ROWS * D + 2 * r) = make_float2(m, l);
                }
            }
            if (!ok) break;
        }
        // ---- tiles that several blocks share: the last of them joins.  One thread decides for all, so that they
        // meet at the same barriers even where a wait has run out.
        __threadfence();
        named_bar_sync(1, 256);
        for (int x = 0; x < 2; ++x) {
            const AttnShared sh = shared_s[x];
            const int bf = share.owner(sh.u_item), bl = share.owner(sh.u_item + sh.units - 1);
            if (threadIdx.x == 0) {
                misc[1] = ok && sh.valid && atomicAdd(a.count + bf, 1) == bl - bf;
                if (misc[1]) a.count[bf] = 0;
                __threadfence();
            }
            named_bar_sync(1, 256);
            if (misc[1]) {
                // The pieces' weights of every row first (into the rings, which are done with), by a thread per row;
                // then a thread per four values of a row, eight of them on their way at once.  (A row per warp, or
                // one value after the other, waits for L2 so often that a joining took 80000 cycles.)
                const int n = bl - bf + 1;
                const float* const p0 = a.part + (size_t)(2 * bf + 1) * PS;  // the first piece; the i-th: p0 + (2 i - 1) PS
                auto piece = [&](int i) { return p0 + (i ? (size_t)(2 * i - 1) * PS : 0); };
                constexpr int WT = 64;  // pieces whose weights fit the rings of every variant; of more they are made again
                float* const wt = reinterpret_cast<float*>(smem + F::oKV);  // [piece][row]
                float* const tops = wt + WT * 256;                          // [row] maxima, [row] sums
                static_assert((WT + 2) * 1024 <= F::oRS - F::oKV, "the joining's table");
                {
                    const int r = threadIdx.x;
                    float m = -INFINITY, l = 0.f;
                    if (r < sh.nr) {
#pragma unroll 4
                        for (int i = 0; i < n; ++i) m = fmaxf(m, __ldcg(piece(i) + ROWS * D + 2 * r));
#pragma unroll 4
                        for (int i = 0; i < n; ++i) {
                            const float2 v = __ldcg(reinterpret_cast<const float2*>(piece(i) + ROWS * D + 2 * r));
                            // a piece that saw nothing has m = -inf and l = 0
                            const float f = v.x == -INFINITY ? (v.y == 0.f ? 0.f : 1.f) : ex2(v.x - m);
                            l += v.y * f;
                            if (i < WT) wt[i * 256 + r] = f;
                        }
                        tops[r] = m;
                        tops[256 + r] = l;
                        attn_store_lse(a, sh.q0, sh.hk, sh.r0 + r, m, l);
                    }
                }
                named_bar_sync(1, 256);
#pragma unroll 1
                for (int e0 = threadIdx.x; e0 < sh.nr * (D / 4); e0 += 8 * 256) {
                    float y[8][4];
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k][0] = y[k][1] = y[k][2] = y[k][3] = 0.f;
#pragma unroll 1
                    for (int i = 0; i < n; i += 2) {  // two pieces at a time, and no branch between their loads
                        float4 o[2][8];
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const int e = e0 + 256 * k;
                                o[j][k] = make_float4(0.f, 0.f, 0.f, 0.f);
                                if (i + j < n && e < sh.nr * (D / 4)) o[j][k] = __ldcg(reinterpret_cast<const float4*>(piece(i + j)) + e);
                            }
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                const int r = min((e0 + 256 * k) / (D / 4), ROWS - 1);
                                float f = 0.f;
                                if (i + j < n) f = i + j < WT ? wt[(i + j) * 256 + r] : ex2(__ldcg(piece(i + j) + ROWS * D + 2 * r) - tops[r]);
                                // a weight of zero takes nothing, whatever the value is
                                const bool none = f == 0.f;
                                y[k][0] = fmaf(none ? 0.f : o[j][k].x, f, y[k][0]), y[k][1] = fmaf(none ? 0.f : o[j][k].y, f, y[k][1]);
                                y[k][2] = fmaf(none ? 0.f : o[j][k].z, f, y[k][2]), y[k][3] = fmaf(none ? 0.f : o[j][k].w, f, y[k][3]);
                            }
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int e = e0 + 256 * k, r = e / (D / 4);
                        if (e < sh.nr * (D / 4)) attn_store<T>(a, sh.q0, sh.hk, sh.r0 + r, D, e % (D / 4) * 4, y[k], tops[256 + r]);
                    }
                }
            }
            named_bar_sync(1, 256);
        }
    } else if (warp < 12) {
        // ================================================================ keys and values in
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyRegsLow));
        // each warp copies RPW rows of 16-byte chunks at a time; lane i owns the address of row(i)
        constexpr int CPR = F::CPR, RPW = 32 / CPR, IT = CPR;
        const int pw = warp - 8;
        const int own = (ln / RPW) * 4 * RPW + pw * RPW + ln % RPW;  // this lane's row of the 128
        const int sub = pw * RPW + ln / CPR, ch = ln % CPR;          // its row (of 4 RPW) and chunk of a copy
        constexpr int AHEAD = 3;      // tiles on their way; the oldest is handed on before another is waited for
        int t_issue = 0, t_done = 0;  // tiles whose copies are issued; tiles handed on
        // A tile has arrived: 16-bit tiles are operands already, codes are converted by the threads that copied them.
        auto hand_on = [&]() {
            const int t = t_done++, buf = t % NB;
            if constexpr (I8) {
                if (t >= NB && !many_wait(b_empty + 8 * buf, ((t / NB) - 1) & 1, ok)) return;
                const uint32_t stg = sb + F::oSTG + (t % F::NSTG) * F::STG;
                const uint32_t dst = sb + F::oKV + buf * TILE;
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    const int r = i * 4 * RPW + sub;
                    uint4 x;
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                                 : "r"(stg + r * D + ch * 16));
                    const uint32_t y[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                    uint32_t h[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        h[2 * k] = hsub2_u32(prmt(y[k], 0x64646464u, 0x4140u), 0x64806480u);
                        h[2 * k + 1] = hsub2_u32(prmt(y[k], 0x64646464u, 0x4342u), 0x64806480u);
                    }
                    // chunk ch holds d = 16 ch ..: two 16-byte places of the tile's row
                    const uint32_t row = dst + (ch >> 2) * HALF + r * 128;
                    const int p = 2 * (ch & 3);
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + ((p ^ (r & 7)) << 4)), "r"(h[0]),
                                 "r"(h[1]), "r"(h[2]), "r"(h[3])
                                 : "memory");
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(row + (((p + 1) ^ (r & 7)) << 4)), "r"(h[4]),
                                 "r"(h[5]), "r"(h[6]), "r"(h[7])
                                 : "memory");
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (ln == 0) mbar_arrive(b_full + 8 * buf);
        };
        for (int n = 0;; ++n) {
            const ManySeg* const sg = segment(n);
            const int lo = sg->lo, hi = sg->hi;
            if (!ok || lo == hi) break;
            const int nvis = sg->nvis, n1 = sg->n1, vlo = sg->vlo, hk = sg->hk;
            const int* const table = a.b.table + sg->s * a.b.table_stride;
            give_back(n);
            // page and row of this lane's position of unit st, and whether it has one (any page number may stand in a table)
            auto page_of = [&](int st, int& r, bool& has) {
                const int v = st * UNIT + own;
                has = v < nvis && st < hi;
                if (!has) return -1;
                const int j = v < n1 ? v : v - n1 + vlo, p = a.by_page(j);
                r = j - p * a.c.page_size;
                return __ldg(table + p);
            };
            int r = 0;
            bool has;
            int pg = page_of(lo, r, has);
            for (int st = lo; st < hi && ok; ++st) {
                uint32_t off = 0xffffffffu;
                float sc[2] = {0.f, 0.f};
                if ((unsigned)pg < (unsigned)a.c.n_pages) {
                    off = (uint32_t)pg * a.c.page + (uint32_t)r * a.c.row + (uint32_t)hk * a.c.head;
                    if constexpr (I8) {
                        const long long so = pg * a.c.spage + (long long)hk * a.c.page_size + r;
                        sc[0] = __ldg(a.c.ks + so);
                        sc[1] = __ldg(a.c.vs + so);
                    }
                } else if (has) {
                    atomicOr(a.b.err, kErrKvRange);
                }
                pg = page_of(st + 1, r, has);
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv) {
                    if (t_issue - t_done == AHEAD) {
                        cp_async_wait(AHEAD - 1);
                        hand_on();
                    }
                    const int t = t_issue++;
                    if constexpr (!I8) {
                        if (t >= NB && !many_wait(b_empty + 8 * (t % NB), ((t / NB) - 1) & 1, ok)) break;
                    } else {
                        // the slot's last readers, of four units before, were done before the tile three before this one
                        // could be handed on (its buffer had held a tile of three units before)
                        reinterpret_cast<float*>(smem + F::oSC + ((t >> 1) & 3) * 1024 + kv * 512)[own] = kv ? sc[1] : sc[0];
                    }
                    const uint32_t dst = I8 ? sb + F::oSTG + (t % max(F::NSTG, 1)) * F::STG : sb + F::oKV + (t % NB) * TILE;
                    const uint8_t* src = kv ? a.c.v : a.c.k;
#pragma unroll
                    for (int i = 0; i < IT; ++i) {
                        const uint32_t o = __shfl_sync(0xffffffffu, off, i * RPW + ln / CPR);
                        const int rr = i * 4 * RPW + sub;
                        const bool have = o != 0xffffffffu;
                        const unsigned long long at = have ? (unsigned long long)o * 64 + ch * 16 : 0;
                        const uint32_t d = I8 ? dst + rr * D + ch * 16
                                              : dst + (ch >> 3) * HALF + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4);
                        cp16_or_zero(d, src + at, have);
                    }
                    cp_async_commit();
                }
            }
        }
        while (t_done < t_issue && ok) {
            cp_async_wait(t_issue - t_done - 1);
            hand_on();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kManyRegsLow));
        if (warp == 12) {
            // ============================================================ the products
            constexpr uint32_t fmt = BF ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t idS = (1u << 4) | fmt | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t idO = (1u << 4) | fmt | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
            uint32_t ph_p[2] = {0, 0}, ph_q[2] = {0, 0};
            int t = 0;  // key and value tiles so far
            for (int n = 0;; ++n) {
                const ManySeg* const sg = segment(n);
                const int nu = sg->hi - sg->lo, halves = sg->nr > 128 ? 2 : 1;
                if (!ok || nu == 0) break;
                give_back(n);
                auto scores = [&](int h, int kt, bool last) {  // S_h = Q_h K^T
                    const uint32_t q = sb + h * TILE, k = sb + F::oKV + (kt % NB) * TILE;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i)
                        many_mma(tmem + h * 128, tc_desc(q + (i >> 2) * HALF + (i & 3) * 32),
                               tc_desc(k + (i >> 2) * HALF + (i & 3) * 32), idS, i ? 1u : 0u);
                    many_commit(b_s + 8 * h);
                    if (last) many_commit(b_qf + 8 * h);
                };
                many_wait(b_full + 8 * (t % NB), (t / NB) & 1, ok);
                for (int h = 0; h < halves; ++h) {
                    if (!many_wait(b_q + 8 * h, ph_q[h], ok)) break;
                    ph_q[h] ^= 1;
                    tc_fence_after();
                    scores(h, t, nu == 1);
                }
                if (!ok) break;
                many_commit(b_empty + 8 * (t % NB));
                for (int u = 0; u < nu && ok; ++u, t += 2) {
                    const int vt = t + 1, kn = t + 2;
                    many_wait(b_full + 8 * (vt % NB), (vt / NB) & 1, ok);
                    if (u + 1 < nu) many_wait(b_full + 8 * (kn % NB), (kn / NB) & 1, ok);
                    for (int h = 0; h < halves; ++h) {
                        if (!many_wait(b_p + 8 * h, ph_p[h], ok)) break;
                        ph_p[h] ^= 1;
                        tc_fence_after();
                        const uint32_t v = sb + F::oKV + (vt % NB) * TILE;
                        if (I8 || !*(volatile int*)&misc[2 + h]) {
#pragma unroll
                            for (int i = 0; i < UNIT / 16; ++i)  // O_h += P_h V
                                many_mma_ta(tmem + 256 + h * 128, tmem + h * 128 + 8 * i, many_v_desc(v + i * 2048, HALF), idO,
                                          u || i ? 1u : 0u);
                        }
                        if (u + 1 < nu) scores(h, kn, u + 2 == nu);
                        else many_commit(b_o + 8 * h);
                    }
                    many_commit(b_empty + 8 * (vt % NB));
                    if (u + 1 < nu) many_commit(b_empty + 8 * (kn % NB));
                }
            }
        } else if (warp == 13) {
            // ============================================================ the segments
            const int b0 = share.begin(c), b1 = share.begin(c + 1);
            AttnIter it;
            it.seek(a, pre_s, b0, ROWS, UNIT);
            int n = 0;
            for (;;) {
                const int lo = max(b0 - it.u_item, 0), hi = min(b1 - it.u_item, it.t.units);
                if (lo < hi) {
                    if (n >= 4 && !many_wait(b_sege + 8 * (n & 3), ((n >> 2) - 1) & 1, ok)) break;
                    if (ln == 0) {
                        const bool whole = lo == 0 && hi == it.t.units;
                        segs[n & 3] = {lo, hi, it.t.nr, it.t.r0, it.q.q0, it.q.q1, it.q.len, it.s, it.hk, it.t.lo, it.t.n1,
                                       it.t.nvis, whole, lo == 0, {0, 0}};
                        if (!whole) shared_s[lo == 0] = {1, it.q.q0, it.hk, it.t.r0, it.t.nr, it.u_item, it.t.units};
                        mbar_arrive(b_seg + 8 * (n & 3));
                    }
                    ++n;
                }
                if (it.u_item + it.t.span >= b1) break;
                it.next(a, ROWS, UNIT);
            }
            if (n < 4 || many_wait(b_sege + 8 * (n & 3), ((n >> 2) - 1) & 1, ok))
                if (ln == 0) {
                    segs[n & 3].lo = segs[n & 3].hi = 0;
                    mbar_arrive(b_seg + 8 * (n & 3));
                }
        } else if (warp > 13) {
            // ============================================================ queries in, and the rows' factors
            constexpr int CH = D / 8, RP = 32 / CH;  // 16-byte chunks of a row; rows a warp takes at a time
            constexpr bool CONV = !__is_same(T, __half) && !BF;  // bf16 rows into f16
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // the scale's sign goes into the queries
            uint32_t ph_qf[2] = {1, 1};  // a half's first queries find it free
            for (int n = 0;; ++n) {
                const ManySeg* const sg = segment(n);
                const int lo = sg->lo, hi = sg->hi, nr = sg->nr, r0 = sg->r0, q0 = sg->q0, hk = sg->hk;
                if (!ok || lo == hi) break;
                give_back(n);
                // the rows come to L2 while the half's place is still in use
                for (int r = (warp - 14) * 32 + ln; r < nr; r += 64) {
                    const int tr = a.by_group(r0 + r);
                    const T* const q = (const T*)a.q + (long long)(q0 + tr) * a.ldq + (hk * a.group + r0 + r - tr * a.group) * D;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(q));
                    if constexpr (D == 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + 64));
                }
                for (int h = 0; h < 2 && h * 128 < nr; ++h) {
                    if (!many_wait(b_qf + 8 * h, ph_qf[h], ok)) break;
                    ph_qf[h] ^= 1;
                    const uint32_t qs = sb + h * TILE;
                    const int ch = ln % CH;
                    auto row_of = [&](int i) { return (warp - 14) * 64 + i * RP + ln / CH; };
                    auto source = [&](int r) {
                        const int row = r0 + h * 128 + r, tr = a.by_group(row);
                        return (const T*)a.q + (long long)(q0 + tr) * a.ldq + (hk * a.group + row - tr * a.group) * D + 8 * ch;
                    };
                    auto place = [&](int r) { return qs + (ch >> 3) * HALF + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
                    const float rs0 = fmaxf(fabsf(a.scale) * 1.44269504f, 1e-30f);  // not 0: 0 * -inf
                    if (!CONV && !flip) {
#pragma unroll 4
                        for (int i = 0; i < 64 / RP; ++i) {
                            const int r = row_of(i);
                            cp16_or_zero(place(r), h * 128 + r < nr ? source(r) : a.q, h * 128 + r < nr);
                            if (ch == 0) rsc[(n & 1) * 256 + h * 128 + r] = rs0;
                        }
                        asm volatile("cp.async.wait_all;" ::: "memory");
                    } else {
#pragma unroll 1
                        for (int i0 = 0; i0 < 64 / RP; i0 += 8) {  // 8 loads on their way
                            uint4 x[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int r = row_of(i0 + i);
                                x[i] = make_uint4(0, 0, 0, 0);
                                if (h * 128 + r < nr) x[i] = __ldg(reinterpret_cast<const uint4*>(source(r)));
                            }
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int r = row_of(i0 + i);
                                float rs = rs0;
                                uint32_t y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                                if constexpr (CONV) {
                                    uint32_t m = 0;
#pragma unroll
                                    for (int k = 0; k < 4; ++k) m = max(m, max(y[k] & 0x7fffu, (y[k] >> 16) & 0x7fffu));
#pragma unroll
                                    for (int o = CH / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                                    const RowSize size(m << 16);
                                    rs = fmaxf(rs * size.back, 1e-30f);
#pragma unroll
                                    for (int k = 0; k < 4; ++k)
                                        y[k] = pack_h2(__uint_as_float(y[k] << 16) * size.by,
                                                       __uint_as_float(y[k] & 0xffff0000u) * size.by);
                                }
                                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(place(r)), "r"(y[0] ^ flip),
                                             "r"(y[1] ^ flip), "r"(y[2] ^ flip), "r"(y[3] ^ flip)
                                             : "memory");
                                if (ch == 0) rsc[(n & 1) * 256 + h * 128 + r] = rs;
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (ln == 0) mbar_arrive(b_q + 8 * h);
                }
            }
        }
    }
    if (!ok) atomicOr(a.b.err, kErrWait);
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

namespace {

template <class T, class C, int D>
cudaError_t launch(const AttnArgs& a, int blocks, cudaStream_t s) {
    constexpr int bytes = ManyCfg<C, D>::BYTES;
    static_assert(bytes <= 227 * 1024, "shared memory of a block");
    static_assert(sizeof(float) * 2 * kManyRows * (D + 2) <= kManyPartBytes, "the workspace of a block");
    static SmemOptIn opted;
    const cudaError_t e = opted(reinterpret_cast<const void*>(attn_many_kernel<T, C, D>), bytes);
    if (e != cudaSuccess) return e;
    AttnArgs b = a;
    b.over = 2;  // a tile's start and end cost about what two of its units do
    attn_many_kernel<T, C, D><<<blocks, kManyThreads, bytes, s>>>(b);
    return cudaGetLastError();
}

template <class T, int D>
cudaError_t by_cache(int ct, const AttnArgs& a, int blocks, cudaStream_t s) {
    if (ct == T_F16) return launch<T, __half, D>(a, blocks, s);
    return launch<T, int8_t, D>(a, blocks, s);
}

}  // namespace

bool attn_many_supported(int ct, int dt) { return (dt == T_F16 && ct != T_BF16) || dt == T_BF16; }

cudaError_t launch_attn_many(int ct, int dt, int D, const AttnArgs& a, int blocks, cudaStream_t s) {
    if (ct == T_BF16)
        return D == 64 ? launch<__nv_bfloat16, __nv_bfloat16, 64>(a, blocks, s)
                       : launch<__nv_bfloat16, __nv_bfloat16, 128>(a, blocks, s);
    if (dt == T_F16) return D == 64 ? by_cache<__half, 64>(ct, a, blocks, s) : by_cache<__half, 128>(ct, a, blocks, s);
    return D == 64 ? by_cache<__nv_bfloat16, 64>(ct, a, blocks, s) : by_cache<__nv_bfloat16, 128>(ct, a, blocks, s);
}

}  // namespace hc
