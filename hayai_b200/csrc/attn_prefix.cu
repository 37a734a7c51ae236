// attn_prefix.cu -- attention for a call with shared prefixes, on the 5th-generation tensor cores: of a group's rows
// over the prefix that its sequences share, which all of them see whole, and of a chunk's rows over what it has behind
// its prefix, up to each row's own position.
//
//     O_i = sum_j 2^(s_ij - m_i) v_j,   l_i = sum_j 2^(s_ij - m_i),   s_ij = scale log2 e q_i . k_j
// over the positions of a piece, with m_i near their maximum (it moves when a score passes it by 8).
//
// Work comes in tiles of up to 256 rows of a kv head (attn_shared.cu) and units of 128 positions.  A wide tile's rows
// are two halves of 128 that take every unit; a narrow one, of up to 128 rows, has its units taken by the two halves in
// turn, each with sums of its own.  Either way a block has two independent chains S = Q K^T -> weights -> O += P V, and
// the tensor cores work on one's products while the other's weights are made: a list of jobs, the j-th on half j & 1.
// One block of 16 warps per SM takes an equal share of the line of units, and leaves a piece for each tile and half;
// attn_shared.cu joins them over the whole GPU.  (A tile joined by the block that comes last, as attn_many.cu does, took
// 100 us of a call with few tiles: one SM reads all its pieces.)
//
//   warps 0-3, 4-7   a thread per row of half 0 and 1: its query in (a row a thread: 256 rows are on their way at
//                    once; one warp for all took 32 us), then S from TMEM to registers, weights back over it in 16
//                    bits, in two parts, so that the first part's product runs while the second is made
//   warps 8-11       16-bit pages: keys and values in by 16-byte asynchronous copies into 128-byte-swizzled operand
//                    tiles; 8-bit pages: staged codes into operands
//   warp 12          the products, one half's after the other's (a warp for each half lets the halves fall into step,
//                    where they wait for the same units in turn: 5000 cycles a unit against 3500 to 4000)
//   warps 13, 14     8-bit pages: codes into the staging ring by bulk copies, a page's rows of a head in one; scales
//   warp 15          is there for the register split, which goes by four warps
//
// Measured: a prefix of 60001 bf16 tokens under 100 single tokens (32 heads on 8 of 128) 132 us, 745 TFLOP/s of the
// visible pairs (45 % of cuBLAS's rate; rows fill 400 of 512 places of their tiles); 65536 tokens under 64 of them 1.3
// times the keys' and values' time at the copy rate from 16-bit pages, and 3 times from 8-bit ones.  A
// unit of a wide tile takes 3500 to 4000 cycles, where its products take 2048 and its exponentials as many: each
// half's chain (scores in, weights 1800, products 800, and the waits between) is the time, not either pipe.  Two threads per row,
// exponentials by polynomials, and scores read twice from a shorter loop took the same time or more.  Chunks that fill
// their tiles run at 470 to 500 TFLOP/s (8 of 256 tokens behind 16384, 577 us at its best; attn_many.cu 560).  A tile's start
// and end take some 12 us (attn_shared.cu, kOver), the block's later tiles' as well as its first: 31 us in all for 64
// sequences behind 4100 8-bit tokens, whose units are 8.  Queries in, the first keys' way, a unit through all roles and O out
// follow one another; which of them it is has not been measured apart.
//
// Formats as in attn_many.cu: products of f16 (f16 and 8-bit caches) or bf16, weights rounded to that type and
// summed in f32; f16 weights are taken 2^7 times as large.  8-bit codes are exact in f16; a K scale multiplies its column of
// S, a V scale its column of P, and m follows the largest score + log2 of its V scale, so that P times scale
// stays within f16 whatever the scales are.  Rows of bf16 on f16 products are scaled by a power of two.
#include <math.h>

#include <type_traits>

#include "attn_rows.cuh"
#include "attn_tc.cuh"

namespace hc {

namespace {

constexpr int kPfxUnit = 128, kPfxThreads = 512, kPfxRegs = 192, kPfxRegsLow = 64;
static_assert(256 * kPfxRegs + 256 * kPfxRegsLow <= 65536, "the registers that the block is launched with, 128 a thread");

template <class C, int D>
struct PfxCfg {
    static constexpr int ES = sizeof(C);
    static constexpr bool I8 = ES == 1, BF = ES == 2 && !__is_same(C, __half);
    static constexpr int TILE = 128 * D * 2;                         // an operand tile: 128 rows of D 16-bit values
    static constexpr int NB = I8 ? 3 : D == 64 ? 8 : 5;              // ring of key and value tiles
    static constexpr int CPR = D * ES / 16;                          // 16-byte chunks of a cache row
    static constexpr int STG = I8 ? 128 * D : 0, NSTG = I8 ? 3 : 0;  // staging ring of tiles of codes
    static constexpr int NSC = 8;                                    // scales: ring of 8 units, K then V
    static constexpr int oKV = 2 * TILE, oSTG = oKV + NB * TILE, oSC = oSTG + NSTG * STG;
    static constexpr int oRS = oSC + (I8 ? NSC * 1024 : 0);  // the rows' score factors, of two runs
    static constexpr int oBAR = oRS + 2048, oMISC = oBAR + 448, BYTES = oMISC + 64;
};

// The block's runs of units, one tile after the other; every role goes through them for itself.
struct PfxWalk {
    const PrefixArgs& p;
    int t, n, b0, b1;
    PrefixTile x;
    int lo, hi;  // units [lo, hi)
    bool wide;
    __device__ __forceinline__ PfxWalk(const PrefixArgs& args, const AttnShares& share, int c) : p(args) {
        t = __ldcg(p.first_tile + c) - 1;
        n = __ldcg(p.line + kLineTiles);
        b0 = share.begin(c);
        b1 = share.begin(c + 1);
    }
    __device__ __forceinline__ bool next() {
        while (++t < n) {
            const int4* const s = reinterpret_cast<const int4*>(p.tiles + t);
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(&x)[i] = __ldcg(s + i);
            if (x.place >= b1) return false;
            wide = x.cost == 2;
            // a unit belongs to the block that has its first place
            lo = max(b0 - x.place, 0), hi = b1 - x.place;
            if (wide) lo = (lo + 1) >> 1, hi = (hi + 1) >> 1;
            hi = min(hi, x.units);
            if (lo < hi) return true;
        }
        return false;
    }
    // The i-th of a run's tiles in the ring, where they lie in the order in which the products need them.  Wide: K0 V0 K1
    // V1 ...; narrow: K0 K1 V0 K2 V1 ... V.
    __device__ __forceinline__ void tile_at(int i, int& unit, bool& v) const {
        const int last = 2 * (hi - lo) - 1;
        if (wide)
            unit = i >> 1, v = i & 1;
        else if (i == 0)
            unit = 0, v = false;
        else if (i == last)
            unit = hi - lo - 1, v = true;
        else
            v = !(i & 1), unit = v ? (i >> 1) - 1 : (i + 1) >> 1;
    }
};

template <class T, class C, int D>
__global__ void __launch_bounds__(kPfxThreads, 1) attn_prefix_kernel(const __grid_constant__ AttnArgs a,
                                                                     const __grid_constant__ PrefixArgs p) {
    using F = PfxCfg<C, D>;
    constexpr bool I8 = F::I8, BF = F::BF;
    constexpr int UNIT = kPfxUnit, NB = F::NB, TILE = F::TILE, HALF = 128 * 128, NSC = F::NSC;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sb = smem_addr(smem), bars = sb + F::oBAR;
    // barriers: key and value tiles full and empty; S ready, P's first and second part ready, O ready (of each half);
    // queries in, queries free; a unit checked (of each half); 8-bit pages: a unit's scales there and done with, a tile of codes there and converted
    const uint32_t b_full = bars, b_empty = b_full + 8 * NB, b_s = b_empty + 8 * NB, b_p = b_s + 16, b_o = b_p + 32,
                   b_q = b_o + 16, b_qf = b_q + 8, b_sc = b_qf + 8, b_scf = b_sc + 8 * NSC, b_stg = b_scf + 8 * NSC,
                   b_stge = b_stg + 8 * F::NSTG, b_chk = b_stge + 8 * F::NSTG;
    float* const rsc = reinterpret_cast<float*>(smem + F::oRS);
    // TMEM base; a zero; [2..3] a half's product is done by hand; [4..9] what its checks found, three in turn
    int* const misc = reinterpret_cast<int*>(smem + F::oMISC);
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), ln = lane_id(), c = blockIdx.x;
    after_previous();
    let_next_start();
    const int U = __ldcg(p.line + kLinePlaces), G = __ldcg(p.line + kLineBlocks);
    if (U <= 0 || c >= G) return;
    const AttnShares share(U, G);
    if (threadIdx.x == 0) {
        for (int i = 1; i < 10; ++i) misc[i] = 0;
        for (int i = 0; i < NB; ++i) {
            mbar_init(b_full + 8 * i, 4);
            mbar_init(b_empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(b_s + 8 * i, 1);
            mbar_init(b_p + 16 * i, 4);
            mbar_init(b_p + 16 * i + 8, 4);
            mbar_init(b_o + 8 * i, 1);
            mbar_init(b_chk + 8 * i, 4);
        }
        mbar_init(b_q, 8);
        mbar_init(b_qf, 1);
        if (I8) {
            for (int i = 0; i < NSC; ++i) {
                mbar_init(b_sc + 8 * i, 1);
                mbar_init(b_scf + 8 * i, 8);  // of a narrow tile's unit the four warps of one half arrive twice
            }
            for (int i = 0; i < F::NSTG; ++i) {
                mbar_init(b_stg + 8 * i, 1);
                mbar_init(b_stge + 8 * i, 4);
            }
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
    PfxWalk w(p, share, c);

    if (warp < 8) {
        // ================================================================ weights, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPfxRegs));
        const int half = warp >> 2, rt = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t tS = tmem + lanes + half * 128, tO = tmem + lanes + 256 + half * 128;
        constexpr float kLift = BF ? 0.f : 7.f;  // log2 of the weights' common factor
        uint32_t ph_s = 0, ph_o = 0;
        int units = 0;   // of the block before this run, for the rings
        int checks = 0;  // units checked for values that are not finite
        // The tile's row r, where the row is this thread's: its query in and its scores' factor, once the products of the
        // run before, n - 1, have read theirs.
        auto queries = [&](int n, int r) {
            constexpr bool CONV = !__is_same(T, __half) && !BF;      // bf16 rows into f16
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // the scale's sign goes into the queries
            float rs = fmaxf(fabsf(a.scale) * 1.44269504f, 1e-30f);  // not 0: 0 * -inf
            const bool mine = w.wide || half == 0;
            uint4 x[D / 8];
#pragma unroll
            for (int i = 0; i < D / 8; ++i) x[i] = make_uint4(0, 0, 0, 0);
            if (mine && r < w.x.nr) {
                const int row = w.x.r0 + r, tr = a.by_group(row);
                const uint4* const q = reinterpret_cast<const uint4*>((const T*)a.q + (long long)(w.x.q0 + tr) * a.ldq +
                                                                      (w.x.hk * a.group + row - tr * a.group) * D);
#pragma unroll
                for (int i = 0; i < D / 8; ++i) x[i] = __ldg(q + i);
            }
            if (n && !many_wait(b_qf, (n - 1) & 1, ok)) return;
            if (mine) {
                float by = 1.f;
                if constexpr (CONV) {
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) m = max(m, top16(x[i]));
                    const RowSize size(m << 16);
                    by = size.by;
                    rs = fmaxf(rs * size.back, 1e-30f);
                }
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    uint32_t y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if constexpr (CONV)
                            y[k] = pack_h2(__uint_as_float(y[k] << 16) * by, __uint_as_float(y[k] & 0xffff0000u) * by);
                        y[k] ^= flip;
                    }
                    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(sb + (r >> 7) * TILE + (i >> 3) * HALF +
                                                                               (r & 127) * 128 + (((i & 7) ^ (r & 7)) << 4)),
                                 "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3])
                                 : "memory");
                }
                rsc[(n & 1) * 256 + r] = rs;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (ln == 0) mbar_arrive(b_q);
        };
        auto row_of = [&]() { return w.wide ? half * 128 + rt : rt; };  // this thread's row of the tile
        bool more = w.next();
        if (more) queries(0, row_of());
        for (int n = 0; more && ok; ++n) {
            const int nu = w.hi - w.lo, step = w.wide ? 1 : 2, first = w.wide ? 0 : half;
            const int r = row_of(), kvt = 2 * units, last = 2 * nu - 1;
            const bool real = r < w.x.nr, wide = w.wide;
            // positions from the run's first on that a row sees: this one's, and the half's first and last row's (whose
            // own are the fewest and the most)
            const int start = w.x.from + w.lo * UNIT;
            auto seen = [&](int row) {
                return (w.x.pos0 == kAllSeen ? w.x.len : min(w.x.len, w.x.pos0 + a.by_group(w.x.r0 + row) + 1)) - start;
            };
            const int r_first = wide ? half * 128 : 0, sees = seen(min(r, w.x.nr - 1)), least = seen(min(r_first, w.x.nr - 1)),
                      most_seen = seen(min(r_first + 127, w.x.nr - 1));
            const bool idle = r_first + 32 * (warp & 3) >= w.x.nr;  // none of the warp's rows is there
            const int piece = w.x.piece + (w.wide ? c - w.x.c0 : 2 * (c - w.x.c0) + half) * w.x.nr + r;
            // a narrow tile's factors are the first half's; they are written over two runs later, when all warps are past this
            if (!many_wait(b_q, n & 1, ok)) break;
            const float rs = rsc[(n & 1) * 256 + r];
            float m = -INFINITY;
            float2 l2 = make_float2(0.f, 0.f);
            for (int u = first; u < nu; u += step) {
                if (!many_wait(b_s + 8 * half, ph_s, ok)) break;
                ph_s ^= 1;
                tc_fence_after();
                const bool full = (u + 1) * UNIT <= least;
                uint32_t odd = 0;
                const uint8_t* vtile = nullptr;
                if constexpr (!I8) {
                    // A value that is not finite, where some row does not see it: 0 * infinity must not reach that row, so
                    // that the unit's product is then done by the rows' threads (rare).  V's tile is not given back before
                    // this half's weights, and the tile that was in its place is before this unit's keys in the ring: its
                    // barrier is at its phase or the one before.
                    if (!full && least < w.x.len - start) {
                        const int vt = kvt + (wide ? 2 * u + 1 : min(2 * u + 2, last));
                        if (!many_wait(b_full + 8 * (vt % NB), (vt / NB) & 1, ok)) break;
                        vtile = smem + F::oKV + (vt % NB) * TILE;
                        constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
                        if (u * UNIT + rt >= least) {
#pragma unroll 4
                            for (int i = 0; i < D / 8; ++i) {
                                const uint4 x = *reinterpret_cast<const uint4*>(vtile + (i >> 3) * HALF + rt * 128 + (((i + rt) & 7) << 4));
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
                    // read by the products' warp after the arrivals; it has read the last unit's before it issued this S
                    if (rt == 0) misc[2 + half] = (int)odd;
                }
                auto arrive = [&](int part) {
                    tc_fence_before();
                    __syncwarp();
                    if (ln == 0) {
                        mbar_arrive(b_p + 16 * half + 8 * part);
                        if (I8 && part == 1) {
                            const uint32_t bar = b_scf + 8 * ((units + u) % NSC);
                            mbar_arrive(bar);
                            if (step == 2) mbar_arrive(bar);
                        }
                    }
                };
                if (idle) {
                    arrive(0);
                    arrive(1);
                    continue;
                }
                float s[128];
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_ld32(tS + 32 * k, s + 32 * k);
                auto size = [](float x) { return fabsf(x) <= 3.4e38f ? fabsf(x) : 0.f; };  // what is not finite has none
                auto size_log2 = [](uint32_t bits) { return max((int)(bits >> 23) - 126, -80); };
                const int left = sees - u * UNIT;  // positions that the row sees from the unit's first on
                float ev = 0.f;
                bool mixed = false;
                const float4 *ksc = nullptr, *vsc = nullptr;
                if constexpr (I8) {
                    const int slot = (units + u) % NSC;
                    if (!many_wait(b_sc + 8 * slot, ((units + u) / NSC) & 1, ok)) break;
                    const uint8_t* const sc = smem + F::oSC + slot * 1024;
                    ksc = reinterpret_cast<const float4*>(sc);
                    vsc = reinterpret_cast<const float4*>(sc + 512);
                    const float4 v = vsc[ln];
                    const float vs[4] = {v.x, v.y, v.z, v.w};
                    uint32_t most = 0, fewest = 0x7f7fffffu;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (4 * ln + i >= most_seen - u * UNIT) continue;
                        const uint32_t b = __float_as_uint(size(vs[i]));
                        most = max(most, b);
                        fewest = min(fewest, b);
                    }
                    const int top = size_log2(__reduce_max_sync(0xffffffffu, most));
                    ev = (float)top;
                    mixed = size_log2(__reduce_min_sync(0xffffffffu, fewest)) < top - 6;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) tc_wait_ld32(s + 32 * k);
                if constexpr (I8) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float4 f = ksc[i];
                        const float2 x = mul2(make_float2(s[4 * i], s[4 * i + 1]), make_float2(f.x, f.y));
                        const float2 y = mul2(make_float2(s[4 * i + 2], s[4 * i + 3]), make_float2(f.z, f.w));
                        s[4 * i] = x.x, s[4 * i + 1] = x.y, s[4 * i + 2] = y.x, s[4 * i + 3] = y.y;
                    }
                }
                if (!full) {
#pragma unroll
                    for (int i = 0; i < 128; ++i)
                        if (i >= left) s[i] = -INFINITY;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 128; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], s[i], s[i + 1]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                float cand = top == -INFINITY ? top : top * rs + ev;
                if constexpr (I8) {
                    if (mixed) {  // rare: the largest score + log2 of its own scale
                        cand = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 128; ++i) {
                            const int e = size_log2(__float_as_uint(size(reinterpret_cast<const float*>(vsc)[i])));
                            cand = fmaxf(cand, s[i] == -INFINITY ? s[i] : fmaf(s[i], rs, (float)e));
                        }
                    }
                }
                if (__any_sync(0xffffffffu, cand > m + 8.f)) {
                    const float mn = fmaxf(m, cand), f = mn == -INFINITY ? 1.f : ex2(m - mn);
                    m = mn;
                    l2.x *= f;
                    l2.y *= f;
                    if (u != first) {  // the unit's S came after the half's last product: O is complete
#pragma unroll 1
                        for (int k = 0; k < D / 16; ++k) {
                            float o[16];
                            tc_ld16(tO + 16 * k, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= f;
                            tc_st16(tO + 16 * k, reinterpret_cast<const uint32_t(&)[16]>(o));
                        }
                    }
                }
                const float mm = m == -INFINITY ? 0.f : m;
                const float2 rs2 = make_float2(rs, rs);
                float2 nm2 = make_float2(kLift - mm, kLift - mm);
                auto weights = [&](auto masked) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    uint32_t pk[16];
                    float4 vs4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int e = 32 * k + 2 * i;
                        const float2 x = fma2(make_float2(s[e], s[e + 1]), rs2, nm2);
                        float2 q = make_float2(ex2(x.x), ex2(x.y));
                        l2 = add2(l2, q);
                        if constexpr (I8) {
                            if ((i & 1) == 0) vs4 = vsc[8 * k + (i >> 1)];
                            q = mul2(q, i & 1 ? make_float2(vs4.z, vs4.w) : make_float2(vs4.x, vs4.y));
                            if constexpr (decltype(masked)::value) {  // whatever a masked position's scale is
                                if (s[e] == -INFINITY) q.x = 0.f;
                                if (s[e + 1] == -INFINITY) q.y = 0.f;
                            }
                        }
                        pk[i] = BF ? pack_b2(q.x, q.y) : pack_h2(q.x, q.y);
                    }
                    tc_st16(tS + 16 * k, pk);
                    if (k & 1) {
                        tc_wait_st();
                        if constexpr (!I8)
                            if (k == 3 && odd) many_product<BF, D>(tO, tS, vtile, u == first);
                        arrive(k >> 1);
                        if (k == 1) {
                            // The second part's arithmetic is not to be moved before the first one's arrival: it takes a
                            // zero that is read behind it.
                            float zero;
                            asm volatile("ld.volatile.shared.f32 %0, [%1];" : "=f"(zero) : "r"(smem_addr(misc + 1)) : "memory");
                            nm2 = add2(nm2, make_float2(zero, zero));
                        }
                    }
                }
                };
                if (I8 && !full)
                    weights(std::true_type());
                else
                    weights(std::false_type());
            }
            units += nu;
            if (!ok) break;
            // ---- the run's end: the next one's queries in, and O out
            more = w.next();
            if (more) queries(n + 1, row_of());
            if (first >= nu) {  // a narrow tile's only unit was the other half's
                if (real) *reinterpret_cast<float2*>(p.part_ml + 2 * (size_t)piece) = make_float2(-INFINITY, 0.f);
                continue;
            }
            if (!many_wait(b_o + 8 * half, ph_o, ok)) break;
            ph_o ^= 1;
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 32; ++k) {
                float o[32];
                tc_ld32(tO + 32 * k, o);
                tc_wait_ld32(o);
                if (!real) continue;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    *reinterpret_cast<float4*>(p.part + (size_t)piece * D + 32 * k + 4 * i) =
                        make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
            tc_fence_before();
            // the sums are of 2^(s - m)
            if (real) *reinterpret_cast<float2*>(p.part_ml + 2 * (size_t)piece) = make_float2(m - kLift, l2.x + l2.y);
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfxRegsLow));
        const int pw = warp - 8;
        if constexpr (I8) {
            // ============================================================ codes into operands
            constexpr int CPR = F::CPR, ROWS = 128 / CPR, IT = 128 / ROWS;  // rows the four warps take at a time
            const int r0 = (pw * 32 + ln) / CPR, ch = ln % CPR;
            uint32_t slot = 0, ph = 0, stage = 0, ph_st = 0;  // the operands' ring and the staging ring
            bool around = false;                              // the ring's places have been used before
            while (ok && w.next()) {
                const int last = 2 * (w.hi - w.lo);
#pragma unroll 1
                for (int i = 0; i < last; ++i) {
                    if (!many_wait(b_stg + 8 * stage, ph_st, ok)) break;
                    if (around && !many_wait(b_empty + 8 * slot, ph ^ 1, ok)) break;
                    const uint32_t src = sb + F::oSTG + stage * F::STG, dst = sb + F::oKV + slot * TILE;
#pragma unroll
                    for (int k0 = 0; k0 < IT; k0 += 4) {  // four reads, then what they give: the trips overlap
                        uint4 code[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                         : "=r"(code[k].x), "=r"(code[k].y), "=r"(code[k].z), "=r"(code[k].w)
                                         : "r"(src + (r0 + (k0 + k) * ROWS) * D + ch * 16));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int r = r0 + (k0 + k) * ROWS;
                            const uint32_t y[4] = {code[k].x ^ 0x80808080u, code[k].y ^ 0x80808080u, code[k].z ^ 0x80808080u,
                                                   code[k].w ^ 0x80808080u};
                            uint32_t h[8];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                h[2 * e] = hsub2_u32(prmt(y[e], 0x64646464u, 0x4140u), 0x64806480u);
                                h[2 * e + 1] = hsub2_u32(prmt(y[e], 0x64646464u, 0x4342u), 0x64806480u);
                            }
                            // chunk ch holds d = 16 ch ..: two 16-byte places of the tile's row, the second first in the
                            // tile's upper half, so that eight lanes meet all banks
                            const uint32_t row = dst + (ch >> 2) * HALF + r * 128;
                            const uint32_t at[2] = {row + (((2 * (ch & 3)) ^ (r & 7)) << 4),
                                                    row + (((2 * (ch & 3) + 1) ^ (r & 7)) << 4)};
#pragma unroll
                            for (int o = 0; o < 2; ++o) {
                                const bool hi = (o ^ (ch >> 2)) & 1;
                                asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(hi ? at[1] : at[0]),
                                             "r"(hi ? h[4] : h[0]), "r"(hi ? h[5] : h[1]), "r"(hi ? h[6] : h[2]),
                                             "r"(hi ? h[7] : h[3])
                                             : "memory");
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (ln == 0) {
                        mbar_arrive(b_full + 8 * slot);
                        mbar_arrive(b_stge + 8 * stage);
                    }
                    if (++slot == NB) slot = 0, ph ^= 1, around = true;
                    if (++stage == F::NSTG) stage = 0, ph_st ^= 1;
                }
            }
        } else {
            // ============================================================ keys and values in
            // each warp copies RPW rows of 16-byte chunks at a time; lane i owns the address of row(i)
            constexpr int CPR = F::CPR, RPW = 32 / CPR, IT = CPR;
            const int mine = (ln / RPW) * 4 * RPW + pw * RPW + ln % RPW;  // this lane's row of the 128
            const int sub = pw * RPW + ln / CPR, ch = ln % CPR;           // its row (of 4 RPW) and chunk of a copy
            constexpr int AHEAD = 3;      // tiles on their way; the oldest is handed on before another is waited for
            int t_issue = 0, t_done = 0;  // tiles whose copies are issued; tiles handed on
            auto hand_on = [&]() {
                const int t = t_done++, buf = t % NB;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (ln == 0) mbar_arrive(b_full + 8 * buf);
            };
            while (ok && w.next()) {
                const int* const table = a.b.table + w.x.row * a.b.table_stride;
                const int last = 2 * (w.hi - w.lo), hk = w.x.hk;
                // page and row of this lane's position of tile i, and whether it has one (any page number may stand in a table)
                auto page_of = [&](int i, int& r, bool& has) {
                    int unit;
                    bool v;
                    has = i < last;
                    if (has) {
                        w.tile_at(i, unit, v);
                        const int j = w.x.from + (w.lo + unit) * UNIT + mine;
                        has = j < w.x.len;
                        if (has) {
                            const int q = a.by_page(j);
                            r = j - q * a.c.page_size;
                            return __ldg(table + q);
                        }
                    }
                    return -1;
                };
                int r = 0;
                bool has;
                int pg = page_of(0, r, has);
#pragma unroll 1
                for (int i = 0; i < last && ok; ++i) {
                    int unit;
                    bool v;
                    w.tile_at(i, unit, v);
                    uint32_t off = 0xffffffffu;
                    if ((unsigned)pg < (unsigned)a.c.n_pages)
                        off = (uint32_t)pg * a.c.page + (uint32_t)r * a.c.row + (uint32_t)hk * a.c.head;
                    else if (has)
                        atomicOr(a.b.err, kErrKvRange);
                    pg = page_of(i + 1, r, has);
                    if (t_issue - t_done == AHEAD) {
                        cp_async_wait(AHEAD - 1);
                        hand_on();
                    }
                    const int t = t_issue++;
                    if (t >= NB && !__all_sync(0xffffffffu, mbar_test(b_empty + 8 * (t % NB), ((t / NB) - 1) & 1))) {
                        // what has come meanwhile is not held back by a place that is not free yet
                        while (t_done < t && ok) {
                            cp_async_wait(t - t_done - 1);
                            hand_on();
                        }
                        if (!many_wait(b_empty + 8 * (t % NB), ((t / NB) - 1) & 1, ok)) break;
                    }
                    const uint32_t dst = sb + F::oKV + (t % NB) * TILE;
                    const uint8_t* const src = v ? a.c.v : a.c.k;
#pragma unroll
                    for (int k = 0; k < IT; ++k) {
                        const uint32_t o = __shfl_sync(0xffffffffu, off, k * RPW + ln / CPR);
                        const int rr = k * 4 * RPW + sub;
                        const bool have = o != 0xffffffffu;
                        const unsigned long long at = have ? (unsigned long long)o * 64 + ch * 16 : 0;
                        cp16_or_zero(dst + (ch >> 3) * HALF + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4), src + at, have);
                    }
                    cp_async_commit();
                }
            }
            while (t_done < t_issue && ok) {
                cp_async_wait(t_issue - t_done - 1);
                hand_on();
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPfxRegsLow));
        if (warp == 12) {
            // ============================================================ the products
            constexpr uint32_t fmt = BF ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t idS = (1u << 4) | fmt | ((128u >> 3) << 17) | ((128u >> 4) << 24);
            constexpr uint32_t idO = (1u << 4) | fmt | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((128u >> 4) << 24);
            // This warp's time is the block's: what it does between two products is kept short.  Barriers are tested before
            // they are waited for (a wait costs a few hundred cycles even where the phase has gone by), the ring's place and
            // phase are counted on, and descriptors advance by constants.
            auto ready = [&](uint32_t bar, uint32_t parity) {
                ok = ok && mbar_wait_spin(bar, parity);
                return ok;
            };
            uint32_t ph_p = 0, ph_q = 0, slot = 0, ph = 0;  // phases of P (a bit for each half) and of the queries; the ring
            auto tile = [&](uint32_t& addr, uint32_t& gone) {  // the next tile, in the ring's order
                const uint32_t s8 = 8 * slot;
                addr = sb + F::oKV + slot * TILE;
                gone = b_empty + s8;
                const uint32_t was = ph;
                if (++slot == NB) slot = 0, ph ^= 1;
                return ready(b_full + s8, was);
            };
            while (ok && w.next()) {
                const bool wide = w.wide;
                const int nj = wide ? 2 * (w.hi - w.lo) : w.hi - w.lo;
                uint32_t k = 0, kgone = 0, v = 0, vgone = 0;
                // S of job j; the keys are done with after it, or after the other half's
                auto scores = [&](int j) {
                    const int h = j & 1;
                    if ((!wide || h == 0) && !tile(k, kgone)) return false;
                    tc_fence_after();
                    const uint64_t qd = tc_desc(sb + (wide ? h * TILE : 0)), kd = tc_desc(k);
                    const uint32_t tS = tmem + h * 128;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const uint64_t off = ((i >> 2) * HALF + (i & 3) * 32) >> 4;
                        many_mma(tS, qd + off, kd + off, idS, i ? 1u : 0u);
                    }
                    many_commit(b_s + 8 * h);
                    if (!wide || h) many_commit(kgone);
                    if (j == nj - 1) many_commit(b_qf);
                    return true;
                };
                if (!ready(b_q, ph_q) || !scores(0) || (nj > 1 && !scores(1))) break;
                ph_q ^= 1;
                for (int j = 0; j < nj; ++j) {
                    const int h = j & 1;
                    if ((!wide || h == 0) && !tile(v, vgone)) break;
                    const uint64_t vd = many_v_desc(v, HALF);
                    const uint32_t tP = tmem + h * 128, tO = tP + 256, bar = b_p + 16 * h, par = (ph_p >> h) & 1;
                    if (!ready(bar, par)) break;
                    tc_fence_after();
                    const bool by_hand = !I8 && *(volatile int*)&misc[2 + h];
                    if (!by_hand)
#pragma unroll
                        for (int i = 0; i < 4; ++i)  // O += P V
                            many_mma_ta(tO, tP + 8 * i, vd + i * 128, idO, j >= 2 || i ? 1u : 0u);
                    if (!ready(bar + 8, par)) break;
                    tc_fence_after();
                    if (!by_hand)
#pragma unroll
                        for (int i = 4; i < 8; ++i) many_mma_ta(tO, tP + 8 * i, vd + i * 128, idO, 1u);
                    ph_p ^= 1u << h;
                    if (!wide || h) many_commit(vgone);
                    if (j + 2 >= nj)
                        many_commit(b_o + 8 * h);
                    else if (!scores(j + 2))
                        break;
                }
            }
        } else if (I8 && warp == 13) {
            // ============================================================ codes in, as they lie
            // A page's rows of a head are one piece where rows follow one another, else a row is.  What is not copied (past the
            // prefix's end, pages out of range) stays whatever codes lay there: numbers, with no weight or a scale of zero.
            constexpr int NS = F::NSTG ? F::NSTG : 1;
            const bool together = a.c.row * 64 == D * F::ES;
            int t = 0;
            while (ok && w.next()) {
                const int* const table = a.b.table + w.x.row * a.b.table_stride;
                const int last = 2 * (w.hi - w.lo);
#pragma unroll 1
                for (int i = 0; i < last; ++i, ++t) {
                    int unit;
                    bool v;
                    w.tile_at(i, unit, v);
                    const int v0 = w.x.from + (w.lo + unit) * UNIT, v1 = min(v0 + UNIT, w.x.len);
                    const uint32_t bar = b_stg + 8 * (t % NS), dst = sb + F::oSTG + (t % NS) * F::STG;
                    if (t >= NS && !many_wait(b_stge + 8 * (t % NS), ((t / NS) - 1) & 1, ok)) break;
                    const uint8_t* const src = (v ? a.c.v : a.c.k) + 64ull * ((uint32_t)w.x.hk * a.c.head);
                    const int p0 = a.by_page(v0), runs = together ? a.by_page(v1 - 1) - p0 + 1 : v1 - v0;
                    // this lane's pieces: from position `from` on, n of them, at row r of page pg
                    auto piece = [&](int k, int& from, int& n, int& pg, int& r) {
                        const int q = together ? p0 + k : a.by_page(v0 + k);
                        from = together ? max(v0, q * a.c.page_size) : v0 + k;
                        n = together ? min(v1, (q + 1) * a.c.page_size) - from : 1;
                        r = from - q * a.c.page_size;
                        pg = __ldg(table + q);
                        return (unsigned)pg < (unsigned)a.c.n_pages;
                    };
                    int from, n, pg, r, rows = 0;
                    for (int k = ln; k < runs; k += 32) {
                        if (piece(k, from, n, pg, r))
                            rows += n;
                        else
                            atomicOr(a.b.err, kErrKvRange);
                    }
                    rows = __reduce_add_sync(0xffffffffu, rows);
                    if (ln == 0) mbar_arrive_expect_tx(bar, (uint32_t)rows * D);
                    __syncwarp();
                    for (int k = ln; k < runs; k += 32)
                        if (piece(k, from, n, pg, r))
                            bulk_g2s(dst + (from - v0) * D, src + 64ull * ((uint32_t)pg * a.c.page + (uint32_t)r * a.c.row),
                                     (uint32_t)n * D, bar);
                    __syncwarp();
                }
            }
            // none of the copies outlives the block, whatever has become of their readers
            bool come = true;
            for (int k = max(t - NS, 0); k < t; ++k) many_wait(b_stg + 8 * (k % NS), (k / NS) & 1, come);
            ok = ok && come;
        } else if (I8 && warp == 14) {
            // ============================================================ the scales
            int q = 0;  // units so far
            while (ok && w.next()) {
                const int* const table = a.b.table + w.x.row * a.b.table_stride;
#pragma unroll 1
                for (int u = w.lo; u < w.hi; ++u, ++q) {
                    float sc[2][4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int j = w.x.from + u * UNIT + 32 * i + ln, p = a.by_page(j);
                        const int pg = j < w.x.len ? __ldg(table + p) : -1;
                        sc[0][i] = sc[1][i] = 0.f;
                        if ((unsigned)pg < (unsigned)a.c.n_pages) {
                            const long long so = pg * a.c.spage + (long long)w.x.hk * a.c.page_size + j - p * a.c.page_size;
                            sc[0][i] = __ldg(a.c.ks + so);
                            sc[1][i] = __ldg(a.c.vs + so);
                        }
                    }
                    const int slot = q % NSC;
                    if (q >= NSC && !many_wait(b_scf + 8 * slot, ((q / NSC) - 1) & 1, ok)) break;
                    float* const at = reinterpret_cast<float*>(smem + F::oSC + slot * 1024);
#pragma unroll
                    for (int i = 0; i < 4; ++i) at[32 * i + ln] = sc[0][i], at[128 + 32 * i + ln] = sc[1][i];
                    __syncwarp();
                    if (ln == 0) mbar_arrive(b_sc + 8 * slot);
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

template <class T, class C, int D>
cudaError_t launch(const AttnArgs& a, const PrefixArgs& p, int blocks, cudaStream_t s) {
    constexpr int bytes = PfxCfg<C, D>::BYTES;
    static_assert(bytes <= 227 * 1024, "shared memory of a block");
    static SmemOptIn opted;
    const cudaError_t e = opted(reinterpret_cast<const void*>(attn_prefix_kernel<T, C, D>), bytes);
    if (e != cudaSuccess) return e;
    return launch_early(attn_prefix_kernel<T, C, D>, blocks, kPfxThreads, bytes, s, a, p);
}

template <class T, int D>
cudaError_t by_cache(int ct, const AttnArgs& a, const PrefixArgs& p, int blocks, cudaStream_t s) {
    if (ct == T_F16) return launch<T, __half, D>(a, p, blocks, s);
    return launch<T, int8_t, D>(a, p, blocks, s);
}

}  // namespace

cudaError_t launch_attn_prefix(int ct, int dt, int D, const AttnArgs& a, const PrefixArgs& p, int blocks, cudaStream_t s) {
    if (ct == T_BF16)
        return D == 64 ? launch<__nv_bfloat16, __nv_bfloat16, 64>(a, p, blocks, s)
                       : launch<__nv_bfloat16, __nv_bfloat16, 128>(a, p, blocks, s);
    if (dt == T_F16) return D == 64 ? by_cache<__half, 64>(ct, a, p, blocks, s) : by_cache<__half, 128>(ct, a, p, blocks, s);
    return D == 64 ? by_cache<__nv_bfloat16, 64>(ct, a, p, blocks, s) : by_cache<__nv_bfloat16, 128>(ct, a, p, blocks, s);
}

}  // namespace hc
