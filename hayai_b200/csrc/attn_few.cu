// attn_few.cu -- attention over the paged cache for sequences with few rows per kv head (single
// tokens, short drafts): bound by reading the cache.
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(c q_i . k_j - m_i),   c = scale log2 e
// in one pass with the running maximum m_i and sum of every row, lse_i = (m_i + log2 sum) ln 2.
// m_i need not be the maximum itself, only near it: it moves when a score passes it by 8 (weights
// up to 2^8), so after the first units a unit's maximum costs one vote.
//
// Both products run on the tensor cores transposed, S^T = K Q^T and O^T = V^T P^T with
// mma.m16n8k16: the cache's rows fill the 16 rows of the first operand, and the 8 query rows of a
// group of heads the 8 columns, where the plain orientation would leave half or more of 16 query
// rows empty.  The order of k inside a product is free as long as both operands agree, so every
// lane takes 16 adjacent bytes of a cache row (8-bit: four k steps; 16-bit: two), and V^T's pairs
// of tokens come from two rows by PRMT, with no transposed copy.  S^T's accumulators become P^T's
// operand with one MOVMATRIX per 8 tokens.
//
// Formats.  8-bit codes are exact in f16 and in bf16.  For 16-bit results V's go in as f16 1152 + code
// (no subtraction: bits 0x6400 + code + 128), and the product's accumulator starts at -1152 sum p of
// the weights as rounded, so that the codes' own product is left.  (The larger sums are rounded to about 1e-4
// of a code, 1e-6 of the values' largest, also where a result is nearly zero; K's codes are taken as they are,
// as the lse is f32 whatever the results are.)  A token's K scale multiplies its score and its V scale its
// weights.  For f32 results the codes are taken as they are, and the weights times scales as bf16 terms.
//
// Query rows are scaled by a power of two to have their largest element in [2^14, 2^15), the top of f16, and
// rounded to the products' type: f16 and bf16 rows are exact to 2^-39 of the largest element; f32 rows are
// split into 2 f16 terms (22 bits, and 2^-39 of the largest) or 3 bf16 terms (24 bits), f16 rows on a bf16
// cache into 2 (11 bits of 16).  Weights are rounded to one term of the cache's type, of the order of the
// 16-bit results' own rounding (f16 results on a bf16 cache: two), for f32 results to two f16 or three bf16
// terms.  Where they go in as f16, a unit's weights of a row are first brought to a fixed size by a power of
// two, which multiplies the unit's product: f16 then holds them however far they are under the row's maximum
// and whatever the scales are (8-bit: to at most 1, and what is under 2^-25 of the unit's largest is lost;
// 16-bit: to 2^15, and 2^-40); bf16 terms need no such care.  All sums are f32; for f32 results and f16
// weights a unit's products are added to zero and then to the running sum in FADD, as the tensor cores' own
// chained additions truncate.
//
// The workers of the line (attn_rows.cuh) are warps, one block of 8 or 12 of them per SM.  A warp
// streams its units through a ring of 16-byte asynchronous copies of its own, whose issue runs ahead
// over tile boundaries, and meets the others only once: a tile that it has whole it writes itself;
// of its first and last tile's pieces it leaves the partial (m, l, O) in shared memory or in the
// workspace, where after one barrier the block joins its warps' pieces, and the last block of a
// tile's row the blocks'.
// Measured: 64 sequences of 300 to 12000 8-bit tokens 100 us (4.2 TB/s, 66 % of the copy rate), one of
// 131071 f16 tokens 58 us (4.6 TB/s, 72 %), one of 1001 8-bit tokens 11.7 us in a graph.
// (Tiles shared by all warps of a block, with a barrier and a joining at each tile's end, took
// 160 us where this takes 100 us: 64 sequences of 300 to 12000 tokens, 64 heads on 8.)
#include <math.h>

#include "attn_rows.cuh"

namespace hc {

template <class T, class C>
struct FewTerms {
    static constexpr bool kBf = sizeof(C) == 2 && !(__is_same(C, __half));  // bf16 products for the scores
    static constexpr int Q = sizeof(T) == 4 ? (kBf ? 3 : 2) : (kBf && __is_same(T, __half)) ? 2 : 1;
    static constexpr bool pBf = kBf || (sizeof(C) == 1 && sizeof(T) == 4);       // bf16 products for the result
    static constexpr int P = sizeof(T) == 4 ? (pBf ? 3 : 2) : (pBf && __is_same(T, __half)) ? 2 : 1;
    static constexpr bool kBias = sizeof(C) == 1 && sizeof(T) == 2;  // V's codes as 1152 + code
    static constexpr bool kNorm = !pBf;                          // f16 products for the result: weights brought to f16's range
    static constexpr int kTop = kBias ? 1 : -14;                 // a unit's largest weight is divided by 2^kTop times its power of two
};

template <class T, class C, int D, int NT>
struct FewCfg {
    static constexpr int ES = sizeof(C), CPR = D * ES / 16;  // 16-byte chunks of a row
    static constexpr int ST = CPR == 16 ? 16 : 32;           // tokens of a unit
    static constexpr int KB = ST * CPR * 16;                 // bytes of a unit's keys (or values)
    static constexpr int SB = 2 * KB + (ES == 1 ? 8 * ST : 0);
    static constexpr int W = NT == 1 && FewTerms<T, C>::Q == 1 ? 12 : 8;  // warps of a block
    static constexpr int NS = CPR == 4 ? 4 : 2;                   // stages of a warp's ring
    static constexpr int QB = D / 16 * NT * FewTerms<T, C>::Q * 256;  // a query tile as B operands
    static constexpr int WB = NS * SB + QB + 32 * NT;  // bytes of a warp: ring, queries, rows' scales
    static constexpr int PS = 8 * NT * (D + 2);  // floats of a partial result: rows of D values, then (m, l) of each
};

// D (+)= A B, 16 x 8 x 16 (mma16816's bf16 twin).
__device__ __forceinline__ void mma16816_bf(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool BF>
__device__ __forceinline__ void mma_any(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (BF)
        mma16816_bf(c, a[0], a[1], a[2], a[3], b0, b1);
    else
        mma16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
// D = A B + (c0, c1, c0, c1).
template <bool BF>
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0,
                                         float c1) {
    if constexpr (BF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%11,%10,%11};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%11,%10,%11};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// The next term of a pair's expansion: (lo, hi) rounded to the products' type, and what is left.
template <bool BF>
__device__ __forceinline__ uint32_t split_pair(float& x, float& y) {
    if constexpr (BF) {
        const uint32_t u = pack_b2(x, y);
        x -= __uint_as_float(u << 16);
        y -= __uint_as_float(u & 0xffff0000u);
        return u;
    } else {
        const uint32_t u = pack_h2(x, y);
        const float2 f = __half22float2(u32_as_h2(u));
        x -= f.x;
        y -= f.y;
        return u;
    }
}

__device__ __forceinline__ void cp4_or_zero(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
    return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
    return r;
}
__device__ __forceinline__ float lds32f(uint32_t a) {
    float r;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(r) : "r"(a));
    return r;
}

// Four adjacent values of a query row, as loaded.
template <class T>
struct FewRaw {
    using type = uint2;
    static __device__ __forceinline__ void values(const uint2& u, float (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t b = (uint16_t)((i < 2 ? u.x : u.y) >> (16 * (i & 1)));
            if constexpr (__is_same(T, __half))
                x[i] = h2f(b);
            else
                x[i] = __uint_as_float((uint32_t)b << 16);
        }
    }
};
template <>
struct FewRaw<float> {
    using type = float4;
    static __device__ __forceinline__ void values(const float4& f, float (&x)[4]) { x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w; }
};

// Places of 16-byte chunks in a stage, permuted so that the 8 lanes of a load's phase (two rows by
// four chunks of K, four rows by two chunks of V) touch all banks once.
template <int CPR>
__device__ __forceinline__ uint32_t few_k_at(int r, int c) {
    return (r * CPR + (CPR == 4 ? c : c ^ ((r & 1) << 2))) * 16;
}
template <int CPR>
__device__ __forceinline__ uint32_t few_v_at(int r, int c) {
    if constexpr (CPR == 4) {
        const int rr = (r & ~3) | ((r & 1) << 1) | ((r >> 1) & 1);
        return (rr * 4 + (c ^ (((r >> 2) & 1) << 1))) * 16;
    } else {
        return (r * CPR + (c ^ (((r >> 1) & 3) << 1))) * 16;
    }
}

// A warp's walk over its units: unit `st` of the item's [0, hi).
struct FewWalk {
    AttnIter it;
    int st, hi, b0, b1;
    bool live;
    __device__ __forceinline__ void enter() {
        st = max(b0 - it.u_item, 0);
        hi = min(b1 - it.u_item, it.t.units);
    }
    // On to the next item with a unit of this warp, if there is one.
    __device__ __forceinline__ void settle(const AttnArgs& a, int rows, int unit) {
        while (st >= hi) {
            if (it.u_item + it.t.span >= b1) {
                live = false;
                return;
            }
            it.next(a, rows, unit);
            enter();
        }
    }
};

template <class T, class C, int D, int NT>
__global__ void __launch_bounds__(32 * FewCfg<T, C, D, NT>::W, 1) attn_few_kernel(const __grid_constant__ AttnArgs a) {
    using F = FewCfg<T, C, D, NT>;
    using X = FewTerms<T, C>;
    constexpr int W = F::W, THREADS = 32 * W, ST = F::ST, CPR = F::CPR, MT = ST / 16, KS = D / 16, ROWS = 8 * NT, I8 = F::ES == 1;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ AttnShared shared_s[W + 1];  // tiles that start in warp w and go on past it; the block's first
    __shared__ __align__(8) int scratch[32];
    const int w = threadIdx.x >> 5, ln = lane_id(), g = ln >> 2, t4 = ln & 3;
    const uint32_t ring = smem_addr(smem) + w * F::WB;
    uint8_t* const qf = smem + w * F::WB + F::NS * F::SB;
    float* const rscale = reinterpret_cast<float*>(qf + F::QB);  // [ROWS]

    __shared__ float* place_s[W][2];  // where a warp's last (0) and first (1) piece of a shared tile is

    // few sequences (a single one above all, whose call is short): every warp schedules for itself
    const bool lanes = a.b.n_seq <= 32 && a.max_rows <= 8 * ROWS;
    int* const pre = reinterpret_cast<int*>(smem);
    AttnLanes lv;
    const int U = lanes ? attn_schedule_lanes(a, ROWS, ST, lv) : attn_schedule<THREADS>(a, ROWS, ST, pre, scratch);
    const int G = min((int)gridDim.x, max(1, U / W)), c = blockIdx.x;
    if (U <= 0 || c >= G) return;
    FewWalk pw;  // the copies' walk: units are issued NS - 1 ahead
    const AttnShares share(U, G * W);
    pw.b0 = share.begin(c * W + w);
    pw.b1 = share.begin(c * W + w + 1);
    pw.live = pw.b0 < pw.b1;
    if (pw.live) {
        if (lanes)
            pw.it.seek(a, lv, pw.b0, ROWS, ST);
        else
            pw.it.seek(a, pre, pw.b0, ROWS, ST);
        pw.enter();
    }
    if (threadIdx.x <= W) shared_s[threadIdx.x].valid = 0;
    __syncthreads();  // `pre` is read
    AttnIter it = pw.it;
    const int b0 = pw.b0, b1 = pw.b1;
    if (pw.live) pw.settle(a, ROWS, ST);
    int pg = -1, pr = 0;  // page and row of this lane's token of the unit to be issued
    auto look_up = [&]() {
        pg = -1;
        if (!pw.live) return;
        const int v = pw.st * ST + ln;
        if (ln < ST && v < pw.it.t.nvis) {
            const int j = v < pw.it.t.n1 ? v : v - pw.it.t.n1 + pw.it.t.lo;
            const int p = a.by_page(j);
            pr = j - p * a.c.page_size;
            pg = __ldg(a.b.table + pw.it.s * a.b.table_stride + p);
            if ((unsigned)pg >= (unsigned)a.c.n_pages) {
                atomicOr(a.b.err, kErrKvRange);
                pg = -1;
            }
        }
    };
    int islot = 0;
    auto issue = [&]() {
        if (pw.live) {
            const uint32_t base = ring + islot * F::SB;
            const bool ok = pg >= 0;
            const uint32_t off = ok ? (uint32_t)pg * a.c.page + (uint32_t)pr * a.c.row + (uint32_t)pw.it.hk * a.c.head
                                    : 0xffffffffu;
#pragma unroll
            for (int i = 0; i < ST * CPR / 32; ++i) {
                const int r = (i * 32 + ln) / CPR, ch = ln % CPR;
                const uint32_t o = __shfl_sync(0xffffffffu, off, r);
                const bool have = o != 0xffffffffu;
                const unsigned long long at = have ? (unsigned long long)o * 64 + ch * 16 : 0;
                cp16_or_zero(base + few_k_at<CPR>(r, ch), a.c.k + at, have);
                cp16_or_zero(base + F::KB + few_v_at<CPR>(r, ch), a.c.v + at, have);
            }
            if constexpr (I8) {
                const long long so = ok ? pg * a.c.spage + (long long)pw.it.hk * a.c.page_size + pr : 0;
                cp4_or_zero(base + 2 * F::KB + ln * 4, a.c.ks + so, ok);
                cp4_or_zero(base + 2 * F::KB + ST * 4 + ln * 4, a.c.vs + so, ok);
            }
            islot = islot + 1 == F::NS ? 0 : islot + 1;
            if (++pw.st >= pw.hi) pw.settle(a, ROWS, ST);
            look_up();
        }
        cp_async_commit();
    };
    // Eight of the tile's query rows as loaded, 4 values to a lane: on their way at once, the first eight before
    // the copies that wait for page numbers.  (All rows of a tile in one straight run are so much code that a short
    // call spends its time fetching instructions.)
    using Raw = typename FewRaw<T>::type;
    Raw raw[8];
    auto load_queries = [&](int r0) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            raw[r] = Raw{};
            if (r0 + r < it.t.nr && ln < D / 4) {
                const int row = it.t.r0 + r0 + r, tr = a.by_group(row);
                raw[r] = __ldg(reinterpret_cast<const Raw*>((const T*)a.q + (long long)(it.q.q0 + tr) * a.ldq +
                                                            (it.hk * a.group + row - tr * a.group) * D + 4 * ln));
            }
        }
    };
    if (b0 < b1) load_queries(0);
    look_up();
#pragma unroll
    for (int i = 0; i < F::NS - 1; ++i) issue();

    int cslot = 0;
    while (b0 < b1) {  // the warp's tiles
        const AttnTile& tl = it.t;
        const int lo = max(b0 - it.u_item, 0), hi = min(b1 - it.u_item, tl.units);
        if (lo >= hi) {
            if (it.u_item + tl.span >= b1) break;
            it.next(a, ROWS, ST);
            load_queries(0);
            continue;
        }
        // ---- the query tile as B operands
#pragma unroll 1
        for (int n = 0; n < NT; ++n) {
            if (n) load_queries(8 * n);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int r = 8 * n + q;
                float x[4];
                FewRaw<T>::values(raw[q], x);
                float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
                m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // not negative: order as bits
                // m brought to [2^14, 2^15) (none for infinity and NaN; the smallest to less)
                const RowSize size(__float_as_uint(m));
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] *= size.by;
                if (ln == 0) rscale[r] = size.back * a.scale * 1.44269504f;
                if (ln < D / 4) {
                    // d = 4 ln + i: 16-byte chunk of the cache row, its k step and the lane that holds it
                    const int ch = I8 ? ln >> 2 : ln >> 1, j = I8 ? 4 * (ch >> 2) + (ln & 3) : 2 * (ch >> 2) + (ln & 1);
                    uint8_t* dst = qf + (j * NT + n) * X::Q * 256 + (q * 4 + (ch & 3)) * 8;
#pragma unroll
                    for (int s = 0; s < X::Q; ++s)
                        *reinterpret_cast<uint2*>(dst + s * 256) =
                            make_uint2(split_pair<X::kBf>(x[0], x[1]), split_pair<X::kBf>(x[2], x[3]));
                }
            }
        }
        __syncwarp();
        float m[NT][2], l[NT][2], o[KS][NT][4], rs[NT][2];
        int lim[NT][2], wlo[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = n * 8 + 2 * t4 + e;
                m[n][e] = -INFINITY;
                l[n][e] = 0.f;
                rs[n][e] = rscale[r];
                const int pos = it.q.len - (it.q.q1 - it.q.q0) + a.by_group(tl.r0 + r);
                lim[n][e] = r >= tl.nr ? -1 : a.causal ? pos : it.q.len - 1;
                wlo[n][e] = a.window ? pos - a.window + 1 : 0;
            }
#pragma unroll
        for (int d = 0; d < KS; ++d)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][n][e] = 0.f;

        for (int st = lo; st < hi; ++st) {
            issue();
            cp_async_wait(F::NS - 1);
            __syncwarp();
            const uint32_t kb = ring + cslot * F::SB, vb = kb + F::KB, sb = kb + 2 * F::KB;
            cslot = cslot + 1 == F::NS ? 0 : cslot + 1;
            // ---- S^T = K Q^T
            float s[MT][NT][4];
#pragma unroll
            for (int cg = 0; cg < CPR / 4; ++cg) {
                uint4 ka[MT], kc[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    ka[i] = lds128(kb + few_k_at<CPR>(16 * i + g, t4 + 4 * cg));
                    kc[i] = lds128(kb + few_k_at<CPR>(16 * i + g + 8, t4 + 4 * cg));
                }
#pragma unroll
                for (int jj = 0; jj < (I8 ? 4 : 2); ++jj) {
                    uint32_t A[MT][4];
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const uint32_t wa[4] = {ka[i].x, ka[i].y, ka[i].z, ka[i].w};
                        const uint32_t wc[4] = {kc[i].x, kc[i].y, kc[i].z, kc[i].w};
                        if constexpr (I8) {
                            const uint32_t fa = wa[jj] ^ 0x80808080u, fc = wc[jj] ^ 0x80808080u;
                            A[i][0] = prmt(fa, 0x64646464u, 0x4140u);
                            A[i][1] = prmt(fc, 0x64646464u, 0x4140u);
                            A[i][2] = prmt(fa, 0x64646464u, 0x4342u);
                            A[i][3] = prmt(fc, 0x64646464u, 0x4342u);
#pragma unroll
                            for (int e = 0; e < 4; ++e) A[i][e] = hsub2_u32(A[i][e], 0x64806480u);
                        } else {
                            A[i][0] = wa[2 * jj];
                            A[i][1] = wc[2 * jj];
                            A[i][2] = wa[2 * jj + 1];
                            A[i][3] = wc[2 * jj + 1];
                        }
                    }
                    const int j = (I8 ? 4 : 2) * cg + jj;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int q = 0; q < X::Q; ++q) {
                            const uint2 b = *reinterpret_cast<const uint2*>(qf + ((j * NT + n) * X::Q + q) * 256 + ln * 8);
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                if (j == 0 && q == 0)
                                    mma_from<X::kBf>(s[i][n], A[i], b.x, b.y, 0.f, 0.f);
                                else
                                    mma_any<X::kBf>(s[i][n], A[i], b.x, b.y);
                            }
                        }
                }
            }
            // ---- scores in units of log 2, masked
            const int v0 = st * ST, v1 = v0 + ST;
            const int j0 = v0 < tl.n1 ? v0 : v0 - tl.n1 + tl.lo, j1 = v1 - tl.n1 + tl.lo - 1;
            const bool full = v1 <= tl.nvis &&
                              (tl.p_lo == tl.p_hi || !a.causal ||
                               (j1 <= tl.p_lo && (!a.window || v1 <= tl.n1 || (v0 >= tl.n1 && j0 > tl.p_hi - a.window))));
            float vsc[MT][2];
            bool vodd = false;  // a V scale that is not finite in a unit that some row does not see whole
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float ksc[2] = {1.f, 1.f};
                vsc[i][0] = vsc[i][1] = 1.f;
                if constexpr (I8) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        ksc[h] = lds32f(sb + (16 * i + 8 * h + g) * 4);
                        vsc[i][h] = lds32f(sb + ST * 4 + (16 * i + 8 * h + g) * 4);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[i][n][e] *= I8 ? rs[n][e & 1] * ksc[e >> 1] : rs[n][e & 1];
                    }
            }
            if (!full) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int v = v0 + 16 * i + 8 * h + g;
                        const int j = v < tl.n1 ? v : v - tl.n1 + tl.lo;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const bool see = v < tl.nvis && j <= lim[n][e] && (j >= wlo[n][e] || j < a.sink);
                                if (!see) s[i][n][2 * h + e] = -INFINITY;
                            }
                        if (I8 && !(fabsf(vsc[i][h]) <= 3e38f)) vodd = true;
                    }
            }
            // ---- move the maxima where a score passes them by 8
            bool up = false;
            float mx[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    mx[n][e] = fmaxf(s[0][n][e], s[0][n][e + 2]);
                    if constexpr (MT == 2) mx[n][e] = fmaxf(mx[n][e], fmaxf(s[MT - 1][n][e], s[MT - 1][n][e + 2]));
                    up |= mx[n][e] > m[n][e] + 8.f;
                }
            if (__any_sync(0xffffffffu, up)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = mx[n][e];
#pragma unroll
                        for (int q = 4; q < 32; q <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, q));
                        x = fmaxf(x, m[n][e]);
                        const float f = x == -INFINITY ? 1.f : ex2(m[n][e] - x);
                        m[n][e] = x;
                        l[n][e] *= f;
#pragma unroll
                        for (int d = 0; d < KS; ++d) {
                            o[d][n][e] *= f;
                            o[d][n][e + 2] *= f;
                        }
                    }
            }
            // ---- weights, and P^T as B operands
            uint32_t pb[MT][NT][X::P][2];
            float unit[NT][2];  // f16: what the unit's weights of a row are divided by
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
                float p[MT][4];
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[i][e] = ex2(s[i][n][e] - (e & 1 ? m1 : m0));
                        l[n][e & 1] += p[i][e];
                        if constexpr (I8) p[i][e] *= vsc[i][e >> 1];
                    }
                if (I8 && vodd) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (s[i][n][e] == -INFINITY) p[i][e] = 0.f;
                }
                unit[n][0] = unit[n][1] = 1.f;
                if constexpr (X::kNorm) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(fmaxf(fabsf(p[0][e]), fabsf(p[0][e + 2])),
                                        fmaxf(fabsf(p[MT - 1][e]), fabsf(p[MT - 1][e + 2])));
#pragma unroll
                        for (int q = 4; q < 32; q <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, q));
                        // exponents that leave the power and its reciprocal normal numbers
                        const uint32_t b = min(max(__float_as_uint(x) >> 23, X::kBias ? 2u : 15u), 252u);
                        unit[n][e] = __uint_as_float((b + X::kTop) << 23);
                        const float inv = __uint_as_float((254 - X::kTop - b) << 23);
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            p[i][e] *= inv;
                            p[i][e + 2] *= inv;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int q = 0; q < X::P; ++q)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            pb[i][n][q][h] = movmatrix(split_pair<X::pBf>(p[i][2 * h], p[i][2 * h + 1]));
            }
            // ---- O^T += V^T P^T
            bool odd = false;  // a value that is not finite in a unit that some row does not see whole
            if constexpr (!I8) {
                if (!full) {
                    constexpr uint32_t E = X::pBf ? 0x7f80u : 0x7c00u;
#pragma unroll 4
                    for (int i = 0; i < F::KB / 512; ++i) {
                        const uint4 x = lds128(vb + i * 512 + ln * 16);
                        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) odd |= (y[k] & E) == E || ((y[k] >> 16) & E) == E;
                    }
                    odd = __any_sync(0xffffffffu, odd);
                }
            }
            if (odd) {  // rare: 0 * infinity must not reach a row that is masked there, so no products
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll 1
                    for (int k = 0; k < 16; ++k) {
                        uint32_t word[KS];
#pragma unroll
                        for (int d = 0; d < KS; ++d) {
                            const uint4 x = lds128(vb + few_v_at<CPR>(16 * i + k, g + 8 * (d >> 2)));
                            word[d] = (d & 3) == 0 ? x.x : (d & 3) == 1 ? x.y : (d & 3) == 2 ? x.z : x.w;
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float sv = k < 8 ? s[i][n][e] : s[i][n][e + 2];
                                const float sc = __shfl_sync(0xffffffffu, sv, 4 * (k & 7) + t4);
                                if (sc == -INFINITY) continue;
                                const float p = ex2(sc - (m[n][e] == -INFINITY ? 0.f : m[n][e]));
#pragma unroll
                                for (int d = 0; d < KS; ++d) {
                                    const uint32_t lo16 = word[d] & 0xffffu, hi16 = word[d] >> 16;
                                    o[d][n][e] += p * (X::pBf ? __uint_as_float(lo16 << 16) : h2f((uint16_t)lo16));
                                    o[d][n][e + 2] += p * (X::pBf ? __uint_as_float(hi16 << 16) : h2f((uint16_t)hi16));
                                }
                            }
                    }
            } else {
                constexpr bool OWN = sizeof(T) == 4 || X::kNorm;  // a unit's products are added to zero, then to the sum
                if constexpr (I8) {
                    uint4 vw[MT][4];  // 16 (D = 128) or 8 (D = 64) adjacent values of four tokens
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int r = 16 * i + 2 * t4 + (k & 1) + 8 * (k >> 1);
                            if constexpr (D == 128) {
                                vw[i][k] = lds128(vb + few_v_at<CPR>(r, g));
                            } else {
                                const uint2 x = lds64(vb + few_v_at<CPR>(r, g >> 1) + 8 * (g & 1));
                                vw[i][k] = make_uint4(x.x, x.y, 0, 0);
                            }
                            if constexpr (X::kBias) {
                                vw[i][k].x ^= 0x80808080u, vw[i][k].y ^= 0x80808080u;
                                vw[i][k].z ^= 0x80808080u, vw[i][k].w ^= 0x80808080u;
                            }
                        }
                    float pbias[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        pbias[n][0] = pbias[n][1] = 0.f;
                        if constexpr (X::kBias) {  // -1152 sum p, by a product with ones
                            const uint32_t one[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
                            float z[4];
                            mma_from<false>(z, one, pb[0][n][0][0], pb[0][n][0][1], 0.f, 0.f);
                            if constexpr (MT == 2) mma_any<false>(z, one, pb[MT - 1][n][0][0], pb[MT - 1][n][0][1]);
                            pbias[n][0] = -1152.f * z[0];
                            pbias[n][1] = -1152.f * z[1];
                        }
                    }
#pragma unroll
                    for (int d = 0; d < KS; ++d) {
                        float z[NT][4];
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            uint32_t A[4];
                            const int wi = d >> 1;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {  // e & 1: value 2 d or 2 d + 1; e >> 1: token pair
                                const uint4 &x = vw[i][2 * (e >> 1)], &y = vw[i][2 * (e >> 1) + 1];
                                const uint32_t xa = wi == 0 ? x.x : wi == 1 ? x.y : wi == 2 ? x.z : x.w;
                                const uint32_t ya = wi == 0 ? y.x : wi == 1 ? y.y : wi == 2 ? y.z : y.w;
                                const uint32_t b = 2 * (d & 1) + (e & 1);
                                const uint32_t u = prmt(xa, ya, b | (b << 4) | ((4 + b) << 8) | ((4 + b) << 12));
                                if constexpr (X::kBias) {
                                    A[e] = lop3_and_or(u, 0x00ff00ffu, 0x64006400u);  // 1152 + code (words flipped)
                                } else {  // code = (128 + low 7 bits) - (128 + 128 * sign bit), exact in bf16
                                    const uint32_t lo7 = lop3_and_or(u, 0x007f007fu, 0x43004300u);
                                    const uint32_t sg = lop3_and_or(u, 0x00800080u, 0x43004300u);
                                    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&lo7),
                                                                     *reinterpret_cast<const __nv_bfloat162*>(&sg));
                                    A[e] = *reinterpret_cast<const uint32_t*>(&v);
                                }
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int q = 0; q < X::P; ++q) {
                                    if (i == 0 && q == 0)
                                        mma_from<X::pBf>(z[n], A, pb[i][n][q][0], pb[i][n][q][1], pbias[n][0], pbias[n][1]);
                                    else
                                        mma_any<X::pBf>(z[n], A, pb[i][n][q][0], pb[i][n][q][1]);
                                }
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[d][n][e] = fmaf(z[n][e], unit[n][e & 1], o[d][n][e]);
                    }
                } else {
#pragma unroll
                    for (int cg = 0; cg < CPR / 8; ++cg) {
                        uint4 vw[MT][4];
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                vw[i][k] = lds128(vb + few_v_at<CPR>(16 * i + 2 * t4 + (k & 1) + 8 * (k >> 1), g + 8 * cg));
#pragma unroll
                        for (int dd = 0; dd < 4; ++dd) {
                            const int d = 4 * cg + dd;
                            float z[NT][4];
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e) z[n][e] = OWN ? 0.f : o[d][n][e];
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                uint32_t A[4];
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const uint4 &x = vw[i][2 * (e >> 1)], &y = vw[i][2 * (e >> 1) + 1];
                                    const uint32_t xa = dd == 0 ? x.x : dd == 1 ? x.y : dd == 2 ? x.z : x.w;
                                    const uint32_t ya = dd == 0 ? y.x : dd == 1 ? y.y : dd == 2 ? y.z : y.w;
                                    A[e] = prmt(xa, ya, e & 1 ? 0x7632u : 0x5410u);
                                }
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int q = 0; q < X::P; ++q)
                                        mma_any<X::pBf>(z[n], A, pb[i][n][q][0], pb[i][n][q][1]);
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    o[d][n][e] = X::kNorm ? fmaf(z[n][e], unit[n][e & 1], o[d][n][e])
                                                 : OWN    ? o[d][n][e] + z[n][e]
                                                          : z[n][e];
                        }
                    }
                }
            }
            __syncwarp();  // the slot is free for the next issue
        }

        // ---- the tile's end: lane (g, t4) holds values 64 cg + 8 g + x (8-bit: (D / 8) g + x) of rows 2 t4 + e
        const bool whole = lo == 0 && hi == tl.units;
        // a piece goes to the workspace, or, the warp's last, to its own ring, which is done with
        const bool done = it.u_item + tl.span >= b1;
        if (done) asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        float* const part = done ? reinterpret_cast<float*>(smem + w * F::WB)
                                 : a.part + (size_t)(2 * (c * W + w) + (lo == 0)) * F::PS;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int q = 4; q < 32; q <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], q);
                const int r = n * 8 + 2 * t4 + e;
                if (r >= tl.nr) continue;
#pragma unroll
                for (int d = 0; d < KS; d += 2) {
                    const int col = I8 ? (D / 8) * g + 2 * d : 64 * (d >> 2) + 8 * g + 2 * (d & 3);
                    const float y[4] = {o[d][n][e], o[d][n][e + 2], o[d + 1][n][e], o[d + 1][n][e + 2]};
                    if (whole)
                        attn_store<T>(a, it.q.q0, it.hk, tl.r0 + r, D, col, y, l[n][e]);
                    else
                        *reinterpret_cast<float4*>(part + r * D + col) = make_float4(y[0], y[1], y[2], y[3]);
                }
                if (g == 0) {
                    if (whole)
                        attn_store_lse(a, it.q.q0, it.hk, tl.r0 + r, m[n][e], l[n][e]);
                    else
                        *reinterpret_cast<float2*>(part + ROWS * D + 2 * r) = make_float2(m[n][e], l[n][e]);
                }
            }
        if (!whole && ln == 0) {
            place_s[w][lo == 0] = part;
            if (lo == 0 || w == 0) shared_s[lo == 0 ? w : W] = {1, it.q.q0, it.hk, tl.r0, tl.nr, it.u_item, tl.units};
        }
        if (done) break;
        it.next(a, ROWS, ST);
        load_queries(0);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();

    // ---- the tiles of several warps: a row per warp at a time, its D values over D / 4 lanes; a tile of several
    // blocks is joined from their results, row by row, by the block whose row comes last
    float* const bpart = a.part + (size_t)2 * gridDim.x * W * F::PS;  // the blocks' partial results, two each
    int turn = 0;
#pragma unroll 1
    for (int x = 0; x <= W; ++x) {
        const AttnShared sh = shared_s[x];
        if (!sh.valid) continue;
        const int wf = share.owner(sh.u_item), wl = share.owner(sh.u_item + sh.units - 1), bf = wf / W, bl = wl / W;
        const int q0 = max(wf, c * W), q1 = min(wl, c * W + W - 1);
#pragma unroll 1
        for (int r = 0; r < sh.nr; ++r) {
            if (turn++ % W != w) continue;
            AttnJoin j;
            auto piece = [&](int i) { return place_s[q0 + i - c * W][q0 + i == wf]; };
            j.join(q1 - q0 + 1, ln < D / 4,
                   [&](int i) { return *reinterpret_cast<const float2*>(piece(i) + ROWS * D + 2 * r); },
                   [&](int i) { return reinterpret_cast<const float4*>(piece(i) + r * D)[ln]; });
            if (bf != bl) {
                float* p = bpart + (size_t)(2 * c + (bf == c)) * F::PS;
                if (ln < D / 4) reinterpret_cast<float4*>(p + r * D)[ln] = make_float4(j.y[0], j.y[1], j.y[2], j.y[3]);
                if (ln == 0) *reinterpret_cast<float2*>(p + ROWS * D + 2 * r) = make_float2(j.m, j.l);
                __threadfence();
                __syncwarp();
                int* const cnt = a.count + bf * 32 + r;
                int last = 0;
                if (ln == 0) {
                    last = atomicAdd(cnt, 1) == bl - bf;
                    if (last) *cnt = 0;
                }
                if (!__shfl_sync(0xffffffffu, last, 0)) continue;
                __threadfence();
                auto block = [&](int i) { return bpart + (size_t)(2 * (bf + i) + (i == 0)) * F::PS; };
                j = AttnJoin();
                j.join(bl - bf + 1, ln < D / 4,
                       [&](int i) { return __ldcg(reinterpret_cast<const float2*>(block(i) + ROWS * D + 2 * r)); },
                       [&](int i) { return __ldcg(reinterpret_cast<const float4*>(block(i) + r * D) + ln); });
            }
            if (ln >= D / 4) continue;
            attn_store<T>(a, sh.q0, sh.hk, sh.r0 + r, D, 4 * ln, j.y, j.l);
            if (ln == 0) attn_store_lse(a, sh.q0, sh.hk, sh.r0 + r, j.m, j.l);
        }
    }
}

namespace {

template <class T, class C, int D, int NT>
cudaError_t launch(const AttnArgs& a, int blocks, cudaStream_t s) {
    using F = FewCfg<T, C, D, NT>;
    constexpr int most = F::W * F::WB;
    static_assert(most <= 227 * 1024 - 1024, "shared memory of a block");
    static_assert(F::WB >= F::PS * 4, "a warp's last piece lies in its own part");
    static_assert(most >= 4 * HC_KV_SEQS, "the schedule's prefix lies in the rings");
    static_assert((size_t)F::PS * 4 * 2 * (F::W + 1) <= kFewPartBytes, "the workspace of a block");
    static SmemOptIn opted;
    const cudaError_t e = opted(reinterpret_cast<const void*>(attn_few_kernel<T, C, D, NT>), most);
    if (e != cudaSuccess) return e;
    attn_few_kernel<T, C, D, NT><<<blocks, 32 * F::W, most, s>>>(a);
    return cudaGetLastError();
}

// Tiles of 8 or 16 rows, by the batch's largest sequence.  (Tiles of 32 need more registers than a thread has.)
template <class T, class C, int D>
cudaError_t by_rows(const AttnArgs& a, int blocks, cudaStream_t s) {
    if (a.max_rows <= 8) return launch<T, C, D, 1>(a, blocks, s);
    return launch<T, C, D, 2>(a, blocks, s);
}

template <class T>
cudaError_t by_cache(int ct, int D, const AttnArgs& a, int blocks, cudaStream_t s) {
    if (D == 64) {
        if (ct == T_F16) return by_rows<T, __half, 64>(a, blocks, s);
        if (ct == T_BF16) return by_rows<T, __nv_bfloat16, 64>(a, blocks, s);
        return by_rows<T, int8_t, 64>(a, blocks, s);
    }
    if (ct == T_F16) return by_rows<T, __half, 128>(a, blocks, s);
    if (ct == T_BF16) return by_rows<T, __nv_bfloat16, 128>(a, blocks, s);
    return by_rows<T, int8_t, 128>(a, blocks, s);
}

}  // namespace

cudaError_t launch_attn_few(int ct, int dt, int D, const AttnArgs& args, int blocks, cudaStream_t s) {
    AttnArgs a = args;
    a.over = 2;  // a tile's start and end cost about what two of its units do
    if (dt == T_F32) return by_cache<float>(ct, D, a, blocks, s);
    if (dt == T_F16) return by_cache<__half>(ct, D, a, blocks, s);
    return by_cache<__nv_bfloat16>(ct, D, a, blocks, s);
}

}  // namespace hc
