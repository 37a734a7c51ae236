// attn_shared.cu -- attention of groups of sequences whose first tokens are the same pages: what has to
// be known of the groups before the attention's kernels run, and the joining after them.
//
// A group's rows see its prefix whole, so that the prefix is one more sequence, of all the group's new tokens and
// not causal: its keys are read once for the group, and its rows fill the tensor cores' tiles.  One call is
//     attn_groups    what every group shares for this step, and the tiles: of the prefixes, then of what every sequence
//                    has behind its own
//     attn_prefix    the tiles (attn_prefix.cu), in pieces
//     attn_few       of many single tokens, what is behind the prefixes (AttnArgs::first), which has no tiles then
//     attn_join      out = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over a row's pieces
// or, of f32 rows, attn_few over the prefixes and again over what is behind them, and the joining.
// attn_groups is one block whose time is its chain of dependent loads and scans (10 to 13 us); attn_join moves the pieces
// once, 10 us for 4096 rows of 128 columns in f32 and 30 us for 28000.
// Where nothing is shared after all, the two others find no tiles, and the paged attention's kernels behind them do the work:
// 16 sequences behind 300 tokens, tables of 32768, 26 us (15 by themselves); 64 behind 1000 60 (43).
#include "attn_rows.cuh"
#include "block_scan.cuh"

namespace hc {

namespace {

// kOver: places of the line that stand for a tile's start and end (queries in, the first unit's way through the roles, O
// out), some 12 us where a unit of a wide tile takes 2.  Tiles behind prefixes have few units, and lie together at the
// line's end, so that too little for them leaves everything to a few blocks.  With 2, 6, 8, 10, 12, 14 of them (us in a
// graph): 8 chunks of 256 bf16 tokens behind 16384, 32 heads on 8 of 128, 1177, 802, 677, 622, 577, 583 (the paged attention
// 560); 6 groups of f16 chunks, 32 heads on 4, 206, 157, 157, 159, 159, 164; 8 chunks of 5 behind 4096 42.6, 37.8, 37.9, 39.8,
// 39.7, 41.3; 64 single tokens behind 4100 8-bit ones, 64 heads on 8, 99, 90, 90, 93, 92, 92.
constexpr int kTileRows = 256, kUnit = 128, kOver = 10;

// Positions that tile k of `tok` tokens sees, at `pos` and following (kAllSeen: the whole of [from, len)).
__device__ __forceinline__ int tile_end(int k, int rows, int group, int len, int pos) {
    if (pos == kAllSeen) return len;
    return min(len, pos + (min((k + 1) * kTileRows, rows) - 1) / group + 1);
}
__device__ __forceinline__ int tile_units(int from, int end) { return end > from ? (end - from + kUnit - 1) / kUnit : 0; }
__device__ __forceinline__ bool tile_narrow(int k, int rows) { return rows - k * kTileRows <= kTileRows / 2; }
// Places of a kv head's first `tiles` tiles.  (Not inlined, as little of the kernel below as can be: its code runs once,
// and fetching it is most of its time.)
__device__ __noinline__ int tile_places(int tiles, int rows, int group, int from, int len, int pos) {
    int w = 0;
#pragma unroll 1
    for (int k = 0; k < tiles; ++k) {
        const int u = tile_units(from, tile_end(k, rows, group, len, pos));
        if (u) w += min((tile_narrow(k, rows) ? u : 2 * u) + kOver, 0x7fffffff - w);
    }
    return w;
}
// The new tokens of sequences [s0, s1), cut as kv_seq cuts them.
__device__ __forceinline__ void group_tokens(const KvBatchDev& b, int s0, int s1, int& q0, int& q1) {
    q0 = min(max(__ldg(b.q_start + s0), 0), b.n_tok);
    q1 = min(max(__ldg(b.q_start + s1), q0), b.n_tok);
}
__device__ __noinline__ long long scan_1024(long long x, long long* scratch, long long& total) { return block_scan(x, scratch, total); }

// A warp per group: how many tokens its sequences share for this step.  All new tokens have to see them all, so that
// they are at most the tokens that every sequence had before; a group of one sequence shares nothing.  Then the
// tiles, in a line whose places the blocks of attn_prefix.cu share equally: a unit of a wide tile is two places, of a narrow
// one one, and starting and finishing a tile counts as kOver more.
__global__ void __launch_bounds__(1024) attn_groups_kernel(KvBatchDev b, KvSharedDev g, int cap) {
    __shared__ long long scratch[33];
    __shared__ unsigned long long saved_s;
    __shared__ int runs_s, chunk_tiles_s;
    extern __shared__ int ent[];
    // entities: the groups' prefixes, then the sequences
    const int E = g.n + b.n_seq, tid = threadIdx.x, ln = lane_id(), group = g.heads / g.kv_heads;
    int *const tok_s = ent, *const from_s = tok_s + E, *const len_s = from_s + E, *const tile_s = len_s + E,
               *const place_s = tile_s + E, *const q0_s = place_s + E, *const w_s = q0_s + E, *const of_s = w_s + E;  // [n_seq] a sequence's group, or -1
    let_next_start();
    if (tid == 0) saved_s = 0, chunk_tiles_s = 0;
    __syncthreads();
#pragma unroll 1
    for (int s = tid; s < b.n_seq; s += 1024) {
        of_s[s] = -1;
        if (!g.rule) continue;
        const KvSeq q = kv_seq(b, cap, s);
        const int rows = (q.q1 - q.q0) * group;
        if (rows > kFewRows) atomicAdd(&chunk_tiles_s, (rows - 1) / kTileRows + 1);
    }
    __syncthreads();
    const long long chunk_tiles = (long long)chunk_tiles_s * g.kv_heads;  // of the paged attention's kernel for many rows
    int *const s0_s = tile_s, *const s1_s = place_s, *const lead_s = w_s;  // the groups' sequences, until the tiles are counted
#pragma unroll 1
    for (int i = tid >> 5; i < g.n; i += 32) {
        const int a0 = __ldg(g.seq_start + i), a1 = __ldg(g.seq_start + i + 1), given = __ldg(g.length + i);
        const int s0 = min(max(a0, 0), b.n_seq), s1 = min(max(a1, s0), b.n_seq);
        int most = min(max(given, 0), cap), seqs = 0, lead = b.n_seq - 1, rows = 0, alone = 0;
        if (s0 != a0 || s1 != a1 || most != given)
            if (ln == 0) atomicOr(b.err, kErrKvRange);
        int q0, q1;
        group_tokens(b, s0, s1, q0, q1);
#pragma unroll 1
        for (int s = s0 + ln; s < s1; s += 32) {
            const KvSeq q = kv_seq(b, cap, s);
            if (q.q1 == q.q0) continue;
            // Offsets that do not ascend (kv_seq reports them): the joining counts a sequence's rows from the group's
            // first, so that a group with others shares nothing.
            if (q.q0 < q0 || q.q1 > q1) most = 0;
            if (seqs++ == 0) lead = s;
            most = min(most, q.len - (q.q1 - q.q0));
            rows += (q.q1 - q.q0) * group;
            alone += ((q.q1 - q.q0) * group - 1) / g.tile + 1;
        }
        most = max(__reduce_min_sync(0xffffffffu, most), 0);
        seqs = __reduce_add_sync(0xffffffffu, seqs);
        lead = __reduce_min_sync(0xffffffffu, lead);
        rows = __reduce_add_sync(0xffffffffu, rows);
        alone = __reduce_add_sync(0xffffffffu, alone);
        if (seqs < 2) most = 0;
        if (ln == 0) {
            len_s[i] = most;
            s0_s[i] = s0;
            s1_s[i] = s1;
            lead_s[i] = lead;
            if (most) {
                // readings of the prefix that sharing saves
                const int together = (rows - 1) / g.tile + 1;
                long long saved = (long long)most * (seqs - 1);
                if (g.rule && g.few)
                    saved = (long long)most * (g.alone * alone - 8 * together) / 5;
                else if (g.rule && chunk_tiles == 0)
                    saved = (long long)most * (seqs - 1 - g.extra);
                else if (g.rule && chunk_tiles >= g.blocks)
                    saved = (long long)most * (25 * alone - 27 * together) / 25;
                atomicAdd(&saved_s, (unsigned long long)saved);
            }
        }
    }
    __syncthreads();
    long long least = g.least;
    if (g.rule && !g.few && chunk_tiles) least = g.chunk;
    if (g.rule && (g.few || chunk_tiles >= g.blocks)) least += g.moved;
    const bool worth = (long long)saved_s >= least;
    if (!worth) {
        if (tid == 0) g.line[kLineTiles] = g.line[kLineOwn] = g.line[kLinePlaces] = 0;
        return;
    }
#pragma unroll 1
    for (int i = tid >> 5; i < g.n; i += 32) {
        const int s0 = s0_s[i], s1 = s1_s[i], most = len_s[i];
        if (most)
#pragma unroll 1
            for (int s = s0 + ln; s < s1; s += 32) of_s[s] = i;
        if (ln == 0) {
            int q0, q1;
            group_tokens(b, s0, s1, q0, q1);
            tok_s[i] = most ? q1 - q0 : 0;
            from_s[i] = 0;
            q0_s[i] = q0;
            g.q_start[i] = q0;
            if (i == g.n - 1) g.q_start[g.n] = q1;
            g.len[i] = most;
            g.row[i] = lead_s[i];  // its pages hold the prefix, whatever became of the others
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int s = tid; s < b.n_seq; s += 1024) {
        const KvSeq q = kv_seq(b, cap, s);
        const int first = of_s[s] >= 0 ? len_s[of_s[s]] : 0;
        g.first[s] = first;
        tok_s[g.n + s] = g.few_behind && !first ? 0 : q.q1 - q.q0;
        from_s[g.n + s] = first;
        len_s[g.n + s] = q.len;
        q0_s[g.n + s] = q.q0;
    }
    __syncthreads();
    // ---- tiles and places of every entity; of those that the kernel for few rows does only what the joining takes
    auto elsewhere = [&](int i) { return i < g.n ? g.few : g.few_behind; };
    auto pos_of = [&](int i) { return i < g.n ? kAllSeen : len_s[i] - tok_s[i]; };
    const int each = (E + 1023) / 1024, e0 = min(tid * each, E), e1 = min(e0 + each, E);
    long long tiles = 0, places = 0, all_tiles, U;
#pragma unroll 1
    for (int i = e0; i < e1; ++i) {  // a kv head's tiles and places
        const int rows = tok_s[i] * group, n = (rows + kTileRows - 1) / kTileRows;
        tile_s[i] = !elsewhere(i) ? n * g.kv_heads : i < g.n ? 0 : (int)(((unsigned)(tok_s[i] * g.heads) + kTileRows - 1) / kTileRows);
        place_s[i] = w_s[i] = elsewhere(i) ? 0 : tile_places(n, rows, group, from_s[i], len_s[i], pos_of(i));
        tiles += tile_s[i];
        places += (long long)w_s[i] * g.kv_heads;
    }
    long long at = scan_1024(tiles, scratch, all_tiles), pl = scan_1024(places, scratch, U);
    const bool fits = all_tiles <= g.max_tiles && U < 0x7fffffff;
#pragma unroll 1
    for (int i = e0; i < e1; ++i) {  // what is before them
        const int n = tile_s[i], w = place_s[i];
        tile_s[i] = (int)at, place_s[i] = (int)pl;
        at += n;
        pl += (long long)w * g.kv_heads;
    }
    const int n_tiles = fits ? (int)all_tiles : 0;
    const int G = fits ? max(1, min(g.blocks, (int)U / 4)) : 1;  // shares of four places and more, so that those within a tile's units have one (others may have none)
    __syncthreads();
    const AttnShares share(max((int)(fits ? U : 0), 1), G);
    long long rows_before = 0;
    int runs = 0;
#pragma unroll 1
    for (int t0 = 0; t0 < n_tiles; t0 += 1024) {
        const int t = t0 + tid;
        PrefixTile x{};
        long long rows = 0;
        if (t < n_tiles) {
            int lo = 0, hi = E - 1;  // the last entity whose tiles start at or before t, of those at one place the last
#pragma unroll 1
            while (lo < hi) {
                const int m = (lo + hi + 1) >> 1;
                if (tile_s[m] <= t) lo = m;
                else hi = m - 1;
            }
            const int r = tok_s[lo] * group, per = (r + kTileRows - 1) / kTileRows, local = t - tile_s[lo], s = lo - g.n;
            const int pos = pos_of(lo);
            const bool all = elsewhere(lo);  // rows of all query heads, for the joining
            x.hk = all ? -1 : local / per;
            const int k = all ? local : local - x.hk * per;
            x.r0 = k * kTileRows;
            x.nr = min(kTileRows, (all ? tok_s[lo] * g.heads : r) - x.r0);
            x.q0 = q0_s[lo];
            x.from = from_s[lo];
            x.len = all ? len_s[lo] : tile_end(k, r, group, len_s[lo], pos);
            x.row = lo < g.n ? g.row[lo] : s;
            x.pos0 = pos;
            x.pre = -1;
            if (s >= 0 && of_s[s] >= 0) {
                const int i = of_s[s], to_head = (tok_s[i] * group + kTileRows - 1) / kTileRows;
                x.pre = tile_s[i] + (all ? 0 : x.hk * to_head);
                x.pre_row = (x.q0 - q0_s[i]) * group;
                x.cost = to_head;
            }
            if (!all) x.cost = tile_narrow(k, r) ? 1 : 2;
            x.units = all ? 0 : tile_units(x.from, x.len);
            if (s >= 0) runs = max(runs, (x.nr + 7) / 8);
            x.place = place_s[lo];
            if (!all) x.place += x.hk * w_s[lo] + (k ? tile_places(k, r, group, x.from, len_s[lo], pos) : 0);
            if (x.units) {
                x.c0 = share.owner(x.place);
                x.pieces = (share.owner(x.place + x.cost * (x.units - 1)) - x.c0 + 1) * (x.cost == 1 ? 2 : 1);
                rows = (long long)x.pieces * x.nr;
                const int end = x.place + x.cost * x.units + kOver;
#pragma unroll 1
                for (int c = x.place ? share.owner(x.place - 1) + 1 : 0; c < G && share.begin(c) < end; ++c) g.first_tile[c] = t;
            }
        }
        long long total;
        x.piece = (int)(rows_before + scan_1024(rows, scratch, total));
        rows_before += total;
        if (t < n_tiles)  // 16 bytes at a time: the tiles are 64 bytes apart, and every store of a warp meets 32 sectors
#pragma unroll
            for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(g.tiles + t)[i] = reinterpret_cast<const int4*>(&x)[i];
    }
    // groups that overlap (offsets that do not ascend) may want more room than any others: nothing is made of them
    const bool room = fits && rows_before <= g.max_pieces;
    runs = __reduce_max_sync(0xffffffffu, runs);
    if (tid == 0) runs_s = 0;
    __syncthreads();
    if (ln == 0) atomicMax(&runs_s, runs);
    __syncthreads();
    if (tid == 0) {
        if (!room) atomicOr(b.err, kErrKvRange);
        g.line[kLineTiles] = room ? n_tiles : 0;
        g.line[kLineOwn] = room ? tile_s[g.n] : 0;
        g.line[kLineRuns] = runs_s;
        g.line[kLinePlaces] = room ? (int)U : 0;
        g.line[kLineBlocks] = G;
    }
}

// A warp per row of a tile behind the prefixes, eight rows of one at a time.  Bound by memory and its latency: four of a
// row's parts are asked for together, the prefix's pieces and then its own, and every lane forms the weights for itself.
template <class T, int D>
__global__ void __launch_bounds__(256, 4) attn_join_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ PrefixArgs p) {
    constexpr int U = 4;
    after_previous();
    let_next_start();
    const int n_tiles = __ldcg(p.line + kLineTiles), own = __ldcg(p.line + kLineOwn), runs = __ldcg(p.line + kLineRuns),
              ln = lane_id();
    const bool mine = ln < D / 4;
    if (n_tiles <= own) return;
    // tile and run (eight rows of the tile), which are a block's distance apart: their product may not fit 32 bits
    const int step = gridDim.x / runs, step_run = gridDim.x - step * runs;
    for (int tile = own + blockIdx.x / runs, run = blockIdx.x % runs; tile < n_tiles;
         run += step_run, tile += step + (run >= runs), run -= run >= runs ? runs : 0) {
        PrefixTile x;
        const int4* const xs = reinterpret_cast<const int4*>(p.tiles + tile);
#pragma unroll
        for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(&x)[i] = __ldcg(xs + i);
        const int r = run * 8 + (threadIdx.x >> 5);
        if (r >= x.nr) continue;
        int row = x.r0 + r, hk = x.hk;
        if (hk < 0) {  // the sequence's row-th of all (token, query head)
            const int t = row / a.heads, h = row - t * a.heads;
            hk = a.by_group(h);
            row = t * a.group + h - hk * a.group;
        }
        const int t = a.by_group(row);
        const long long at = (long long)(x.q0 + t) * a.heads + hk * a.group + row - t * a.group;
        // the row's places among its own pieces and its prefix's, and from one piece to the next
        size_t p_own = (size_t)x.piece + r, p_pre = 0;
        int s_own = x.nr, s_pre = 0, n_own = x.pieces, n_pre = 0;
        bool w_own = false, w_pre = false;  // one result, divided by its sum
        if (a.base) n_own = 1, p_own = at, w_own = true;
        if (p.few) {
            n_pre = 1, p_pre = at, w_pre = true;
        } else if (x.pre >= 0) {
            const int pr = x.pre_row + row;
            const PrefixTile* const z = p.tiles + x.pre + (x.hk < 0 ? hk * x.cost : 0) + pr / kTileRows;
            s_pre = __ldcg(&z->nr), n_pre = __ldcg(&z->pieces);
            p_pre = (size_t)__ldcg(&z->piece) + pr % kTileRows;
        }
        float m = -INFINITY, l = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
        const int n = n_pre + n_own;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += U) {
            float2 ml[U];
            float4 o[U];
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int i = i0 + k;
                ml[k] = make_float2(-INFINITY, 0.f);
                o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < n) {
                    const bool pre = i < n_pre, whole = pre ? w_pre : w_own;
                    const size_t q = pre ? p_pre + (size_t)i * s_pre : p_own + (size_t)(i - n_pre) * s_own;
                    if (whole) {
                        const float e = __ldcg((pre ? p.few_lse : a.base_lse) + q);
                        ml[k] = make_float2(e, e == -INFINITY ? 0.f : 1.f);
                    } else {
                        ml[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml) + q);
                    }
                    if (mine) o[k] = __ldcg(reinterpret_cast<const float4*>((whole ? (pre ? p.few : a.base) : p.part) + q * D) + ln);
                }
            }
            float top = m;
#pragma unroll
            for (int k = 0; k < U; ++k) top = fmaxf(top, ml[k].x);
            // a part that saw nothing has m = -inf and l = 0; one of scores that are not numbers has m = -inf only
            const float old = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - top);
            m = top;
            l *= old;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = old == 0.f ? 0.f : y[e] * old;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const float f = ml[k].x == -INFINITY ? (ml[k].y == 0.f ? 0.f : 1.f) : ex2(ml[k].x - top);
                l += ml[k].y * f;
                if (f == 0.f) continue;  // a weight of zero takes nothing, whatever the value is
                y[0] = fmaf(o[k].x, f, y[0]), y[1] = fmaf(o[k].y, f, y[1]);
                y[2] = fmaf(o[k].z, f, y[2]), y[3] = fmaf(o[k].w, f, y[3]);
            }
        }
        if (mine) attn_store<T>(a, x.q0, hk, row, D, 4 * ln, y, l, false);
        if (ln == 0) attn_store_lse(a, x.q0, hk, row, m, l, false);
    }
}

template <class T>
cudaError_t join(int head_dim, const AttnArgs& a, const PrefixArgs& p, int sms, cudaStream_t s) {
    return launch_early(head_dim == 64 ? attn_join_kernel<T, 64> : attn_join_kernel<T, 128>, sms * 8, 256, 0, s, a, p);
}

}  // namespace

cudaError_t launch_attn_groups(const KvBatchDev& b, const KvSharedDev& g, int cap, cudaStream_t s) {
    const int bytes = (7 * (g.n + b.n_seq) + b.n_seq) * 4;
    static SmemOptIn opted;
    const cudaError_t e = opted(reinterpret_cast<const void*>(attn_groups_kernel), (7 * 2 * HC_KV_SEQS + HC_KV_SEQS) * 4);
    if (e != cudaSuccess) return e;
    attn_groups_kernel<<<1, 1024, bytes, s>>>(b, g, cap);
    return cudaGetLastError();
}

cudaError_t launch_attn_join(int dtype, int head_dim, const AttnArgs& a, const PrefixArgs& p, int sms, cudaStream_t s) {
    if (dtype == T_F32) return join<float>(head_dim, a, p, sms, s);
    if (dtype == T_F16) return join<__half>(head_dim, a, p, sms, s);
    return join<__nv_bfloat16>(head_dim, a, p, sms, s);
}

}  // namespace hc
