// kv_launch.h -- launchers of the paged key/value cache's kernels.
#pragma once

#include <atomic>

#include "kv.cuh"

namespace hc {

constexpr int HC_KV_SEQS = 2048;  // sequences of a batch (HC_KV_MAX_SEQ)
constexpr int T_I8 = 24;  // GgmlType id of plain int8 (crates/hayai-model/src/gguf_types.rs:6-40)

// A pair of packed row arrays [n_tok][heads * dim] with their own token strides (elements).
struct KvRows {
    void *k, *v;
    long long ldk, ldv;
};

cudaError_t launch_kv_append(int cache_type, int dtype, int head_dim, const KvDev& c, const KvBatchDev& b,
                             const KvRows& r, cudaStream_t s);
cudaError_t launch_kv_read(int cache_type, int dtype, int head_dim, const KvDev& c, const KvBatchDev& b,
                           const KvRows& r, cudaStream_t s);

// hc_rope as the kernels get it.
struct RopeDev {
    int pairs, dim, rot;
    float amplitude;
    unsigned long long turns[128];
};
struct RopeRows {
    const int* pos;
    const void* x;
    void* out;
    long long ldx, ldo;
    int n_tok, heads;
};
struct RopeAppend {
    const void *q, *k, *v;
    void* q_out;
    long long ldq, ldqo, ldk, ldv;
    int heads;
};
// wide: sizes, strides and addresses in whole 16 bytes and chunks of 8 values.
cudaError_t launch_rope(int dtype, const RopeDev& r, const RopeRows& a, bool wide, int sms, cudaStream_t s);
cudaError_t launch_kv_append_rope(int cache_type, int dtype, int head_dim, const RopeDev& r, const KvDev& c,
                                  const KvBatchDev& b, const RopeAppend& a, int sms, cudaStream_t s);

// Division of 0 <= n < 2^31 by d >= 1 as a multiplication: with 2^k >= d and m = ceil(2^(31+k) / d),
// floor(n m / 2^(31+k)) = floor(n / d), as m d - 2^(31+k) < d <= 2^k.
struct FastDiv {
    uint32_t d, m, k;
    explicit FastDiv(uint32_t div = 1) : d(div) {
        k = 0;
        while (k < 31 && (1u << k) < div) ++k;
        m = (uint32_t)(((1ull << (31 + k)) + div - 1) / div);
    }
    __device__ __forceinline__ int operator()(int n) const {
        return (int)(((unsigned long long)(uint32_t)n * m) >> (31 + k));
    }
};

// A launch that may start while the kernel before it on the stream still runs (programmatic dependent launch): the
// kernel waits with after_previous() before it reads what that one wrote, and of such data uses no __ldg, which may
// be moved before the wait.  A kernel calls let_next_start() where its successor is such a launch.
template <class... P, class... A>
cudaError_t launch_early(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, args...);
}
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A kernel's shared-memory opt-in, once per device (a call of it costs about a microsecond).
struct SmemOptIn {
    std::atomic<unsigned long long> done{0};
    cudaError_t operator()(const void* kernel, int bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        const unsigned long long bit = 1ull << (dev & 63);
        if (e != cudaSuccess || (done.load() & bit)) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done.fetch_or(bit);
        return e;
    }
};

// hc_kv_pages as the kernels get it, with its scratch divided.
struct PagesDev {
    int* table;  // [n_slots][stride]
    long long stride;
    int *len, *refs;  // [n_slots], [n_pages]
    int n_slots, max_pages, n_pages, page_size;
    FastDiv by_page;
    int* moves;             // the number of copies
    int* item;              // 4 x HC_KV_SEQS
    int *src, *dst, *rows;  // the copies: pages, and rows from the first (null: all)
    int* free;              // free pages that the call takes
    int* err;
};
constexpr size_t kv_pages_scratch(int n_pages) {
    return 16 + 4 * (size_t)HC_KV_SEQS + 3 * (size_t)(n_pages > HC_KV_SEQS ? n_pages : HC_KV_SEQS) + n_pages;
}
// Layers of one shape: strides in 64-byte units as in KvDev.
constexpr int kMaxLayers = 64;
struct KvLayers {
    uint8_t *k[kMaxLayers], *v[kMaxLayers];
    float *ks[kMaxLayers], *vs[kMaxLayers];  // null: 16-bit pages
    uint32_t page, head, row;
    long long spage;
    int n, n_heads, row_bytes;
};
cudaError_t launch_kv_fork(const PagesDev& p, const KvLayers* layers, int groups, int n, const int* parents,
                           const int* children, int sms, cudaStream_t s);
cudaError_t launch_kv_resize(const PagesDev& p, const KvLayers* layers, int groups, int n, const int* slots,
                             const int* lens, int sms, cudaStream_t s);
cudaError_t launch_kv_compact(const PagesDev& p, const KvLayers* layers, int groups, int* moved, int sms, cudaStream_t s);

struct AttnArgs {
    KvDev c;
    KvBatchDev b;
    const void* q;
    void* out;
    float* lse;
    long long ldq, ldo;
    int heads, group;  // query heads, and query heads per kv head
    FastDiv by_group, by_page;
    int causal, window, sink;
    float scale;
    int max_rows;          // the host's bound on a sequence's rows of one kv head (new tokens x group)
    int row_min, row_max;  // sequences with fewer or more rows are left to another kernel
    int over;              // places of the line that stand for a tile's start and end
    int shared;            // one of the kernels of a call with shared prefixes; 0: nothing behind `count` is read
    float* part;           // partial results: 2 slots per block of rows * (head_dim + 2) floats
    int* count;            // 32 counters per block, zero between calls
    // A shared prefix (attn_shared.cu): results over a part of the positions go to `base`, to be joined.
    const int* first;        // [n_seq] positions that a sequence leaves out, or null
    const int* table_row;    // [n_seq] rows of the page table, or null: a sequence's own
    float *base, *base_lse;  // [n_tok * heads][head_dim] and log 2 of the weights' sums
    int to_base;             // the sequences are prefixes: all their results, but nothing of empty ones
    int early;               // a launch_early
    const int *unless, *only;  // nothing is done where the one is not 0, or the other is
};
// Those of a call of its own, for a kernel in which nothing asks for shared prefixes.
struct AttnAlone : AttnArgs {
    static constexpr int shared = 0;
};

// hc_kv_shared as the kernels get it, and what is made of it.
struct KvSharedDev {
    const int *seq_start, *length;
    int n;
    long long least;           // tokens that sharing has to save, or nothing is shared
    // Without a bound of the program's (rule) what it saves is counted by what kernels take (capi_kv.cu):
    int rule;
    int tile;         // rows that read a prefix together: 256, or 16 of the kernel for few rows
    int extra;        // single tokens: readings that the prefix's kernel costs more than it saves
    int alone;        // f32 rows: what a sequence's reading by itself costs, in eighths of one by 16 rows
    long long chunk;  // where sequences have more rows than the kernel for few takes, their bound
    long long moved;  // and tokens whose reading takes as long as moving all rows' parts
    int heads, kv_heads;       // query heads, and those that the keys have
    int few, few_behind;       // the prefixes, or what is behind them, go to the kernel for few rows, else to attn_prefix.cu
    int *first;                // few_behind: [n_seq] shared tokens, where what is behind them starts
    int *q_start, *len, *row;  // few: [n + 1], [n], [n]: the prefixes as sequences
    int blocks;                // of attn_prefix.cu
    int max_tiles, max_pieces;  // tiles, and rows of pieces, that there is room for
    struct PrefixTile* tiles;
    int *line, *first_tile;  // kLine...; [blocks] the tile that a block starts in
};
// Rows of a kv head, up to 256 of them, and the positions that they see together: those of a prefix all of them, those
// behind one up to each row's own.
struct alignas(16) PrefixTile {
    int place, units;    // the first of its places on the line (attn_prefix.cu); units of 128 positions
    int cost;            // places of a unit: 2, or 1 for up to 128 rows
    int q0;              // the first token of the group, or of the sequence
    int hk, r0, nr;      // the kv head; the tile's first row and number of rows.  hk = -1: (token, query head) rows, only for
                         // the joining (what is behind the prefix has a result from elsewhere)
    int from, len;       // positions [from, len)
    int row;             // of the page table
    int piece, pieces;   // its first row in the pieces, and how many there are
    int c0;              // the block that has its first unit
    int pos0;            // position of token q0, or kAllSeen
    int pre, pre_row;    // behind a prefix: its first tile of this kv head (or -1), and the row there of row 0; hk = -1: its
                         // first tile, `cost` of them to a kv head
};
constexpr int kAllSeen = 1 << 30;
// Tiles; the first behind a prefix; what there is of those rows by eights, at most; places; blocks.
enum { kLineTiles, kLineOwn, kLineRuns, kLinePlaces, kLineBlocks, kLineInts = 16 };
// What attn_prefix.cu and the joining get besides: pieces (O, then m and l of a row), and where the kernel for few rows
// made them the prefixes' results (what is behind them: AttnArgs::base).
struct PrefixArgs {
    const PrefixTile* tiles;
    const int *line, *first_tile;
    float *part, *part_ml;
    const float *few, *few_lse;
};
// Rows of a kv head up to which a sequence goes to the kernel for few rows.
constexpr int kFewRows = 16;
cudaError_t launch_attn_groups(const KvBatchDev& b, const KvSharedDev& g, int cap, cudaStream_t s);
cudaError_t launch_attn_prefix(int cache_type, int dtype, int head_dim, const AttnArgs& a, const PrefixArgs& p, int blocks,
                               cudaStream_t s);
// out and lse of all tiles' rows, from their own and their prefixes' pieces, or from `base` and PrefixArgs::few.
cudaError_t launch_attn_join(int dtype, int head_dim, const AttnArgs& a, const PrefixArgs& p, int sms, cudaStream_t s);

// Partial results of the kernel for few rows: bytes for each block.
constexpr size_t kFewPartBytes = 2 * 13 * 16 * (128 + 2) * 4;
constexpr size_t kManyPartBytes = 2 * 256 * (128 + 2) * 4;
constexpr size_t kAttnPartBytes = kFewPartBytes > kManyPartBytes ? kFewPartBytes : kManyPartBytes;

// Sequences with few rows of a kv head, on mma.sync; any types.
cudaError_t launch_attn_few(int cache_type, int dtype, int head_dim, const AttnArgs& a, int blocks, cudaStream_t s);
cudaError_t launch_attn_few_shared(int cache_type, int dtype, int head_dim, const AttnArgs& a, int blocks, cudaStream_t s);
// Sequences with many rows of a kv head, on tcgen05; 16-bit rows.
bool attn_many_supported(int cache_type, int dtype);
cudaError_t launch_attn_many(int cache_type, int dtype, int head_dim, const AttnArgs& a, int blocks, cudaStream_t s);

}  // namespace hc
