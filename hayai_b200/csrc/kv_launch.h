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
    float* part;           // partial results: 2 slots per block of rows * (head_dim + 2) floats
    int* count;            // 32 counters per block, zero between calls
};

// Partial results of the kernel for few rows: bytes for each block.
constexpr size_t kFewPartBytes = 2 * 13 * 16 * (128 + 2) * 4;
constexpr size_t kManyPartBytes = 2 * 256 * (128 + 2) * 4;
constexpr size_t kAttnPartBytes = kFewPartBytes > kManyPartBytes ? kFewPartBytes : kManyPartBytes;

// Sequences with few rows of a kv head, on mma.sync; any types.
cudaError_t launch_attn_few(int cache_type, int dtype, int head_dim, const AttnArgs& a, int blocks, cudaStream_t s);
// Sequences with many rows of a kv head, on tcgen05; 16-bit rows.
bool attn_many_supported(int cache_type, int dtype);
cudaError_t launch_attn_many(int cache_type, int dtype, int head_dim, const AttnArgs& a, int blocks, cudaStream_t s);

}  // namespace hc
