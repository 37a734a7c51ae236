// kv_launch.h -- launchers of the paged key/value cache's kernels.
#pragma once

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

struct AttnArgs {
    KvDev c;
    KvBatchDev b;
    const void* q;
    void* out;
    float* lse;
    long long ldq, ldo;
    int heads, group;  // query heads, and query heads per kv head
    int causal, window, sink;
    float scale;
    int max_rows;          // the host's bound on a sequence's rows of one kv head (new tokens x group)
    int row_min, row_max;  // sequences with fewer or more rows are left to another kernel
    float* part;           // partial results: 2 slots per block of rows * (head_dim + 2) floats
    int* count;            // one counter per block, zero between calls
};

// Rows per tile of the kernel for few rows, by the batch's largest sequence.
inline int attn_few_tile(int max_rows) { return max_rows <= 8 ? 8 : max_rows <= 16 ? 16 : 32; }
inline size_t attn_few_part_bytes(int rows, int head_dim, int blocks) {
    return (size_t)blocks * 2 * rows * (head_dim + 2) * sizeof(float);
}
cudaError_t launch_attn_few(int cache_type, int dtype, int head_dim, const AttnArgs& a, int blocks, cudaStream_t s);

}  // namespace hc
