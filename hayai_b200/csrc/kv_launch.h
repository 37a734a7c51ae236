// kv_launch.h -- launchers of the paged key/value cache's kernels.
#pragma once

#include "kv.cuh"

namespace hc {

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
};
cudaError_t launch_attn_paged(int cache_type, int dtype, int head_dim, const AttnArgs& a, cudaStream_t s);

}  // namespace hc
