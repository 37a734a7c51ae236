// attn_few_shared.cu -- the kernel for few rows, as a part of attention over shared prefixes.
#include "attn_few.cuh"

namespace hc {

cudaError_t launch_attn_few_shared(int ct, int dt, int D, const AttnArgs& a, int blocks, cudaStream_t s) {
    return by_type(ct, dt, D, a, blocks, s);
}

}  // namespace hc
