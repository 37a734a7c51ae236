// attn_few.cu -- the kernel for few rows, for calls without shared prefixes.
#include "attn_few.cuh"

namespace hc {

cudaError_t launch_attn_few(int ct, int dt, int D, const AttnArgs& a, int blocks, cudaStream_t s) {
    if (a.shared) return launch_attn_few_shared(ct, dt, D, a, blocks, s);
    return by_type(ct, dt, D, AttnAlone{a}, blocks, s);
}

}  // namespace hc
