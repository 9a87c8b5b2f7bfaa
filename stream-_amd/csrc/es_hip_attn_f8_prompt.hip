// Attention of prompts over caches in 8 bits: attn_prompt_kernel where it turns K and V into 16 bits on their way.
#include "es_hip_attn_kernels.h"

namespace {

template <bool BF, int NQ, bool SINKS> AttnKernel kernel_of(int dim) {
    return dim <= 64    ? attn_prompt_kernel<BF, NQ, 64, true, SINKS>
           : dim <= 128 ? attn_prompt_kernel<BF, NQ, 128, true, SINKS>
                        : attn_prompt_kernel<BF, NQ, 256, true, SINKS>;
}
template <bool BF, int NQ> AttnKernel kernel_of(int dim, bool sinks) { return sinks ? kernel_of<BF, NQ, true>(dim) : kernel_of<BF, NQ, false>(dim); }

}  // namespace

namespace esq {

AttnKernel attn_f8_prompt_kernel(uint32_t type, int dim, bool sinks) {
    return type == ES_HIP_F32 ? kernel_of<false, 2>(dim, sinks) : type == ES_HIP_BF16 ? kernel_of<true, 1>(dim, sinks) : kernel_of<false, 1>(dim, sinks);
}

}  // namespace esq
