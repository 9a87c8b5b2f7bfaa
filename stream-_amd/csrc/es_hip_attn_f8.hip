// Attention over caches in 8 bits: the kernels of es_hip_attn_kernels.h that turn K and V into 16 bits on their way.
#include "es_hip_attn_kernels.h"

namespace {

template <bool BF, int NQ, int DP> AttnKernel kernel_of(bool prompt, bool sinks) {
    if (prompt) return sinks ? attn_prompt_kernel<BF, NQ, DP, true, true> : attn_prompt_kernel<BF, NQ, DP, true, false>;
    return sinks ? attn_decode_kernel<BF, NQ, DP, true, true> : attn_decode_kernel<BF, NQ, DP, true, false>;
}
template <bool BF, int NQ> AttnKernel kernel_of(bool prompt, bool sinks, int dim) {
    return dim <= 64 ? kernel_of<BF, NQ, 64>(prompt, sinks) : dim <= 128 ? kernel_of<BF, NQ, 128>(prompt, sinks) : kernel_of<BF, NQ, 256>(prompt, sinks);
}

}  // namespace

namespace esq {

AttnKernel attn_f8_kernel(bool prompt, uint32_t type, int dim, bool sinks) {
    return type == ES_HIP_F32    ? kernel_of<false, 2>(prompt, sinks, dim)
           : type == ES_HIP_BF16 ? kernel_of<true, 1>(prompt, sinks, dim)
                                 : kernel_of<false, 1>(prompt, sinks, dim);
}

}  // namespace esq
