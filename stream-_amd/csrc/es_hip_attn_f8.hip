// Attention over caches in 8 bits: the kernels of es_hip_attn_kernels.h that turn K and V into bf16 on their way.
#include "es_hip_attn_kernels.h"

namespace {

template <int NQ, int DP> AttnKernel kernel_of(bool prompt, bool sinks) {
    if (prompt) return sinks ? attn_prompt_kernel<true, NQ, DP, true, true> : attn_prompt_kernel<true, NQ, DP, true, false>;
    return sinks ? attn_decode_kernel<true, NQ, DP, true, true> : attn_decode_kernel<true, NQ, DP, true, false>;
}

}  // namespace

namespace esq {

AttnKernel attn_f8_kernel(bool prompt, bool fp32, int dim, bool sinks) {
    if (fp32) return dim <= 64 ? kernel_of<3, 64>(prompt, sinks) : dim <= 128 ? kernel_of<3, 128>(prompt, sinks) : kernel_of<3, 256>(prompt, sinks);
    return dim <= 64 ? kernel_of<1, 64>(prompt, sinks) : dim <= 128 ? kernel_of<1, 128>(prompt, sinks) : kernel_of<1, 256>(prompt, sinks);
}

}  // namespace esq
