// Attention over 16-bit caches through a window that leaves a few first tokens in sight: those of the kernels of
// es_hip_attn_kernels.h.
#include "es_hip_attn_kernels.h"

namespace {

template <bool BF, int NQ> AttnKernel kernel_of(bool prompt, int dim) {
    if (prompt)
        return dim <= 64    ? attn_prompt_kernel<BF, NQ, 64, false, true>
               : dim <= 128 ? attn_prompt_kernel<BF, NQ, 128, false, true>
                            : attn_prompt_kernel<BF, NQ, 256, false, true>;
    return dim <= 64 ? attn_decode_kernel<BF, NQ, 64, false, true> : dim <= 128 ? attn_decode_kernel<BF, NQ, 128, false, true> : attn_decode_kernel<BF, NQ, 256, false, true>;
}

}  // namespace

namespace esq {

AttnKernel attn_sinks_kernel(bool prompt, bool bf16, bool fp32, int dim) {
    if (bf16) return fp32 ? kernel_of<true, 3>(prompt, dim) : kernel_of<true, 1>(prompt, dim);
    return fp32 ? kernel_of<false, 2>(prompt, dim) : kernel_of<false, 1>(prompt, dim);
}

}  // namespace esq
