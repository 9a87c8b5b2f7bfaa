// Attention of single tokens over caches in 8 bits: attn_decode_kernel where it turns K and V into 16 bits on their way.
#include "es_hip_attn_kernels.h"

namespace {

template <bool BF, int NQ, int DP> AttnKernel kernel_of(bool sinks, int nseq) {
    if (DP == 64 || decode_ahead(DP, nseq) == 2) return sinks ? attn_decode_kernel<BF, NQ, DP, true, true, 2> : attn_decode_kernel<BF, NQ, DP, true, false, 2>;
    if constexpr (DP > 64) return sinks ? attn_decode_kernel<BF, NQ, DP, true, true> : attn_decode_kernel<BF, NQ, DP, true, false>;
    return nullptr;
}
template <bool BF, int NQ> AttnKernel kernel_of(int dim, bool sinks, int nseq) {
    return dim <= 64 ? kernel_of<BF, NQ, 64>(sinks, nseq) : dim <= 128 ? kernel_of<BF, NQ, 128>(sinks, nseq) : kernel_of<BF, NQ, 256>(sinks, nseq);
}

}  // namespace

namespace esq {

AttnKernel attn_f8_decode_kernel(uint32_t type, int dim, bool sinks, int nseq) {
    return type == ES_HIP_F32    ? kernel_of<false, 2>(dim, sinks, nseq)
           : type == ES_HIP_BF16 ? kernel_of<true, 1>(dim, sinks, nseq)
                                 : kernel_of<false, 1>(dim, sinks, nseq);
}

}  // namespace esq
