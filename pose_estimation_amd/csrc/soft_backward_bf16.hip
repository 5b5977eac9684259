// Soft correspondence, backward kernels on bfloat16 MFMAs.
#include "soft_backward_impl.h"

namespace ispa_soft {
int backward_bf16(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream) {
    return backward_channels<BF16>(p, dq, dkv, stream);
}
}  // namespace ispa_soft
