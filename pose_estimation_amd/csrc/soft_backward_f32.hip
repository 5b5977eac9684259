// Soft correspondence, backward kernels of float32 maps (bfloat16 MFMAs on three planes, float32 MFMAs: see Arithmetic).
#include "soft_backward_impl.h"

namespace ispa_soft {
int backward_f32(const Params &p, const Plan &dq, const Plan &dkv, hipStream_t stream) {
    return backward_channels<F32>(p, dq, dkv, stream);
}
}  // namespace ispa_soft
