// Soft correspondence, forward kernels: bfloat16 maps.
#include "soft_forward_impl.h"

namespace ispa_soft {
int forward_bf16(const Params &p, int waves, hipStream_t stream) { return forward_channels<BF16, BF16>(p, waves, stream); }
}  // namespace ispa_soft
