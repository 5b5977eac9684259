// Soft correspondence, forward kernels on bfloat16 MFMAs.
#include "soft_forward_impl.h"

namespace ispa_soft {
int forward_bf16(const Params &p, int source, int waves, hipStream_t stream) {
    return forward_source<BF16>(p, source, waves, stream);
}
}  // namespace ispa_soft
