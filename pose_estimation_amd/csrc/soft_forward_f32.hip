// Soft correspondence, forward kernels on float32 MFMAs.
#include "soft_forward_impl.h"

namespace ispa_soft {
int forward_f32(const Params &p, int source, int waves, hipStream_t stream) {
    return forward_source<F32>(p, source, waves, stream);
}
}  // namespace ispa_soft
