// Soft correspondence, forward kernels: float32 maps.
#include "soft_forward_impl.h"

namespace ispa_soft {
int forward_f32(const Params &p, int waves, hipStream_t stream) {
    return arithmetic(true, false, padded_channels(p.D, p.Dv), waves) == kSplit ? forward_channels<F32S, F32S>(p, waves, stream)
                                                                               : forward_channels<F32, F32>(p, waves, stream);
}
}  // namespace ispa_soft
