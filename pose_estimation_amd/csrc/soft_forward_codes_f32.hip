// Soft correspondence, forward kernels: float32 queries against stored codes.
#include "soft_forward_impl.h"

namespace ispa_soft {
int forward_codes_f32(const Params &p, bool fp8, int waves, hipStream_t stream) {
    if (few_columns(true, p.nq)) return fp8 ? forward_channels<F32Q, FP8>(p, waves, stream) : forward_channels<F32Q, I8>(p, waves, stream);
    return fp8 ? forward_channels<F32C, FP8>(p, waves, stream) : forward_channels<F32C, I8>(p, waves, stream);
}
}  // namespace ispa_soft
