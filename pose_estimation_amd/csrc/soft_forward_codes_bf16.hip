// Soft correspondence, forward kernels: bfloat16 queries against stored codes.
#include "soft_forward_impl.h"

namespace ispa_soft {
int forward_codes_bf16(const Params &p, bool fp8, int waves, hipStream_t stream) {
    return fp8 ? forward_channels<BF16, FP8>(p, waves, stream) : forward_channels<BF16, I8>(p, waves, stream);
}
}  // namespace ispa_soft
