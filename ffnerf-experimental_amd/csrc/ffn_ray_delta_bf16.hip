// ffn_ray_delta_bf16.hip -- the delta rule along rays, __bf16.
#include "ffn_ray_delta.h"

namespace ffn {

hipError_t delta_bf16(const ffn_ray_delta& a, bool back, hipStream_t st) { return delta_of_type<__bf16>(a, back, st); }

}  // namespace ffn
