// ffn_ray_delta_f16.hip -- the delta rule along rays, _Float16.
#include "ffn_ray_delta.h"

namespace ffn {

hipError_t delta_f16(const ffn_ray_delta& a, bool back, hipStream_t st) { return delta_of_type<_Float16>(a, back, st); }

}  // namespace ffn
