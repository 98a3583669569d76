// ffn_ray_delta_f32.hip -- the delta rule along rays, float; sizes and the choice of the type.
#include "ffn_ray_delta.h"

namespace ffn {

hipError_t delta_f32(const ffn_ray_delta& a, bool back, hipStream_t st) { return delta_of_type<float>(a, back, st); }

uint64_t delta_marks(const ffn_ray_delta& a) {
  return ((uint64_t)a.rays.n + DL_MARK - 1) / DL_MARK * a.v_heads * delta_rows(a.key_dim) * delta_waves(a.val_dim) * 16 * sizeof(float);
}
uint64_t delta_workspace(const ffn_ray_delta& a) {
  return a.heads == a.v_heads ? 0 : 2ull * a.rays.n * a.v_heads * a.key_dim * sizeof(float);
}

hipError_t launch_delta(const ffn_ray_delta& a, bool back, hipStream_t st) {
  if (!a.rays.num_rays && !a.rays.n) return hipSuccess;
  if (a.dtype == FFN_F32) return delta_f32(a, back, st);
  if (a.dtype == FFN_F16) return delta_f16(a, back, st);
  return delta_bf16(a, back, st);
}

}  // namespace ffn
