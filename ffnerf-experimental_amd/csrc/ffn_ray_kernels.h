// ffn_ray_kernels.h -- launchers of the operators along rays and of the expert layers (internal to the library).
// Their arguments have been checked (ffn_ray_capi.hip).
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/ffnerf_hip.h"

namespace ffn {

uint64_t attn_workspace(const ffn_ray_attn& a, bool backward);
hipError_t launch_attn(const ffn_ray_attn& a, bool backward, hipStream_t st);

uint64_t scan_marks(const ffn_ray_scan& a);
uint64_t scan_workspace(const ffn_ray_scan& a, bool backward);
hipError_t launch_scan(const ffn_ray_scan& a, bool backward, hipStream_t st);

uint64_t delta_marks(const ffn_ray_delta& a);
uint64_t delta_workspace(const ffn_ray_delta& a);
hipError_t launch_delta(const ffn_ray_delta& a, bool backward, hipStream_t st);

uint64_t expert_plan_words(uint32_t n, int experts);
uint64_t expert_plan_workspace(uint32_t n, int experts);
// slots: the inverse of the plan's rows, or NULL
hipError_t launch_expert_plan(const int32_t* ids, uint32_t n, int experts, uint32_t* plan, uint32_t* slots, uint32_t* workspace,
                              hipStream_t st);
uint64_t expert_workspace(const ffn_experts& a);
hipError_t launch_experts(const ffn_experts& a, bool backward, hipStream_t st);

uint64_t norm_workspace(const ffn_norm& a);
hipError_t launch_norm(const ffn_norm& a, bool backward, hipStream_t st);

hipError_t launch_dispatch(const ffn_route& a, hipStream_t st);
hipError_t launch_combine(const ffn_route& a, hipStream_t st);
hipError_t launch_combine_bwd(const ffn_route& a, hipStream_t st);

// the message of ffn_last_error; returns code
int set_error(int code, const char* msg);

}  // namespace ffn
