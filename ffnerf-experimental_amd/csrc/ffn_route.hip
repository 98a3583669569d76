// ffn_route.hip -- rows to several experts and back: copies in the experts' order, weighted sums, their gradients.
//
// A plan (ffn_expert_plan) over the n k places (place i k + j: row i's j-th expert) says which place each slot holds; here
// its inverse, the slot of each place, is kept beside it.  Everything then goes by rows: a team of lanes takes a row, its k
// slots, and for each of them reads or writes one row of the slots' array.  So the rows' own array is passed over once,
// and no sum is split: no atomics, one order.  A place of no expert has a slot behind all groups; it is written as 0 and
// never read.  Memory bounds all of it.
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int RT_NT = 256;

__global__ __launch_bounds__(RT_NT) void k_route_slots(const uint32_t* __restrict__ places, uint32_t n, uint32_t* __restrict__ slots) {
  const int64_t s = block_number() * RT_NT + threadIdx.x;
  if (s < n) slots[places[s]] = (uint32_t)s;
}

// EL neighbouring columns: 16 bytes, or one column where rows are not aligned
template <typename T, int EL> struct Part {
  typedef T type __attribute__((ext_vector_type(EL)));
};
template <typename T> struct Part<T, 1> {
  typedef T type;
};
template <typename T, int EL> __device__ __forceinline__ float part_at(const typename Part<T, EL>::type& v, int e) {
  if constexpr (EL == 1) return (float)v;
  else return (float)v[e];
}
template <typename T, int EL> __device__ __forceinline__ void part_set(typename Part<T, EL>::type& v, int e, float f) {
  if constexpr (EL == 1) v = (T)f;
  else v[e] = (T)f;
}

constexpr int RT_AT_ONCE = 4;  // rows of slots a lane has on their way

enum { ROUTE_OUT, ROUTE_BACK, ROUTE_GRAD };

// OUT: slots_out[slot] = rows_in[i];  BACK: rows_out[i] = sum_j w_ij slots_in[slot_ij];
// GRAD: slots_out[slot_ij] = w_ij rows_in[i], dweights_ij = rows_in[i] . slots_in[slot_ij]
template <typename T, int EL, int WHAT>
__global__ __launch_bounds__(RT_NT) void k_route(const ffn_route a, int team) {
  typedef typename Part<T, EL>::type vec;
  const int lane = threadIdx.x & (team - 1), k = a.k;
  const int64_t i = block_number() * (RT_NT / team) + threadIdx.x / team;
  const bool there = i < a.n;  // every lane goes on: the sums of GRAD are exchanged between them
  const uint32_t kept = a.plan[a.n_experts + 1 + a.n_experts];  // slots before those of no expert
  const uint32_t* slots = a.slots + (there ? i : 0) * k;
  const float* weights = a.weights ? a.weights + (there ? i : 0) * k : nullptr;
  const T* in = (const T*)a.rows_in + (there ? i : 0) * a.rows_stride;
  const T* from = (const T*)a.slots_in;
  const int width = there ? a.width : 0;
  for (int j0 = 0; j0 < k; j0 += WHAT == ROUTE_GRAD ? RT_AT_ONCE : k) {
    uint32_t slot[RT_AT_ONCE];
    float w[RT_AT_ONCE], dot[RT_AT_ONCE];
    if constexpr (WHAT == ROUTE_GRAD) {
#pragma unroll
      for (int u = 0; u < RT_AT_ONCE; ++u) {
        slot[u] = j0 + u < k ? slots[j0 + u] : 0xFFFFFFFFu;
        w[u] = weights && j0 + u < k ? weights[j0 + u] : 1.f;
        dot[u] = 0.f;
      }
    }
    for (int c = lane * EL; c < width; c += team * EL) {
      if constexpr (WHAT == ROUTE_OUT) {
        const vec x = *reinterpret_cast<const vec*>(in + c);
        for (int j = 0; j < k; ++j) {
          const uint32_t s = slots[j];
          *reinterpret_cast<vec*>((T*)a.slots_out + (int64_t)s * a.width + c) = s < kept ? x : vec{};
        }
      } else if constexpr (WHAT == ROUTE_BACK) {
        float sum[EL];
#pragma unroll
        for (int e = 0; e < EL; ++e) sum[e] = 0.f;
        for (int j = 0; j < k; j += RT_AT_ONCE) {
          vec y[RT_AT_ONCE];
          float f[RT_AT_ONCE];
#pragma unroll
          for (int u = 0; u < RT_AT_ONCE; ++u) {
            const uint32_t s = j + u < k ? slots[j + u] : 0xFFFFFFFFu;
            y[u] = vec{};
            f[u] = 0.f;
            if (s < kept) {
              y[u] = *reinterpret_cast<const vec*>(from + (int64_t)s * a.slots_stride + c);
              f[u] = weights ? weights[j + u] : 1.f;
            }
          }
#pragma unroll
          for (int u = 0; u < RT_AT_ONCE; ++u) {
#pragma unroll
            for (int e = 0; e < EL; ++e) sum[e] = __builtin_fmaf(f[u], part_at<T, EL>(y[u], e), sum[e]);
          }
        }
        vec out;
#pragma unroll
        for (int e = 0; e < EL; ++e) part_set<T, EL>(out, e, sum[e]);
        *reinterpret_cast<vec*>((T*)a.rows_out + i * a.width + c) = out;
      } else {
        const vec x = *reinterpret_cast<const vec*>(in + c);
        vec y[RT_AT_ONCE];
#pragma unroll
        for (int u = 0; u < RT_AT_ONCE; ++u) {
          y[u] = vec{};
          if (a.dweights && slot[u] < kept) y[u] = *reinterpret_cast<const vec*>(from + (int64_t)slot[u] * a.slots_stride + c);
        }
#pragma unroll
        for (int u = 0; u < RT_AT_ONCE; ++u) {
          vec d{};
          if (slot[u] < kept) {
#pragma unroll
            for (int e = 0; e < EL; ++e) {
              const float g = part_at<T, EL>(x, e);
              dot[u] = __builtin_fmaf(g, part_at<T, EL>(y[u], e), dot[u]);
              part_set<T, EL>(d, e, w[u] * g);
            }
          }
          if (j0 + u < k) *reinterpret_cast<vec*>((T*)a.slots_out + (int64_t)slot[u] * a.width + c) = d;
        }
      }
    }
    if constexpr (WHAT == ROUTE_GRAD) {
      if (a.dweights) {
#pragma unroll
        for (int u = 0; u < RT_AT_ONCE; ++u) {
          for (int d = 1; d < team; d *= 2) dot[u] += __shfl_xor(dot[u], d);
          if (lane == 0 && there && j0 + u < k) a.dweights[i * k + j0 + u] = slot[u] < kept ? dot[u] : 0.f;
        }
      }
    }
  }
}

namespace {

bool fits(const void* p, int64_t row, int64_t n, int size) { return !((uintptr_t)p & 15) && (n < 2 || row * size % 16 == 0); }

template <typename T, int EL, int WHAT>
void start(const ffn_route& a, hipStream_t st) {
  int team = 1;  // a power of two, so that it divides a wavefront
  while (team < 64 && team * EL < a.width) team *= 2;
  const int64_t rows = RT_NT / team;
  k_route<T, EL, WHAT><<<grid_of((a.n + rows - 1) / rows), RT_NT, 0, st>>>(a, team);
}

template <typename T, int WHAT>
void choose(const ffn_route& a, hipStream_t st) {
  constexpr int EL = 16 / (int)sizeof(T), S = (int)sizeof(T);
  const int64_t places = (int64_t)a.n * a.k;
  const bool vec = a.width % EL == 0 && fits(a.rows_in, a.rows_stride, a.n, S) && fits(a.slots_in, a.slots_stride, places, S) &&
                   fits(a.rows_out, 0, 0, S) && fits(a.slots_out, 0, 0, S);
  if (vec) start<T, EL, WHAT>(a, st);
  else start<T, 1, WHAT>(a, st);
}

template <int WHAT>
hipError_t by_type(const ffn_route& a, hipStream_t st) {
  if (a.n) {
    if (a.dtype == FFN_F32) choose<float, WHAT>(a, st);
    else if (a.dtype == FFN_F16) choose<_Float16, WHAT>(a, st);
    else choose<__bf16, WHAT>(a, st);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t launch_route_slots(const uint32_t* plan, uint32_t places, int n_experts, uint32_t* slots, hipStream_t st) {
  if (places)
    k_route_slots<<<grid_of(((int64_t)places + RT_NT - 1) / RT_NT), RT_NT, 0, st>>>(
        plan + expert_plan_words(places, n_experts) - places, places, slots);
  return hipGetLastError();
}

hipError_t launch_dispatch(const ffn_route& a, hipStream_t st) { return by_type<ROUTE_OUT>(a, st); }
hipError_t launch_combine(const ffn_route& a, hipStream_t st) { return by_type<ROUTE_BACK>(a, st); }
hipError_t launch_combine_bwd(const ffn_route& a, hipStream_t st) { return by_type<ROUTE_GRAD>(a, st); }

}  // namespace ffn
