// ffn_route.hip -- rows to several experts and back: copies in the experts' order, weighted sums, their gradients.
//
// The plan over the n k places (place i k + j: row i's j-th expert) says which place each slot holds, and its move writes
// the inverse, the slot of each place, in the places' order as it goes.  Everything then goes by rows: a team of lanes takes a row, its k
// slots, and for each of them reads or writes one row of the slots' array.  So the rows' own array is passed over once,
// and no sum is split: no atomics, one order.  A place of no expert has a slot behind all groups; it is written as 0 and
// never read.  Memory bounds all of it: 2^20 rows of 128 bytes to 2 of 64 experts out 64 us, back 96 (6.3 and 4.2 TB/s with
// what the last-level cache gives); 50,021 rows of 2 KiB to 4 of 128 out 79, back 119, gradient 160; 300,007 rows of 64 bytes
// to 8 of 27, half lines, 44, 53 and 89 (4.0, 3.3 and 3.8 TB/s).
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int RT_NT = 256;

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

enum { ROUTE_OUT, ROUTE_BACK, ROUTE_GRAD };

// OUT: slots_out[slot] = rows_in[i];  BACK: rows_out[i] = sum_j w_ij slots_in[slot_ij];
// GRAD: slots_out[slot_ij] = w_ij rows_in[i], dweights_ij = rows_in[i] . slots_in[slot_ij]
// U: rows of slots that a lane has on their way
template <typename T, int EL, int WHAT, int U>
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
  T* to = (T*)a.slots_out;
  const int width = there ? a.width : 0;
  // U places at a time, every load of them on its way before the first is waited for: places past k are the last one
  // again, slots of no expert the first one; what is loaded there is dropped
  for (int c0 = 0; c0 < (WHAT == ROUTE_BACK ? width : 1); c0 += team * EL) {
    const int cb = c0 + lane * EL;  // of BACK
    const bool in_row = cb < width;
    float sum[EL];
#pragma unroll
    for (int e = 0; e < EL; ++e) sum[e] = 0.f;
    for (int j = 0; j < k; j += U) {
      uint32_t slot[U];
      float w[U], dot[U];
      bool kept_u[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        slot[u] = slots[min(j + u, k - 1)];
        w[u] = WHAT != ROUTE_OUT && weights ? weights[min(j + u, k - 1)] : 1.f;
        dot[u] = 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) kept_u[u] = slot[u] < kept && j + u < k;
      if constexpr (WHAT == ROUTE_BACK) {
        vec y[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          y[u] = *reinterpret_cast<const vec*>(from + (int64_t)(kept_u[u] ? slot[u] : 0) * a.slots_stride + (in_row ? cb : 0));
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
          for (int e = 0; e < EL; ++e) sum[e] = kept_u[u] ? __builtin_fmaf(w[u], part_at<T, EL>(y[u], e), sum[e]) : sum[e];
        }
      } else {
        for (int c = lane * EL; c < width; c += team * EL) {
          const vec x = *reinterpret_cast<const vec*>(in + c);
          vec y[U];
          if (WHAT == ROUTE_GRAD && a.dweights) {
#pragma unroll
            for (int u = 0; u < U; ++u)
              y[u] = *reinterpret_cast<const vec*>(from + (int64_t)(kept_u[u] ? slot[u] : 0) * a.slots_stride + c);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            vec d{};
            if constexpr (WHAT == ROUTE_OUT) {
              if (kept_u[u]) d = x;
            } else {
#pragma unroll
              for (int e = 0; e < EL; ++e) {
                const float g = part_at<T, EL>(x, e);
                if (a.dweights) dot[u] = __builtin_fmaf(g, part_at<T, EL>(y[u], e), dot[u]);
                part_set<T, EL>(d, e, kept_u[u] ? w[u] * g : 0.f);
              }
            }
            if (j + u < k) *reinterpret_cast<vec*>(to + (int64_t)slot[u] * a.width + c) = d;
          }
        }
        if (WHAT == ROUTE_GRAD && a.dweights) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            for (int d = 1; d < team; d *= 2) dot[u] += __shfl_xor(dot[u], d);
            if (lane == 0 && there && j + u < k) a.dweights[i * k + j + u] = kept_u[u] ? dot[u] : 0.f;
          }
        }
      }
    }
    if (WHAT == ROUTE_BACK && in_row) {
      vec out;
#pragma unroll
      for (int e = 0; e < EL; ++e) part_set<T, EL>(out, e, sum[e]);
      *reinterpret_cast<vec*>((T*)a.rows_out + i * a.width + cb) = out;
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
  const dim3 grid = grid_of((a.n + rows - 1) / rows);
  // 300,007 rows of 64 bytes to 8 experts, us: out 44 with eight places at once, 53 with four; back 60 and 53
  constexpr int MOST = WHAT == ROUTE_OUT ? 8 : 4;
  if (a.k <= 2) k_route<T, EL, WHAT, 2><<<grid, RT_NT, 0, st>>>(a, team);
  else if (a.k <= 4) k_route<T, EL, WHAT, 4><<<grid, RT_NT, 0, st>>>(a, team);
  else k_route<T, EL, WHAT, MOST><<<grid, RT_NT, 0, st>>>(a, team);
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

hipError_t launch_dispatch(const ffn_route& a, hipStream_t st) { return by_type<ROUTE_OUT>(a, st); }
hipError_t launch_combine(const ffn_route& a, hipStream_t st) { return by_type<ROUTE_BACK>(a, st); }
hipError_t launch_combine_bwd(const ffn_route& a, hipStream_t st) { return by_type<ROUTE_GRAD>(a, st); }

}  // namespace ffn
