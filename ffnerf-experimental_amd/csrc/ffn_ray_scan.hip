// ffn_ray_scan.hip -- the gated recurrence h_t = (1 - z_t) h_{t-1} + z_t x_t, z = sigmoid(gate), along rays.
//
// Per channel and in float.  A thread takes V neighbouring channels of one ray and walks it; the loads do not depend on
// the state, so a block of rows is in flight while the one before it is combined.
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int SC_NT = 256;
constexpr int SC_MARK = 16;  // a state is kept every so many rows of a ray for the backward pass

struct RayPath {
  int64_t first;  // row of place 0
  int64_t at;     // place 0 counted in the direction of the walk (marks)
  int len, step;
};
// ray r's rows in the direction of the walk; rows past n are cut off
__device__ __forceinline__ RayPath path_of(const ffn_ray_scan& a, uint32_t r) {
  const int64_t n = a.rays.n, o = min((int64_t)a.rays.offsets[r], n), len = min((int64_t)a.rays.counts[r], n - o);
  if (a.reverse) return {o + len - 1, n - o - len, (int)len, -1};
  return {o, o, (int)len, 1};
}

// V neighbouring channels
template <typename T, int V> struct Chan {
  typedef T vec __attribute__((ext_vector_type(V)));
};
template <typename T> struct Chan<T, 1> {
  typedef T vec;
};
template <int V, typename X> __device__ __forceinline__ float get(const X& x, int i) {
  if constexpr (V == 1) return (float)x;
  else return (float)x[i];
}
template <typename T, int V> __device__ __forceinline__ void put(typename Chan<T, V>::vec& x, int i, float v) {
  if constexpr (V == 1) x = (T)v;
  else x[i] = (T)v;
}

__device__ __forceinline__ float sigmoid_f(float g) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(g * -1.4426950408889634f));
}

// a row that no ray holds gets 0
template <typename T>
__device__ void clear_outside(const ffn_ray_scan& a, int64_t i, T* p0, T* p1) {
  if (i >= a.rays.n) return;
  const uint32_t r = a.rays.ray_ids[i];
  if (r < a.rays.num_rays) {
    const int64_t o = a.rays.offsets[r];
    if (i >= o && i - o < (int64_t)a.rays.counts[r]) return;
  }
  for (int c = 0; c < a.channels; ++c) {
    p0[i * a.channels + c] = (T)0.f;
    if (p1) p1[i * a.channels + c] = (T)0.f;
  }
}

template <typename T, int V>
__global__ __launch_bounds__(SC_NT) void k_scan_fwd(ffn_ray_scan a, int64_t ray_blocks) {
  if (blockIdx.x >= ray_blocks) {
    clear_outside<T>(a, (blockIdx.x - ray_blocks) * SC_NT + threadIdx.x, (T*)a.h, nullptr);
    return;
  }
  typedef typename Chan<T, V>::vec vec;
  constexpr int U = SC_MARK / 2;
  const int lanes = a.channels / V;
  const int64_t id = (int64_t)blockIdx.x * SC_NT + threadIdx.x;
  const int64_t ray = id / lanes;
  if (ray >= a.rays.num_rays) return;
  const int ch = (int)(id % lanes) * V;
  const RayPath p = path_of(a, (uint32_t)ray);
  const T* gp = (const T*)a.gate + p.first * a.gate_row + ch;
  const T* xp = (const T*)a.x + p.first * a.x_row + ch;
  T* hp = (T*)a.h + p.first * a.channels + ch;
  const int64_t gs = p.step * a.gate_row, xs = p.step * a.x_row, hs = (int64_t)p.step * a.channels;
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = a.h0 ? a.h0[ray * a.channels + ch + v] : 0.f;
  vec g[U], x[U];
  auto fetch = [&](int k) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < p.len) {
        g[u] = *reinterpret_cast<const vec*>(gp + (k + u) * gs);
        x[u] = *reinterpret_cast<const vec*>(xp + (k + u) * xs);
      }
  };
  fetch(0);
  for (int k = 0; k < p.len; k += U) {
    vec gc[U], xc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) gc[u] = g[u], xc[u] = x[u];
    fetch(k + U);
    if (a.marks && k && k % SC_MARK == 0) {
      float* m = a.marks + (p.at + k) / SC_MARK * a.channels + ch;
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = h[v];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u < p.len) {
        vec out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float z = sigmoid_f(get<V>(gc[u], v));
          h[v] = __builtin_fmaf(1.f - z, h[v], z * get<V>(xc[u], v));
          put<T, V>(out, v, h[v]);
        }
        *reinterpret_cast<vec*>(hp + (k + u) * hs) = out;
      }
  }
  if (a.last) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.last[ray * a.channels + ch + v] = h[v];
  }
}

// The ray is walked back in pieces of SC_MARK rows: a piece's states come again from the mark before it, in registers,
// so the backward pass does not read h (which is rounded) and writes the gradients in one pass.
template <typename T, int V>
__global__ __launch_bounds__(SC_NT) void k_scan_bwd(ffn_ray_scan a, int64_t ray_blocks) {
  if (blockIdx.x >= ray_blocks) {
    clear_outside<T>(a, (blockIdx.x - ray_blocks) * SC_NT + threadIdx.x, (T*)a.dgate, (T*)a.dx);
    return;
  }
  typedef typename Chan<T, V>::vec vec;
  constexpr int L = SC_MARK;
  const int lanes = a.channels / V;
  const int64_t id = (int64_t)blockIdx.x * SC_NT + threadIdx.x;
  const int64_t ray = id / lanes;
  if (ray >= a.rays.num_rays) return;
  const int ch = (int)(id % lanes) * V;
  const RayPath p = path_of(a, (uint32_t)ray);
  const T* gp = (const T*)a.gate + p.first * a.gate_row + ch;
  const T* xp = (const T*)a.x + p.first * a.x_row + ch;
  const T* dp = (const T*)a.dh + p.first * a.dh_row + ch;
  T* dgp = (T*)a.dgate + p.first * a.channels + ch;
  T* dxp = (T*)a.dx + p.first * a.channels + ch;
  const int64_t gs = p.step * a.gate_row, xs = p.step * a.x_row, ds = p.step * a.dh_row, os = (int64_t)p.step * a.channels;
  float d[V];
#pragma unroll
  for (int v = 0; v < V; ++v) d[v] = a.dlast ? a.dlast[ray * a.channels + ch + v] : 0.f;
  for (int k = p.len > 0 ? (p.len - 1) / L * L : -1; k >= 0; k -= L) {
    vec g[L], x[L], dh[L];
#pragma unroll
    for (int u = 0; u < L; ++u)
      if (k + u < p.len) {
        g[u] = *reinterpret_cast<const vec*>(gp + (k + u) * gs);
        x[u] = *reinterpret_cast<const vec*>(xp + (k + u) * xs);
        dh[u] = *reinterpret_cast<const vec*>(dp + (k + u) * ds);
      }
    float z[L][V], before[L][V], h[V];
    const float* m = k ? a.marks + (p.at + k) / L * a.channels + ch : (a.h0 ? a.h0 + ray * a.channels + ch : nullptr);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = m ? m[v] : 0.f;
#pragma unroll
    for (int u = 0; u < L; ++u)
      if (k + u < p.len) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          z[u][v] = sigmoid_f(get<V>(g[u], v));
          before[u][v] = h[v];
          h[v] = __builtin_fmaf(1.f - z[u][v], h[v], z[u][v] * get<V>(x[u], v));
        }
      }
#pragma unroll
    for (int u = L - 1; u >= 0; --u)
      if (k + u < p.len) {
        vec og, ox;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float D = get<V>(dh[u], v) + d[v], zz = z[u][v], keep = 1.f - zz;
          put<T, V>(ox, v, zz * D);
          put<T, V>(og, v, D * (get<V>(x[u], v) - before[u][v]) * (zz * keep));
          d[v] = keep * D;
        }
        *reinterpret_cast<vec*>(dgp + (k + u) * os) = og;
        *reinterpret_cast<vec*>(dxp + (k + u) * os) = ox;
      }
  }
  if (a.dh0) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.dh0[ray * a.channels + ch + v] = d[v];
  }
}

static bool aligned(const void* p, int64_t row, int bytes, int size) {
  return ((uintptr_t)p | (uintptr_t)(row * size)) % bytes == 0;
}

template <typename T, int V>
static hipError_t run(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  const int64_t rb = ((int64_t)a.rays.num_rays * (a.channels / V) + SC_NT - 1) / SC_NT;
  const int64_t cb = ((int64_t)a.rays.n + SC_NT - 1) / SC_NT;
  if (rb + cb == 0) return hipSuccess;
  if (backward) k_scan_bwd<T, V><<<(unsigned)(rb + cb), SC_NT, 0, st>>>(a, rb);
  else k_scan_fwd<T, V><<<(unsigned)(rb + cb), SC_NT, 0, st>>>(a, rb);
  return hipGetLastError();
}

template <typename T>
static hipError_t by_width(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  constexpr int S = sizeof(T), V = sizeof(T) == 4 ? 2 : 4;
  bool wide = a.channels % V == 0 && aligned(a.gate, a.gate_row, V * S, S) && aligned(a.x, a.x_row, V * S, S);
  if (backward)
    wide = wide && aligned(a.dh, a.dh_row, V * S, S) && aligned(a.dgate, 0, V * S, S) && aligned(a.dx, 0, V * S, S);
  else wide = wide && aligned(a.h, 0, V * S, S);
  return wide ? run<T, V>(a, backward, st) : run<T, 1>(a, backward, st);
}

uint64_t scan_marks(const ffn_ray_scan& a) {
  return ((uint64_t)a.rays.n + SC_MARK - 1) / SC_MARK * a.channels * sizeof(float);
}
uint64_t scan_workspace(const ffn_ray_scan&, bool) { return 0; }

hipError_t launch_scan(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  if (a.dtype == FFN_BF16) return by_width<__bf16>(a, backward, st);
  if (a.dtype == FFN_F16) return by_width<_Float16>(a, backward, st);
  return by_width<float>(a, backward, st);
}

}  // namespace ffn
