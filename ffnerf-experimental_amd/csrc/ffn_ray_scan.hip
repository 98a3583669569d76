// ffn_ray_scan.hip -- the gated recurrence h_t = (1 - z_t) h_{t-1} + z_t x_t, z = sigmoid(gate), along rays.
//
// Per channel and in float.  A thread takes V neighbouring channels and walks rows in order; nothing it loads depends on
// the state, so the rows of one step are in flight while those of the step before are combined.  What a thread walks:
//   * by rays: one whole ray.  One launch, every value read once.
//   * by parts: a part of the packed rows of a fixed length, whatever rays it holds, so that few long rays fill the GPU
//     too.  A part that begins inside a ray needs the state there: k_scan_ends composes, per part, the steps of the ray
//     that leaves it (h -> A h + B), k_scan_chain the parts of a ray, in a fixed order.  That reads gate and x a second
//     time, but only of rays that cross a part's end.
// The backward pass walks the other way with D_t = dh_t + (1 - z_{t+1}) D_{t+1}.
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int SC_NT = 256;
constexpr int SC_MARK = 16;  // a state is kept every so many rows of a walk for the backward pass

// Places are counted in the direction of the walk: place p is row p, or row n - 1 - p.
struct Walk {
  int64_t n;
  int step;
  __device__ __forceinline__ explicit Walk(const ffn_ray_scan& a) : n(a.rays.n), step(a.reverse ? -1 : 1) {}
  __device__ __forceinline__ int64_t row(int64_t p) const { return step < 0 ? n - 1 - p : p; }
};

// the places of ray r; rows past n are cut off
struct Span64 {
  int64_t from, to;
};
__device__ __forceinline__ Span64 places_of(const ffn_ray_scan& a, uint32_t r) {
  const int64_t n = a.rays.n, o = min((int64_t)a.rays.offsets[r], n), e = o + min((int64_t)a.rays.counts[r], n - o);
  if (a.reverse) return {n - e, n - o};
  return {o, e};
}

// the ray that holds place p, and its places; -1 and {p, p + 1} where none does
__device__ __forceinline__ int64_t ray_at(const ffn_ray_scan& a, const Walk& w, int64_t p, Span64& s) {
  const uint32_t r = a.rays.ray_ids[w.row(p)];
  if (r < a.rays.num_rays) {
    s = places_of(a, r);
    if (p >= s.from && p < s.to) return r;
  }
  s = {p, p + 1};
  return -1;
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

// N rows from p on, of which `left` are there: the last one again for the others, so that no lane branches
template <typename T, int V, int N>
__device__ __forceinline__ void load_rows(typename Chan<T, V>::vec (&to)[N], const T* p, int64_t stride, int left) {
#pragma unroll
  for (int u = 0; u < N; ++u) {
    to[u] = *reinterpret_cast<const typename Chan<T, V>::vec*>(p);
    p += u + 1 < left ? stride : 0;
  }
}

// the columns of one thread
template <typename T, int V>
struct Cols {
  typedef typename Chan<T, V>::vec vec;
  int ch;
  Walk w;
  const T *gate, *x;
  int64_t gs, xs;
  __device__ __forceinline__ Cols(const ffn_ray_scan& a, int c)
      : ch(c), w(a), gate((const T*)a.gate + c), x((const T*)a.x + c), gs(w.step * a.gate_row), xs(w.step * a.x_row) {}
};

// h over `len` > 0 places from `from` on; marks are kept at multiples of SC_MARK of the walk, and at its start if `mark0`
template <typename T, int V>
__device__ __forceinline__ void walk_fwd(const ffn_ray_scan& a, const Cols<T, V>& c, int64_t from, int len, bool mark0,
                                         float (&h)[V]) {
  typedef typename Cols<T, V>::vec vec;
  constexpr int U = 8;
  const int64_t row = c.w.row(from);
  const T* gp = c.gate + row * a.gate_row;
  const T* xp = c.x + row * a.x_row;
  T* hp = (T*)a.h + row * a.channels + c.ch;
  const int64_t hs = (int64_t)c.w.step * a.channels;
  vec g[U], x[U];
  load_rows<T, V, U>(g, gp, c.gs, len);
  load_rows<T, V, U>(x, xp, c.xs, len);
  for (int k = 0; k < len; k += U) {
    vec gc[U], xc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) gc[u] = g[u], xc[u] = x[u];
    if (k + U < len) {
      gp += U * c.gs;
      xp += U * c.xs;
      load_rows<T, V, U>(g, gp, c.gs, len - k - U);
      load_rows<T, V, U>(x, xp, c.xs, len - k - U);
    }
    if (a.marks && k % SC_MARK == 0 && (k || mark0)) {
      float* m = a.marks + (from + k) / SC_MARK * a.channels + c.ch;
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = h[v];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u < len) {
        vec out;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float z = sigmoid_f(get<V>(gc[u], v));
          h[v] = __builtin_fmaf(1.f - z, h[v], z * get<V>(xc[u], v));
          put<T, V>(out, v, h[v]);
        }
        *reinterpret_cast<vec*>(hp) = out;
      }
      hp += hs;
    }
  }
}

// Gradients over `len` > 0 places from `from` on, last to first, in pieces of SC_MARK: a piece's states come again from
// the mark before it, so that the backward pass neither reads h nor takes its rounding.  Of them it keeps z and
// q = (x - h_{t-1}) z (1 - z):  dx = z D, dgate = q D, and D goes on as (1 - z) D.  start: the state before a walk
// whose first piece has no mark (NULL: 0).
template <typename T, int V>
__device__ __forceinline__ void walk_bwd(const ffn_ray_scan& a, const Cols<T, V>& c, int64_t from, int len, bool mark0,
                                         const float* start, float (&d)[V]) {
  typedef typename Cols<T, V>::vec vec;
  constexpr int L = SC_MARK;
  int k = (len - 1) / L * L;
  const int64_t row = c.w.row(from + k), ds = c.w.step * a.dh_row, os = (int64_t)c.w.step * a.channels;
  const T* gp = c.gate + row * a.gate_row;
  const T* xp = c.x + row * a.x_row;
  const T* dp = (const T*)a.dh + row * a.dh_row + c.ch;
  T* og = (T*)a.dgate + row * a.channels + c.ch;
  T* ox = (T*)a.dx + row * a.channels + c.ch;
  vec g[L], x[L], dh[L];
  load_rows<T, V, L>(g, gp, c.gs, len - k);
  load_rows<T, V, L>(x, xp, c.xs, len - k);
  load_rows<T, V, L>(dh, dp, ds, len - k);
  for (; k >= 0; k -= L) {
    const float* m = k || mark0 ? a.marks + (from + k) / L * a.channels + c.ch : start;
    float h[V], z[L][V], q[L][V];
    vec dc[L];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = m ? m[v] : 0.f;
#pragma unroll
    for (int u = 0; u < L; ++u) {
      dc[u] = dh[u];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float zz = sigmoid_f(get<V>(g[u], v)), keep = 1.f - zz, xx = get<V>(x[u], v);
        z[u][v] = zz;
        q[u][v] = (xx - h[v]) * (zz * keep);
        h[v] = __builtin_fmaf(keep, h[v], zz * xx);
      }
    }
    const int left = len - k;
    T *wg = og + (L - 1) * os, *wx = ox + (L - 1) * os;
    if (k > 0) {
      gp -= L * c.gs, xp -= L * c.xs, dp -= L * ds;
      og -= L * os, ox -= L * os;
      load_rows<T, V, L>(g, gp, c.gs, L);
      load_rows<T, V, L>(x, xp, c.xs, L);
      load_rows<T, V, L>(dh, dp, ds, L);
    }
#pragma unroll
    for (int u = L - 1; u >= 0; --u) {
      if (u < left) {
        vec vg, vx;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float D = get<V>(dc[u], v) + d[v];
          put<T, V>(vx, v, z[u][v] * D);
          put<T, V>(vg, v, q[u][v] * D);
          d[v] = (1.f - z[u][v]) * D;
        }
        *reinterpret_cast<vec*>(wx) = vx;
        *reinterpret_cast<vec*>(wg) = vg;
      }
      wx -= os, wg -= os;
    }
  }
}

template <int V>
__device__ __forceinline__ void load_state(float (&s)[V], const float* from, int64_t ray, int channels, int ch) {
#pragma unroll
  for (int v = 0; v < V; ++v) s[v] = from ? from[ray * channels + ch + v] : 0.f;
}
template <int V>
__device__ __forceinline__ void store_state(float* to, int64_t ray, int channels, int ch, const float (&s)[V]) {
  if (!to) return;
#pragma unroll
  for (int v = 0; v < V; ++v) to[ray * channels + ch + v] = s[v];
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

// By rays: a thread a ray and V channels; the blocks past ray_blocks clear the rows of no ray.
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(SC_NT) void k_scan_rays(ffn_ray_scan a, int64_t ray_blocks) {
  if (blockIdx.x >= ray_blocks) {
    const int64_t i = (blockIdx.x - ray_blocks) * SC_NT + threadIdx.x;
    if (BACK) clear_outside<T>(a, i, (T*)a.dgate, (T*)a.dx);
    else clear_outside<T>(a, i, (T*)a.h, nullptr);
    return;
  }
  const int lanes = a.channels / V;
  const int64_t id = (int64_t)blockIdx.x * SC_NT + threadIdx.x;
  const int64_t ray = id / lanes;
  if (ray >= a.rays.num_rays) return;
  const Cols<T, V> c(a, (int)(id % lanes) * V);
  const Span64 s = places_of(a, (uint32_t)ray);
  const int len = (int)(s.to - s.from);
  float h[V];
  if constexpr (BACK) {
    load_state<V>(h, a.dlast, ray, a.channels, c.ch);
    if (len > 0) walk_bwd<T, V>(a, c, s.from, len, false, a.h0 ? a.h0 + ray * a.channels + c.ch : nullptr, h);
    store_state<V>(a.dh0, ray, a.channels, c.ch, h);
  } else {
    load_state<V>(h, a.h0, ray, a.channels, c.ch);
    if (len > 0) walk_fwd<T, V>(a, c, s.from, len, false, h);
    store_state<V>(a.last, ray, a.channels, c.ch, h);
  }
}

// By parts of `size` places (a multiple of SC_MARK): carry[part][channel] is the state at the part's start (BACK: D at
// its end).  The blocks past part_blocks give the rays without rows their last state.  Large inputs: parts in falling
// order, since k_scan_ends has just read the last ones (they are still in the last-level cache).
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(SC_NT) void k_scan_parts(ffn_ray_scan a, int size, int64_t parts, int64_t part_blocks,
                                                      const float* __restrict__ carry) {
  const int lanes = a.channels / V;
  if (blockIdx.x >= part_blocks) {
    const int64_t id = (blockIdx.x - part_blocks) * SC_NT + threadIdx.x, ray = id / lanes;
    if (ray >= a.rays.num_rays) return;
    const Span64 s = places_of(a, (uint32_t)ray);
    if (s.to > s.from) return;
    const int ch = (int)(id % lanes) * V;
    float h[V];
    load_state<V>(h, BACK ? a.dlast : a.h0, ray, a.channels, ch);
    store_state<V>(BACK ? a.dh0 : a.last, ray, a.channels, ch, h);
    return;
  }
  const int64_t id = (part_blocks - 1 - blockIdx.x) * SC_NT + threadIdx.x;
  const int64_t part = id / lanes;
  if (part >= parts) return;
  const Cols<T, V> c(a, (int)(id % lanes) * V);
  const int64_t p0 = part * size, p1 = min(p0 + size, (int64_t)a.rays.n);
  float h[V];
  int64_t p = BACK ? p1 - 1 : p0;
  while (BACK ? p >= p0 : p < p1) {
    Span64 s;
    const int64_t ray = ray_at(a, c.w, p, s);
    if (ray < 0) {
      typename Cols<T, V>::vec zero;
#pragma unroll
      for (int v = 0; v < V; ++v) put<T, V>(zero, v, 0.f);
      const int64_t at = c.w.row(p) * a.channels + c.ch;
      *reinterpret_cast<typename Cols<T, V>::vec*>((BACK ? (T*)a.dx : (T*)a.h) + at) = zero;
      if (BACK) *reinterpret_cast<typename Cols<T, V>::vec*>((T*)a.dgate + at) = zero;
      p += BACK ? -1 : 1;
      continue;
    }
    const int64_t from = max(s.from, p0), to = min(s.to, p1);
    const int len = (int)(to - from);
    const bool inside = from > s.from;  // the walk begins inside the ray
    if constexpr (BACK) {
      if (to < s.to) load_state<V>(h, carry, part, a.channels, c.ch);
      else load_state<V>(h, a.dlast, ray, a.channels, c.ch);
      walk_bwd<T, V>(a, c, from, len, inside, a.h0 ? a.h0 + ray * a.channels + c.ch : nullptr, h);
      if (!inside) store_state<V>(a.dh0, ray, a.channels, c.ch, h);
      p = from - 1;
    } else {
      if (inside) load_state<V>(h, carry, part, a.channels, c.ch);
      else load_state<V>(h, a.h0, ray, a.channels, c.ch);
      walk_fwd<T, V>(a, c, from, len, inside, h);
      if (to == s.to) store_state<V>(a.last, ray, a.channels, c.ch, h);
      p = to;
    }
  }
}

// The ray that leaves each part in the direction of the walk: the part's steps of it as h -> A h + B, with A = 0 where
// the ray begins (BACK: ends) in the part, so that B is the state.  A = B = 0 where none leaves.
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(SC_NT) void k_scan_ends(ffn_ray_scan a, int size, int64_t parts, float* __restrict__ A_of,
                                                     float* __restrict__ B_of) {
  constexpr int U = 8;
  typedef typename Chan<T, V>::vec vec;
  const int lanes = a.channels / V;
  const int64_t id = (int64_t)blockIdx.x * SC_NT + threadIdx.x;
  const int64_t part = id / lanes;
  if (part >= parts) return;
  const Cols<T, V> c(a, (int)(id % lanes) * V);
  const int64_t p0 = part * size, p1 = min(p0 + size, (int64_t)a.rays.n);
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = B[v] = 0.f;
  Span64 s;
  const int64_t ray = ray_at(a, c.w, BACK ? p0 : p1 - 1, s);
  if (ray >= 0 && (BACK ? s.from < p0 : s.to > p1)) {
    const int64_t from = max(s.from, p0), to = min(s.to, p1);
    const bool whole = BACK ? to == s.to : from == s.from;
    const int len = (int)(to - from);
    if (whole) load_state<V>(B, BACK ? a.dlast : a.h0, ray, a.channels, c.ch);
    else {
#pragma unroll
      for (int v = 0; v < V; ++v) A[v] = 1.f;
    }
    const int64_t row = c.w.row(BACK ? to - 1 : from), dir = BACK ? -1 : 1;
    const T* gp = c.gate + row * a.gate_row;
    const T* xp = BACK ? (const T*)a.dh + row * a.dh_row + c.ch : c.x + row * a.x_row;
    const int64_t gs = dir * c.gs, xs = BACK ? -c.w.step * a.dh_row : c.xs;
    vec g[U], x[U];
    load_rows<T, V, U>(g, gp, gs, len);
    load_rows<T, V, U>(x, xp, xs, len);
    for (int k = 0; k < len; k += U) {
      vec gc[U], xc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) gc[u] = g[u], xc[u] = x[u];
      if (k + U < len) {
        gp += U * gs;
        xp += U * xs;
        load_rows<T, V, U>(g, gp, gs, len - k - U);
        load_rows<T, V, U>(x, xp, xs, len - k - U);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u < len) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float z = sigmoid_f(get<V>(gc[u], v)), keep = 1.f - z;
            A[v] *= keep;
            // BACK: the D that leaves a step is (1 - z) (dh + D)
            B[v] = BACK ? keep * (B[v] + get<V>(xc[u], v)) : __builtin_fmaf(keep, B[v], z * get<V>(xc[u], v));
          }
        }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A_of[part * a.channels + c.ch + v] = A[v];
    B_of[part * a.channels + c.ch + v] = B[v];
  }
}

// carry[j]: what enters part j (BACK: from the part after it).  A block a channel: a thread composes its run of parts, the
// runs are scanned in LDS, and the thread walks its run again.
constexpr int CH_NT = 1024;
template <bool BACK>
__global__ __launch_bounds__(CH_NT) void k_scan_chain(int channels, int64_t parts, const float* __restrict__ A_of,
                                                      const float* __restrict__ B_of, float* __restrict__ carry) {
  __shared__ float sa[CH_NT], sb[CH_NT];
  const int ch = blockIdx.x, tid = threadIdx.x;
  const int64_t run = (parts + CH_NT - 1) / CH_NT, j0 = min(tid * run, parts), j1 = min(j0 + run, parts);
  auto at = [&](int64_t j) { return (BACK ? parts - 1 - j : j) * channels + ch; };
  float A = 1.f, B = 0.f;
  for (int64_t j = j0; j < j1; ++j) {
    const float a = A_of[at(j)], b = B_of[at(j)];
    A *= a;
    B = __builtin_fmaf(a, B, b);
  }
  sa[tid] = A;
  sb[tid] = B;
  __syncthreads();
  for (int d = 1; d < CH_NT; d *= 2) {
    float a = 1.f, b = 0.f;
    if (tid >= d) a = sa[tid - d], b = sb[tid - d];
    __syncthreads();
    B = __builtin_fmaf(A, b, B);
    A *= a;
    sa[tid] = A;
    sb[tid] = B;
    __syncthreads();
  }
  float h = tid ? sb[tid - 1] : 0.f;
  for (int64_t j = j0; j < j1; ++j) {
    carry[at(j)] = h;
    h = __builtin_fmaf(A_of[at(j)], h, B_of[at(j)]);
  }
}

static bool aligned(const void* p, int64_t row, int bytes, int size) {
  return ((uintptr_t)p | (uintptr_t)(row * size)) % bytes == 0;
}

// Which walk: by rays where they are many and short.  PLAN_THREADS: threads (of channels / 2 lanes a ray or part) that
// fill the GPU.
constexpr int64_t SC_THREADS = 262144;
static bool by_rays(const ffn_ray_scan& a) {
  const int64_t lanes = (a.channels + 1) / 2, avg = a.rays.num_rays ? (int64_t)a.rays.n / a.rays.num_rays : 0;
  return avg <= 64 || (avg <= 512 && a.rays.num_rays * lanes >= SC_THREADS / 2);
}
static int part_size(const ffn_ray_scan& a) {
  const int64_t lanes = (a.channels + 1) / 2;
  int64_t s = (int64_t)a.rays.n * lanes / SC_THREADS;
  s = (s + SC_MARK - 1) / SC_MARK * SC_MARK;
  return (int)(s < 64 ? 64 : s > 4096 ? 4096 : s);
}

template <typename T, int V, bool BACK>
static hipError_t run(const ffn_ray_scan& a, hipStream_t st) {
  const int64_t lanes = a.channels / V;
  if (by_rays(a)) {
    const int64_t rb = (a.rays.num_rays * lanes + SC_NT - 1) / SC_NT, cb = ((int64_t)a.rays.n + SC_NT - 1) / SC_NT;
    if (rb + cb) k_scan_rays<T, V, BACK><<<(unsigned)(rb + cb), SC_NT, 0, st>>>(a, rb);
    return hipGetLastError();
  }
  const int size = part_size(a);
  const int64_t parts = ((int64_t)a.rays.n + size - 1) / size, states = parts * a.channels;
  float *A = (float*)a.workspace, *B = A + states, *carry = B + states;
  const int64_t pb = (parts * lanes + SC_NT - 1) / SC_NT, rb = (a.rays.num_rays * lanes + SC_NT - 1) / SC_NT;
  k_scan_ends<T, V, BACK><<<(unsigned)pb, SC_NT, 0, st>>>(a, size, parts, A, B);
  k_scan_chain<BACK><<<a.channels, CH_NT, 0, st>>>(a.channels, parts, A, B, carry);
  k_scan_parts<T, V, BACK><<<(unsigned)(pb + rb), SC_NT, 0, st>>>(a, size, parts, pb, carry);
  return hipGetLastError();
}

template <typename T, int V, bool BACK>
static hipError_t by_width(const ffn_ray_scan& a, hipStream_t st) {
  constexpr int S = sizeof(T);
  if constexpr (V > 1) {
    bool wide = a.channels % V == 0 && aligned(a.gate, a.gate_row, V * S, S) && aligned(a.x, a.x_row, V * S, S);
    if (BACK)
      wide = wide && aligned(a.dh, a.dh_row, V * S, S) && aligned(a.dgate, 0, V * S, S) && aligned(a.dx, 0, V * S, S);
    else wide = wide && aligned(a.h, 0, V * S, S);
    if (wide) return run<T, V, BACK>(a, st);
  }
  return run<T, 1, BACK>(a, st);
}

uint64_t scan_marks(const ffn_ray_scan& a) {
  return ((uint64_t)a.rays.n + SC_MARK - 1) / SC_MARK * a.channels * sizeof(float);
}
uint64_t scan_workspace(const ffn_ray_scan& a, bool) {
  if (by_rays(a)) return 0;
  const int size = part_size(a);
  return ((uint64_t)a.rays.n + size - 1) / size * a.channels * 3 * sizeof(float);
}

template <typename T>
static hipError_t by_direction(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  return backward ? by_width<T, 2, true>(a, st) : by_width<T, sizeof(T) == 4 ? 2 : 4, false>(a, st);
}

hipError_t launch_scan(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  if (a.dtype == FFN_BF16) return by_direction<__bf16>(a, backward, st);
  if (a.dtype == FFN_F16) return by_direction<_Float16>(a, backward, st);
  return by_direction<float>(a, backward, st);
}

}  // namespace ffn
