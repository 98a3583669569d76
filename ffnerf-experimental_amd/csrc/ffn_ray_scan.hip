// ffn_ray_scan.hip -- the gated recurrence h_t = (1 - z_t) h_{t-1} + z_t x_t, z = sigmoid(gate), along rays.
//
// Per channel and in float.  A thread takes V neighbouring channels and walks rows in order; nothing it loads depends on
// the state, so the rows of one step are in flight while those of the step before are combined.  What a thread walks:
//   * by rays: one whole ray.  One launch, every value read once.
//   * by parts: a part of the packed rows of a fixed length, whatever rays it holds, so that few long rays fill the GPU
//     too.  A part that begins inside a ray needs the state there: k_scan_ends composes, per part, the steps of the ray
//     that leaves it (h -> A h + B), k_scan_groups those of neighbouring parts, in a fixed order.  That reads gate and x a
//     second time, but only of rays that cross a part's end.
// The backward pass walks the other way with D_t = dh_t + (1 - z_{t+1}) D_{t+1}.
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int SC_NT = 256;
constexpr int SC_MARK = 8;  // a state is kept every so many rows of a walk for the backward pass

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

// V neighbouring channels as they lie in memory: kept as words until they are used (as vectors of 16-bit elements the
// compiler spreads them over a register each)
template <int BYTES> struct Words;
template <> struct Words<2> { typedef uint16_t type; };
template <> struct Words<4> { typedef uint32_t type; };
template <> struct Words<8> { typedef uint2 type; };
template <typename T, int V> struct Chan {
  typedef typename Words<V * (int)sizeof(T)>::type vec;
};
template <typename T, int V> __device__ __forceinline__ float get(const typename Chan<T, V>::vec& x, int i) {
  uint32_t w;
  if constexpr (V * sizeof(T) == 8) w = sizeof(T) == 4 ? (i ? x.y : x.x) : (i >> 1 ? x.y : x.x);
  else w = x;
  if constexpr (sizeof(T) == 4) return __uint_as_float(w);
  else if constexpr (__is_same(T, __bf16)) return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w >> 16 : w & 0xFFFFu));
}
template <typename T, int V> __device__ __forceinline__ typename Chan<T, V>::vec pack(const float (&f)[V]) {
  typedef T tvec __attribute__((ext_vector_type(V)));
  if constexpr (V == 1) {
    const T t = (T)f[0];
    return __builtin_bit_cast(typename Chan<T, V>::vec, t);
  } else {
    tvec t;
#pragma unroll
    for (int v = 0; v < V; ++v) t[v] = (T)f[v];
    return __builtin_bit_cast(typename Chan<T, V>::vec, t);
  }
}

// z = sigmoid(g) and 1 - z, each to its own size: with e = exp(-|g|) they are 1 / (1 + e) and e / (1 + e), whichever is
// which.  1 - z by subtraction would be off by 5e-4 of itself at g = 10, and 0 from 17 on.
__device__ __forceinline__ void gates(float g, float& z, float& keep) {
  const float e = __builtin_amdgcn_exp2f(fabsf(g) * -1.4426950408889634f);
  const float most = __builtin_amdgcn_rcpf(1.f + e), least = e * most;
  z = g < 0.f ? least : most;
  keep = g < 0.f ? most : least;
}

// N rows from p on, `step` bytes apart.  Addresses are opaque to the compiler: else all N are formed, and held, before the
// first load.
template <typename T, int V, int N>
__device__ __forceinline__ void load_rows(typename Chan<T, V>::vec (&to)[N], const T* p, int step) {
  const char* at = reinterpret_cast<const char*>(p);
#pragma unroll
  for (int u = 0; u < N; ++u) {
    to[u] = *reinterpret_cast<const typename Chan<T, V>::vec*>(at);
    at += step;
    asm volatile("" : "+v"(at));
  }
}
// the same where `left` of them are there: the last one again for the others, so that no lane branches
template <typename T, int V, int N>
__device__ __forceinline__ void load_rows(typename Chan<T, V>::vec (&to)[N], const T* p, int step, int left) {
  const int last = (min(left, N) - 1) * step;
#pragma unroll
  for (int u = 0; u < N; ++u) {
    // between 0 and the last row, whichever way the rows go
    int off = max(min(u * step, last), min(max(u * step, last), 0));
    if (u) asm volatile("" : "+v"(off));
    to[u] = *reinterpret_cast<const typename Chan<T, V>::vec*>(reinterpret_cast<const char*>(p) + off);
  }
}

// the columns of one thread
template <typename T, int V>
struct Cols {
  typedef typename Chan<T, V>::vec vec;
  int ch;
  Walk w;
  const T *gate, *x;
  int64_t gs, xs;  // from a place to the next, in elements
  int gb, xb;      // in bytes
  __device__ __forceinline__ Cols(const ffn_ray_scan& a, int c)
      : ch(c), w(a), gate((const T*)a.gate + c), x((const T*)a.x + c), gs(w.step * a.gate_row), xs(w.step * a.x_row),
        gb((int)(gs * (int)sizeof(T))), xb((int)(xs * (int)sizeof(T))) {}
};

// h over `len` > 0 places from `from` on; marks are kept at multiples of SC_MARK of the walk, and at its start if `mark0`
template <typename T, int V>
__device__ __forceinline__ void walk_fwd(const ffn_ray_scan& a, const Cols<T, V>& c, int64_t from, int len, bool mark0,
                                         float (&h)[V]) {
  typedef typename Cols<T, V>::vec vec;
  constexpr int U = SC_MARK;
  const int64_t row = c.w.row(from);
  const T* gp = c.gate + row * a.gate_row;
  const T* xp = c.x + row * a.x_row;
  T* hp = (T*)a.h + row * a.channels + c.ch;
  const int64_t hs = (int64_t)c.w.step * a.channels;
  vec g[U], x[U];
  load_rows<T, V, U>(g, gp, c.gb, len);
  load_rows<T, V, U>(x, xp, c.xb, len);
  for (int k = 0; k < len; k += U) {
    vec gc[U], xc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) gc[u] = g[u], xc[u] = x[u];
    if (k + U < len) {
      gp += U * c.gs;
      xp += U * c.xs;
      load_rows<T, V, U>(g, gp, c.gb, len - k - U);
      load_rows<T, V, U>(x, xp, c.xb, len - k - U);
    }
    if (a.marks && (k || mark0)) {
      float* m = a.marks + (from + k) / SC_MARK * a.channels + c.ch;
#pragma unroll
      for (int v = 0; v < V; ++v) m[v] = h[v];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k + u < len) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float z, keep;
          gates(get<T, V>(gc[u], v), z, keep);
          h[v] = __builtin_fmaf(keep, h[v], z * get<T, V>(xc[u], v));
        }
        *reinterpret_cast<vec*>(hp) = pack<T, V>(h);
      }
      hp += hs;
    }
  }
}

// Gradients over `len` > 0 places from `from` on, last to first, in pieces of SC_MARK: a piece's states come again from
// the mark before it, so that the backward pass neither reads h nor takes its rounding.  Of them it keeps z, 1 - z
// and q = (x - h_{t-1}) z (1 - z):  dx = z D, dgate = q D, and D goes on as (1 - z) D.  start: the state before a walk
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
  load_rows<T, V, L>(g, gp, c.gb, len - k);
  load_rows<T, V, L>(x, xp, c.xb, len - k);
  load_rows<T, V, L>(dh, dp, (int)(ds * sizeof(T)), len - k);
  for (; k >= 0; k -= L) {
    const float* m = k || mark0 ? a.marks + (from + k) / L * a.channels + c.ch : start;
    float h[V], z[L][V], keep[L][V], q[L][V];
    vec dc[L];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = m ? m[v] : 0.f;
#pragma unroll
    for (int u = 0; u < L; ++u) {
      dc[u] = dh[u];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float xx = get<T, V>(x[u], v);
        float zz, kk;
        gates(get<T, V>(g[u], v), zz, kk);
        z[u][v] = zz;
        keep[u][v] = kk;
        q[u][v] = (xx - h[v]) * (zz * kk);
        h[v] = __builtin_fmaf(kk, h[v], zz * xx);
        // opaque: formed here, before the next piece's rows are asked for (else both pieces' rows are held)
        asm volatile("" : "+v"(z[u][v]), "+v"(keep[u][v]), "+v"(q[u][v]));
      }
    }
    const int left = len - k;
    T *wg = og + (L - 1) * os, *wx = ox + (L - 1) * os;
    if (k > 0) {
      gp -= L * c.gs, xp -= L * c.xs, dp -= L * ds;
      og -= L * os, ox -= L * os;
      load_rows<T, V, L>(g, gp, c.gb);
      load_rows<T, V, L>(x, xp, c.xb);
      load_rows<T, V, L>(dh, dp, (int)(ds * sizeof(T)));
    }
#pragma unroll
    for (int u = L - 1; u >= 0; --u) {
      if (u < left) {
        float vg[V], vx[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float D = get<T, V>(dc[u], v) + d[v];
          vx[v] = z[u][v] * D;
          vg[v] = q[u][v] * D;
          d[v] = keep[u][v] * D;
        }
        *reinterpret_cast<vec*>(wx) = pack<T, V>(vx);
        *reinterpret_cast<vec*>(wg) = pack<T, V>(vg);
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

// By rays: a thread a ray and V channels; the blocks past ray_blocks clear the rows of no ray.  Bound by memory, with the
// vector ALU 89 % busy beside it: 4.7 million rows of 2^18 rays, 64 channels, bf16, repeated: forward 387 us (4.7 TB/s),
// backward 690 (4.4 TB/s; the marks are read too); by turns they take 1075.
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(SC_NT) void k_scan_rays(ffn_ray_scan a, int64_t ray_blocks) {
  const int64_t block = block_number();
  if (block >= ray_blocks) {
    const int64_t i = (block - ray_blocks) * SC_NT + threadIdx.x;
    if (BACK) clear_outside<T>(a, i, (T*)a.dgate, (T*)a.dx);
    else clear_outside<T>(a, i, (T*)a.h, nullptr);
    return;
  }
  const int lanes = a.channels / V;
  const int64_t id = block * SC_NT + threadIdx.x;
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

constexpr int GROUP = 64, GR_C = 16;
// k_scan_ends' and k_scan_groups' results: [parts][channels], [runs][channels]
struct Ends {
  float *A, *B, *run_A, *run_B;
};

// h -> A h + B over some parts.  FORGET in the place of A: the walk of the ray that leaves them began in them, or none
// leaves, and B is the state whatever entered; a factor of 0 would let another ray's infinity or NaN through.  Factors of
// a ray's own steps are +0 or more, so that a product that underflows still multiplies, and the ray's own NaN stays in it.
constexpr float FORGET = -0.f;
__device__ __forceinline__ bool forgets(float A) { return __float_as_uint(A) == 0x80000000u; }
__device__ __forceinline__ float over(float A, float B, float h) { return forgets(A) ? B : __builtin_fmaf(A, h, B); }

// The ray that leaves each part in the direction of the walk: the part's steps of it, FORGET where the ray begins (BACK:
// ends) in the part or none leaves.
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(SC_NT) void k_scan_ends(ffn_ray_scan a, int size, int64_t parts, float* __restrict__ A_of,
                                                     float* __restrict__ B_of) {
  constexpr int U = 8;
  typedef typename Chan<T, V>::vec vec;
  const int lanes = a.channels / V;
  const int64_t id = block_number() * SC_NT + threadIdx.x;
  const int64_t part = id / lanes;
  if (part >= parts) return;
  const Cols<T, V> c(a, (int)(id % lanes) * V);
  const int64_t p0 = part * size, p1 = min(p0 + size, (int64_t)a.rays.n);
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
  Span64 s;
  const int64_t ray = ray_at(a, c.w, BACK ? p0 : p1 - 1, s);
  bool whole = true;
  if (ray >= 0 && (BACK ? s.from < p0 : s.to > p1)) {
    const int64_t from = max(s.from, p0), to = min(s.to, p1);
    whole = BACK ? to == s.to : from == s.from;
    const int len = (int)(to - from);
    if (whole) load_state<V>(B, BACK ? a.dlast : a.h0, ray, a.channels, c.ch);
    const int64_t row = c.w.row(BACK ? to - 1 : from), dir = BACK ? -1 : 1;
    const T* gp = c.gate + row * a.gate_row;
    const T* xp = BACK ? (const T*)a.dh + row * a.dh_row + c.ch : c.x + row * a.x_row;
    const int64_t gs = dir * c.gs, xs = BACK ? -c.w.step * a.dh_row : c.xs;
    vec g[U], x[U];
    load_rows<T, V, U>(g, gp, (int)(gs * sizeof(T)), len);
    load_rows<T, V, U>(x, xp, (int)(xs * sizeof(T)), len);
    for (int k = 0; k < len; k += U) {
      vec gc[U], xc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) gc[u] = g[u], xc[u] = x[u];
      if (k + U < len) {
        gp += U * gs;
        xp += U * xs;
        load_rows<T, V, U>(g, gp, (int)(gs * sizeof(T)), len - k - U);
        load_rows<T, V, U>(x, xp, (int)(xs * sizeof(T)), len - k - U);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u < len) {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            float z, keep;
            gates(get<T, V>(gc[u], v), z, keep);
            A[v] *= keep;
            // BACK: the D that leaves a step is (1 - z) (dh + D)
            B[v] = BACK ? keep * (B[v] + get<T, V>(xc[u], v)) : __builtin_fmaf(keep, B[v], z * get<T, V>(xc[u], v));
          }
        }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A_of[part * a.channels + c.ch + v] = whole ? FORGET : A[v];
    B_of[part * a.channels + c.ch + v] = B[v];
  }
}

// Runs of GROUP parts, in the order of the walk: what the parts before each one in its run make of a state, in place, and
// what the whole run makes of it.  A block takes a run and 16 channels (a cache line of the parts' rows).
template <bool BACK>
__global__ __launch_bounds__(GR_C * GROUP) void k_scan_groups(int channels, int64_t parts, float* __restrict__ A_of,
                                                              float* __restrict__ B_of, float* __restrict__ run_A,
                                                              float* __restrict__ run_B) {
  __shared__ float sa[GROUP][GR_C], sb[GROUP][GR_C];
  const int c = threadIdx.x % GR_C, t = threadIdx.x / GR_C, ch = blockIdx.y * GR_C + c;
  const int64_t j = (int64_t)blockIdx.x * GROUP + t, at = (BACK ? parts - 1 - j : j) * channels + ch;
  const bool there = j < parts && ch < channels;
  float A = there ? A_of[at] : 1.f, B = there ? B_of[at] : 0.f;
  sa[t][c] = A;
  sb[t][c] = B;
  __syncthreads();
  for (int d = 1; d < GROUP; d *= 2) {
    float a = 1.f, b = 0.f;
    if (t >= d) a = sa[t - d][c], b = sb[t - d][c];
    __syncthreads();
    if (!forgets(A)) {
      B = __builtin_fmaf(A, b, B);
      A = forgets(a) ? FORGET : A * a;
    }
    sa[t][c] = A;
    sb[t][c] = B;
    __syncthreads();
  }
  if (!there) return;
  A_of[at] = t ? sa[t - 1][c] : 1.f;
  B_of[at] = t ? sb[t - 1][c] : 0.f;
  if (t == GROUP - 1 || j == parts - 1) {
    run_A[(int64_t)blockIdx.x * channels + ch] = A;
    run_B[(int64_t)blockIdx.x * channels + ch] = B;
  }
}

// What enters part j inside a ray whose walk began in part j0: the runs since then, then the parts of j's own run.
template <int V, bool BACK>
__device__ __forceinline__ void enter(float (&h)[V], const Ends& e, int64_t parts, int64_t j, int64_t j0, int channels,
                                      int ch) {
  const int64_t r0 = (BACK ? parts - 1 - j0 : j0) / GROUP, r1 = (BACK ? parts - 1 - j : j) / GROUP;
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.f;  // the run, or the parts of it, in which the walk began forget it
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r)
#pragma unroll
    for (int v = 0; v < V; ++v)
      h[v] = over(e.run_A[r * channels + ch + v], e.run_B[r * channels + ch + v], h[v]);
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = over(e.A[j * channels + ch + v], e.B[j * channels + ch + v], h[v]);
}

// By parts of `size` places (a multiple of SC_MARK).  The blocks past part_blocks give the rays without rows their last
// state.  Parts in falling order, since k_scan_ends has just read the last ones: 204 us for all three launches instead of
// 209 in rising order, with 710137 rows of three rays, 128 channels, fp16; 94 us of them k_scan_ends, 5 and 102, where one
// read of gate and x and one write would take 116.  Registers are held for four wavefronts a SIMD (backward of 200,000 rows of 37
// float channels: 41 us, with three 44).
template <typename T, int V, bool BACK>
__global__ __launch_bounds__(SC_NT, 4) void k_scan_parts(ffn_ray_scan a, int size, int64_t parts, int64_t part_blocks,
                                                      Ends e) {
  const int lanes = a.channels / V;
  const int64_t block = block_number();
  if (block >= part_blocks) {
    const int64_t id = (block - part_blocks) * SC_NT + threadIdx.x, ray = id / lanes;
    if (ray >= a.rays.num_rays) return;
    const Span64 s = places_of(a, (uint32_t)ray);
    if (s.to > s.from) return;
    const int ch = (int)(id % lanes) * V;
    float h[V];
    load_state<V>(h, BACK ? a.dlast : a.h0, ray, a.channels, ch);
    store_state<V>(BACK ? a.dh0 : a.last, ray, a.channels, ch, h);
    return;
  }
  const int64_t id = (part_blocks - 1 - block) * SC_NT + threadIdx.x;
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
      const typename Cols<T, V>::vec zero{};
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
      if (to < s.to) enter<V, true>(h, e, parts, part, (s.to - 1) / size, a.channels, c.ch);
      else load_state<V>(h, a.dlast, ray, a.channels, c.ch);
      walk_bwd<T, V>(a, c, from, len, inside, a.h0 ? a.h0 + ray * a.channels + c.ch : nullptr, h);
      if (!inside) store_state<V>(a.dh0, ray, a.channels, c.ch, h);
      p = from - 1;
    } else {
      if (inside) enter<V, false>(h, e, parts, part, s.from / size, a.channels, c.ch);
      else load_state<V>(h, a.h0, ray, a.channels, c.ch);
      walk_fwd<T, V>(a, c, from, len, inside, h);
      if (to == s.to) store_state<V>(a.last, ray, a.channels, c.ch, h);
      p = to;
    }
  }
}

static bool aligned(const void* p, int64_t row, int bytes, int size) {
  return ((uintptr_t)p | (uintptr_t)(row * size)) % bytes == 0;
}

// Which walk.  By rays, the longest one is the least that a call takes (about 0.1 us a row); that is hidden where there
// are rays for several rounds of threads, and short where there are few rows.  By parts it takes two more launches and a
// second read of what crosses parts.  196,000 samples of 5003 rays, 37 channels: 97 us by rays, 45 by parts; 4.6 million
// samples of 2^18 rays, 64 channels: 418 and 590; 1000 samples of 64 rays: 8 and 33.
constexpr int64_t SC_THREADS = 262144;  // threads at work at once
static int64_t words_a_row(const ffn_ray_scan& a) {  // of 4 bytes: threads a ray or part
  return a.dtype == FFN_F32 ? a.channels : (a.channels + 1) / 2;
}
static bool by_rays(const ffn_ray_scan& a) {
  if (a.rays.n <= 4096) return (int64_t)a.rays.n <= 64 * (int64_t)a.rays.num_rays;
  return a.rays.num_rays * words_a_row(a) >= 4 * SC_THREADS && a.rays.n <= 256 * (int64_t)a.rays.num_rays;
}
static int part_size(const ffn_ray_scan& a) {
  int64_t s = (int64_t)a.rays.n * words_a_row(a) / SC_THREADS;
  s = (s + SC_MARK - 1) / SC_MARK * SC_MARK;
  return (int)(s < 32 ? 32 : s > 4096 ? 4096 : s);
}

template <typename T, int V, bool BACK>
static hipError_t run(const ffn_ray_scan& a, hipStream_t st) {
  const int64_t lanes = a.channels / V;
  if (by_rays(a)) {
    const int64_t rb = (a.rays.num_rays * lanes + SC_NT - 1) / SC_NT, cb = ((int64_t)a.rays.n + SC_NT - 1) / SC_NT;
    if (rb + cb) k_scan_rays<T, V, BACK><<<grid_of(rb + cb), SC_NT, 0, st>>>(a, rb);
    return hipGetLastError();
  }
  const int size = part_size(a);
  const int64_t parts = ((int64_t)a.rays.n + size - 1) / size, runs = (parts + GROUP - 1) / GROUP;
  float* w = (float*)a.workspace;
  const Ends e{w, w + parts * a.channels, w + 2 * parts * a.channels, w + (2 * parts + runs) * a.channels};
  const int64_t pb = (parts * lanes + SC_NT - 1) / SC_NT, rb = (a.rays.num_rays * lanes + SC_NT - 1) / SC_NT;
  if (parts) {
    k_scan_ends<T, V, BACK><<<grid_of(pb), SC_NT, 0, st>>>(a, size, parts, e.A, e.B);
    k_scan_groups<BACK><<<dim3((unsigned)runs, (a.channels + GR_C - 1) / GR_C), GR_C * GROUP, 0, st>>>(
        a.channels, parts, e.A, e.B, e.run_A, e.run_B);
  }
  if (pb + rb) k_scan_parts<T, V, BACK><<<grid_of(pb + rb), SC_NT, 0, st>>>(a, size, parts, pb, e);
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
  const uint64_t parts = ((uint64_t)a.rays.n + size - 1) / size, runs = (parts + GROUP - 1) / GROUP;
  return 2 * (parts + runs) * a.channels * sizeof(float);
}

template <typename T>
static hipError_t by_direction(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  constexpr int V = 4 / (int)sizeof(T);  // 4 bytes a lane: with 8 the forward of 2^18 rays takes 524 us instead of 418
  return backward ? by_width<T, V, true>(a, st) : by_width<T, V, false>(a, st);
}

hipError_t launch_scan(const ffn_ray_scan& a, bool backward, hipStream_t st) {
  if (a.dtype == FFN_BF16) return by_direction<__bf16>(a, backward, st);
  if (a.dtype == FFN_F16) return by_direction<_Float16>(a, backward, st);
  return by_direction<float>(a, backward, st);
}

}  // namespace ffn
