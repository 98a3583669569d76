// ffn_ray_attn.hip -- attention among the samples of a ray, forward and backward.
//
// A wavefront keeps 16 rows (queries; keys in the dk/dv kernel) and walks the rows that they may see.  Products are
// formed transposed, with the kept rows along the lanes: lane (g, c) then holds four values of kept row c, the softmax's
// maxima and sums need two exchanges over the four lane groups, and the weights are already the operand of the second
// product (product_frag).  Whatever mask applies, the rows that a row sees are one contiguous range (a ray's rows, cut
// at the causal edge or the prefix), so a mask is one unsigned comparison and whole tiles are skipped or left unmasked
// by the wavefront's ranges.
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int AT_NT = 256, AT_TILE = 64;  // four wavefronts of 16 kept rows; rows of a streamed tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Range {
  int lo, hi;
};

// the keys that query i sees
__device__ __forceinline__ Range keys_of(const ffn_ray_attn& a, int64_t i) {
  if (i >= a.q_rays.n) return {0, 0};
  const uint32_t r = a.q_rays.ray_ids[i];
  if (r >= a.q_rays.num_rays) return {0, 0};
  const int64_t qo = a.q_rays.offsets[r], nq = a.q_rays.counts[r];
  if (i < qo || i - qo >= nq) return {0, 0};
  const int64_t ko = a.k_rays.offsets[r], nk = a.k_rays.counts[r], n = a.k_rays.n;
  int64_t seen = nk;
  if (a.causal) {
    seen = i - qo + nk - nq + 1;
    if (a.prefix) seen = max(seen, (int64_t)a.prefix[r]);
    seen = min(max(seen, (int64_t)0), nk);
  }
  return {(int)min(ko, n), (int)min(ko + seen, n)};
}

// the queries that see key j: keys_of from the other side
__device__ __forceinline__ Range queries_of(const ffn_ray_attn& a, int64_t j) {
  if (j >= a.k_rays.n) return {0, 0};
  const uint32_t r = a.k_rays.ray_ids[j];
  if (r >= a.k_rays.num_rays) return {0, 0};
  const int64_t ko = a.k_rays.offsets[r], nk = a.k_rays.counts[r];
  if (j < ko || j - ko >= nk) return {0, 0};
  const int64_t qo = a.q_rays.offsets[r], nq = a.q_rays.counts[r], n = a.q_rays.n;
  int64_t from = 0;
  if (a.causal && !(a.prefix && j - ko < (int64_t)a.prefix[r])) from = min(max(j - ko - nk + nq, (int64_t)0), nq);
  return {(int)min(qo + from, n), (int)min(qo + nq, n)};
}

__device__ __forceinline__ float swap_add(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float swap_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// What the wavefront's 16 rows see: lane c holds row c's range.  [lo, hi) covers all of them; a tile inside
// [all_lo, all_hi) is seen by every row.
struct Span {
  int lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ Span span_of(const Range& r) {
  const bool none = r.hi <= r.lo;
  Span s{none ? INT_MAX : r.lo, none ? 0 : r.hi, none ? INT_MAX : r.lo, none ? 0 : r.hi};
#pragma unroll
  for (int m = 1; m < 16; m *= 2) {
    s.lo = min(s.lo, __shfl_xor(s.lo, m));
    s.hi = max(s.hi, __shfl_xor(s.hi, m));
    s.all_lo = max(s.all_lo, __shfl_xor(s.all_lo, m));
    s.all_hi = min(s.all_hi, __shfl_xor(s.all_hi, m));
  }
  s.lo = __builtin_amdgcn_readfirstlane(s.lo);
  s.hi = __builtin_amdgcn_readfirstlane(s.hi);
  s.all_lo = __builtin_amdgcn_readfirstlane(s.all_lo);
  s.all_hi = __builtin_amdgcn_readfirstlane(s.all_hi);
  return s;
}

// AT_TILE rows of one head on their way to LDS (rows outside [row0, end) and columns past dim as 0)
template <typename T, int DP, int NT = AT_NT>
struct Staged {
  static constexpr int EL = 16 / (int)sizeof(T), CPR = DP / EL, N = AT_TILE * CPR / NT;
  uint4 v[N];
  __device__ __forceinline__ void load(const T* __restrict__ base, int64_t stride, int row0, int end, int dim, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT, row = row0 + c / CPR, col = (c % CPR) * EL;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < end && col < dim) v[i] = *reinterpret_cast<const uint4*>(base + row * stride + col);
    }
  }
  // returns whether any of this thread's values is infinite or NaN
  __device__ __forceinline__ bool store(T* tile, int tid) const {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = tid + i * NT;
      *reinterpret_cast<uint4*>(tile + (c / CPR) * lds_row<T, DP> + (c % CPR) * EL) = v[i];
      bad |= any_nonfinite<T>(v[i]);
    }
    return bad;
  }
};

// one row of one head as KS fragments (lane group g holds columns 32 ks + 8 g ..)
template <typename T, int KS>
__device__ __forceinline__ void load_frags(typename Mat<T>::frag (&f)[KS], const T* __restrict__ row, bool there, int dim,
                                           int g) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int col = ks * 32 + g * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[ks][j] = (T)0.f;
    if (there && col < dim) f[ks] = *reinterpret_cast<const typename Mat<T>::frag*>(row + col);
  }
}

// tanh to single precision: the odd series where 1 - 2 / (1 + e^2x) would cancel
__device__ __forceinline__ float tanh_f(float x) {
  const float x2 = x * x;
  float p = __builtin_fmaf(x2, 62.f / 2835.f, -17.f / 315.f);
  p = __builtin_fmaf(x2, p, 2.f / 15.f);
  p = __builtin_fmaf(x2, p, -1.f / 3.f);
  const float small = __builtin_fmaf(x * x2, p, x);
  const float e = __builtin_amdgcn_exp2f(x * (2.f * LOG2E));
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e);
  return fabsf(x) < 0.25f ? small : big;
}

// Products of 16 x 64 rows -> logits in units of log 2; th: tanh of the capped scores (only with a cap).  x: the streamed
// rows' depths in LDS.  The unit lets every exponential be one v_exp_f32.
struct Logits {
  float scale2, cap, inv_cap, cap2, slope2;
  bool bias;
  __device__ __forceinline__ Logits(const ffn_ray_attn& a, int head)
      : scale2(a.scale * LOG2E), cap(a.cap), inv_cap(a.cap > 0.f ? a.scale / a.cap : 0.f), cap2(a.cap * LOG2E),
        slope2(a.slopes ? a.slopes[head] * LOG2E : 0.f), bias(a.slopes != nullptr) {}
  __device__ __forceinline__ void operator()(f32x4 (&s)[4], f32x4 (&th)[4], float t, const float* x, int g) const {
    if (cap > 0.f) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          th[b][r] = tanh_f(s[b][r] * inv_cap);
          s[b][r] = cap2 * th[b][r];
        }
    } else {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] *= scale2;
    }
    if (bias) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4 tx = *reinterpret_cast<const f32x4*>(x + 16 * b + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] = __builtin_fmaf(-slope2, fabsf(t - tx[r]), s[b][r]);
      }
    }
  }
};

__device__ __forceinline__ bool sees(int row, const Range& r) {
  return (unsigned)(row - r.lo) < (unsigned)(r.hi - r.lo);
}

// acc += tile^T w over the tile's 64 rows, where a row of the tile holds an infinity or a NaN: pair by pair, so that a
// weight of 0 that only a mask made does not meet it
template <typename T, int DP>
__device__ __noinline__ void add_careful(f32x4* acc, const f32x4* w, const T* tile, int row0, Range seen, int lane) {
  const int g = lane >> 4, c = lane & 15;
  for (int row = 0; row < AT_TILE; ++row) {
    const float mine = w[row >> 4][row & 3];
    const float ww = __shfl(mine, 16 * ((row >> 2) & 3) + c);
    if (!sees(row0 + row, seen)) continue;
    for (int db = 0; db < DP / 16; ++db)
      for (int r = 0; r < 4; ++r)
        acc[db][r] = __builtin_fmaf(ww, (float)tile[row * lds_row<T, DP> + 16 * db + 4 * g + r], acc[db][r]);
  }
}

// acc += tile^T w: the tile's 64 rows are the K of the product
template <typename T, int DP>
__device__ __forceinline__ void add_weighted(f32x4 (&acc)[DP / 16], const f32x4 (&w)[4], const T* tile, bool careful,
                                             int row0, const Range& seen, int lane) {
  if (careful) {
    f32x4 a2[DP / 16], w2[4];
    for (int i = 0; i < DP / 16; ++i) a2[i] = acc[i];
    for (int i = 0; i < 4; ++i) w2[i] = w[i];
    add_careful<T, DP>(a2, w2, tile, row0, seen, lane);
    for (int i = 0; i < DP / 16; ++i) acc[i] = a2[i];
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const typename Mat<T>::frag f = product_frag<T>(w[2 * h], w[2 * h + 1]);
#pragma unroll
    for (int db = 0; db < DP / 16; ++db)
      acc[db] = Mat<T>::mma(col_frag<T, DP>(tile, 32 * h, 16 * db, lane), f, acc[db]);
  }
}

// s = tile rows . kept rows
template <typename T, int DP>
__device__ __forceinline__ void products(f32x4 (&s)[4], const T* tile, const typename Mat<T>::frag (&kept)[DP / 32],
                                         int lane) {
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < DP / 32; ++ks)
      s[b] = Mat<T>::mma(row_frag<T, DP>(tile, 16 * b + (lane & 15), ks, lane), kept[ks], s[b]);
  }
}

template <typename T, int DP>
__device__ __forceinline__ void store_row(T* __restrict__ row, const f32x4 (&acc)[DP / 16], float by, int dim, int g) {
#pragma unroll
  for (int db = 0; db < DP / 16; ++db) {
    const int col = 16 * db + 4 * g;
    if (col < dim) {
      typename Mat<T>::quad v;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = (T)(acc[db][r] * by);
      *reinterpret_cast<typename Mat<T>::quad*>(row + col) = v;
    }
  }
}

// Weights carry a factor of 2^14, which the sums' division (forward) or the final factor takes out again: fp16's normal
// numbers end at 2^-14, and the exponential's at 2^-126 (it gives 0 below).
constexpr float W_SHIFT = 14.f, W_UNSHIFT = 1.f / 16384.f;

// Running softmax of one row, its sum still apart by lane group
struct Softmax {
  float m = -INFINITY, l = 0.f;
  // weights in place of the logits
  template <int NACC>
  __device__ __forceinline__ void step(f32x4 (&s)[4], f32x4 (&acc)[NACC]) {
    float mx = s[0][0];
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[b][r]);
    mx = fmaxf(m, swap_max(mx));
    const float base = mx == -INFINITY ? 0.f : mx;
    if (__any(mx != m)) {
      const float f = __builtin_amdgcn_exp2f(m - base);
      l *= f;
#pragma unroll
      for (int i = 0; i < NACC; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= f;
      m = mx;
    }
    const float from = base - W_SHIFT;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - from);
        l += s[b][r];
      }
  }
  // factor of the sums, and the logarithm of the sum of exponentials
  __device__ __forceinline__ float finish(float& lse) {
    l = swap_add(l);
    lse = l == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(l) - W_SHIFT) * LN2;
    return l == 0.f ? 0.f : 1.f / l;
  }
};

// Blocks in launch order go round the eight dies; this gives each die a contiguous part of the work, whose tiles share
// keys in its L2.
__device__ __forceinline__ int64_t die_order(int64_t total) {
  const int64_t per = (total + 7) / 8;
  return (blockIdx.x & 7) * per + (blockIdx.x >> 3);
}

template <typename T, int DP>
__global__ __launch_bounds__(AT_NT) void k_attn_fwd(ffn_ray_attn a, int64_t total) {
  constexpr int KS = DP / 32, NB = DP / 16;
  __shared__ T ks[AT_TILE * lds_row<T, DP>], vs[AT_TILE * lds_row<T, DP>];
  __shared__ float ts[AT_TILE];
  __shared__ int s_lo[4], s_hi[4], s_bad[4];
  const int64_t work = die_order(total);
  if (work >= total) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int head = (int)(work % a.heads), kh = head / (a.heads / a.kv_heads);
  const int64_t i = work / a.heads * AT_TILE + wave * 16 + c;
  const bool there = i < a.q_rays.n;
  const Range seen = keys_of(a, i);
  const Span w = span_of(seen);
  if (lane == 0) s_lo[wave] = w.lo, s_hi[wave] = w.hi;
  typename Mat<T>::frag qf[KS];
  load_frags<T, KS>(qf, (const T*)a.q + i * a.q_row + head * a.q_head, there, a.dim, g);
  const Logits logits(a, head);
  const float t = logits.bias && there ? a.t_q[i * a.t_q_row] : 0.f;
  __syncthreads();
  const int lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
  const T* kb = (const T*)a.k + kh * a.k_head;
  const T* vb = (const T*)a.v + kh * a.v_head;
  f32x4 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  Softmax sm;
  Staged<T, DP> kst, vst;
  float tst = 0.f;
  auto fetch = [&](int row0) {
    kst.load(kb, a.k_row, row0, hi, a.dim, tid);
    vst.load(vb, a.v_row, row0, hi, a.dim, tid);
    if (logits.bias && tid < AT_TILE && row0 + tid < hi) tst = a.t_k[(int64_t)(row0 + tid) * a.t_k_row];
  };
  if (lo < hi) fetch(lo);
  for (int row0 = lo; row0 < hi; row0 += AT_TILE) {
    kst.store(ks, tid);
    const bool bad = __any(vst.store(vs, tid));
    if (lane == 0) s_bad[wave] = bad;
    if (tid < AT_TILE) ts[tid] = tst;
    __syncthreads();
    if (hi - row0 > AT_TILE) fetch(row0 + AT_TILE);
    if (row0 < w.hi && row0 + AT_TILE > w.lo) {
      f32x4 s[4], th[4];
      products<T, DP>(s, ks, qf, lane);
      logits(s, th, t, ts, g);
      if (row0 < w.all_lo || row0 + AT_TILE > w.all_hi) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!sees(row0 + 16 * b + 4 * g + r, seen)) s[b][r] = -INFINITY;
      }
      sm.step(s, acc);
      add_weighted<T, DP>(acc, s, vs, s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3], row0, seen, lane);
    }
    __syncthreads();
  }
  float lse;
  const float by = sm.finish(lse);
  if (there) {
    const int64_t at = i * a.heads + head;
    store_row<T, DP>((T*)a.o + at * a.dim, acc, by, a.dim, g);
    if (g == 0) a.lse[at] = lse;
  }
}

// Factor of one row's gradient weights.  fp16's exponent is too narrow for them (a probability times an upstream
// gradient of any size): each kept row's are scaled by a power of two that puts the largest so far into [2^13, 2^15],
// and its sums are rescaled when a larger one comes.  The other types take them as they are.
template <typename T>
struct GradScale {
  float f = 0.f;
  template <int NACC>
  __device__ __forceinline__ void apply(f32x4 (&s)[4], f32x4 (&acc)[NACC]) {
    if constexpr (__is_same(T, _Float16)) {
      float mx = 0.f;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, fabsf(s[b][r]));
      mx = swap_max(mx);
      const bool grow = mx > 0.f && (f == 0.f || mx * f > 32768.f);
      if (__any(grow)) {
        const int e = min(max(140 - (int)(__float_as_uint(mx) >> 23), -100), 100);  // 13 - exponent
        const float to = __uint_as_float((unsigned)(127 + e) << 23);
        const float by = grow ? (f == 0.f ? 0.f : to / f) : 1.f;
        if (grow) f = to;
#pragma unroll
        for (int i = 0; i < NACC; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][r] *= by;
      }
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] *= f;
    }
  }
  __device__ __forceinline__ float undo() const {
    if constexpr (__is_same(T, _Float16)) return f == 0.f ? 0.f : 1.f / f;
    return 1.f;
  }
};

// dq; also leaves D = sum_d do o of its rows in the workspace for k_attn_dkv
template <typename T, int DP>
__global__ __launch_bounds__(AT_NT) void k_attn_dq(ffn_ray_attn a, int64_t total) {
  constexpr int KS = DP / 32, NB = DP / 16;
  __shared__ T ks[AT_TILE * lds_row<T, DP>], vs[AT_TILE * lds_row<T, DP>];
  __shared__ float ts[AT_TILE];
  __shared__ int s_lo[4], s_hi[4], s_bad[4];
  const int64_t work = die_order(total);
  if (work >= total) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int head = (int)(work % a.heads), kh = head / (a.heads / a.kv_heads);
  const int64_t i = work / a.heads * AT_TILE + wave * 16 + c, at = i * a.heads + head;
  const bool there = i < a.q_rays.n;
  const Range seen = keys_of(a, i);
  const Span w = span_of(seen);
  if (lane == 0) s_lo[wave] = w.lo, s_hi[wave] = w.hi;
  typename Mat<T>::frag qf[KS], df[KS];
  load_frags<T, KS>(qf, (const T*)a.q + i * a.q_row + head * a.q_head, there, a.dim, g);
  load_frags<T, KS>(df, (const T*)a.dout + i * a.do_row + head * a.do_head, there, a.dim, g);
  float delta = 0.f;
  {
    typename Mat<T>::frag of[KS];
    load_frags<T, KS>(of, (const T*)a.o + at * a.dim, there, a.dim, g);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)of[k][j], (float)df[k][j], delta);
    delta = swap_add(delta);
  }
  const Logits logits(a, head);
  const float t = logits.bias && there ? a.t_q[i * a.t_q_row] : 0.f;
  float lse2 = there ? a.lse[at] * LOG2E : 0.f;
  if (lse2 == -INFINITY) lse2 = 0.f;
  const float from = lse2 - W_SHIFT;
  if (there && g == 0) ((float*)a.workspace)[at] = delta;
  __syncthreads();
  const int lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
  const T* kb = (const T*)a.k + kh * a.k_head;
  const T* vb = (const T*)a.v + kh * a.v_head;
  f32x4 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  GradScale<T> gs;
  Staged<T, DP> kst, vst;
  float tst = 0.f;
  auto fetch = [&](int row0) {
    kst.load(kb, a.k_row, row0, hi, a.dim, tid);
    vst.load(vb, a.v_row, row0, hi, a.dim, tid);
    if (logits.bias && tid < AT_TILE && row0 + tid < hi) tst = a.t_k[(int64_t)(row0 + tid) * a.t_k_row];
  };
  if (lo < hi) fetch(lo);
  for (int row0 = lo; row0 < hi; row0 += AT_TILE) {
    const bool bad = __any(kst.store(ks, tid));
    vst.store(vs, tid);
    if (lane == 0) s_bad[wave] = bad;
    if (tid < AT_TILE) ts[tid] = tst;
    __syncthreads();
    if (hi - row0 > AT_TILE) fetch(row0 + AT_TILE);
    if (row0 < w.hi && row0 + AT_TILE > w.lo) {
      f32x4 s[4], dp[4], th[4];
      products<T, DP>(s, ks, qf, lane);
      products<T, DP>(dp, vs, df, lane);
      logits(s, th, t, ts, g);
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - from) * (dp[b][r] - delta);
      if (logits.cap > 0.f) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[b][r] *= 1.f - th[b][r] * th[b][r];
      }
      if (row0 < w.all_lo || row0 + AT_TILE > w.all_hi) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!sees(row0 + 16 * b + 4 * g + r, seen)) s[b][r] = 0.f;
      }
      gs.apply(s, acc);
      add_weighted<T, DP>(acc, s, ks, s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3], row0, seen, lane);
    }
    __syncthreads();
  }
  if (there) store_row<T, DP>((T*)a.dq + at * a.dim, acc, gs.undo() * (a.scale * W_UNSHIFT), a.dim, g);
}

// dk and dv of 64 keys of one key head: the queries of the heads that share it stream past
template <typename T, int DP>
__global__ __launch_bounds__(AT_NT) void k_attn_dkv(ffn_ray_attn a, int64_t total) {
  constexpr int KS = DP / 32, NB = DP / 16;
  __shared__ T qs[AT_TILE * lds_row<T, DP>], ds[AT_TILE * lds_row<T, DP>];
  __shared__ float ts[AT_TILE], ls[AT_TILE], es[AT_TILE];
  __shared__ int s_lo[4], s_hi[4], s_bad[8];
  const int64_t work = die_order(total);
  if (work >= total) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int kh = (int)(work % a.kv_heads), group = a.heads / a.kv_heads;
  const int64_t j = work / a.kv_heads * AT_TILE + wave * 16 + c;
  const bool there = j < a.k_rays.n;
  const Range seen = queries_of(a, j);
  const Span w = span_of(seen);
  if (lane == 0) s_lo[wave] = w.lo, s_hi[wave] = w.hi;
  typename Mat<T>::frag kf[KS], vf[KS];
  load_frags<T, KS>(kf, (const T*)a.k + j * a.k_row + kh * a.k_head, there, a.dim, g);
  load_frags<T, KS>(vf, (const T*)a.v + j * a.v_row + kh * a.v_head, there, a.dim, g);
  const bool bias = a.slopes != nullptr;
  const float t = bias && there ? a.t_k[j * a.t_k_row] : 0.f;
  __syncthreads();
  const int lo = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), hi = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
  f32x4 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dk[b] = dv[b] = f32x4{0.f, 0.f, 0.f, 0.f};
  GradScale<T> gs;
  Staged<T, DP> qst, dst;
  float tst = 0.f, lst = 0.f, est = 0.f;
  auto fetch = [&](int head, int row0) {
    qst.load((const T*)a.q + head * a.q_head, a.q_row, row0, hi, a.dim, tid);
    dst.load((const T*)a.dout + head * a.do_head, a.do_row, row0, hi, a.dim, tid);
    if (tid < AT_TILE && row0 + tid < hi) {
      const int64_t i = row0 + tid;
      if (bias) tst = a.t_q[i * a.t_q_row];
      lst = a.lse[i * a.heads + head] * LOG2E;
      est = ((const float*)a.workspace)[i * a.heads + head];
      if (lst == -INFINITY) lst = 0.f;
    }
  };
  const int first = kh * group, end = first + group;
  if (lo < hi) fetch(first, lo);
  for (int head = first; head < end && lo < hi; ++head) {
    const Logits logits(a, head);
    for (int row0 = lo; row0 < hi; row0 += AT_TILE) {
      const bool bad_q = __any(qst.store(qs, tid)), bad_d = __any(dst.store(ds, tid));
      if (lane == 0) s_bad[wave] = bad_q, s_bad[4 + wave] = bad_d;
      if (tid < AT_TILE) ts[tid] = tst, ls[tid] = lst, es[tid] = est;
      __syncthreads();
      if (hi - row0 > AT_TILE) fetch(head, row0 + AT_TILE);
      else if (head + 1 < end) fetch(head + 1, lo);
      if (row0 < w.hi && row0 + AT_TILE > w.lo) {
        f32x4 s[4], dp[4], th[4];
        products<T, DP>(s, qs, kf, lane);
        products<T, DP>(dp, ds, vf, lane);
        logits(s, th, t, ts, g);
        const bool masked = row0 < w.all_lo || row0 + AT_TILE > w.all_hi;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const f32x4 l = *reinterpret_cast<const f32x4*>(ls + 16 * b + 4 * g);
          const f32x4 e = *reinterpret_cast<const f32x4*>(es + 16 * b + 4 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[b][r] = __builtin_amdgcn_exp2f(s[b][r] - (l[r] - W_SHIFT));
            dp[b][r] = s[b][r] * (dp[b][r] - e[r]);
          }
        }
        if (logits.cap > 0.f) {
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) dp[b][r] *= 1.f - th[b][r] * th[b][r];
        }
        if (masked) {
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!sees(row0 + 16 * b + 4 * g + r, seen)) s[b][r] = dp[b][r] = 0.f;
        }
        add_weighted<T, DP>(dv, s, ds, s_bad[4] | s_bad[5] | s_bad[6] | s_bad[7], row0, seen, lane);
        gs.apply(dp, dk);
        add_weighted<T, DP>(dk, dp, qs, s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3], row0, seen, lane);
      }
      __syncthreads();
    }
  }
  if (there) {
    const int64_t at = (j * a.kv_heads + kh) * a.dim;
    store_row<T, DP>((T*)a.dk + at, dk, gs.undo() * (a.scale * W_UNSHIFT), a.dim, g);
    store_row<T, DP>((T*)a.dv + at, dv, W_UNSHIFT, a.dim, g);
  }
}

// One query at a time: a wavefront takes query i, the heads of one key head along its columns, and part `split` of the
// query's keys.  K comes straight into the operand's registers, V through the wavefront's own LDS rows (for the
// transposing read).  Nothing is shared, so nothing waits.
template <typename T, int DP>
__global__ __launch_bounds__(AT_NT) void k_attn_row(ffn_ray_attn a, int splits, int64_t total) {
  constexpr int KS = DP / 32, NB = DP / 16;
  __shared__ T vs_all[4][AT_TILE * lds_row<T, DP>];
  __shared__ float ts_all[4][AT_TILE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int64_t work = (int64_t)blockIdx.x * 4 + wave;
  if (work >= total) return;  // no barriers below
  T* vs = vs_all[wave];
  float* ts = ts_all[wave];
  const int group = a.heads / a.kv_heads;
  const int kh = (int)(work % a.kv_heads);
  const int split = (int)(work / a.kv_heads % splits);
  const int64_t i = work / a.kv_heads / splits;
  Range seen = keys_of(a, i);
  if (splits > 1) {  // whole tiles
    const int tiles = (seen.hi - seen.lo + AT_TILE - 1) / AT_TILE;
    const int from = (int)((int64_t)tiles * split / splits), to = (int)((int64_t)tiles * (split + 1) / splits);
    seen = {seen.lo + from * AT_TILE, min(seen.hi, seen.lo + to * AT_TILE)};
  }
  const T* kb = (const T*)a.k + kh * a.k_head;
  const T* vb = (const T*)a.v + kh * a.v_head;
  for (int h0 = 0; h0 < group; h0 += 16) {
    const bool there = h0 + c < group;
    const int head = kh * group + min(h0 + c, group - 1);
    typename Mat<T>::frag qf[KS];
    load_frags<T, KS>(qf, (const T*)a.q + i * a.q_row + head * a.q_head, there, a.dim, g);
    const Logits logits(a, head);
    const float t = logits.bias ? a.t_q[i * a.t_q_row] : 0.f;
    f32x4 acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = f32x4{0.f, 0.f, 0.f, 0.f};
    Softmax sm;
    Staged<T, DP, 64> vst;
    typename Mat<T>::frag kf[4][KS];
    float tst = 0.f;
    auto fetch = [&](int row0) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int row = row0 + 16 * b + c;
        load_frags<T, KS>(kf[b], kb + row * a.k_row, row < seen.hi, a.dim, g);
      }
      vst.load(vb, a.v_row, row0, seen.hi, a.dim, lane);
      if (logits.bias && row0 + lane < seen.hi) tst = a.t_k[(int64_t)(row0 + lane) * a.t_k_row];
    };
    if (seen.lo < seen.hi) fetch(seen.lo);
    for (int row0 = seen.lo; row0 < seen.hi; row0 += AT_TILE) {
      f32x4 s[4], th[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) s[b] = Mat<T>::mma(kf[b][k], qf[k], s[b]);
      }
      vst.store(vs, lane);
      ts[lane] = tst;
      if (seen.hi - row0 > AT_TILE) fetch(row0 + AT_TILE);
      wave_sync();
      logits(s, th, t, ts, g);
      if (seen.hi - row0 < AT_TILE) {
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (row0 + 16 * b + 4 * g + r >= seen.hi) s[b][r] = -INFINITY;
      }
      sm.step(s, acc);
      add_weighted<T, DP>(acc, s, vs, false, row0, seen, lane);
      wave_sync();
    }
    if (splits == 1) {
      float lse;
      const float by = sm.finish(lse);
      if (there) {
        const int64_t at = i * a.heads + head;
        store_row<T, DP>((T*)a.o + at * a.dim, acc, by, a.dim, g);
        if (g == 0) a.lse[at] = lse;
      }
    } else {
      const float l = swap_add(sm.l);
      if (there) {
        const int64_t rows = (int64_t)a.q_rays.n * a.heads, at = split * rows + i * a.heads + head;
        float* part = (float*)a.workspace;
        store_row<float, DP>(part + at * a.dim, acc, 1.f, a.dim, g);
        if (g == 0) reinterpret_cast<float2*>(part + splits * rows * a.dim)[at] = make_float2(sm.m, l);
      }
    }
  }
}

// Joins the splits of k_attn_row: a wavefront a (query, head)
template <typename T>
__global__ __launch_bounds__(AT_NT) void k_attn_join(ffn_ray_attn a, int splits) {
  const int lane = threadIdx.x & 63;
  const int64_t rows = (int64_t)a.q_rays.n * a.heads, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= rows) return;
  const float* part = (const float*)a.workspace;
  const float2* ml = reinterpret_cast<const float2*>(part + splits * rows * a.dim);
  float m = -INFINITY;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[s * rows + at].x);
  const float base = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float2 x = ml[s * rows + at];
    l = __builtin_fmaf(x.y, __builtin_amdgcn_exp2f(x.x - base), l);
  }
  const float by = l == 0.f ? 0.f : 1.f / l;
  for (int d = lane; d < a.dim; d += 64) {
    float o = 0.f;
    for (int s = 0; s < splits; ++s) {
      const float f = __builtin_amdgcn_exp2f(ml[s * rows + at].x - base);
      // an empty split's sums are 0; where the others made f infinite or NaN, theirs already are
      o = __builtin_fmaf(part[(s * rows + at) * a.dim + d], f, o);
    }
    ((T*)a.o)[at * a.dim + d] = (T)(o * by);
  }
  if (lane == 0) a.lse[at] = l == 0.f ? -INFINITY : (base + __builtin_amdgcn_logf(l) - W_SHIFT) * LN2;
}

// Few rows are split over their keys until about this many wavefronts have work: 16 a CU
constexpr int64_t ROW_WAVES = 4096;
// one wavefront a row and no tile shared between rows, where rays have at most one query each (on average)
static bool by_row(const ffn_ray_attn& a) { return a.q_rays.n <= a.q_rays.num_rays; }
static int row_splits(const ffn_ray_attn& a) {
  const int64_t waves = (int64_t)a.q_rays.n * a.kv_heads;
  const int64_t tiles = ((int64_t)a.k_rays.n / a.q_rays.n + AT_TILE - 1) / AT_TILE;  // of an average row
  int64_t s = (ROW_WAVES + waves - 1) / waves;
  s = s < tiles ? s : tiles;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

uint64_t attn_workspace(const ffn_ray_attn& a, bool backward) {
  const uint64_t rows = (uint64_t)a.q_rays.n * a.heads;
  if (backward) return rows * sizeof(float);
  if (a.q_rays.n == 0 || !by_row(a)) return 0;
  const uint64_t s = row_splits(a);
  return s > 1 ? s * rows * (a.dim + 2) * sizeof(float) : 0;
}

static unsigned die_grid(int64_t total) { return (unsigned)((total + 7) / 8 * 8); }

template <typename T, int DP>
static hipError_t fwd(const ffn_ray_attn& a, hipStream_t st) {
  if (by_row(a)) {
    const int splits = row_splits(a);
    const int64_t total = (int64_t)a.q_rays.n * a.kv_heads * splits;
    k_attn_row<T, DP><<<(unsigned)((total + 3) / 4), AT_NT, 0, st>>>(a, splits, total);
    if (splits > 1) k_attn_join<T><<<(unsigned)(((int64_t)a.q_rays.n * a.heads + 3) / 4), AT_NT, 0, st>>>(a, splits);
  } else {
    const int64_t total = ((int64_t)a.q_rays.n + AT_TILE - 1) / AT_TILE * a.heads;
    k_attn_fwd<T, DP><<<die_grid(total), AT_NT, 0, st>>>(a, total);
  }
  return hipGetLastError();
}

template <typename T, int DP>
static hipError_t bwd(const ffn_ray_attn& a, hipStream_t st) {
  if (a.q_rays.n) {
    const int64_t total = ((int64_t)a.q_rays.n + AT_TILE - 1) / AT_TILE * a.heads;
    k_attn_dq<T, DP><<<die_grid(total), AT_NT, 0, st>>>(a, total);
  }
  if (a.k_rays.n) {
    const int64_t total = ((int64_t)a.k_rays.n + AT_TILE - 1) / AT_TILE * a.kv_heads;
    k_attn_dkv<T, DP><<<die_grid(total), AT_NT, 0, st>>>(a, total);
  }
  return hipGetLastError();
}

template <typename T>
static hipError_t by_dim(const ffn_ray_attn& a, bool backward, hipStream_t st) {
  if (a.dim <= 32) return backward ? bwd<T, 32>(a, st) : fwd<T, 32>(a, st);
  if (a.dim <= 64) return backward ? bwd<T, 64>(a, st) : fwd<T, 64>(a, st);
  return backward ? bwd<T, 128>(a, st) : fwd<T, 128>(a, st);
}

hipError_t launch_attn(const ffn_ray_attn& a, bool backward, hipStream_t st) {
  if (a.dtype == FFN_BF16) return by_dim<__bf16>(a, backward, st);
  if (a.dtype == FFN_F16) return by_dim<_Float16>(a, backward, st);
  return by_dim<float>(a, backward, st);
}

}  // namespace ffn
