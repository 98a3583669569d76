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

constexpr int AT_NT = 256, AT_TILE = 64;  // four wavefronts; rows of a streamed tile
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Wavefronts a SIMD that the registers are held to: a wavefront waits more than it computes, so that one more is worth more
// than a few registers (16 bits; dk and dv of 8192 short rays: 139 us with three, 117 with four).
constexpr int least_waves(int size, int dim, int sets, bool cap) {
  return size == 2 && dim == 32 ? 5 - sets : size == 2 && dim == 64 && sets == 2 && !cap ? 3 : 1;
}
constexpr int least_waves_dkv(int size, int dim, int sets, bool cap) {
  return size == 2 && sets == 1 && dim == 32 ? 4 : size == 2 && sets == 1 && dim == 64 && !cap ? 3 : 1;
}

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

// sums and maxima over the four lane groups
__device__ __forceinline__ float swap_add(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float swap_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}

// What 16 kept rows see: lane c holds row c's range.  [lo, hi) covers all of them; a piece inside [all_lo, all_hi) is
// seen by every row.
struct Span {
  int lo, hi, all_lo, all_hi;
};
// v of the lane N further on among the same 16
template <int N> __device__ __forceinline__ int turn16(int v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xF, 0xF, true);  // row_ror:N
}
template <int N> __device__ __forceinline__ void span_step(Span& s) {
  s.lo = min(s.lo, turn16<N>(s.lo));
  s.hi = max(s.hi, turn16<N>(s.hi));
  s.all_lo = max(s.all_lo, turn16<N>(s.all_lo));
  s.all_hi = min(s.all_hi, turn16<N>(s.all_hi));
}
__device__ __forceinline__ Span span_of(const Range& r) {
  const bool none = r.hi <= r.lo;
  Span s{none ? INT_MAX : r.lo, none ? 0 : r.hi, none ? INT_MAX : r.lo, none ? 0 : r.hi};
  span_step<8>(s);
  span_step<4>(s);
  span_step<2>(s);
  span_step<1>(s);
  s.lo = __builtin_amdgcn_readfirstlane(s.lo);
  s.hi = __builtin_amdgcn_readfirstlane(s.hi);
  s.all_lo = __builtin_amdgcn_readfirstlane(s.all_lo);
  s.all_hi = __builtin_amdgcn_readfirstlane(s.all_hi);
  return s;
}
__device__ __forceinline__ bool sees(int row, const Range& r) {
  return (unsigned)(row - r.lo) < (unsigned)(r.hi - r.lo);
}

// ROWS rows of one head on their way to LDS, tile after tile (rows outside [row, end) and columns past dim as 0)
template <typename T, int DP, int NT = AT_NT, int ROWS = AT_TILE>
struct Staged {
  static constexpr int EL = 16 / (int)sizeof(T), CPR = DP / EL, N = ROWS * CPR / NT, STEP = NT / CPR;
  uint4 v[N];
  const T* p;   // this thread's first 16 bytes of the next tile
  int64_t row_step, tile_step;
  int row;      // and their row; past any end where the column is past dim
  __device__ __forceinline__ void begin(const T* __restrict__ base, int64_t stride, int row0, int dim, int tid) {
    const int col = tid % CPR * EL;
    row = col < dim ? row0 + tid / CPR : INT_MAX;
    p = base + (int64_t)(row0 + tid / CPR) * stride + col;
    row_step = STEP * stride;
    tile_step = ROWS * stride;
  }
  __device__ __forceinline__ void load(int end) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < end - i * STEP) v[i] = *reinterpret_cast<const uint4*>(p + i * row_step);
    }
    p += tile_step;
    row += row == INT_MAX ? 0 : ROWS;
  }
  __device__ __forceinline__ void store(T* tile, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i)
      *reinterpret_cast<uint4*>(tile + (tid / CPR + i * STEP) * lds_row<T, DP> + (tid % CPR) * EL) = v[i];
  }
  // whether any of this thread's values is infinite or NaN: their largest magnitude, as integers
  __device__ __forceinline__ bool nonfinite() const {
    if constexpr (sizeof(T) == 4) {
      unsigned m = 0u;
#pragma unroll
      for (int i = 0; i < N; ++i)
        m = max(max(m, max(v[i].x & 0x7FFFFFFFu, v[i].y & 0x7FFFFFFFu)), max(v[i].z & 0x7FFFFFFFu, v[i].w & 0x7FFFFFFFu));
      return m >= 0x7F800000u;
    } else {
      typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
      u16x2 m = {0, 0};
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const unsigned w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[k] & 0x7FFF7FFFu));
      }
      constexpr unsigned short e = __is_same(T, __bf16) ? 0x7F80 : 0x7C00;
      return max(m[0], m[1]) >= e;
    }
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

// tanh to single precision.  Pieces whose arguments all lie within NEAR, the usual ones, take a minimax polynomial of
// x^2 (relative error 3e-8); others 1 - 2 / (1 + e^2x), and the odd series where that would cancel.
constexpr float NEAR = 0.75f;
__device__ __forceinline__ float tanh_near(float x) {
  const float x2 = x * x;
  float p = __builtin_fmaf(x2, -0.004716258f, 0.019582909f);
  p = __builtin_fmaf(x2, p, -0.053344432f);
  p = __builtin_fmaf(x2, p, 0.13325407f);
  p = __builtin_fmaf(x2, p, -0.33332959f);
  return __builtin_fmaf(x * x2, p, x);
}
__device__ __forceinline__ float tanh_any(float x) {
  const float x2 = x * x;
  float p = __builtin_fmaf(x2, 62.f / 2835.f, -17.f / 315.f);
  p = __builtin_fmaf(x2, p, 2.f / 15.f);
  p = __builtin_fmaf(x2, p, -1.f / 3.f);
  const float small = __builtin_fmaf(x * x2, p, x);
  const float e = __builtin_amdgcn_exp2f(x * (2.f * LOG2E));
  const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e);
  return fabsf(x) < 0.25f ? small : big;
}

// Streamed rows are scored, masked and skipped in pieces of 32: B = 2 product tiles at once (4 in k_attn_row).  Whole tiles
// of 64 at once take a third more registers, and the wavefronts that costs are worth more: 108 us instead of 81 for the
// forward of 8192 short rays, 692 instead of 594 for dk and dv of long ones.
constexpr int PIECE = 32;
template <int B, typename F> __device__ __forceinline__ void each(F f) {
#pragma unroll
  for (int b = 0; b < B; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) f(b, r);
}

// Products -> logits: the exponential is 2^(mul s - ...), so that without a cap the scale and the unit cost nothing.
// x: the streamed rows' depths in LDS.
template <bool CAP>
struct Logits {
  float mul, pre, inv_cap, cap2, slope;
  bool bias;
  __device__ __forceinline__ Logits(const ffn_ray_attn& a, int head) {
    const float scale2 = a.scale * LOG2E;
    inv_cap = CAP ? a.scale / a.cap : 0.f;
    cap2 = a.cap * LOG2E;
    bias = a.slopes != nullptr;
    // s stays the bare product while mul is positive (maxima are taken of s)
    const bool bare = !CAP && scale2 > 1e-30f;
    mul = bare ? scale2 : 1.f;
    pre = bare ? 1.f : scale2;
    slope = bias ? a.slopes[head] * LOG2E / mul : 0.f;
  }
  template <int B>
  __device__ __forceinline__ void operator()(f32x4 (&s)[B], f32x4 (&th)[B], float t, const float* x, int g) const {
    if constexpr (CAP) {
      float top = 0.f;
      each<B>([&](int b, int r) {
        th[b][r] = s[b][r] * inv_cap;
        top = fmaxf(top, fabsf(th[b][r]));
      });
      if (__any(!(top <= NEAR))) each<B>([&](int b, int r) { th[b][r] = tanh_any(th[b][r]); });
      else each<B>([&](int b, int r) { th[b][r] = tanh_near(th[b][r]); });
      each<B>([&](int b, int r) { s[b][r] = cap2 * th[b][r]; });
    } else if (pre != 1.f) {
      each<B>([&](int b, int r) { s[b][r] *= pre; });
    }
    if (bias) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const f32x4 tx = *reinterpret_cast<const f32x4*>(x + 16 * b + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[b][r] = __builtin_fmaf(-slope, fabsf(t - tx[r]), s[b][r]);
      }
    }
  }
};

// s[q] = from(q, b) + 16 B tile rows . kept rows of set q
template <typename T, int DP, int NQ, int B, typename F>
__device__ __forceinline__ void products(f32x4 (&s)[NQ][B], const T* tile, const typename Mat<T>::frag (&kept)[NQ][DP / 32],
                                         int lane, F from) {
#pragma unroll
  for (int b = 0; b < B; ++b) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) s[q][b] = from(q, b);
#pragma unroll
    for (int ks = 0; ks < DP / 32; ++ks) {
      const typename Mat<T>::frag f = row_frag<T, DP>(tile, 16 * b + (lane & 15), ks, lane);
#pragma unroll
      for (int q = 0; q < NQ; ++q) s[q][b] = Mat<T>::mma(f, kept[q][ks], s[q][b]);
    }
  }
}

template <typename T, int DP, int NQ, int B>
__device__ __forceinline__ void products(f32x4 (&s)[NQ][B], const T* tile, const typename Mat<T>::frag (&kept)[NQ][DP / 32],
                                         int lane) {
  products<T, DP, NQ, B>(s, tile, kept, lane, [](int, int) { return f32x4{0.f, 0.f, 0.f, 0.f}; });
}

// a fragment with its infinities and NaN as 0
template <typename T>
__device__ __forceinline__ typename Mat<T>::frag finite_frag(typename Mat<T>::frag f) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (!(fabsf((float)f[j]) < INFINITY)) f[j] = (T)0.f;
  return f;
}

// acc[q] += tile^T w[q]: the 16 B tile rows are the K of the product.  Where the tile holds infinities or NaN (bad), pairs
// that do not see each other must not meet, since a weight of 0 times them is not 0: the product takes them as 0, and the
// pairs that do see each other are added one by one.
template <typename T, int DP, int NQ, int B>
__device__ __forceinline__ void add_weighted(f32x4 (&acc)[NQ][DP / 16], const f32x4 (&w)[NQ][B], const T* tile, bool bad,
                                             int row0, const Range (&seen)[NQ], int lane) {
#pragma unroll
  for (int h = 0; h < B / 2; ++h) {
    typename Mat<T>::frag f[NQ], m[DP / 16];
#pragma unroll
    for (int db = 0; db < DP / 16; ++db) m[db] = col_frag<T, DP>(tile, PIECE * h, 16 * db, lane);
    if (bad) {
#pragma unroll
      for (int db = 0; db < DP / 16; ++db) m[db] = finite_frag<T>(m[db]);
    }
#pragma unroll
    for (int q = 0; q < NQ; ++q) f[q] = product_frag<T>(w[q][2 * h], w[q][2 * h + 1]);
#pragma unroll
    for (int db = 0; db < DP / 16; ++db)
#pragma unroll
      for (int q = 0; q < NQ; ++q) acc[q][db] = Mat<T>::mma(m[db], f[q], acc[q][db]);
  }
  if (bad) {
    const int g = lane >> 4, c = lane & 15;
#pragma unroll 1
    for (int row = 0; row < 16 * B; ++row) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float mine = 0.f;
        each<B>([&](int b, int r) { mine = row >> 4 == b && (row & 3) == r ? w[q][b][r] : mine; });
        const float ww = __shfl(mine, 16 * ((row >> 2) & 3) + c);
        const bool see = sees(row0 + row, seen[q]);
#pragma unroll
        for (int db = 0; db < DP / 16; ++db) {
          const f32x4 x = __builtin_convertvector(
              *reinterpret_cast<const typename Mat<T>::quad*>(tile + row * lds_row<T, DP> + 16 * db + 4 * g), f32x4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (see && !(fabsf(x[k]) < INFINITY)) acc[q][db][k] = __builtin_fmaf(ww, x[k], acc[q][db][k]);
        }
      }
    }
  }
}

// what is not seen gets `v`
template <int B>
__device__ __forceinline__ void mask(f32x4 (&s)[B], int row0, const Span& w, const Range& seen, int g, float v) {
  if (row0 < w.all_lo || row0 + 16 * B > w.all_hi)
    each<B>([&](int b, int r) {
      if (!sees(row0 + 16 * b + 4 * g + r, seen)) s[b][r] = v;
    });
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

// log(l 2^(m - W_SHIFT)); the exponent of l goes to m, so that the logarithm is not rounded at its size
__device__ __forceinline__ float log_sum(float m, float l) {
  const float e = (float)__builtin_amdgcn_frexp_expf(l);
  return l == 0.f ? -INFINITY : (m + (e - W_SHIFT) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(l))) * LN2;
}

// Running softmax of one row, its sum still apart by lane group.  m is a maximum that lags: it is raised, and the sums are
// rescaled, only when a logit passes it by more than SLACK (which fp16's weights, 2^14 and more, have room for), so that
// most pieces need no exchange between lanes.  The rows of a wavefront are raised together, so that a row's last bits depend on
// its neighbours (each by its own logits alone: forward of 24 long rays 297 us instead of 278).
template <typename T>
struct Softmax {
  static constexpr float SLACK = __is_same(T, _Float16) ? 1.f : 8.f;
  float m = -INFINITY, l = 0.f;
  // weights in place of the logits
  template <int B, int NACC>
  __device__ __forceinline__ void step(f32x4 (&s)[B], float mul, f32x4 (&acc)[NACC]) {
    float mx = s[0][0];
    each<B>([&](int b, int r) { mx = fmaxf(mx, s[b][r]); });
    mx *= mul;
    if (__any(mx > m + SLACK)) {
      mx = fmaxf(m, swap_max(mx));
      const float f = __builtin_amdgcn_exp2f(m - (mx == -INFINITY ? 0.f : mx));
      l *= f;
#pragma unroll
      for (int i = 0; i < NACC; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= f;
      m = mx;
    }
    const float from = (m == -INFINITY ? 0.f : m) - W_SHIFT;
    each<B>([&](int b, int r) {
      s[b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], mul, -from));
      l += s[b][r];
    });
  }
  // factor of the sums, and the logarithm of the sum of exponentials
  __device__ __forceinline__ float finish(float& lse) {
    l = swap_add(l);
    lse = log_sum(m, l);
    return l == 0.f ? 0.f : 1.f / l;
  }
};

// Blocks in launch order go round the eight dies; this gives each die runs of 2^run neighbouring pieces of work, whose
// tiles share keys in its L2.
__device__ __forceinline__ int64_t die_order(int run) {
  const int64_t n = block_number(), b = n >> 3;
  return (((b >> run) * 8 + (n & 7)) << run) + (b & ((1 << run) - 1));
}

// the kept rows of a wavefront, NQ sets of 16: row number, what it sees, and the ranges over all of them
template <int NQ>
struct Kept {
  int64_t row[NQ];
  bool there[NQ];
  Range seen[NQ];
  Span span[NQ];
  int lo, hi;
  template <typename F>
  __device__ __forceinline__ Kept(int64_t first, int64_t n, int c, F sees_of) {
    lo = INT_MAX, hi = 0;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      row[q] = first + 16 * q + c;
      there[q] = row[q] < n;
      seen[q] = sees_of(row[q]);
      span[q] = span_of(seen[q]);
      lo = min(lo, span[q].lo);
      hi = max(hi, span[q].hi);
    }
  }
};

// Waits for the kept rows' fragments where it stands.  Without it their loads are still pending, as far as the compiler
// knows, when the streaming loop begins, and their first use there waits for the rows asked for ahead as well.
template <typename F, int N>
__device__ __forceinline__ void arrived(F (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// [lo, hi) over the block's four wavefronts
__device__ __forceinline__ Range block_range(int lo, int hi, int wave, int lane, int (&s)[8]) {
  if (lane == 0) s[wave] = lo, s[4 + wave] = hi;
  __syncthreads();
  return {min(min(s[0], s[1]), min(s[2], s[3])), max(max(s[4], s[5]), max(s[6], s[7]))};
}

// the pieces of a tile that the wavefront needs
template <typename F>
__device__ __forceinline__ void take_tile(F& take, int tile, int lo, int hi) {
  const bool one = tile < hi && tile + PIECE > lo, two = tile + PIECE < hi && tile + AT_TILE > lo;
  if (one) take(0);
  if (two) take(PIECE);
}

// o and lse by a running softmax.  NQ: sets of 16 queries a wavefront.  Two sets read each fragment of K and V once; short
// rays lose more to pieces that only one of the sets sees.
// Bound by the vector ALU (about a dozen instructions a visible pair; 70 % busy and the matrix cores 22 % on long rays) and,
// where rays are short, by the wavefronts' start.  24 rays of up to 4096 rows, 4 heads of 64 with 2 of keys, causal, bf16:
// 310 us, 395 TFLOP/s; 8192 rays of 23, 4 heads of 32, every option: 82 us.
template <typename T, int DP, int NQ, bool CAP>
__global__ __launch_bounds__(AT_NT, least_waves(sizeof(T), DP, NQ, CAP)) void k_attn_fwd(ffn_ray_attn a, int64_t total, int run) {
  constexpr int KS = DP / 32, NB = DP / 16, TILE = AT_TILE * lds_row<T, DP>;
  __shared__ __align__(16) T ks[2][TILE];
  __shared__ __align__(16) T vs[2][TILE];
  __shared__ __align__(16) float ts[2][AT_TILE];
  __shared__ int s_range[8], s_bad[2][4];
  const int64_t work = die_order(run);
  if (work >= total) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const unsigned item = (unsigned)work;
  const int head = (int)(item % (unsigned)a.heads), kh = head / (a.heads / a.kv_heads);
  const Kept<NQ> kept((int64_t)(item / (unsigned)a.heads) * (64 * NQ) + wave * 16 * NQ, a.q_rays.n, c, [&](int64_t i) { return keys_of(a, i); });
  const Logits<CAP> logits(a, head);
  typename Mat<T>::frag qf[NQ][KS];
  float t[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    load_frags<T, KS>(qf[q], (const T*)a.q + kept.row[q] * a.q_row + head * a.q_head, kept.there[q], a.dim, g);
    t[q] = logits.bias && kept.there[q] ? a.t_q[kept.row[q] * a.t_q_row] : 0.f;
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) arrived(qf[q]);
  arrived(t);
  const Range range = block_range(kept.lo, kept.hi, wave, lane, s_range);
  f32x4 acc[NQ][NB];
  Softmax<T> sm[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  Staged<T, DP> kst, vst;
  kst.begin((const T*)a.k + kh * a.k_head, a.k_row, range.lo, a.dim, tid);
  vst.begin((const T*)a.v + kh * a.v_head, a.v_row, range.lo, a.dim, tid);
  float tst = 0.f;
  auto fetch = [&](int row0) {
    kst.load(range.hi);
    vst.load(range.hi);
    if (logits.bias && tid < AT_TILE && row0 + tid < range.hi) tst = a.t_k[(int64_t)(row0 + tid) * a.t_k_row];
  };
  auto put = [&](int to) {
    kst.store(ks[to], tid);
    vst.store(vs[to], tid);
    const bool bad = __any(vst.nonfinite());
    if (lane == 0) s_bad[to][wave] = bad;
    if (tid < AT_TILE) ts[to][tid] = tst;
  };
  if (range.lo < range.hi) {
    fetch(range.lo);
    put(0);
  }
  int at = 0;
  for (int tile = range.lo; tile < range.hi; tile += AT_TILE, at ^= 1) {
    __syncthreads();
    const bool more = range.hi - tile > AT_TILE;
    if (more) fetch(tile + AT_TILE);
    const bool bad = s_bad[at][0] | s_bad[at][1] | s_bad[at][2] | s_bad[at][3];
    constexpr int B = PIECE / 16;
    auto take = [&](int p) {
      const int row0 = tile + p;
      f32x4 s[NQ][B], th[B];
      products<T, DP, NQ, B>(s, ks[at] + p * lds_row<T, DP>, qf, lane);
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        logits(s[q], th, t[q], ts[at] + p, g);
        mask(s[q], row0, kept.span[q], kept.seen[q], g, -INFINITY);
        sm[q].step(s[q], logits.mul, acc[q]);
      }
      add_weighted<T, DP, NQ, B>(acc, s, vs[at] + p * lds_row<T, DP>, bad, row0, kept.seen, lane);
    };
    take_tile(take, tile, kept.lo, kept.hi);
    if (more) put(at ^ 1);
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    float lse;
    const float by = sm[q].finish(lse);
    if (kept.there[q]) {
      const int64_t to = kept.row[q] * a.heads + head;
      store_row<T, DP>((T*)a.o + to * a.dim, acc[q], by, a.dim, g);
      if (g == 0) a.lse[to] = lse;
    }
  }
}

// Factor of one row's gradient weights.  fp16's exponent is too narrow for them (a probability times an upstream
// gradient of any size): each kept row's are scaled by a power of two that puts the largest so far into [2^13, 2^15],
// and its sums are rescaled when a larger one comes.  The other types take them as they are.
template <typename T>
struct GradScale {
  float f = 0.f;
  template <int B, int NACC>
  __device__ __forceinline__ void apply(f32x4 (&s)[B], f32x4 (&acc)[NACC]) {
    if constexpr (__is_same(T, _Float16)) {
      float mx = 0.f;
      each<B>([&](int b, int r) { mx = fmaxf(mx, fabsf(s[b][r])); });
      if (__any(mx * f > 32768.f || (f == 0.f && mx > 0.f))) {
        mx = swap_max(mx);
        const bool grow = mx > 0.f && (f == 0.f || mx * f > 32768.f);
        const int e = min(max(140 - (int)(__float_as_uint(mx) >> 23), -100), 100);  // 13 - exponent
        const float to = __uint_as_float((unsigned)(127 + e) << 23);
        const float by = grow ? (f == 0.f ? 0.f : to / f) : 1.f;
        if (grow) f = to;
#pragma unroll
        for (int i = 0; i < NACC; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][r] *= by;
      }
      each<B>([&](int b, int r) { s[b][r] *= f; });
    }
  }
  __device__ __forceinline__ float undo() const {
    if constexpr (__is_same(T, _Float16)) return f == 0.f ? 0.f : 1.f / f;
    return 1.f;
  }
};

// dq; also leaves D of its rows in the workspace for k_attn_dkv.  D = sum_d do o takes o's rounding in 16 bits, which puts dq of
// short rays a fifth further off, of long ones of up to 32 columns a twentieth.  There it is only a first value D': the
// products begin at -D', the sums are those of P (dP - D'), and beside them sum_j P (dP - D') = D - D' and sum_j P k, whose
// fragments of K are there already, set dq right (102 -> 110 us for 8192 rays; 65536 rows in rays of 2048, 32 columns,
// backward 373 -> 437).  Long rays of more columns (two sets of rows) keep D', which does not show there: 328 us instead of
// 472.  Bound as k_attn_fwd is; on the rays named there 335 us (550 TFLOP/s) and 109 us.
template <typename T, int DP, int NQ, bool CAP>
__global__ __launch_bounds__(AT_NT, least_waves(sizeof(T), DP, NQ, CAP)) void k_attn_dq(ffn_ray_attn a, int64_t total, int run) {
  constexpr int KS = DP / 32, NB = DP / 16, TILE = AT_TILE * lds_row<T, DP>;
  __shared__ __align__(16) T ks[2][TILE];
  __shared__ __align__(16) T vs[2][TILE];
  __shared__ __align__(16) float ts[2][AT_TILE];
  __shared__ int s_range[8], s_bad[2][4];
  const int64_t work = die_order(run);
  if (work >= total) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const unsigned item = (unsigned)work;
  const int head = (int)(item % (unsigned)a.heads), kh = head / (a.heads / a.kv_heads);
  const Kept<NQ> kept((int64_t)(item / (unsigned)a.heads) * (64 * NQ) + wave * 16 * NQ, a.q_rays.n, c, [&](int64_t i) { return keys_of(a, i); });
  const Logits<CAP> logits(a, head);
  typename Mat<T>::frag qf[NQ][KS], df[NQ][KS];
  float t[NQ], delta[NQ], from[NQ], exact[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t i = kept.row[q], to = i * a.heads + head;
    load_frags<T, KS>(qf[q], (const T*)a.q + i * a.q_row + head * a.q_head, kept.there[q], a.dim, g);
    load_frags<T, KS>(df[q], (const T*)a.dout + i * a.do_row + head * a.do_head, kept.there[q], a.dim, g);
    typename Mat<T>::frag of[KS];
    load_frags<T, KS>(of, (const T*)a.o + to * a.dim, kept.there[q], a.dim, g);
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) d = __builtin_fmaf((float)of[k][j], (float)df[q][k][j], d);
    d = swap_add(d);
    delta[q] = kept.seen[q].hi > kept.seen[q].lo ? d : 0.f;  // a row that sees nothing gets 0 whatever it holds
    exact[q] = 0.f;
    t[q] = logits.bias && kept.there[q] ? a.t_q[i * a.t_q_row] : 0.f;
    const float lse2 = kept.there[q] ? a.lse[to] * LOG2E : 0.f;
    from[q] = (lse2 == -INFINITY ? 0.f : lse2) - W_SHIFT;
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    arrived(qf[q]);
    arrived(df[q]);
  }
  arrived(t);
  arrived(from);
  arrived(delta);
  const Range range = block_range(kept.lo, kept.hi, wave, lane, s_range);
  constexpr bool EXACT = sizeof(T) == 2 && NQ == 1;
  constexpr int SETS = EXACT ? 2 * NQ : NQ;  // sums of P (dP - D') k, and of P k
  f32x4 acc[SETS][NB];
  GradScale<T> gs[NQ];
  Range seen[SETS];
#pragma unroll
  for (int q = 0; q < SETS; ++q) {
    seen[q] = kept.seen[q % NQ];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  Staged<T, DP> kst, vst;
  kst.begin((const T*)a.k + kh * a.k_head, a.k_row, range.lo, a.dim, tid);
  vst.begin((const T*)a.v + kh * a.v_head, a.v_row, range.lo, a.dim, tid);
  float tst = 0.f;
  auto fetch = [&](int row0) {
    kst.load(range.hi);
    vst.load(range.hi);
    if (logits.bias && tid < AT_TILE && row0 + tid < range.hi) tst = a.t_k[(int64_t)(row0 + tid) * a.t_k_row];
  };
  auto put = [&](int to) {
    kst.store(ks[to], tid);
    vst.store(vs[to], tid);
    const bool bad = __any(kst.nonfinite());
    if (lane == 0) s_bad[to][wave] = bad;
    if (tid < AT_TILE) ts[to][tid] = tst;
  };
  if (range.lo < range.hi) {
    fetch(range.lo);
    put(0);
  }
  int at = 0;
  for (int tile = range.lo; tile < range.hi; tile += AT_TILE, at ^= 1) {
    __syncthreads();
    const bool more = range.hi - tile > AT_TILE;
    if (more) fetch(tile + AT_TILE);
    const bool bad = s_bad[at][0] | s_bad[at][1] | s_bad[at][2] | s_bad[at][3];
    constexpr int B = PIECE / 16;
    auto take = [&](int p) {
      const int row0 = tile + p;
      f32x4 dp[NQ][B], th[B], s[SETS][B];  // s: the products, then the weights; the sets' logits come last
      f32x4(&x)[NQ][B] = *reinterpret_cast<f32x4(*)[NQ][B]>(&s[SETS - NQ]);
      products<T, DP, NQ, B>(x, ks[at] + p * lds_row<T, DP>, qf, lane);
      products<T, DP, NQ, B>(dp, vs[at] + p * lds_row<T, DP>, df, lane,
                             [&](int q, int) { return f32x4{-delta[q], -delta[q], -delta[q], -delta[q]}; });
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        logits(x[q], th, t[q], ts[at] + p, g);
        each<B>([&](int b, int r) { x[q][b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[q][b][r], logits.mul, -from[q])); });
        if constexpr (EXACT) {
          mask(x[q], row0, kept.span[q], kept.seen[q], g, 0.f);
          mask(dp[q], row0, kept.span[q], kept.seen[q], g, 0.f);
          if (CAP) mask(th, row0, kept.span[q], kept.seen[q], g, 0.f);  // a weight of 0 times a slope of NaN is NaN
          each<B>([&](int b, int r) { exact[q] = __builtin_fmaf(x[q][b][r], dp[q][b][r], exact[q]); });
        }
        // the slope of the cap
        if (CAP) each<B>([&](int b, int r) { x[q][b][r] *= __builtin_fmaf(-th[b][r], th[b][r], 1.f); });
        each<B>([&](int b, int r) { s[q][b][r] = x[q][b][r] * dp[q][b][r]; });
        if constexpr (!EXACT) mask(s[q], row0, kept.span[q], kept.seen[q], g, 0.f);
        gs[q].apply(s[q], acc[q]);
      }
      add_weighted<T, DP, SETS, B>(acc, s, ks[at] + p * lds_row<T, DP>, bad, row0, seen, lane);
    };
    take_tile(take, tile, kept.lo, kept.hi);
    if (more) put(at ^ 1);
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t to = kept.row[q] * a.heads + head;
    const float off = EXACT ? -swap_add(exact[q]) * W_UNSHIFT : 0.f, D = delta[q] - off, by = gs[q].undo();
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[q][b][r] = EXACT ? __builtin_fmaf(acc[q][b][r], by, off * acc[SETS - NQ + q][b][r]) : acc[q][b][r] * by;
    if (kept.there[q]) {
      store_row<T, DP>((T*)a.dq + to * a.dim, acc[q], a.scale * W_UNSHIFT, a.dim, g);
      if (g == 0) ((float*)a.workspace)[to] = D;
    }
  }
}

// dk and dv of the kept keys of one key head: the queries of the heads that share it stream past, so that the sums over heads
// and queries stay in registers.  Four products a pair instead of dq's three; bound on long rays by the chain of products and
// weights at two wavefronts a SIMD (vector ALU 46 %, matrix cores 27 % busy); on k_attn_fwd's rays 540 us (455 TFLOP/s) and
// 118 us.
template <typename T, int DP, int NQ, bool CAP>
__global__ __launch_bounds__(AT_NT, least_waves_dkv(sizeof(T), DP, NQ, CAP)) void k_attn_dkv(ffn_ray_attn a, int64_t total, int run) {
  constexpr int KS = DP / 32, NB = DP / 16, TILE = AT_TILE * lds_row<T, DP>;
  __shared__ __align__(16) T qs[2][TILE];
  __shared__ __align__(16) T ds[2][TILE];
  __shared__ __align__(16) float ts[2][AT_TILE], ls[2][AT_TILE], es[2][AT_TILE];
  __shared__ int s_range[8], s_bad[2][8];
  const int64_t work = die_order(run);
  if (work >= total) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const unsigned item = (unsigned)work;
  const int kh = (int)(item % (unsigned)a.kv_heads), group = a.heads / a.kv_heads;
  const Kept<NQ> kept((int64_t)(item / (unsigned)a.kv_heads) * (64 * NQ) + wave * 16 * NQ, a.k_rays.n, c, [&](int64_t j) { return queries_of(a, j); });
  const bool bias = a.slopes != nullptr;
  typename Mat<T>::frag kf[NQ][KS], vf[NQ][KS];
  float t[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int64_t j = kept.row[q];
    load_frags<T, KS>(kf[q], (const T*)a.k + j * a.k_row + kh * a.k_head, kept.there[q], a.dim, g);
    load_frags<T, KS>(vf[q], (const T*)a.v + j * a.v_row + kh * a.v_head, kept.there[q], a.dim, g);
    t[q] = bias && kept.there[q] ? a.t_k[j * a.t_k_row] : 0.f;
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    arrived(kf[q]);
    arrived(vf[q]);
  }
  arrived(t);
  const Range range = block_range(kept.lo, kept.hi, wave, lane, s_range);
  f32x4 dk[NQ][NB], dv[NQ][NB];
  GradScale<T> gs[NQ];
#pragma unroll
  for (int q = 0; q < NQ; ++q)
#pragma unroll
    for (int b = 0; b < NB; ++b) dk[q][b] = dv[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};
  Staged<T, DP> qst, dst;
  float tst = 0.f, lst = 0.f, est = 0.f;
  auto fetch = [&](int head, int row0) {
    if (row0 == range.lo) {
      qst.begin((const T*)a.q + head * a.q_head, a.q_row, row0, a.dim, tid);
      dst.begin((const T*)a.dout + head * a.do_head, a.do_row, row0, a.dim, tid);
    }
    qst.load(range.hi);
    dst.load(range.hi);
    if (tid < AT_TILE && row0 + tid < range.hi) {
      const int64_t i = row0 + tid;
      if (bias) tst = a.t_q[i * a.t_q_row];
      lst = a.lse[i * a.heads + head] * LOG2E;
      est = -((const float*)a.workspace)[i * a.heads + head];
      lst = (lst == -INFINITY ? 0.f : lst) - W_SHIFT;
    }
  };
  auto put = [&](int to) {
    qst.store(qs[to], tid);
    dst.store(ds[to], tid);
    const bool bad_q = __any(qst.nonfinite()), bad_d = __any(dst.nonfinite());
    if (lane == 0) s_bad[to][wave] = bad_q, s_bad[to][4 + wave] = bad_d;
    if (tid < AT_TILE) ts[to][tid] = tst, ls[to][tid] = lst, es[to][tid] = est;
  };
  const int first = kh * group, end = first + group;
  if (range.lo < range.hi) {
    fetch(first, range.lo);
    put(0);
  }
  int at = 0;
  for (int head = first; head < end && range.lo < range.hi; ++head) {
    const Logits<CAP> logits(a, head);
    for (int tile = range.lo; tile < range.hi; tile += AT_TILE, at ^= 1) {
      __syncthreads();
      const bool rest = range.hi - tile > AT_TILE, more = rest || head + 1 < end;
      if (more) fetch(rest ? head : head + 1, rest ? tile + AT_TILE : range.lo);
      const bool bad_q = s_bad[at][0] | s_bad[at][1] | s_bad[at][2] | s_bad[at][3];
      const bool bad_d = s_bad[at][4] | s_bad[at][5] | s_bad[at][6] | s_bad[at][7];
      constexpr int B = PIECE / 16;
      auto take = [&](int p) {
        const int row0 = tile + p;
        f32x4 s[NQ][B], dp[NQ][B], th[B];
        products<T, DP, NQ, B>(s, qs[at] + p * lds_row<T, DP>, kf, lane);
        products<T, DP, NQ, B>(dp, ds[at] + p * lds_row<T, DP>, vf, lane,
                               [&](int, int b) { return *reinterpret_cast<const f32x4*>(es[at] + p + 16 * b + 4 * g); });
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          logits(s[q], th, t[q], ts[at] + p, g);
#pragma unroll
          for (int b = 0; b < B; ++b) {
            const f32x4 l = *reinterpret_cast<const f32x4*>(ls[at] + p + 16 * b + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              s[q][b][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[q][b][r], logits.mul, -l[r]));
              dp[q][b][r] *= s[q][b][r];
            }
          }
          if (CAP) each<B>([&](int b, int r) { dp[q][b][r] *= __builtin_fmaf(-th[b][r], th[b][r], 1.f); });
          mask(s[q], row0, kept.span[q], kept.seen[q], g, 0.f);
          mask(dp[q], row0, kept.span[q], kept.seen[q], g, 0.f);
          gs[q].apply(dp[q], dk[q]);
        }
        add_weighted<T, DP, NQ, B>(dv, s, ds[at] + p * lds_row<T, DP>, bad_d, row0, kept.seen, lane);
        add_weighted<T, DP, NQ, B>(dk, dp, qs[at] + p * lds_row<T, DP>, bad_q, row0, kept.seen, lane);
      };
      take_tile(take, tile, kept.lo, kept.hi);
      if (more) put(at ^ 1);
    }
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q)
    if (kept.there[q]) {
      const int64_t to = (kept.row[q] * a.kv_heads + kh) * a.dim;
      store_row<T, DP>((T*)a.dk + to, dk[q], gs[q].undo() * (a.scale * W_UNSHIFT), a.dim, g);
      store_row<T, DP>((T*)a.dv + to, dv[q], W_UNSHIFT, a.dim, g);
    }
}

// part `split` of one query's keys, in whole tiles
template <int ROWS>
__device__ __forceinline__ Range split_keys(Range r, int split, int splits) {
  r = {__builtin_amdgcn_readfirstlane(r.lo), __builtin_amdgcn_readfirstlane(r.hi)};
  if (splits == 1) return r;
  const int tiles = (r.hi - r.lo + ROWS - 1) / ROWS;
  const int from = (int)((int64_t)tiles * split / splits), to = (int)((int64_t)tiles * (split + 1) / splits);
  return {r.lo + from * ROWS, min(r.hi, r.lo + to * ROWS)};
}

// One query at a time: a wavefront takes query i, the heads of one key head along its columns, and part `split` of the
// query's keys.  K comes straight into the operand's registers, V through the wavefront's own LDS rows (for the
// transposing read), 64 at a time where the registers hold them.  Nothing is shared, so nothing waits.  Bound by memory: 96
// rays of up to 4096 keys, 8 heads of 64, fp16: 122 us and 5 to join, 4.9 TB/s.
template <typename T, int DP> constexpr int row_tile = sizeof(T) * DP > 256 ? 32 : 64;
template <typename T, int DP, bool CAP>
__global__ __launch_bounds__(AT_NT) void k_attn_row(ffn_ray_attn a, int splits, int64_t total) {
  constexpr int KS = DP / 32, NB = DP / 16, ROWS = row_tile<T, DP>, B = ROWS / 16;
  __shared__ __align__(16) T vs_all[4][ROWS * lds_row<T, DP>];
  __shared__ __align__(16) float ts_all[4][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int64_t work = block_number() * 4 + wave;
  if (work >= total) return;  // no barriers below
  T* vs = vs_all[wave];
  float* ts = ts_all[wave];
  const int group = a.heads / a.kv_heads;
  const int kh = (int)(work % a.kv_heads);
  const int split = (int)(work / a.kv_heads % splits);
  const int64_t i = work / a.kv_heads / splits;
  const Range seen[1] = {split_keys<ROWS>(keys_of(a, i), split, splits)};
  const int lo = seen[0].lo, hi = seen[0].hi;
  const T* kb = (const T*)a.k + kh * a.k_head;
  for (int h0 = 0; h0 < group; h0 += 16) {
    const bool there = h0 + c < group;
    const int head = kh * group + min(h0 + c, group - 1);
    typename Mat<T>::frag qf[KS];
    load_frags<T, KS>(qf, (const T*)a.q + i * a.q_row + head * a.q_head, there, a.dim, g);
    const Logits<CAP> logits(a, head);
    const float t = logits.bias ? a.t_q[i * a.t_q_row] : 0.f;
    f32x4 acc[1][NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[0][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    Softmax<T> sm;
    Staged<T, DP, 64, ROWS> vst;
    typename Mat<T>::frag kf[B][KS];
    vst.begin((const T*)a.v + kh * a.v_head, a.v_row, lo, a.dim, lane);
    float tst = 0.f;
    auto fetch = [&](int row0) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int row = row0 + 16 * b + c;
        load_frags<T, KS>(kf[b], kb + row * a.k_row, row < hi, a.dim, g);
      }
      vst.load(hi);
      if (logits.bias && lane < ROWS && row0 + lane < hi) tst = a.t_k[(int64_t)(row0 + lane) * a.t_k_row];
    };
    if (lo < hi) fetch(lo);
    for (int row0 = lo; row0 < hi; row0 += ROWS) {
      f32x4 s[1][B], th[B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        s[0][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) s[0][b] = Mat<T>::mma(kf[b][k], qf[k], s[0][b]);
      }
      vst.store(vs, lane);
      if (lane < ROWS) ts[lane] = tst;
      if (hi - row0 > ROWS) fetch(row0 + ROWS);
      wave_sync();
      logits(s[0], th, t, ts, g);
      if (hi - row0 < ROWS)
        each<B>([&](int b, int r) {
          if (row0 + 16 * b + 4 * g + r >= hi) s[0][b][r] = -INFINITY;
        });
      sm.step(s[0], logits.mul, acc[0]);
      add_weighted<T, DP, 1, B>(acc, s, vs, false, row0, seen, lane);
      wave_sync();
    }
    if (splits == 1) {
      float lse;
      const float by = sm.finish(lse);
      if (there) {
        const int64_t at = i * a.heads + head;
        store_row<T, DP>((T*)a.o + at * a.dim, acc[0], by, a.dim, g);
        if (g == 0) a.lse[at] = lse;
      }
    } else {
      const float l = swap_add(sm.l);
      if (there) {
        const int64_t rows = (int64_t)a.q_rays.n * a.heads, at = split * rows + i * a.heads + head;
        float* part = (float*)a.workspace;
        store_row<float, DP>(part + at * a.dim, acc[0], 1.f, a.dim, g);
        if (g == 0) reinterpret_cast<float2*>(part + splits * rows * a.dim)[at] = make_float2(sm.m, l);
      }
    }
  }
}

// Sum over the splits s of factor[s] p[s step + 4 lane ..] by one wavefront: the lanes take four columns each of every G-th
// split, and the G sums are added in order.  factor null: 1.
__device__ __forceinline__ f32x4 sum_splits(const float* p, int64_t step, int splits, int dim, const float* factor, f32x4* sums,
                                            int lane) {
  const int quads = dim / 4, groups = 64 / quads, quad = lane % quads, group = lane / quads;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  if (group < groups) {
#pragma unroll 4
    for (int s = group; s < splits; s += groups) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + s * step + 4 * quad);
      const float f = factor ? factor[s] : 1.f;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = __builtin_fmaf(x[r], f, o[r]);
    }
  }
  sums[lane] = o;
  wave_sync();
  for (int s = 1; s < groups && lane < quads; ++s) {
    const f32x4 x = sums[s * quads + lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] += x[r];
  }
  wave_sync();
  return o;
}

// Joins the splits of k_attn_row: a wavefront a (query, head), its lanes the splits for the maximum and the sum.  An empty
// split's sums are 0; where the others made its factor infinite or NaN, theirs already are.
constexpr int MAX_SPLITS = 256;
template <typename T>
__global__ __launch_bounds__(AT_NT) void k_attn_join(ffn_ray_attn a, int splits) {
  __shared__ float factor[4][MAX_SPLITS];
  __shared__ f32x4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rows = (int64_t)a.q_rays.n * a.heads, at = (int64_t)blockIdx.x * 4 + wave;
  if (at >= rows) return;  // no barriers below
  const float* part = (const float*)a.workspace;
  const float2* ml = reinterpret_cast<const float2*>(part + splits * rows * a.dim);
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < splits; s += 64) m = fmaxf(m, ml[s * rows + at].x);
#pragma unroll
  for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const float base = m == -INFINITY ? 0.f : m;
  for (int s = lane; s < splits; s += 64) {
    const float2 x = ml[s * rows + at];
    const float f = __builtin_amdgcn_exp2f(x.x - base);
    factor[wave][s] = f;
    l = __builtin_fmaf(x.y, f, l);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
  wave_sync();
  const f32x4 o = sum_splits(part + at * a.dim, rows * a.dim, splits, a.dim, factor[wave], sums[wave], lane);
  if (lane < a.dim / 4) {
    const float by = l == 0.f ? 0.f : 1.f / l;
    typename Mat<T>::quad q;
#pragma unroll
    for (int r = 0; r < 4; ++r) q[r] = (T)(o[r] * by);
    *reinterpret_cast<typename Mat<T>::quad*>((T*)a.o + at * a.dim + 4 * lane) = q;
  }
  if (lane == 0) a.lse[at] = log_sum(base, l);
}

// words of D before the parts, which are 16-byte aligned
__host__ __device__ inline int64_t dq_parts(int64_t rows) { return (rows + 3) / 4 * 4; }

// k_attn_dq for the queries that k_attn_row takes: K through the wavefront's LDS rows, V straight into the operand.  The
// workspace holds D, then (splits) the sums of each part, and {sum P (dP - D'), D'}.
template <typename T, int DP, bool CAP>
__global__ __launch_bounds__(AT_NT) void k_attn_dq_row(ffn_ray_attn a, int splits, int64_t total) {
  constexpr int KS = DP / 32, NB = DP / 16, ROWS = row_tile<T, DP>, B = ROWS / 16;
  constexpr bool EXACT = sizeof(T) == 2;
  constexpr int SETS = EXACT ? 2 : 1;
  __shared__ __align__(16) T ks_all[4][ROWS * lds_row<T, DP>];
  __shared__ __align__(16) float ts_all[4][ROWS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int64_t work = block_number() * 4 + wave;
  if (work >= total) return;  // no barriers below
  T* ks = ks_all[wave];
  float* ts = ts_all[wave];
  const int group = a.heads / a.kv_heads;
  const int kh = (int)(work % a.kv_heads);
  const int split = (int)(work / a.kv_heads % splits);
  const int64_t i = work / a.kv_heads / splits;
  const Range all = keys_of(a, i), mine = split_keys<ROWS>(all, split, splits);
  const Range seen[2] = {mine, mine};
  const Range(&seen_by)[SETS] = *reinterpret_cast<const Range(*)[SETS]>(seen);
  const int lo = mine.lo, hi = mine.hi;
  const T* vb = (const T*)a.v + kh * a.v_head;
  for (int h0 = 0; h0 < group; h0 += 16) {
    const bool there = h0 + c < group;
    const int head = kh * group + min(h0 + c, group - 1);
    const int64_t at = i * a.heads + head;
    typename Mat<T>::frag qf[KS], df[KS], of[KS];
    load_frags<T, KS>(qf, (const T*)a.q + i * a.q_row + head * a.q_head, there, a.dim, g);
    load_frags<T, KS>(df, (const T*)a.dout + i * a.do_row + head * a.do_head, there, a.dim, g);
    load_frags<T, KS>(of, (const T*)a.o + at * a.dim, there, a.dim, g);
    float delta = 0.f, exact = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)of[k][j], (float)df[k][j], delta);
    delta = swap_add(delta);
    if (all.hi <= all.lo) delta = 0.f;
    const float lse2 = there ? a.lse[at] * LOG2E : 0.f, from = (lse2 == -INFINITY ? 0.f : lse2) - W_SHIFT;
    const Logits<CAP> logits(a, head);
    const float t = logits.bias ? a.t_q[i * a.t_q_row] : 0.f;
    f32x4 acc[SETS][NB];
#pragma unroll
    for (int q = 0; q < SETS; ++q)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[q][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    GradScale<T> gs;
    Staged<T, DP, 64, ROWS> kst;
    typename Mat<T>::frag vf[B][KS];
    kst.begin((const T*)a.k + kh * a.k_head, a.k_row, lo, a.dim, lane);
    float tst = 0.f;
    auto fetch = [&](int row0) {
      kst.load(hi);
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int row = row0 + 16 * b + c;
        load_frags<T, KS>(vf[b], vb + row * a.v_row, row < hi, a.dim, g);
      }
      if (logits.bias && lane < ROWS && row0 + lane < hi) tst = a.t_k[(int64_t)(row0 + lane) * a.t_k_row];
    };
    if (lo < hi) fetch(lo);
    for (int row0 = lo; row0 < hi; row0 += ROWS) {
      f32x4 dp[B], th[B], s[SETS][B], x[1][B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        dp[b] = f32x4{-delta, -delta, -delta, -delta};
#pragma unroll
        for (int k = 0; k < KS; ++k) dp[b] = Mat<T>::mma(vf[b][k], df[k], dp[b]);
      }
      kst.store(ks, lane);
      if (lane < ROWS) ts[lane] = tst;
      if (hi - row0 > ROWS) fetch(row0 + ROWS);
      wave_sync();
      const typename Mat<T>::frag(&q1)[1][KS] = *reinterpret_cast<const typename Mat<T>::frag(*)[1][KS]>(&qf);
      products<T, DP, 1, B>(x, ks, q1, lane);
      logits(x[0], th, t, ts, g);
      const bool ends = hi - row0 < ROWS;
      each<B>([&](int b, int r) {
        float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[0][b][r], logits.mul, -from));
        if (ends && row0 + 16 * b + 4 * g + r >= hi) w = 0.f;
        if (EXACT) exact = __builtin_fmaf(w, dp[b][r], exact);
        if (CAP) w *= __builtin_fmaf(-th[b][r], th[b][r], 1.f);
        s[SETS - 1][b][r] = w;
        s[0][b][r] = w * dp[b][r];
      });
      gs.apply(s[0], acc[0]);
      add_weighted<T, DP, SETS, B>(acc, s, ks, false, row0, seen_by, lane);
      wave_sync();
    }
    const float by = gs.undo();
    exact = swap_add(exact) * W_UNSHIFT;
    if (splits == 1) {
      each<NB>([&](int b, int r) {
        acc[0][b][r] = EXACT ? __builtin_fmaf(acc[0][b][r], by, -exact * acc[SETS - 1][b][r]) : acc[0][b][r] * by;
      });
      if (there) {
        store_row<T, DP>((T*)a.dq + at * a.dim, acc[0], a.scale * W_UNSHIFT, a.dim, g);
        if (g == 0) ((float*)a.workspace)[at] = EXACT ? delta + exact : delta;
      }
    } else if (there) {
      const int64_t rows = (int64_t)a.q_rays.n * a.heads, to = split * rows + at;
      float* part = (float*)a.workspace + dq_parts(rows);
      store_row<float, DP>(part + to * (SETS * a.dim), acc[0], by, a.dim, g);
      if (EXACT) store_row<float, DP>(part + to * (SETS * a.dim) + a.dim, acc[SETS - 1], 1.f, a.dim, g);
      if (g == 0) reinterpret_cast<float2*>(part + splits * rows * (SETS * a.dim))[to] = make_float2(exact, delta);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(AT_NT) void k_attn_dq_join(ffn_ray_attn a, int splits) {
  constexpr bool EXACT = sizeof(T) == 2;
  constexpr int SETS = EXACT ? 2 : 1;
  __shared__ f32x4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rows = (int64_t)a.q_rays.n * a.heads, at = (int64_t)blockIdx.x * 4 + wave;
  if (at >= rows) return;  // no barriers below
  const float* part = (const float*)a.workspace + dq_parts(rows);
  const float2* ed = reinterpret_cast<const float2*>(part + splits * rows * (SETS * a.dim));
  const float delta = ed[at].y;
  float exact = 0.f;
  for (int s = lane; EXACT && s < splits; s += 64) exact += ed[s * rows + at].x;
#pragma unroll
  for (int d = 32; d; d >>= 1) exact += __shfl_xor(exact, d);
  const int64_t step = rows * (SETS * a.dim);
  const float* p = part + at * (SETS * a.dim);
  f32x4 o = sum_splits(p, step, splits, a.dim, nullptr, sums[wave], lane);
  if (EXACT) {
    const f32x4 x = sum_splits(p + a.dim, step, splits, a.dim, nullptr, sums[wave], lane);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = __builtin_fmaf(x[r], -exact, o[r]);
  }
  if (lane < a.dim / 4) {
    typename Mat<T>::quad q;
#pragma unroll
    for (int r = 0; r < 4; ++r) q[r] = (T)(o[r] * (a.scale * W_UNSHIFT));
    *reinterpret_cast<typename Mat<T>::quad*>((T*)a.dq + at * a.dim + 4 * lane) = q;
  }
  if (lane == 0) ((float*)a.workspace)[at] = delta + exact;
}

// Averages that the host knows: rays with queries, and the keys of one
static int64_t rays_with_queries(const ffn_ray_attn& a) {
  const int64_t rays = a.q_rays.num_rays < a.q_rays.n ? a.q_rays.num_rays : a.q_rays.n;
  return rays < 1 ? 1 : rays;
}

// Whether one query at a time is the faster.  Its time is about 1.6 ns a (query, key head) and tile of keys, one more for
// the start, for every 16 heads that share the key head: k_attn_row passes over the keys once for each.  k_attn_fwd's is a
// chain over the keys of a block's 64 queries, 1.1 us a tile, or 1.6 ns a block and tile and 10 ns a block if there are many
// blocks; k_attn_dq's is 1.4 times that, where k_attn_dq_row's is hardly more than k_attn_row's.  Measured, bf16, dim 64, 8
// heads with 2 of keys, us (row / tile): 65536 rays of 8 keys and a query 303 / 154; 8192 of 128 102 / 202, with four
// queries each 257 / 213; 64 of 16384 106 / 17505, with four 196 / 4395, with sixteen 782 / 1008, and 1642 / 1008 where each
// head has its own keys.  Backward, mostly dk and dv: 1001 / 489, 675 / 893, 1045 / 840, 618 / 22772, 699 / 6128, 1186 / 1701,
// 2061 / 1879.  64 heads on one key head, forward and backward: 24 rays of 2500 among themselves 10138 + 28308 / 3672 +
// 20712; 64 of 8192 with 16 queries 778 + 2001 / 692 + 2420, with 32 1332 + 2539 / 748 + 2211; 64 of 16384 with one query
// 177 + 2559 (32 heads 92 + 1350).
static bool by_row(const ffn_ray_attn& a, bool backward) {
  const double n = (double)a.q_rays.n, keys = (double)a.k_rays.n, mean = keys / rays_with_queries(a);
  // 16 rows that share a few tiles of keys: k_attn_fwd's own case, though its chain may be a few us longer if all is small
  if (n > 16. * rays_with_queries(a) && mean <= 16. * AT_TILE) return false;
  const int passes = (a.heads / a.kv_heads + 15) / 16;  // over the keys, 16 heads a pass
  const double row = 1.6 * n * a.kv_heads * passes * (2. + floor(mean / AT_TILE));
  const double blocks = ceil(n / AT_TILE) * a.heads;
  const double a_block = (a.q_rays.n < AT_TILE ? keys : keys * AT_TILE / n) / AT_TILE;
  const double tiles = fmax(a_block, mean / AT_TILE) + 1.;
  return row < (backward ? 1.4 : 1.) * fmax(1100. * tiles, (1.6 * tiles + 10.) * blocks);
}
// Few rows are split over their keys until ROW_WAVES wavefronts have work, 16 a CU: 64 rays of 16384 keys, us with 512, 1024,
// 2048 and 4096 of them: 126, 104, 104, 106; with four queries each 453, 325, 327, 195.
constexpr int64_t ROW_WAVES = 4096;
static int row_splits(const ffn_ray_attn& a) {
  const int64_t waves = (int64_t)a.q_rays.n * a.kv_heads;
  const int64_t tiles = (int64_t)a.k_rays.n / rays_with_queries(a) / AT_TILE + 1;
  int64_t s = (ROW_WAVES + waves - 1) / waves;
  s = s < tiles ? s : tiles;
  return (int)(s < 1 ? 1 : s > MAX_SPLITS ? MAX_SPLITS : s);
}

uint64_t attn_workspace(const ffn_ray_attn& a, bool backward) {
  const uint64_t rows = (uint64_t)a.q_rays.n * a.heads;
  const uint64_t splits = a.q_rays.n && by_row(a, backward) ? row_splits(a) : 1;
  const uint64_t sets = backward && a.dtype != FFN_F32 ? 2 : 1;
  const uint64_t parts = splits > 1 ? splits * rows * (sets * a.dim + 2) : 0;
  return ((backward ? (uint64_t)dq_parts(rows) : 0) + parts) * sizeof(float);
}

// Runs of 16 pieces of work a die, of 4 where rays are so long that runs of 16 would leave the dies with unequal work (4 / 16,
// forward + backward, us: 65536 rows in rays of 4000 266 + 788 / 326 + 880; 131072 in rays of 1000, 8 heads 305 + 911 /
// 301 + 862; 131072 in rays of 512 119 + 346 / 93 + 287; 400000 in rays of 40 195 + 492 / 193 + 489)
static int die_run(const ffn_ray_set& kept) { return kept.n >= 2048 * (int64_t)kept.num_rays ? 2 : 4; }
static dim3 die_grid(int64_t total, int run) { return grid_of(((total + (8 << run) - 1) >> (3 + run)) << (3 + run)); }

// Sets of 16 kept rows a wavefront: two where rays are long on both sides, the registers hold them and `least` blocks of 128
// rows have work.  One set / two, us, forward and backward of bf16, dim 64, 4 heads, causal: 400000 rows in rays of 48
// 189 + 483 / 194 + 499, of 96 192 + 486 / 191 + 496; 262144 in rays of 128 124 + 351 / 120 + 325; 65536 in rays of 1024
// 114 + 361 / 105 + 267; in rays of 1500 72000 132 + 409 / 136 + 363, 36000 79 + 235 / 86 + 214, 18000 49 + 175 / 58 + 196.
constexpr int64_t FWD_BLOCKS = 1536, DQ_BLOCKS = 1024, DKV_BLOCKS = 512;
template <typename T, int DP> constexpr int MAX_SETS = sizeof(T) == 2 && DP <= 64 ? 2 : 1;
template <typename T, int DP> constexpr int DQ_SETS = DP > 32 ? MAX_SETS<T, DP> : 1;
template <int MOST>
static int sets(const ffn_ray_set& kept, const ffn_ray_set& streamed, int heads, int64_t least) {
  const int64_t rays = kept.num_rays;
  return kept.n >= 128 * rays && streamed.n >= 128 * rays && kept.n / 128 * heads >= least ? MOST : 1;
}

template <typename T, int DP, bool CAP>
static hipError_t fwd(const ffn_ray_attn& a, hipStream_t st) {
  if (by_row(a, false)) {
    const int splits = row_splits(a);
    const int64_t total = (int64_t)a.q_rays.n * a.kv_heads * splits;
    k_attn_row<T, DP, CAP><<<grid_of((total + 3) / 4), AT_NT, 0, st>>>(a, splits, total);
    if (splits > 1) k_attn_join<T><<<(unsigned)(((int64_t)a.q_rays.n * a.heads + 3) / 4), AT_NT, 0, st>>>(a, splits);
  } else {
    const int run = die_run(a.q_rays);
    const int64_t rows = 64 * sets<MAX_SETS<T, DP>>(a.q_rays, a.k_rays, a.heads, FWD_BLOCKS), total = ((int64_t)a.q_rays.n + rows - 1) / rows * a.heads;
    if (rows > 64) k_attn_fwd<T, DP, MAX_SETS<T, DP>, CAP><<<die_grid(total, run), AT_NT, 0, st>>>(a, total, run);
    else k_attn_fwd<T, DP, 1, CAP><<<die_grid(total, run), AT_NT, 0, st>>>(a, total, run);
  }
  return hipGetLastError();
}

template <typename T, int DP, bool CAP>
static hipError_t bwd(const ffn_ray_attn& a, hipStream_t st) {
  if (a.q_rays.n && by_row(a, true)) {
    const int splits = row_splits(a);
    const int64_t total = (int64_t)a.q_rays.n * a.kv_heads * splits;
    k_attn_dq_row<T, DP, CAP><<<grid_of((total + 3) / 4), AT_NT, 0, st>>>(a, splits, total);
    if (splits > 1) k_attn_dq_join<T><<<(unsigned)(((int64_t)a.q_rays.n * a.heads + 3) / 4), AT_NT, 0, st>>>(a, splits);
  } else if (a.q_rays.n) {
    const int run = die_run(a.q_rays);
    const int64_t rows = 64 * sets<DQ_SETS<T, DP>>(a.q_rays, a.k_rays, a.heads, DQ_BLOCKS), total = ((int64_t)a.q_rays.n + rows - 1) / rows * a.heads;
    if (rows > 64) k_attn_dq<T, DP, DQ_SETS<T, DP>, CAP><<<die_grid(total, run), AT_NT, 0, st>>>(a, total, run);
    else k_attn_dq<T, DP, 1, CAP><<<die_grid(total, run), AT_NT, 0, st>>>(a, total, run);
  }
  if (a.k_rays.n) {
    const int run = die_run(a.k_rays);
    const int64_t rows = 64 * sets<MAX_SETS<T, DP>>(a.k_rays, a.q_rays, a.kv_heads, DKV_BLOCKS), total = ((int64_t)a.k_rays.n + rows - 1) / rows * a.kv_heads;
    if (rows > 64) k_attn_dkv<T, DP, MAX_SETS<T, DP>, CAP><<<die_grid(total, run), AT_NT, 0, st>>>(a, total, run);
    else k_attn_dkv<T, DP, 1, CAP><<<die_grid(total, run), AT_NT, 0, st>>>(a, total, run);
  }
  return hipGetLastError();
}

template <typename T, int DP>
static hipError_t by_cap(const ffn_ray_attn& a, bool backward, hipStream_t st) {
  if (a.cap > 0.f) return backward ? bwd<T, DP, true>(a, st) : fwd<T, DP, true>(a, st);
  return backward ? bwd<T, DP, false>(a, st) : fwd<T, DP, false>(a, st);
}

template <typename T>
static hipError_t by_dim(const ffn_ray_attn& a, bool backward, hipStream_t st) {
  if (a.dim <= 32) return by_cap<T, 32>(a, backward, st);
  if (a.dim <= 64) return by_cap<T, 64>(a, backward, st);
  return by_cap<T, 128>(a, backward, st);
}

hipError_t launch_attn(const ffn_ray_attn& a, bool backward, hipStream_t st) {
  if (a.dtype == FFN_BF16) return by_dim<__bf16>(a, backward, st);
  if (a.dtype == FFN_F16) return by_dim<_Float16>(a, backward, st);
  return by_dim<float>(a, backward, st);
}

}  // namespace ffn
