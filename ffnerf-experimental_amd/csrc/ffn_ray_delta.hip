// ffn_ray_delta.hip -- a matrix state a ray and head, written by the delta rule with decay, and its gradients.
//
//   S_t = a_t S_{t-1} + k_t n_t^T,  n_t = b_t (v_t - a_t S_{t-1}^T k_t),  a_t = exp(decay_t),  o_t = scale S_t^T q_t
//
// In chunks of 16 rows, one matrix tile.  Inside a chunk, with D_ij = exp(decay_{j+1} + .. + decay_i) and e_i the same
// from the chunk's start, the rows' writes n solve a unit triangular system, and everything else is a matrix product:
//   A_ij = b_i D_ij k_i.k_j (j < i),  T = (I + A)^-1,  n = T R,  R_i = b_i (v_i - e_i S^T k_i)
//   P_ij = scale D_ij q_i.k_j (j <= i),  o_i = scale e_i S^T q_i + sum_j P_ij n_j,  S' = e_15 S + sum_j D_15,j k_j n_j^T
// Marched rays are short: a chunk of 16 wastes less of their last tile than a longer one, and its triangle is solved by
// substitution (sums of powers of A would cancel where neighbouring keys are alike, as they are along a ray).  Sums of
// decays are taken anew for every pair, so that neither a reset (decay = -infinity) nor a strong decay before a row costs
// the pairs after it their accuracy.
//
// A block is a ray and head; its wavefronts each hold 16 columns of S, whose columns do not touch each other, in product
// layout (lane c + 16 g: column c, rows 4 g + r of each 16), which is that of a product's second operand as well.  T and P
// belong to the rows alone: the wavefronts make those of a segment's chunks side by side and share them through LDS.
// Products are made in float.
#include <algorithm>

#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int DL_C = 16;              // rows of a chunk
constexpr int DL_SEG = 2;             // chunks between two states that are kept for the backward pass
constexpr int DL_MARK = DL_C * DL_SEG;
constexpr int DL_LD = 20;             // LDS row of a 16 x 16 matrix
constexpr int DL_VEC = 64;            // a chunk's b, e, D_15 and (first of the last 16) e_15
constexpr float DL_RESET = -1e30f;    // stands for a decay of -infinity, which must not meet a zero in a product
constexpr int DL_CLEAR = 1024;        // rows that one block looks through for those of no ray

__device__ __forceinline__ f32x4 mma4(float a, float b, const f32x4& c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// a b^T with both operands' K values in fragments of four a tile
template <int N>
__device__ __forceinline__ f32x4 dot_tiles(const f32x4 (&a)[N], const f32x4 (&b)[N]) {
  f32x4 even = {0.f, 0.f, 0.f, 0.f}, odd = even;
#pragma unroll
  for (int t = 0; t < N; ++t) {
#pragma unroll
    for (int r = 0; r < 4; r += 2) {
      even = mma4(a[t][r], b[t][r], even);
      odd = mma4(a[t][r + 1], b[t][r + 1], odd);
    }
  }
  return even + odd;
}
// A b for a 16 x 16 A, this lane's four values of its row c and columns 4 g + s, on a product
__device__ __forceinline__ f32x4 mul16(const f32x4& a, const f32x4& b, f32x4 to) {
#pragma unroll
  for (int s = 0; s < 4; ++s) to = mma4(a[s], b[s], to);
  return to;
}

template <typename T> __device__ __forceinline__ f32x4 load4(const T* p) {
  typedef T tvec __attribute__((ext_vector_type(4)));
  return __builtin_convertvector(*reinterpret_cast<const tvec*>(p), f32x4);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const f32x4& x) {
  typedef T tvec __attribute__((ext_vector_type(4)));
  *reinterpret_cast<tvec*>(p) = __builtin_convertvector(x, tvec);
}

// sum over the 16 lanes of a group
__device__ __forceinline__ f32x4 sum16(f32x4 x) {
#pragma unroll
  for (int d = 1; d < 16; d *= 2) {
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] += __shfl_xor(x[r], d);
  }
  return x;
}

// the rows of a ray in the order of the recurrence.
struct Chain {
  int64_t from;  // row of place 0
  int64_t first; // lowest row
  int step, count;
  __device__ __forceinline__ int64_t row(int p) const { return from + (int64_t)step * p; }
};
__device__ __forceinline__ Chain chain_of(const ffn_ray_delta& a, int64_t ray) {
  const int64_t n = a.rays.n, o = min((int64_t)a.rays.offsets[ray], n), c = min((int64_t)a.rays.counts[ray], n - o);
  return {a.reverse ? o + c - 1 : o, o, a.reverse ? -1 : 1, (int)c};
}
// where the state before place p (a multiple of DL_MARK above 0) is kept: places of one ray, and of rays that do not
// overlap, never share a slot
__device__ __forceinline__ int64_t mark_slot(const Chain& ch, int p) { return (ch.first + p) / DL_MARK; }

// Loads go to the last row, or the first columns, where a place is past the ray's end or the columns, and their values are
// dropped then: under a branch each would wait for the one before it.

// this lane's part of a chunk's rows p0 + c: four values of every 16 columns, 0 past the ray's end or the columns
template <typename T, int N>
__device__ __forceinline__ void load_rows(f32x4 (&to)[N], const T* base, int64_t row_stride, const Chain& ch, int p0, int c,
                                          int g, int cols) {
  typedef T tvec __attribute__((ext_vector_type(4)));
  const T* p = base + ch.row(min(p0 + c, ch.count - 1)) * row_stride;
  const bool there = p0 + c < ch.count;
  tvec x[N];
#pragma unroll
  for (int t = 0; t < N; ++t) x[t] = *reinterpret_cast<const tvec*>(p + (16 * t + 4 * g < cols ? 16 * t + 4 * g : 0));
#pragma unroll
  for (int t = 0; t < N; ++t) {
    const f32x4 f = __builtin_convertvector(x[t], f32x4), zero = {0.f, 0.f, 0.f, 0.f};
    to[t] = there && 16 * t + 4 * g < cols ? f : zero;
  }
}
// column `col` of the chunk's rows 4 g + r
template <typename T>
__device__ __forceinline__ f32x4 load_col(const T* base, int64_t row_stride, const Chain& ch, int p0, int g, int col, int cols) {
  T x[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) x[r] = base[ch.row(min(p0 + 4 * g + r, ch.count - 1)) * row_stride + (col < cols ? col : 0)];
  f32x4 y;
#pragma unroll
  for (int r = 0; r < 4; ++r) y[r] = p0 + 4 * g + r < ch.count && col < cols ? (float)x[r] : 0.f;
  return y;
}

// the decays of the chunk's rows 4 g + r and the strength of its row c
template <typename T>
__device__ __forceinline__ void load_gates(const ffn_ray_delta& a, int h, const Chain& ch, int p0, int c, int g, f32x4& decay,
                                           float& beta) {
  const T *d = (const T*)a.decay + h * a.decay_head, *b = (const T*)a.beta + h * a.beta_head;
  const T bx = b[ch.row(min(p0 + c, ch.count - 1)) * a.beta_row];
  T dx[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) dx[r] = d[ch.row(min(p0 + 4 * g + r, ch.count - 1)) * a.decay_row];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const float x = p0 + 4 * g + r < ch.count ? (float)dx[r] : 0.f;
    decay[r] = x < DL_RESET ? DL_RESET : x;
  }
  beta = p0 + c < ch.count ? (float)bx : 0.f;
}

// A state's 16 columns from `w16` on, in product layout, from or to [dk][dv].
template <int NT>
__device__ __forceinline__ void load_state(f32x4 (&S)[NT], const float* from, const ffn_ray_delta& a, int c, int g, int w16) {
#pragma unroll
  for (int t = 0; t < NT; ++t) S[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!from) return;
  const int v = min(w16 + c, a.val_dim - 1);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) S[t][r] = from[(int64_t)min(16 * t + 4 * g + r, a.key_dim - 1) * a.val_dim + v];
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (16 * t + 4 * g + r >= a.key_dim || w16 + c >= a.val_dim) S[t][r] = 0.f;
  }
}
template <int NT>
__device__ __forceinline__ void store_state(float* to, const f32x4 (&S)[NT], const ffn_ray_delta& a, int c, int g, int w16) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = 16 * t + 4 * g + r, v = w16 + c;
      if (k < a.key_dim && v < a.val_dim) to[(int64_t)k * a.val_dim + v] = S[t][r];
    }
  }
}

// x of lane L of this lane's group of 16
template <int L> __device__ __forceinline__ float of_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x150 + L, 0xF, 0xF, true));
}

// exp(x): the product with log2(e) in two parts, so that the result is as accurate as the hardware's 2^x
__device__ __forceinline__ float exp_of(float x) {
  const float hi = x * 1.442695041f, lo = __builtin_fmaf(x, 1.442695041f, -hi);
  const float y = __builtin_amdgcn_exp2f(hi);
  return __builtin_fmaf(y, lo * 0.6931471806f, y);
}

// Column c of X with (I + A) X = I: x[J] is done when the rows before it have been taken off.  a[j] = A[c][j].  (By rows of X
// a NaN in a row of A would meet the zeros of the rows before it.)
template <int J, int I> __device__ __forceinline__ void take_off_row(const float (&a)[DL_C], float (&x)[DL_C]) {
  x[I] = __builtin_fmaf(-of_lane<I>(a[J]), x[J], x[I]);
  if constexpr (I + 1 < DL_C) take_off_row<J, I + 1>(a, x);
}
template <int J> __device__ __forceinline__ void take_off(const float (&a)[DL_C], float (&x)[DL_C]) {
  take_off_row<J, J + 1>(a, x);
  if constexpr (J + 2 < DL_C) take_off<J + 1>(a, x);
}

// What a chunk's rows do to each other, by one wavefront: T, P and (if Dm) D as [row i][column j], and the rows' vectors.
// decay: those of rows 4 g + r (at least DL_RESET), beta: that of row c.  Sums of decays are products with zeros and ones.
template <int NT>
__device__ __forceinline__ void prepare_chunk(const f32x4 (&kf)[NT], const f32x4 (&qf)[NT], const f32x4& decay, float beta,
                                              float scale, int c, int g, float* Tm, float* Pm, float* Dm, float* vec) {
  // row j = 4 g + r, column i = c: the sum of decays from j + 1 to i
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < 4; ++s) sum = mma4(4 * g + s > c ? 1.f : 0.f, 4 * g + s <= c ? decay[s] : 0.f, sum);
  const f32x4 kk = dot_tiles(kf, kf), kq = dot_tiles(kf, qf);
  f32x4 D, P, A;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = 4 * g + r;
    const float d = exp_of(sum[r]);
    D[r] = j <= c ? d : 0.f;
    P[r] = j <= c ? scale * d * kq[r] : 0.f;
    A[r] = j < c ? beta * d * kk[r] : 0.f;
  }
  *reinterpret_cast<f32x4*>(Tm + c * DL_LD + 4 * g) = A;
  *reinterpret_cast<f32x4*>(Pm + c * DL_LD + 4 * g) = P;
  if (Dm) *reinterpret_cast<f32x4*>(Dm + c * DL_LD + 4 * g) = D;
  const float e = exp_of(decay[0] + sum[0]);  // in the first group, from the chunk's start to row c
  if (g == 0) {
    vec[c] = beta;
    vec[16 + c] = e;
    if (c == DL_C - 1) vec[48] = e;
  }
  if (c == DL_C - 1) *reinterpret_cast<f32x4*>(vec + 32 + 4 * g) = D;
  wave_sync();
  float a[DL_C], x[DL_C];
#pragma unroll
  for (int i = 0; i < DL_C; i += 4) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(Tm + c * DL_LD + i);
#pragma unroll
    for (int r = 0; r < 4; ++r) a[i + r] = v[r], x[i + r] = i + r == c ? 1.f : 0.f;
  }
  take_off<0>(a, x);
  wave_sync();
#pragma unroll
  for (int r = 0; r < 4; ++r) Tm[(4 * g + r) * DL_LD + c] = g == 0 ? x[r] : g == 1 ? x[4 + r] : g == 2 ? x[8 + r] : x[12 + r];
}

__device__ __forceinline__ bool finite4(const f32x4& x) {
  return fabsf(x[0]) <= 3.4e38f && fabsf(x[1]) <= 3.4e38f && fabsf(x[2]) <= 3.4e38f && fabsf(x[3]) <= 3.4e38f;
}
// A x for a lower triangular A where x holds infinities or NaN: they must not meet the zeros above the diagonal, so they
// are left out, and the rows from the first of them on are NaN.
__device__ __forceinline__ f32x4 mul16_sick(const f32x4& A, f32x4 x, const f32x4& to, int g) {
  int first = DL_C;
#pragma unroll
  for (int r = 3; r >= 0; --r) {
    if (!(fabsf(x[r]) <= 3.4e38f)) {
      first = 4 * g + r;
      x[r] = 0.f;
    }
  }
  first = min(first, __shfl_xor(first, 16));
  first = min(first, __shfl_xor(first, 32));
  f32x4 y = mul16(A, x, to);
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (4 * g + r >= first) y[r] = __builtin_nanf("");
  return y;
}

// rows of no ray: 0 in `heads` x `cols` of each output
template <typename T>
__device__ __forceinline__ void clear_rows(const ffn_ray_delta& a, int64_t block, T* p, int64_t width) {
  for (int64_t i = block * DL_CLEAR + threadIdx.x; i < min((block + 1) * DL_CLEAR, (int64_t)a.rays.n); i += blockDim.x) {
    const uint32_t r = a.rays.ray_ids[i];
    if (r < a.rays.num_rays) {
      const int64_t o = a.rays.offsets[r];
      if (i >= o && i - o < (int64_t)a.rays.counts[r]) continue;
    }
    for (int64_t j = 0; j < width; ++j) p[i * width + j] = (T)0.f;
  }
}

template <typename T, int DK, int CH>
__global__ __launch_bounds__(512) void k_delta_fwd(const ffn_ray_delta a) {
  constexpr int NT = DK / 16, LDK = DK + 16 / (int)sizeof(T);
  __shared__ float Tm[CH][DL_C * DL_LD], Pm[CH][DL_C * DL_LD], vec[CH][DL_VEC];
  __shared__ __align__(16) T Kl[CH * DL_C * LDK];
  const int64_t block = block_number(), teams = (int64_t)a.rays.num_rays * a.v_heads;
  if (block >= teams) {
    clear_rows(a, block - teams, (T*)a.o, (int64_t)a.v_heads * a.val_dim);
    return;
  }
  const int64_t ray = block / a.v_heads;
  const int h = (int)(block - ray * a.v_heads), hk = h / (a.v_heads / a.heads);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, W = blockDim.x >> 6, w16 = 16 * w;
  int c = lane & 15, g = lane >> 4;
  const Chain ch = chain_of(a, ray);
  const T* q = (const T*)a.q + hk * a.q_head;
  const T* k = (const T*)a.k + hk * a.k_head;
  const T* v = (const T*)a.v + h * a.v_head;
  T* o = (T*)a.o + (int64_t)h * a.val_dim;
  const int64_t size = (int64_t)a.key_dim * a.val_dim;
  f32x4 S[NT];
  load_state(S, a.h0 ? a.h0 + block * size : nullptr, a, c, g, w16);
  for (int p0 = 0; p0 < ch.count; p0 += CH * DL_C) {
    if (p0) __syncthreads();
    for (int i = w; i < CH; i += W) {
      const int p = p0 + DL_C * i;
      if (p >= ch.count) break;
      asm volatile("" : "+v"(c), "+v"(g));  // opaque: else all that goes by the lane alone is formed ahead, and held
      f32x4 kf[NT], qf[NT];
      load_rows(kf, k, a.k_row, ch, p, c, g, a.key_dim);
      load_rows(qf, q, a.q_row, ch, p, c, g, a.key_dim);
      f32x4 decay;
      float beta;
      load_gates<T>(a, h, ch, p, c, g, decay, beta);
#pragma unroll
      for (int t = 0; t < NT; ++t) store4(&Kl[(DL_C * i + c) * LDK + 16 * t + 4 * g], kf[t]);
      prepare_chunk(kf, qf, decay, beta, a.scale, c, g, Tm[i], Pm[i], (float*)nullptr, vec[i]);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < CH; ++i) {
      const int p = p0 + DL_C * i;
      if (p >= ch.count) break;
      asm volatile("" : "+v"(c), "+v"(g));
      if (a.marks && p && p % DL_MARK == 0)
        store_state(a.marks + (mark_slot(ch, p) * a.v_heads + h) * size, S, a, c, g, w16);
      const T* Kc = Kl + DL_C * i * LDK;
      f32x4 kf[NT], qf[NT];
      load_rows(qf, q, a.q_row, ch, p, c, g, a.key_dim);
      const f32x4 vv = load_col(v, a.v_row, ch, p, g, w16 + c, a.val_dim);
#pragma unroll
      for (int t = 0; t < NT; ++t) kf[t] = load4(Kc + c * LDK + 16 * t + 4 * g);
      const f32x4 beta = *reinterpret_cast<const f32x4*>(&vec[i][4 * g]);
      const f32x4 e = *reinterpret_cast<const f32x4*>(&vec[i][16 + 4 * g]);
      const f32x4 left = *reinterpret_cast<const f32x4*>(&vec[i][32 + 4 * g]);
      const float all = vec[i][48];
      const f32x4 Tr = *reinterpret_cast<const f32x4*>(&Tm[i][c * DL_LD + 4 * g]);
      const f32x4 Pr = *reinterpret_cast<const f32x4*>(&Pm[i][c * DL_LD + 4 * g]);
      const f32x4 R = beta * (vv - e * dot_tiles(kf, S)), zero = {0.f, 0.f, 0.f, 0.f};
      const f32x4 qs = a.scale * e * dot_tiles(qf, S);
      f32x4 n = mul16(Tr, R, zero), y;
      if (__any(!finite4(n))) {
        n = mul16_sick(Tr, R, zero, g);
        y = mul16_sick(Pr, n, qs, g);
      } else {
        y = mul16(Pr, n, qs);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = p + 4 * g + r;
        if (at < ch.count && w16 + c < a.val_dim) o[ch.row(at) * a.v_heads * a.val_dim + w16 + c] = (T)y[r];
      }
      const f32x4 nl = left * n;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 kt;
#pragma unroll
        for (int s = 0; s < 4; ++s) kt[s] = (float)Kc[(4 * g + s) * LDK + 16 * t + c];
        S[t] = mul16(kt, nl, all * S[t]);
      }
    }
  }
  if (a.last) store_state(a.last + block * size, S, a, c, g, w16);
}

// Few rows a ray (one more sample of each): the state goes through once, row by row on the vector ALU, and memory bounds
// it.  A wavefront takes 32 columns of a state: 8 lanes of four columns, 8 groups of rows dk = 8 i + group.
template <typename T, int DK>
__global__ __launch_bounds__(256) void k_delta_step(const ffn_ray_delta a) {
  constexpr int N = DK / 8;
  const int parts = (a.val_dim + 31) / 32;
  const int64_t teams = (int64_t)a.rays.num_rays * a.v_heads * parts, blocks = (teams + 3) / 4;
  if (block_number() >= blocks) {
    clear_rows(a, block_number() - blocks, (T*)a.o, (int64_t)a.v_heads * a.val_dim);
    return;
  }
  const int64_t team = block_number() * 4 + (threadIdx.x >> 6);
  if (team >= teams) return;
  const int64_t state = team / parts, ray = state / a.v_heads;
  const int h = (int)(state - ray * a.v_heads), hk = h / (a.v_heads / a.heads);
  const int lane = threadIdx.x & 63, rg = lane >> 3, col = (int)(team - state * parts) * 32 + 4 * (lane & 7);
  const bool in = col < a.val_dim;
  const Chain ch = chain_of(a, ray);
  const int64_t at = state * a.key_dim * a.val_dim;
  f32x4 S[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int kd = 8 * i + rg;
    S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.h0 && in && kd < a.key_dim) S[i] = load4(a.h0 + at + (int64_t)kd * a.val_dim + col);
  }
  for (int p = 0; p < ch.count; ++p) {
    const int64_t row = ch.row(p);
    const T* q = (const T*)a.q + row * a.q_row + hk * a.q_head;
    const T* k = (const T*)a.k + row * a.k_row + hk * a.k_head;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (in) v = load4((const T*)a.v + row * a.v_row + h * a.v_head + col);
    const float decay = expf((float)((const T*)a.decay)[row * a.decay_row + h * a.decay_head]);
    const float beta = (float)((const T*)a.beta)[row * a.beta_row + h * a.beta_head];
    float kk[N], qq[N], qk = 0.f;
    f32x4 ks = {0.f, 0.f, 0.f, 0.f}, qs = ks;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int kd = 8 * i + rg;
      kk[i] = kd < a.key_dim ? (float)k[kd] : 0.f;
      qq[i] = kd < a.key_dim ? (float)q[kd] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      S[i] = decay * S[i];
      qk = __builtin_fmaf(qq[i], kk[i], qk);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] = __builtin_fmaf(kk[i], S[i][e], ks[e]);
        qs[e] = __builtin_fmaf(qq[i], S[i][e], qs[e]);
      }
    }
#pragma unroll
    for (int d = 8; d < 64; d *= 2) {
      qk += __shfl_xor(qk, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        ks[e] += __shfl_xor(ks[e], d);
        qs[e] += __shfl_xor(qs[e], d);
      }
    }
    const f32x4 n = beta * (v - ks);
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) S[i][e] = __builtin_fmaf(kk[i], n[e], S[i][e]);
    }
    if (rg == 0 && in) store4((T*)a.o + (row * a.v_heads + h) * a.val_dim + col, a.scale * (qs + qk * n));
  }
  if (!a.last) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int kd = 8 * i + rg;
    if (in && kd < a.key_dim) store4(a.last + at + (int64_t)kd * a.val_dim + col, S[i]);
  }
}

// The backward pass.  Segments of two chunks from the ray's end, each from the state that the forward kept: its chunks'
// states and writes again, then the chunks back to front.  With dS the gradient of the state after a chunk:
//   dn = P^T do + D_15 K dS,  dR = T^T dn,  dv = b dR,  X = D (do n^T) (j <= i),  Y = -D (dR n^T) (j < i)
//   dq_i = scale (e_i S do_i + sum_j X_ij k_j),  left_i = -e_i S dR_i + sum_j Y_ij k_j
//   right_j = D_15,j dS n_j + sum_i (scale X_ij q_i + b_i Y_ij k_i),  dk = b left + right,  db_i = k_i.left_i + v_i.dR_i
//   dS' = e_15 dS + sum_i (scale e_i q_i do_i^T - b_i e_i k_i dR_i^T)
// Every factor e or D a row i was multiplied with gives its sum of products to the decays up to i:
//   ddecay = sums, from each row to the chunk's end, of q.dq + b k.left - k.right, and at the end dS.S
// dn, dR, dv and dS go by columns, as S does; dq and dk are sums over the columns: S, dS, n and dR pass through LDS, and a
// wavefront takes 16 columns of dq and dk.
__host__ __device__ constexpr int delta_lds(int DK, int W, int size) {
  return (DL_SEG * (3 * DL_C * DL_LD + DL_VEC) + 2 * DL_C * DL_LD + (2 * DL_C + DK) * (16 * W + 4) + W * 32) * 4 +
         2 * DL_MARK * (DK + 16 / size) * size;
}

template <typename T, int DK, int TP>
__global__ __launch_bounds__(512) void k_delta_bwd(const ffn_ray_delta a) {
  constexpr int NT = DK / 16, LDK = DK + 16 / (int)sizeof(T), SQ = DL_C * DL_LD;
  extern __shared__ __align__(16) float lds[];
  const int64_t block = block_number(), teams = (int64_t)a.rays.num_rays * a.v_heads;
  const bool shared = a.heads != a.v_heads;
  if (block >= teams) {
    clear_rows(a, block - teams, (T*)a.dq, (int64_t)a.heads * a.key_dim);
    clear_rows(a, block - teams, (T*)a.dk, (int64_t)a.heads * a.key_dim);
    clear_rows(a, block - teams, (T*)a.dv, (int64_t)a.v_heads * a.val_dim);
    clear_rows(a, block - teams, (T*)a.ddecay, (int64_t)a.v_heads);
    clear_rows(a, block - teams, (T*)a.dbeta, (int64_t)a.v_heads);
    return;
  }
  const int64_t ray = block / a.v_heads;
  const int h = (int)(block - ray * a.v_heads), hk = h / (a.v_heads / a.heads);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, W = blockDim.x >> 6, w16 = 16 * w;
  int c = lane & 15, g = lane >> 4;
  const int LDV = 16 * W + 4, vcol = w16 + c;
  float* Tm = lds;
  float* Pm = Tm + DL_SEG * SQ;
  float* Dm = Pm + DL_SEG * SQ;
  float* vecs = Dm + DL_SEG * SQ;
  float* Xm = vecs + DL_SEG * DL_VEC;
  float* Ym = Xm + SQ;
  float* Nl = Ym + SQ;
  float* Rl = Nl + DL_C * LDV;
  float* Sl = Rl + DL_C * LDV;
  float* sums = Sl + DK * LDV;
  T* Kl = (T*)(sums + W * 32);
  T* Ql = Kl + DL_MARK * LDK;
  const Chain ch = chain_of(a, ray);
  const T* q = (const T*)a.q + hk * a.q_head;
  const T* k = (const T*)a.k + hk * a.k_head;
  const T* v = (const T*)a.v + h * a.v_head;
  const T* dout = (const T*)a.dout + h * a.do_head;
  const int64_t size = (int64_t)a.key_dim * a.val_dim;
  f32x4 dS[NT];
  load_state(dS, a.dlast ? a.dlast + block * size : nullptr, a, c, g, w16);
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  const int last = ch.count ? (ch.count - 1) / DL_MARK * DL_MARK : -1;
#pragma unroll 1
  for (int p0 = last; p0 >= 0; p0 -= DL_MARK) {
    if (p0 != last) __syncthreads();
    for (int i = w; i < DL_SEG; i += W) {
      const int p = p0 + DL_C * i;
      if (p >= ch.count) break;
      asm volatile("" : "+v"(c), "+v"(g));  // opaque: else all that goes by the lane alone is formed ahead, and held
      f32x4 kf[NT], qf[NT];
      load_rows(kf, k, a.k_row, ch, p, c, g, a.key_dim);
      load_rows(qf, q, a.q_row, ch, p, c, g, a.key_dim);
      f32x4 decay;
      float beta;
      load_gates<T>(a, h, ch, p, c, g, decay, beta);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        store4(&Kl[(DL_C * i + c) * LDK + 16 * t + 4 * g], kf[t]);
        store4(&Ql[(DL_C * i + c) * LDK + 16 * t + 4 * g], qf[t]);
      }
      prepare_chunk(kf, qf, decay, beta, a.scale, c, g, Tm + i * SQ, Pm + i * SQ, Dm + i * SQ, vecs + i * DL_VEC);
    }
    // the segment's states S[0] .. S[DL_SEG] and writes n
    f32x4 S[DL_SEG + 1][NT], n[DL_SEG], vv[DL_SEG];
    const float* from = p0 ? a.marks + (mark_slot(ch, p0) * a.v_heads + h) * size : a.h0 ? a.h0 + block * size : nullptr;
    load_state(S[0], from, a, c, g, w16);
#pragma unroll
    for (int i = 0; i < DL_SEG; ++i) vv[i] = load_col(v, a.v_row, ch, p0 + DL_C * i, g, vcol, a.val_dim);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < DL_SEG; ++i) {
      if (p0 + DL_C * i < ch.count) {
        const T* Kc = Kl + DL_C * i * LDK;
        const float* vec = vecs + i * DL_VEC;
        f32x4 kf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) kf[t] = load4(Kc + c * LDK + 16 * t + 4 * g);
        const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + 4 * g), e = *reinterpret_cast<const f32x4*>(vec + 16 + 4 * g);
        const f32x4 R = beta * (vv[i] - e * dot_tiles(kf, S[i]));
        n[i] = mul16(*reinterpret_cast<const f32x4*>(Tm + i * SQ + c * DL_LD + 4 * g), R, zero);
        const f32x4 nl = *reinterpret_cast<const f32x4*>(vec + 32 + 4 * g) * n[i];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          f32x4 kt;
#pragma unroll
          for (int s = 0; s < 4; ++s) kt[s] = (float)Kc[(4 * g + s) * LDK + 16 * t + c];
          S[i + 1][t] = mul16(kt, nl, vec[48] * S[i][t]);
        }
      } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) S[i + 1][t] = zero;
        n[i] = zero;
      }
    }
#pragma unroll
    for (int i = DL_SEG - 1; i >= 0; --i) {
      const int p = p0 + DL_C * i;
      if (p >= ch.count) continue;
      asm volatile("" : "+v"(c), "+v"(g));
      const T *Kc = Kl + DL_C * i * LDK, *Qc = Ql + DL_C * i * LDK;
      const float *vec = vecs + i * DL_VEC, *Tc = Tm + i * SQ, *Pc = Pm + i * SQ, *Dc = Dm + i * SQ;
      const f32x4 beta = *reinterpret_cast<const f32x4*>(vec + 4 * g), e = *reinterpret_cast<const f32x4*>(vec + 16 + 4 * g);
      const f32x4 left = *reinterpret_cast<const f32x4*>(vec + 32 + 4 * g);
      // by columns: dn, dR, dv
      const f32x4 go = load_col(dout, a.do_row, ch, p, g, vcol, a.val_dim);
      f32x4 dn, dR, col;
      {
        f32x4 kf[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) kf[t] = load4(Kc + c * LDK + 16 * t + 4 * g);
        dn = left * dot_tiles(kf, dS);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) col[s] = Pc[(4 * g + s) * DL_LD + c];
      dn = mul16(col, go, dn);
#pragma unroll
      for (int s = 0; s < 4; ++s) col[s] = Tc[(4 * g + s) * DL_LD + c];
      dR = mul16(col, dn, zero);
      f32x4 to_beta = vv[i] * dR, to_decay = zero;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = p + 4 * g + r;
        if (at < ch.count && vcol < a.val_dim)
          ((T*)a.dv)[(ch.row(at) * a.v_heads + h) * a.val_dim + vcol] = (T)(beta[r] * dR[r]);
        Nl[(4 * g + r) * LDV + vcol] = n[i][r];
        Rl[(4 * g + r) * LDV + vcol] = dR[r];
      }
      float inner = 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          inner = __builtin_fmaf(dS[t][r], S[i + 1][t][r], inner);
          Sl[(16 * t + 4 * g + r) * LDV + vcol] = S[i][t][r];
        }
      }
      inner += __shfl_xor(inner, 16);
      inner += __shfl_xor(inner, 32);
      if (g == 3) to_decay[3] = inner;  // the chunk's last row
      __syncthreads();
      // X and Y (the first and the second wavefront, where there are two); products with S
      const bool there = p + c < ch.count;
      const T* dorow = dout + (there ? ch.row(p + c) : ch.from) * a.do_row + 4 * g;
      if (w == 0 || (w == 1 && W > 1)) {
        f32x4 x = zero, y = zero;  // rows j, column i
        for (int u = 0; u < W; ++u) {
          const f32x4 nj = *reinterpret_cast<const f32x4*>(Nl + c * LDV + 16 * u + 4 * g);
          f32x4 d = zero;
          if (w == 0) {
            if (there && 16 * u + 4 * g < a.val_dim) d = load4(dorow + 16 * u);
            x = mul16(nj, d, x);
          }
          if (w == W - 1 || w == 1) y = mul16(nj, *reinterpret_cast<const f32x4*>(Rl + c * LDV + 16 * u + 4 * g), y);
        }
        const f32x4 D = *reinterpret_cast<const f32x4*>(Dc + c * DL_LD + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = 4 * g + r <= c ? D[r] * x[r] : 0.f;
          y[r] = 4 * g + r < c ? -D[r] * y[r] : 0.f;
        }
        if (w == 0) *reinterpret_cast<f32x4*>(Xm + c * DL_LD + 4 * g) = x;
        if (w == 1 || W == 1) *reinterpret_cast<f32x4*>(Ym + c * DL_LD + 4 * g) = y;
      }
      f32x4 dq[TP], lf[TP];
#pragma unroll
      for (int j = 0; j < TP; ++j) {
        dq[j] = lf[j] = zero;
        const int t = w + j * W;
        if (t < NT) {
          for (int u = 0; u < W; ++u) {
            const f32x4 s = *reinterpret_cast<const f32x4*>(Sl + (16 * t + c) * LDV + 16 * u + 4 * g);
            f32x4 d = zero;
            if (there && 16 * u + 4 * g < a.val_dim) d = load4(dorow + 16 * u);
            dq[j] = mul16(d, s, dq[j]);
            lf[j] = mul16(*reinterpret_cast<const f32x4*>(Rl + c * LDV + 16 * u + 4 * g), s, lf[j]);
          }
        }
      }
      __syncthreads();
      // dS out, and back to the chunk's start
      const f32x4 fo = a.scale * e * go, fr = -(beta * e) * dR;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        f32x4 kt, qt;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          Sl[(16 * t + 4 * g + r) * LDV + vcol] = dS[t][r];
          kt[r] = (float)Kc[(4 * g + r) * LDK + 16 * t + c];
          qt[r] = (float)Qc[(4 * g + r) * LDK + 16 * t + c];
        }
        dS[t] = mul16(kt, fr, mul16(qt, fo, vec[48] * dS[t]));
      }
      __syncthreads();
      f32x4 xr = *reinterpret_cast<const f32x4*>(Xm + c * DL_LD + 4 * g), yr = *reinterpret_cast<const f32x4*>(Ym + c * DL_LD + 4 * g);
      f32x4 xc, yc;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        xc[s] = a.scale * Xm[(4 * g + s) * DL_LD + c];
        yc[s] = beta[s] * Ym[(4 * g + s) * DL_LD + c];
      }
#pragma unroll
      for (int j = 0; j < TP; ++j) {
        const int t = w + j * W, kcol = 16 * t + c;
        if (t < NT) {
          f32x4 kt, qt, right = zero;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            kt[s] = (float)Kc[(4 * g + s) * LDK + kcol];
            qt[s] = (float)Qc[(4 * g + s) * LDK + kcol];
          }
          for (int u = 0; u < W; ++u)
            right = mul16(*reinterpret_cast<const f32x4*>(Nl + c * LDV + 16 * u + 4 * g),
                          *reinterpret_cast<const f32x4*>(Sl + kcol * LDV + 16 * u + 4 * g), right);
          const f32x4 gq = a.scale * mul16(xr, kt, e * dq[j]);
          const f32x4 gl = mul16(yr, kt, -(e * lf[j]));
          right = mul16(yc, kt, mul16(xc, qt, left * right));
          const f32x4 gk = beta * gl + right;
          to_beta += kt * gl;
          to_decay += qt * gq + beta * (kt * gl) - kt * right;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = p + 4 * g + r;
            if (at < ch.count && kcol < a.key_dim) {
              if (shared) {
                const int64_t to = (ch.row(at) * a.v_heads + h) * a.key_dim + kcol;
                ((float*)a.workspace)[to] = gq[r];
                ((float*)a.workspace)[to + (int64_t)a.rays.n * a.v_heads * a.key_dim] = gk[r];
              } else {
                const int64_t to = (ch.row(at) * a.heads + h) * a.key_dim + kcol;
                ((T*)a.dq)[to] = (T)gq[r];
                ((T*)a.dk)[to] = (T)gk[r];
              }
            }
          }
        }
      }
      to_beta = sum16(to_beta);
      to_decay = sum16(to_decay);
      if (c == 0) {
        *reinterpret_cast<f32x4*>(sums + w * 32 + 4 * g) = to_beta;
        *reinterpret_cast<f32x4*>(sums + w * 32 + 16 + 4 * g) = to_decay;
      }
      __syncthreads();
      if (w == 0 && g == 0) {
        float db = 0.f, dd = 0.f;
        for (int u = 0; u < W; ++u) {
          db += sums[u * 32 + c];
          dd += sums[u * 32 + 16 + c];
        }
#pragma unroll
        for (int d = 1; d < DL_C; d *= 2) {
          const float x = __shfl_down(dd, d);
          dd += c + d < DL_C ? x : 0.f;
        }
        if (there) {
          const int64_t to = ch.row(p + c) * a.v_heads + h;
          ((T*)a.ddecay)[to] = (T)dd;
          ((T*)a.dbeta)[to] = (T)db;
        }
      }
    }
  }
  if (a.dh0) store_state(a.dh0 + block * size, dS, a, c, g, w16);
}

// dq and dk of key heads that value heads share, in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void k_delta_join(const ffn_ray_delta a) {
  const int64_t all = (int64_t)a.rays.n * a.heads * a.key_dim, i = block_number() * 256 + threadIdx.x;
  if (i >= 2 * all) return;
  const int64_t j = i < all ? i : i - all, row = j / ((int64_t)a.heads * a.key_dim);
  const uint32_t r = a.rays.ray_ids[row];
  if (r >= a.rays.num_rays) return;  // written as 0
  const int64_t o = a.rays.offsets[r];
  if (row < o || row - o >= (int64_t)a.rays.counts[r]) return;
  const int x = (int)(j - row * a.heads * a.key_dim), hk = x / a.key_dim, col = x - hk * a.key_dim, per = a.v_heads / a.heads;
  const float* from = (const float*)a.workspace + (i < all ? 0 : (int64_t)a.rays.n * a.v_heads * a.key_dim) +
                      (row * a.v_heads + hk * per) * a.key_dim + col;
  float s = 0.f;
  for (int u = 0; u < per; ++u) s += from[(int64_t)u * a.key_dim];
  ((T*)(i < all ? a.dq : a.dk))[j] = (T)s;
}

uint64_t delta_marks(const ffn_ray_delta& a) {
  return ((uint64_t)a.rays.n + DL_MARK - 1) / DL_MARK * a.v_heads * a.key_dim * a.val_dim * sizeof(float);
}
uint64_t delta_workspace(const ffn_ray_delta& a) {
  return a.heads == a.v_heads ? 0 : 2ull * a.rays.n * a.v_heads * a.key_dim * sizeof(float);
}

namespace {

int64_t clear_blocks(const ffn_ray_delta& a) { return ((int64_t)a.rays.n + DL_CLEAR - 1) / DL_CLEAR; }

template <typename T, int DK>
hipError_t forward(const ffn_ray_delta& a, hipStream_t st) {
  const int64_t states = (int64_t)a.rays.num_rays * a.v_heads;
  if (!a.marks && a.rays.n <= 4ull * a.rays.num_rays) {
    const int64_t teams = states * ((a.val_dim + 31) / 32);
    k_delta_step<T, DK><<<grid_of((teams + 3) / 4 + clear_blocks(a)), 256, 0, st>>>(a);
    return hipGetLastError();
  }
  const int W = (a.val_dim + 15) / 16;
  k_delta_fwd<T, DK, 4><<<grid_of(states + clear_blocks(a)), 64 * W, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T, int DK, int TP>
hipError_t start_bwd(const ffn_ray_delta& a, int W, hipStream_t st) {
  const int bytes = delta_lds(DK, W, (int)sizeof(T));
  // more than 64 KiB has to be allowed, on the device that is current
  const hipError_t e = hipFuncSetAttribute((const void*)k_delta_bwd<T, DK, TP>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return e;
  k_delta_bwd<T, DK, TP><<<grid_of((int64_t)a.rays.num_rays * a.v_heads + clear_blocks(a)), 64 * W, bytes, st>>>(a);
  return hipGetLastError();
}

template <typename T, int DK>
hipError_t backward(const ffn_ray_delta& a, hipStream_t st) {
  const int W = (a.val_dim + 15) / 16, tiles = (DK / 16 + W - 1) / W;  // tiles of dq and dk a wavefront
  hipError_t e;
  if (tiles <= 1) e = start_bwd<T, DK, 1>(a, W, st);
  else if (tiles <= 2) e = start_bwd<T, DK, 2>(a, W, st);
  else if (tiles <= 4) e = start_bwd<T, DK, (DK >= 64 ? 4 : 1)>(a, W, st);
  else e = start_bwd<T, DK, (DK >= 128 ? 8 : 1)>(a, W, st);
  if (e != hipSuccess || a.heads == a.v_heads || !a.rays.n) return e;
  k_delta_join<T><<<grid_of((2 * (int64_t)a.rays.n * a.heads * a.key_dim + 255) / 256), 256, 0, st>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t by_dim(const ffn_ray_delta& a, bool back, hipStream_t st) {
  if (a.key_dim <= 32) return back ? backward<T, 32>(a, st) : forward<T, 32>(a, st);
  if (a.key_dim <= 64) return back ? backward<T, 64>(a, st) : forward<T, 64>(a, st);
  return back ? backward<T, 128>(a, st) : forward<T, 128>(a, st);
}

}  // namespace

hipError_t launch_delta(const ffn_ray_delta& a, bool back, hipStream_t st) {
  if (!a.rays.num_rays && !a.rays.n) return hipSuccess;
  if (a.dtype == FFN_F32) return by_dim<float>(a, back, st);
  if (a.dtype == FFN_F16) return by_dim<_Float16>(a, back, st);
  return by_dim<__bf16>(a, back, st);
}

}  // namespace ffn
