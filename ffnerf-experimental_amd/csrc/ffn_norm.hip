// ffn_norm.hip -- layer norm of rows, y = (x - mean) rstd w + b, and its gradients.
//
// Memory bounds it: a row is read once and held in registers between its statistics and its result.  A row is worked on
// by a team of lanes: 1 to 64 of a wavefront, so that narrow rows fill it (64 columns of 16 bits: 8 lanes a row, 8 rows a
// wavefront), or a whole block where a row has more columns than a wavefront's registers are given.  Teams walk over the
// rows, so that a lane's parameters are loaded once and its share of their gradients stays in registers.
// Rates: 2^22 rows of 64 in bf16 255 us forward, 343 backward (4.2 and 4.7 TB/s); 20,011 rows of 4096 71 and 134 + 12 (4.6 and
// 3.7); 100,003 rows of 333 floats, which start anywhere, 64 and 83 + 7 (4.2 and 4.8).  A copy reaches 4.63.
#include <algorithm>

#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

constexpr int NM_NT = 256;
constexpr int NM_BLOCK_COLS = 16;     // a lane's columns where a block takes a row: rows of up to 16384
constexpr int NM_BLOCKS = 2048;       // of the forward: 8 blocks a CU
constexpr int NM_GRAD_BLOCKS = 1024;  // of the backward: as many partial sums of the parameters' gradients

// What a lane holds of a row: P pieces of EL neighbouring columns (16 bytes, or one column where rows are not aligned);
// piece p is at column (lane + p team) EL.
template <typename T, int EL> struct Piece {
  typedef T type __attribute__((ext_vector_type(EL)));
};
template <typename T> struct Piece<T, 1> {
  typedef T type;
};

template <typename T, int EL, int P>
struct RowPart {
  typedef typename Piece<T, EL>::type vec;
  vec v[P];
  __device__ __forceinline__ void load(const T* __restrict__ row, int lane, int team, int width) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (lane + p * team) * EL;
      v[p] = vec{};
      if (c < width) v[p] = *reinterpret_cast<const vec*>(row + c);
    }
  }
  __device__ __forceinline__ float at(int p, int e) const {
    if constexpr (EL == 1) return (float)v[p];
    else return (float)v[p][e];
  }
  __device__ __forceinline__ void set(int p, int e, float f) {
    if constexpr (EL == 1) v[p] = (T)f;
    else v[p][e] = (T)f;
  }
  __device__ __forceinline__ void store(T* __restrict__ row, int lane, int team, int width) const {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (lane + p * team) * EL;
      if (c < width) *reinterpret_cast<vec*>(row + c) = v[p];
    }
  }
};

// parameters of this lane's columns as floats, `none` where there are none
template <typename T, int EL, int P>
__device__ __forceinline__ void load_params(const void* p, bool f32, float none, int lane, int team, int width,
                                            float (&to)[P * EL]) {
  if constexpr (EL > 1) {
    if (p && !((uintptr_t)p & 15)) {  // whole pieces; rows of pieces end with one
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const int c = (lane + i * team) * EL < width ? (lane + i * team) * EL : 0;
        if (f32) {
#pragma unroll
          for (int e = 0; e < EL; e += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>((const float*)p + c + e);
#pragma unroll
            for (int q = 0; q < 4; ++q) to[i * EL + e + q] = v[q];
          }
        } else {
          const typename Piece<T, EL>::type v = *reinterpret_cast<const typename Piece<T, EL>::type*>((const T*)p + c);
#pragma unroll
          for (int e = 0; e < EL; ++e) to[i * EL + e] = (float)v[e];
        }
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < P; ++i) {
#pragma unroll
    for (int e = 0; e < EL; ++e) {
      const int c = (lane + i * team) * EL + e;
      to[i * EL + e] = !p ? none : c >= width ? 0.f : f32 ? ((const float*)p)[c] : (float)((const T*)p)[c];
    }
  }
}

// sums over a team: by exchange within a wavefront, and over the wavefronts of a block through LDS
template <int N, bool BLOCK>
__device__ __forceinline__ void team_sum(float (&s)[N], int team, float (*part)[4]) {
  for (int d = 1; d < (BLOCK ? 64 : team); d *= 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor(s[i], d);
  }
  if constexpr (BLOCK) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) part[wave][i] = s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = 0.f;
    for (int w = 0; w < waves; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] += part[w][i];
    }
  }
}

// the rows of a team: `first`, and every `step` on
struct Team {
  int lane;
  int64_t first, step;
  template <bool BLOCK> static __device__ __forceinline__ Team of(int team) {
    if (BLOCK) return {(int)threadIdx.x, (int64_t)blockIdx.x, (int64_t)gridDim.x};
    const int per = (int)blockDim.x / team;
    return {(int)threadIdx.x & (team - 1), (int64_t)blockIdx.x * per + (int)threadIdx.x / team, (int64_t)gridDim.x * per};
  }
};

// The variance is that of d = x - m about its own mean, m the first sum's quotient: d is exact where x is near m, so that
// neither m's rounding nor a large mean costs anything.
template <typename T, int EL, int P, int U, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? 1024 : NM_NT) void k_norm_fwd(const ffn_norm a, int team) {
  __shared__ float part[16][4];
  constexpr int N = P * EL;
  const Team t = Team::of<BLOCK>(team);
  const int width = a.width;
  const float inv = 1.f / (float)width;
  float w[N], b[N];
  load_params<T, EL, P>(a.weight, a.param_dtype == FFN_F32, 1.f, t.lane, team, width, w);
  load_params<T, EL, P>(a.bias, a.param_dtype == FFN_F32, 0.f, t.lane, team, width, b);
  // all lanes of a wavefront make the same trips (the exchanges need them), those past the last row without effect
  const int64_t trips = (a.n + t.step * U - 1) / (t.step * U);
  for (int64_t k = 0; k < trips; ++k) {
    RowPart<T, EL, P> x[U];
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      row[u] = t.first + (k * U + u) * t.step;
      x[u].load((const T*)a.x + min(row[u], (int64_t)a.n - 1) * a.x_row, t.lane, team, width);
    }
    float m[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) m[u] += x[u].at(i / EL, i % EL);
    }
    team_sum<U, BLOCK>(m, team, part);
    float s[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] *= inv;
      s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int c = (t.lane + i / EL * team) * EL;
        const float d = c < width ? x[u].at(i / EL, i % EL) - m[u] : 0.f;
        s[2 * u] += d;
        s[2 * u + 1] = __builtin_fmaf(d, d, s[2 * u + 1]);
      }
    }
    team_sum<2 * U, BLOCK>(s, team, part);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float off = s[2 * u] * inv;
      const float var = __builtin_fmaf(-off, off, s[2 * u + 1] * inv);
      const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + a.eps);  // a NaN stays one
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = (x[u].at(i / EL, i % EL) - m[u]) - off;
        x[u].set(i / EL, i % EL, __builtin_fmaf(d * rstd, w[i], b[i]));
      }
      if (row[u] < (int64_t)a.n) {
        x[u].store((T*)a.y + row[u] * width, t.lane, team, width);
        if (t.lane == 0) {
          a.mean[row[u]] = m[u] + off;
          a.rstd[row[u]] = rstd;
        }
      }
    }
  }
}

// g = dy w, xhat = (x - mean) rstd:  dx = rstd (g - mean(g) - xhat mean(g xhat)), dw = sum of dy xhat, db = sum of dy.
// The saved mean is rounded: what the row's x - mean still has as its mean is taken off as well.
// BT: threads of a block that takes a row, 0 where a wavefront's team does.  Blocks of 1024 leave a lane 128 registers: the
// next row then waits for the last one, and the weights are read again for every row.
template <typename T, int EL, int P, int BT>
__global__ __launch_bounds__(BT ? BT : NM_NT) void k_norm_bwd(const ffn_norm a, int team) {
  __shared__ float part[16][4];
  constexpr int N = P * EL;
  constexpr bool BLOCK = BT > 0, AHEAD = BT < 1024;
  const Team t = Team::of<BLOCK>(team);
  const int width = a.width;
  const float inv = 1.f / (float)width;
  float w[N], dw[N], db[N];
  load_params<T, EL, P>(a.weight, a.param_dtype == FFN_F32, 1.f, t.lane, team, width, w);
#pragma unroll
  for (int i = 0; i < N; ++i) dw[i] = db[i] = 0.f;
  const int64_t trips = (a.n + t.step - 1) / t.step;
  RowPart<T, EL, P> nx, ny;
  float nmean, nrstd;
  const auto fetch = [&](int64_t r) {
    const int64_t at = min(r, (int64_t)a.n - 1);
    nx.load((const T*)a.x + at * a.x_row, t.lane, team, width);
    ny.load((const T*)a.dy + at * a.dy_row, t.lane, team, width);
    nmean = a.mean[at];
    nrstd = a.rstd[at];
  };
  if (AHEAD && trips) fetch(t.first);
  for (int64_t k = 0; k < trips; ++k) {
    const int64_t row = t.first + k * t.step;
    if (!AHEAD) {
      fetch(row);
      load_params<T, EL, P>(a.weight, a.param_dtype == FFN_F32, 1.f, t.lane, team, width, w);
    }
    RowPart<T, EL, P> x = nx;
    const RowPart<T, EL, P> y = ny;
    const float mean = nmean, rstd = nrstd;
    if (AHEAD && k + 1 < trips) fetch(row + t.step);
    float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t.lane + i / EL * team) * EL;
      const float d = c < width ? x.at(i / EL, i % EL) - mean : 0.f;
      const float g = y.at(i / EL, i % EL) * w[i];
      s[0] += d;
      s[1] += g;
      s[2] = __builtin_fmaf(g, d, s[2]);
    }
    team_sum<3, BLOCK>(s, team, part);
    const float off = s[0] * inv, mg = s[1] * inv;
    const float mgx = (s[2] - off * s[1]) * inv * rstd;  // mean of g xhat
    const bool there = row < (int64_t)a.n;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float dy = y.at(i / EL, i % EL);
      const float xhat = ((x.at(i / EL, i % EL) - mean) - off) * rstd;
      x.set(i / EL, i % EL, rstd * (__builtin_fmaf(dy, w[i], -mg) - xhat * mgx));
      dw[i] = there ? __builtin_fmaf(dy, xhat, dw[i]) : dw[i];
      db[i] = there ? db[i] + dy : db[i];
    }
    if (there && a.dx) x.store((T*)a.dx + row * width, t.lane, team, width);
  }
  if (!a.workspace) return;
  // the block's sums, in a fixed order: teams of a wavefront by exchange, then the wavefronts one after the other
  float* out = (float*)a.workspace + (int64_t)blockIdx.x * 2 * width;
  if constexpr (BLOCK) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = (t.lane + i / EL * team) * EL + i % EL;
      if (c < width) out[c] = dw[i], out[width + c] = db[i];
    }
  } else {
    __shared__ float sums[NM_NT / 64][64 * N];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = team; d < 64; d *= 2) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dw[i] += __shfl_xor(dw[i], d);
        db[i] += __shfl_xor(db[i], d);
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
      if (lane < team) {
#pragma unroll
        for (int i = 0; i < N; ++i) sums[wave][i * team + lane] = half ? db[i] : dw[i];
      }
      __syncthreads();
      for (int j = threadIdx.x; j < N * team; j += NM_NT) {
        const int i = j / team, l = j % team, c = (l + i / EL * team) * EL + i % EL;
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < NM_NT / 64; ++v) s += sums[v][j];
        if (c < width) out[half * width + c] = s;
      }
    }
  }
}

// dw and db from the blocks' sums: 16 threads a column, each every 16th block, joined in a fixed order
__global__ __launch_bounds__(NM_NT) void k_norm_join(const float* __restrict__ part, int blocks, int width, float* dw, float* db) {
  __shared__ float sums[16][17];
  const int col = threadIdx.x & 15, from = threadIdx.x >> 4, c = blockIdx.x * 16 + col;
  float s = 0.f;
  if (c < 2 * width) {
    for (int b = from; b < blocks; b += 128) {
      float x[8];  // on their way at once
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = b + 16 * i < blocks ? part[(int64_t)(b + 16 * i) * 2 * width + c] : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += x[i];
    }
  }
  sums[from][col] = s;
  __syncthreads();
  if (from || c >= 2 * width) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sums[i][col];
  float* to = c < width ? dw : db;
  if (to) to[c < width ? c : c - width] = s;
}

namespace {

struct Shape {
  bool vec, block;
  int pieces, team, threads;
};

bool fits(const void* p, int64_t row, int64_t n, int size) { return !((uintptr_t)p & 15) && (n < 2 || row * size % 16 == 0); }

// A piece is 16 bytes where every row allows it.  The fewest pieces a lane that a wavefront covers the row with, up to
// four (16 columns a lane where pieces are columns); then blocks of 4 to 16 wavefronts with 16 columns a lane.  Blocks of 16,
// past 8192 columns, have 128 registers a lane, and the backward's parameters and their sums do not fit into them (6 to 79
// are spilled); nor do two rows of single columns in the forward, whose blocks of any size are held to that (2 to 6).
Shape shape_of(const ffn_norm& a, bool backward) {
  const int size = a.dtype == FFN_F32 ? 4 : 2, el = 16 / size;
  Shape s;
  s.vec = a.width % el == 0 && fits(a.x, a.x_row, a.n, size) &&
          (backward ? fits(a.dy, a.dy_row, a.n, size) && fits(a.dx, 0, 0, size) : fits(a.y, 0, 0, size));
  const int e = s.vec ? el : 1, first = s.vec ? 1 : 4, most = s.vec ? 4 : 16;
  const int pieces = (a.width + e - 1) / e;
  s.pieces = first;
  while (s.pieces < most && pieces > 64 * s.pieces) s.pieces *= 2;
  s.block = pieces > 64 * s.pieces;
  s.threads = NM_NT;
  if (s.block) {
    s.pieces = NM_BLOCK_COLS / e;
    while (s.threads < 1024 && pieces > s.threads * s.pieces) s.threads *= 2;
    s.team = s.threads;
  } else {
    s.team = 1;
    while (s.team * s.pieces < pieces) s.team *= 2;
  }
  return s;
}

int grad_blocks(const ffn_norm& a, const Shape& s) {
  const int64_t rows = s.block ? 1 : s.threads / s.team;
  return (int)std::min<int64_t>(NM_GRAD_BLOCKS, (a.n + rows - 1) / rows);
}

template <typename T, int EL, int P>
void start(const ffn_norm& a, bool backward, const Shape& s, hipStream_t st) {
  const int64_t rows = s.block ? 1 : s.threads / s.team;
  const dim3 grid(backward ? grad_blocks(a, s) : (int)std::min<int64_t>(NM_BLOCKS, (a.n + rows - 1) / rows));
  if (s.block) {
    if constexpr (P * EL == NM_BLOCK_COLS) {
      if (backward && s.threads <= 512) k_norm_bwd<T, EL, P, 512><<<grid, s.threads, 0, st>>>(a, s.team);
      else if (backward) k_norm_bwd<T, EL, P, 1024><<<grid, s.threads, 0, st>>>(a, s.team);
      else k_norm_fwd<T, EL, P, 2, true><<<grid, s.threads, 0, st>>>(a, s.team);
    }
  } else if (backward) {
    k_norm_bwd<T, EL, P, 0><<<grid, s.threads, 0, st>>>(a, s.team);
  } else {
    // short parts take several rows at once, so that a lane has 64 bytes on their way
    constexpr int U = P * EL * sizeof(T) >= 64 ? 1 : P * EL * sizeof(T) >= 32 ? 2 : 4;
    k_norm_fwd<T, EL, P, U, false><<<grid, s.threads, 0, st>>>(a, s.team);
  }
}

template <typename T>
void choose(const ffn_norm& a, bool backward, const Shape& s, hipStream_t st) {
  constexpr int EL = 16 / (int)sizeof(T);
  if (s.vec) {
    if (s.pieces == 1) start<T, EL, 1>(a, backward, s, st);
    else if (s.pieces == 2) start<T, EL, 2>(a, backward, s, st);
    else start<T, EL, 4>(a, backward, s, st);
  } else {
    if (s.pieces == 4) start<T, 1, 4>(a, backward, s, st);
    else if (s.pieces == 8) start<T, 1, 8>(a, backward, s, st);
    else start<T, 1, 16>(a, backward, s, st);
  }
}

}  // namespace

// enough for any alignment of the buffers, so that it may be asked for before they are there
uint64_t norm_workspace(const ffn_norm& a) { return a.n ? (uint64_t)NM_GRAD_BLOCKS * 2 * a.width * sizeof(float) : 0; }

hipError_t launch_norm(const ffn_norm& a, bool backward, hipStream_t st) {
  const Shape s = shape_of(a, backward);
  ffn_norm b = a;
  const bool params = backward && (a.dweight || a.dbias);
  if (!params) b.workspace = nullptr;
  if (a.n && (!backward || a.dx || params)) {
    if (a.dtype == FFN_F32) choose<float>(b, backward, s, st);
    else if (a.dtype == FFN_F16) choose<_Float16>(b, backward, s, st);
    else choose<__bf16>(b, backward, s, st);
  }
  if (params)
    k_norm_join<<<(2 * a.width + 15) / 16, NM_NT, 0, st>>>((const float*)a.workspace, a.n ? grad_blocks(a, s) : 0, a.width,
                                                           a.dweight, a.dbias);
  return hipGetLastError();
}

}  // namespace ffn
