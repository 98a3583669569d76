// ffn_experts.hip -- layers of experts on ragged groups of rows: the grouping, the product, its gradients.
#include "ffn_ray_common.h"
#include "ffn_ray_kernels.h"

namespace ffn {

// ---------------------------------------------------------------------------
// The grouping: a stable counting sort of row indices by expert.  Counts per block of 2048 rows, a scan per expert over
// the blocks, and a move in which a row's place comes from ballots over the lanes that hold equal ids, so the order
// depends on the ids alone.

constexpr int PL_NT = 256, PL_ITEMS = 8, PL_BLOCK = PL_NT * PL_ITEMS, PL_BINS = FFN_MAX_EXPERTS + 1;
constexpr int EX_ROWS = 128;  // slots of a product tile

// where the parts of a plan are, in words
struct PlanView {
  int bins;  // experts + 1: the last bin is that of the rows of no expert
  uint32_t n;
  uint64_t counts, offsets, rows, tiles, n_tiles, words;
};
__host__ __device__ inline PlanView plan_view(uint32_t n, int experts) {
  PlanView v;
  v.bins = experts + 1;
  v.n = n;
  v.counts = 0;
  v.offsets = v.bins;
  v.tiles = 2 * (uint64_t)v.bins;
  v.n_tiles = ((uint64_t)n + EX_ROWS - 1) / EX_ROWS + v.bins;
  v.rows = v.tiles + 2 * v.n_tiles;
  v.words = v.rows + n;
  return v;
}

__device__ __forceinline__ uint32_t bin_of(const int32_t* ids, int64_t i, int bins) {
  return min((uint32_t)ids[i], (uint32_t)(bins - 1));
}

__global__ __launch_bounds__(PL_NT) void k_plan_count(const int32_t* __restrict__ ids, PlanView v,
                                                      uint32_t* __restrict__ block_counts) {
  __shared__ uint32_t cnt[PL_BINS];
  for (int b = threadIdx.x; b < v.bins; b += PL_NT) cnt[b] = 0u;
  __syncthreads();
  const int64_t b0 = (int64_t)blockIdx.x * PL_BLOCK;
#pragma unroll
  for (int q = 0; q < PL_ITEMS; ++q) {
    const int64_t i = b0 + q * PL_NT + threadIdx.x;
    if (i < v.n) atomicAdd(&cnt[bin_of(ids, i, v.bins)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < v.bins; b += PL_NT) block_counts[(int64_t)b * gridDim.x + blockIdx.x] = cnt[b];
}

// inclusive sum over a wavefront
__device__ __forceinline__ uint32_t wave_scan(uint32_t x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// one wavefront a bin: exclusive sums over the blocks in place, the total to the plan's counts
__global__ __launch_bounds__(64) void k_plan_scan(uint32_t* __restrict__ block_counts, int blocks,
                                                  uint32_t* __restrict__ plan, PlanView v) {
  const int lane = threadIdx.x;
  uint32_t* c = block_counts + (int64_t)blockIdx.x * blocks;
  constexpr int PER = 8;
  uint32_t sum = 0u;
  for (int b0 = 0; b0 < blocks; b0 += 64 * PER) {
    uint32_t x[PER], mine = 0u;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int b = b0 + lane * PER + q;
      x[q] = b < blocks ? c[b] : 0u;
      mine += x[q];
    }
    const uint32_t s = wave_scan(mine, lane);
    uint32_t at = sum + s - mine;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int b = b0 + lane * PER + q;
      if (b < blocks) c[b] = at;
      at += x[q];
    }
    sum += __shfl(s, 63);
  }
  if (lane == 0) plan[v.counts + blockIdx.x] = sum;
}

// out[b] = sum of f(in[a]) over a < b, for all bins and (out[bins]) the total; in may be global, out is in LDS
template <int NT, typename F>
__device__ __forceinline__ void bin_scan(const uint32_t* in, int bins, uint32_t* out, uint32_t* part, F f) {
  constexpr int PER = (PL_BINS + NT - 1) / NT;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t x[PER], sum = 0u;
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int b = tid * PER + q;
    x[q] = b < bins ? f(in[b]) : 0u;
    sum += x[q];
  }
  const uint32_t s = wave_scan(sum, lane);
  if (lane == 63) part[wave] = s;
  __syncthreads();
  uint32_t at = s - sum;
  for (int w = 0; w < wave; ++w) at += part[w];
#pragma unroll
  for (int q = 0; q < PER; ++q) {
    const int b = tid * PER + q;
    if (b < bins) out[b] = at;
    at += x[q];
    if (b == bins - 1) out[bins] = at;
  }
  __syncthreads();
}

// entries {bin, index of the piece among its bin's} of a table of pieces, of which bin b has first[b + 1] - first[b]
template <int NT>
__device__ __forceinline__ void fill_table(uint2* table, uint64_t n, uint64_t from, uint64_t count, const uint32_t* first,
                                           int bins) {
  for (uint64_t t = from + threadIdx.x; t < from + count && t < n; t += NT) {
    uint2 e = make_uint2(0xFFFFFFFFu, 0u);
    if (t < first[bins]) {
      int lo = 0, hi = bins - 1;  // the last bin whose first piece is not past t
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      e = make_uint2((uint32_t)lo, (uint32_t)(t - first[lo]));
    }
    table[t] = e;
  }
}

// The bins of this wavefront's rows w0 + 64 q + lane, and how many rows of the same bin the wavefront has before each.
// cnt: the wavefront's counts so far, 0 at first.
template <int ITEMS>
__device__ __forceinline__ void rank_rows(const int32_t* __restrict__ ids, const PlanView& v, int64_t w0, int bits,
                                          uint32_t* cnt, uint32_t (&bin)[ITEMS], uint32_t (&rank)[ITEMS]) {
  const int lane = threadIdx.x & 63;
  const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const int64_t i = w0 + q * 64 + lane;
    bin[q] = i < v.n ? bin_of(ids, i, v.bins) : 0u;
  }
#pragma unroll
  for (int q = 0; q < ITEMS; ++q) {
    const bool there = w0 + q * 64 + lane < v.n;
    uint64_t same = __ballot(there);
    for (int b = 0; b < bits; ++b) {
      const uint64_t m = __ballot((bin[q] >> b) & 1u);
      same &= ((bin[q] >> b) & 1u) ? m : ~m;
    }
    const uint32_t before = cnt[bin[q]];
    rank[q] = before + (uint32_t)__popcll(same & below);
    wave_sync();
    if (there && (same & below) == 0ull) cnt[bin[q]] = before + (uint32_t)__popcll(same);
    wave_sync();
  }
}

// Few rows: the whole plan by one block, in one launch, us, one / three launches: 2048 rows with 8 experts 9.1 / 11.0, with 256
// 12.1 / 13.3; 8192 rows 11.4 / 11.4 and 15.8 / 14.0, where three still cost the host more.
constexpr int PS_NT = 1024, PS_ITEMS = 8, PS_ROWS = PS_NT * PS_ITEMS;
__global__ __launch_bounds__(PS_NT) void k_plan_small(const int32_t* __restrict__ ids, PlanView v, int bits,
                                                      uint32_t* __restrict__ plan) {
  constexpr int NW = PS_NT / 64;
  __shared__ uint32_t first[PL_BINS + 1], total[PL_BINS], part[NW], cnt[NW][PL_BINS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int b = lane; b < v.bins; b += 64) cnt[wave][b] = 0u;
  wave_sync();
  const int64_t w0 = (int64_t)wave * (PS_ROWS / NW);
  uint32_t bin[PS_ITEMS], rank[PS_ITEMS];
  rank_rows<PS_ITEMS>(ids, v, w0, bits, cnt[wave], bin, rank);
  __syncthreads();
  for (int b = tid; b < v.bins; b += PS_NT) {
    uint32_t sum = 0u;
    for (int w = 0; w < NW; ++w) {
      const uint32_t c = cnt[w][b];
      cnt[w][b] = sum;
      sum += c;
    }
    total[b] = sum;
    plan[v.counts + b] = sum;
  }
  __syncthreads();
  bin_scan<PS_NT>(total, v.bins, first, part, [](uint32_t c) { return c; });
  for (int b = tid; b < v.bins; b += PS_NT) plan[v.offsets + b] = first[b];
#pragma unroll
  for (int q = 0; q < PS_ITEMS; ++q) {
    const int64_t i = w0 + q * 64 + lane;
    if (i < v.n) plan[v.rows + first[bin[q]] + cnt[wave][bin[q]] + rank[q]] = (uint32_t)i;
  }
  __syncthreads();
  bin_scan<PS_NT>(total, v.bins, first, part, [](uint32_t c) { return (c + EX_ROWS - 1) / EX_ROWS; });
  fill_table<PS_NT>((uint2*)(plan + v.tiles), v.n_tiles, 0, v.n_tiles, first, v.bins);
}

__global__ __launch_bounds__(PL_NT) void k_plan_move(const int32_t* __restrict__ ids, PlanView v, int bits, int blocks,
                                                     const uint32_t* __restrict__ block_counts,
                                                     uint32_t* __restrict__ plan) {
  constexpr int NW = PL_NT / 64;
  __shared__ uint32_t first[PL_BINS + 1], part[NW], cnt[NW][PL_BINS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t* counts = plan + v.counts;
  if ((int)blockIdx.x >= blocks) {
    bin_scan<PL_NT>(counts, v.bins, first, part, [](uint32_t c) { return (c + EX_ROWS - 1) / EX_ROWS; });
    fill_table<PL_NT>((uint2*)(plan + v.tiles), v.n_tiles, (uint64_t)(blockIdx.x - blocks) * PL_BLOCK, PL_BLOCK, first, v.bins);
    return;
  }
  bin_scan<PL_NT>(counts, v.bins, first, part, [](uint32_t c) { return c; });
  if (blockIdx.x == 0)
    for (int b = tid; b < v.bins; b += PL_NT) plan[v.offsets + b] = first[b];
  for (int b = tid; b < NW * PL_BINS; b += PL_NT) (&cnt[0][0])[b] = 0u;
  __syncthreads();
  // wavefront w holds rows [w PL_BLOCK / NW, ...) of the block, 64 consecutive ones per trip
  const int64_t w0 = (int64_t)blockIdx.x * PL_BLOCK + (int64_t)wave * (PL_BLOCK / NW);
  uint32_t bin[PL_ITEMS], rank[PL_ITEMS];
  rank_rows<PL_ITEMS>(ids, v, w0, bits, cnt[wave], bin, rank);
  __syncthreads();
  for (int b = tid; b < v.bins; b += PL_NT) {
    uint32_t at = first[b] + block_counts[(int64_t)b * blocks + blockIdx.x];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const uint32_t c = cnt[w][b];
      cnt[w][b] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < PL_ITEMS; ++q) {
    const int64_t i = w0 + q * 64 + lane;
    if (i < v.n) plan[v.rows + cnt[wave][bin[q]] + rank[q]] = (uint32_t)i;
  }
}

static int plan_blocks(uint32_t n) { return (int)(((uint64_t)n + PL_BLOCK - 1) / PL_BLOCK); }

uint64_t expert_plan_words(uint32_t n, int experts) { return plan_view(n, experts).words; }
uint64_t expert_plan_workspace(uint32_t n, int experts) {
  return n <= PS_ROWS ? 0 : (uint64_t)plan_blocks(n) * (experts + 1) * sizeof(uint32_t);
}

hipError_t launch_expert_plan(const int32_t* ids, uint32_t n, int experts, uint32_t* plan, uint32_t* workspace,
                              hipStream_t st) {
  const PlanView v = plan_view(n, experts);
  const int blocks = plan_blocks(n);
  int bits = 1;
  while ((1 << bits) < v.bins) ++bits;
  if (n <= PS_ROWS) {
    k_plan_small<<<1, PS_NT, 0, st>>>(ids, v, bits, plan);
    return hipGetLastError();
  }
  k_plan_count<<<blocks, PL_NT, 0, st>>>(ids, v, workspace);
  k_plan_scan<<<v.bins, 64, 0, st>>>(workspace, blocks, plan, v);
  const int tile_blocks = (int)((v.n_tiles + PL_BLOCK - 1) / PL_BLOCK);
  k_plan_move<<<blocks + tile_blocks, PL_NT, 0, st>>>(ids, v, bits, blocks, workspace, plan);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// The products.

constexpr int EX_NT = 256, EX_K = 64;  // the products' sums go in steps of 64

// One step's part of W_e on its way to LDS: R x C values from [r0][c0], 0 past the matrix.  PERM: row m = 8 g + j of each
// 32 goes where col_frag reads slot j of lane group g, so that the K order is that of the other operand's 16-byte loads.
template <typename T, int R, int C, bool PERM>
struct StageW {
  static constexpr int EL = 16 / (int)sizeof(T), CPR = C / EL, N = R * CPR / EX_NT;
  uint4 v[N];
  __device__ __forceinline__ void load(const T* __restrict__ W, int rows, int cols, int r0, int c0) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = threadIdx.x + i * EX_NT, row = r0 + c / CPR, col = c0 + (c % CPR) * EL;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < rows && col < cols) v[i] = *reinterpret_cast<const uint4*>(W + (int64_t)row * cols + col);
    }
  }
  __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = threadIdx.x + i * EX_NT, row = c / CPR;
      int to = row;
      if (PERM) {
        const int g = (row & 31) >> 3, j = row & 7;
        to = (row & ~31) + (j < 4 ? 4 * g + j : 16 + 4 * g + j - 4);
      }
      *reinterpret_cast<uint4*>(tile + to * lds_row<T, C> + (c % CPR) * EL) = v[i];
    }
  }
};

// Keeps the values of g whose y is positive (16 bytes or a fragment of either type).  In 16 bits, two at a time on the
// bits: y - 1 is below infinity's bits exactly where y is positive and no NaN; the saturating sum puts that into the sign.
template <typename T, typename V>
__device__ __forceinline__ V where_positive(V g, V y) {
  constexpr int N = sizeof(V) / 4;
  typedef uint32_t words __attribute__((ext_vector_type(N)));
  words a = __builtin_bit_cast(words, g);
  const words b = __builtin_bit_cast(words, y);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = __uint_as_float(b[i]) > 0.f ? a[i] : 0u;
  } else {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    constexpr unsigned short up = 0x8000 - (__is_same(T, __bf16) ? 0x7F80 : 0x7C00);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t word = b[i];
      const u16x2 below = __builtin_bit_cast(u16x2, word) - (u16x2){1, 1};
      const u16x2 sign = __builtin_elementwise_add_sat(below, (u16x2){up, up});
      a[i] &= ~__builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, sign) >> (i16x2){15, 15});
    }
  }
  return __builtin_bit_cast(V, a);
}

// row r of a tensor whose rows are `stride` bytes apart
template <typename T>
__device__ __forceinline__ const T* row_at(const T* base, uint32_t r, uint32_t stride) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + (uint64_t)r * stride);
}

// Wavefronts a SIMD that the products' registers are held to (dx of a million rows of 128 x 128 values in bf16: 147 us with
// two, 131 with three)
constexpr int ex_waves(int size, int nb) { return size == 4 || nb == 16 ? 2 : nb == 8 ? 3 : 4; }

// BACK = false: y = act(x W_e^T + b_e);  true: dx = (dy where y > 0) W_e.  128 slots by 16 NB columns a block, 32 slots a
// wavefront.  The product is formed transposed (slots along the lanes), so that a lane's rows come by 16-byte loads
// straight into the operand; W_e goes through LDS.  Results turn in LDS, so that rows go out whole: stored from the
// product's own layout (8 bytes a lane, 32 in a row) a write-bound layer takes nearly twice as long.  Bound by memory, and by
// its latency where W is wide: two million rows of 64 x 64 values in bf16 140 us (3.9 TB/s), dx of 500009 rows of 256 x 256
// values 193 us (4.0 TB/s).
template <typename T, bool BACK, int NB>
__global__ __launch_bounds__(EX_NT, ex_waves(sizeof(T), NB)) void k_expert(ffn_experts a, PlanView v, int64_t total, int col_tiles) {
  typedef typename Mat<T>::frag frag;
  constexpr int C = 16 * NB, EL = 16 / (int)sizeof(T);
  constexpr int W_SIZE = BACK ? EX_K * lds_row<T, C> : C * lds_row<T, EX_K>, OUT_SIZE = 4 * 16 * lds_row<T, C>;
  __shared__ __align__(16) T lds[W_SIZE > OUT_SIZE ? W_SIZE : OUT_SIZE];
  const int64_t block = block_number(), per = (total + 7) / 8, work = (block & 7) * per + (block >> 3);
  if (block >= 8 * per || work >= total) return;
  const uint2 tile = reinterpret_cast<const uint2*>(a.plan + v.tiles)[work / col_tiles];
  if (tile.x >= (uint32_t)v.bins) return;
  const int col0 = (int)(work % col_tiles) * C;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
  const uint32_t off = a.plan[v.offsets + tile.x], first = off + tile.y * EX_ROWS, end = off + a.plan[v.counts + tile.x];
  const bool none = tile.x == (uint32_t)v.bins - 1;
  const int depth = BACK ? a.out : a.in, width = BACK ? a.in : a.out;
  const bool in_slots = a.flags & (BACK ? FFN_EXPERTS_Y_SLOTS : FFN_EXPERTS_X_SLOTS);
  const bool out_slots = a.flags & (BACK ? FFN_EXPERTS_X_SLOTS : FFN_EXPERTS_Y_SLOTS);
  uint32_t slot[2], row[2];
  bool there[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    slot[s] = first + wave * 32 + s * 16 + c;
    there[s] = slot[s] < end;
    row[s] = there[s] ? a.plan[v.rows + slot[s]] : 0u;
  }
  f32x4 acc[NB][2];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b][0] = acc[b][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (!none) {
    const T* W = (const T*)a.W + (int64_t)tile.x * a.out * a.in;
    StageW<T, BACK ? EX_K : C, BACK ? C : EX_K, BACK> w;
    uint32_t r[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) r[s] = in_slots && there[s] ? slot[s] : row[s];
    const T* in = (const T*)(BACK ? a.dy : a.x) + 8 * g;
    const T* gate = (const T*)a.y + 8 * g;
    const uint32_t in_step = (uint32_t)(BACK ? a.dy_row : a.x_row) * sizeof(T), gate_step = (uint32_t)a.out * sizeof(T);
    // The rows of the next step as they are, without predicates (rows past the end are row 0, their results are not stored;
    // past the last column, the last ones again), so that nothing waits for them here.
    frag f[2][2], y[2][2];
    const bool gated = BACK && a.relu;
    auto fetch = [&](int k0) {
      if (BACK) w.load(W, a.out, a.in, k0, col0);
      else w.load(W, a.out, a.in, col0, k0);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        asm("" : "+v"(r[s]));  // the addresses are formed again each time: registers are what is short
        const T* row_in = row_at(in, r[s], in_step);
        const T* row_gate = row_at(gate, r[s], gate_step);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
          if (k0 + 32 * ks < depth) {
            const int k = min(k0 + 32 * ks, depth - 8 - 8 * g);
            f[s][ks] = *reinterpret_cast<const frag*>(row_in + k);
            if (gated) y[s][ks] = *reinterpret_cast<const frag*>(row_gate + k);
          }
      }
    };
    fetch(0);
    for (int k0 = 0; k0 < depth; k0 += EX_K) {
      w.store(lds);
      frag x[2][2];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          x[s][ks] = f[s][ks];
          if (gated) x[s][ks] = where_positive<T>(x[s][ks], y[s][ks]);
          if (depth - k0 < EX_K && k0 + 32 * ks + 8 * g >= depth) x[s][ks] = frag{};
        }
      __syncthreads();
      if (k0 + EX_K < depth) fetch(k0 + EX_K);
      auto half = [&](int ks) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const frag m = BACK ? col_frag<T, C>(lds, 32 * ks, 16 * b, lane) : row_frag<T, EX_K>(lds, 16 * b + c, ks, lane);
#pragma unroll
          for (int s = 0; s < 2; ++s) acc[b][s] = Mat<T>::mma(m, x[s][ks], acc[b][s]);
        }
      };
      half(0);
      if (depth - k0 > 32) half(1);
      __syncthreads();
    }
  }
  // 16 rows of the wavefront at a time; no other wavefront touches its part of the LDS
  T* turn = lds + wave * 16 * lds_row<T, C>;
  const int cols = min(width - col0, C);
  T* out = (BACK ? (T*)a.dx : (T*)a.y) + col0;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int col = 16 * b + 4 * g;
      f32x4 bias = f32x4{0.f, 0.f, 0.f, 0.f};
      if (!BACK && a.b && !none && col < cols)
        bias = __builtin_convertvector(*reinterpret_cast<const typename Mat<T>::quad*>((const T*)a.b + (int64_t)tile.x * a.out + col0 + col), f32x4);
      typename Mat<T>::quad q;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float val = acc[b][s][r] + bias[r];
        if (!BACK && a.relu) val = val < 0.f ? 0.f : val;  // a NaN stays one
        q[r] = (T)val;
      }
      *reinterpret_cast<typename Mat<T>::quad*>(turn + c * lds_row<T, C> + col) = q;
    }
    wave_sync();
    const uint32_t to = out_slots ? slot[s] : row[s];
#pragma unroll
    for (int i = 0; i < 16 * C / EL / 64; ++i) {
      const int at = i * 64 + lane, r = at / (C / EL), col = at % (C / EL) * EL;
      const uint32_t dest = __shfl(to, r);  // of lane r: row r of the 16
      const bool live = first + wave * 32 + s * 16 + r < end;
      if (live && col < cols)
        *reinterpret_cast<uint4*>(out + (int64_t)dest * width + col) = *reinterpret_cast<const uint4*>(turn + r * lds_row<T, C> + col);
    }
    wave_sync();
  }
}

// Shares of the weight gradient: `groups` runs of `len` slots, whatever experts they hold, so that all blocks have the same
// work.  The part of run j and expert e has index j + e: parts follow each other with j, e or both one up.
// (Equal pieces of each expert, eight to a block: 255 us instead of 204 for 500009 rows of 24 uneven experts.)
struct Shares {
  uint32_t groups, len;
};

// Sums over runs of an expert's slots of g^T x, g = dy where y > 0: TM x TK values a block in four wavefronts.  The slots
// are the K of the product, so both operands are columns of their LDS tiles.  g against ones gives db's share.  500009 rows of
// 256 x 256 values: 205 us (3.7 TB/s of each input read once; 320 TFLOP/s), bound by the wait of each step for its rows.
template <typename T, int TM, int TK>
__global__ __launch_bounds__(EX_NT) void k_expert_dw(ffn_experts a, PlanView v, int64_t total, int m_tiles, int k_tiles,
                                                     Shares shares) {
  typedef typename Mat<T>::frag frag;
  constexpr int EL = 16 / (int)sizeof(T), S = 64;  // slots of a step
  constexpr int GC = TM / EL, XC = TK / EL, NG = S * GC / EX_NT, NX = S * XC / EX_NT, NM = TM / 32, NK = TK / 32;
  __shared__ __align__(16) T gs[S * lds_row<T, TM>];
  __shared__ __align__(16) T xs[S * lds_row<T, TK>];
  const int64_t per = (total + 7) / 8, work = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (work >= total) return;
  const uint32_t run = (uint32_t)(work / (m_tiles * k_tiles));
  const int k0 = (int)(work % k_tiles) * TK, m0 = (int)(work / k_tiles % m_tiles) * TM;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, c = lane & 15;
  const int mw = (wave >> 1) * (TM / 2), kw = (wave & 1) * (TK / 2);
  const uint32_t* offsets = a.plan + v.offsets;  // the last bin's: the end of the experts' slots
  const int experts = v.bins - 1;
  uint32_t from = run * shares.len, to = 0;
  const uint32_t end = min(from + shares.len, offsets[experts]);
  if (from >= end) return;
  int e = -1;  // to the expert that holds `from`: the last one that does not begin past it
  for (int b = 0; b < experts; b += 64)
    e += (int)__popcll(__ballot(b + lane < experts && offsets[min(b + lane, experts)] <= from));
  uint4 gv[NG], yv[NG], xv[NX];
  const bool x_slots = a.flags & FFN_EXPERTS_X_SLOTS, y_slots = a.flags & FFN_EXPERTS_Y_SLOTS;
  uint32_t gr[NG], xr[NX];  // the rows of the next step
  auto rows = [&](uint32_t s0) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const uint32_t slot = min(s0 + (tid + i * EX_NT) / GC, to - 1);
      gr[i] = y_slots ? slot : a.plan[v.rows + slot];
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const uint32_t slot = min(s0 + (tid + i * EX_NT) / XC, to - 1);
      xr[i] = x_slots ? slot : a.plan[v.rows + slot];
    }
  };
  // this thread's columns; past the matrix, the last ones again (what comes of them is not stored)
  const T* gp = (const T*)a.dy + min(m0 + tid % GC * EL, a.out - EL);
  const T* yp = (const T*)a.y + min(m0 + tid % GC * EL, a.out - EL);
  const T* xp = (const T*)a.x + min(k0 + tid % XC * EL, a.in - EL);
  const uint32_t g_step = (uint32_t)a.dy_row * sizeof(T), y_step = (uint32_t)a.out * sizeof(T), x_step = (uint32_t)a.x_row * sizeof(T);
  auto fetch = [&](uint32_t s0) {
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      gv[i] = *reinterpret_cast<const uint4*>(row_at(gp, gr[i], g_step));
      if (a.relu) yv[i] = *reinterpret_cast<const uint4*>(row_at(yp, gr[i], y_step));
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) xv[i] = *reinterpret_cast<const uint4*>(row_at(xp, xr[i], x_step));
    if (to - s0 < (uint32_t)S) {  // rows past the part (the last one again) as 0
#pragma unroll
      for (int i = 0; i < NG; ++i)
        if (s0 + (tid + i * EX_NT) / GC >= to) gv[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int i = 0; i < NX; ++i)
        if (s0 + (tid + i * EX_NT) / XC >= to) xv[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  };
  const bool sums = k0 == 0 && kw == 0;
  frag ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = (T)1.f;
  const int64_t size = (int64_t)a.out * a.in + a.out;
  for (; from < end; from = to) {
    while (offsets[e + 1] <= from) ++e;
    to = min(offsets[e + 1], end);
    f32x4 acc[NM][NK], sum[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NK; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    rows(from);
    fetch(from);
    rows(from + S);
    for (uint32_t s0 = from; s0 < to; s0 += S) {
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        const int ch = tid + i * EX_NT;
        if (a.relu) gv[i] = where_positive<T>(gv[i], yv[i]);
        *reinterpret_cast<uint4*>(gs + ch / GC * lds_row<T, TM> + ch % GC * EL) = gv[i];
      }
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int ch = tid + i * EX_NT;
        *reinterpret_cast<uint4*>(xs + ch / XC * lds_row<T, TK> + ch % XC * EL) = xv[i];
      }
      __syncthreads();
      if (to - s0 > S) {
        fetch(s0 + S);
        rows(s0 + 2 * S);
      }
#pragma unroll
      for (int h = 0; h < S / 32; ++h) {
        frag gf[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) gf[i] = col_frag<T, TM>(gs, 32 * h, mw + 16 * i, lane);
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const frag xf = col_frag<T, TK>(xs, 32 * h, kw + 16 * j, lane);
#pragma unroll
          for (int i = 0; i < NM; ++i) acc[i][j] = Mat<T>::mma(gf[i], xf, acc[i][j]);
        }
        if (sums) {
#pragma unroll
          for (int i = 0; i < NM; ++i) sum[i] = Mat<T>::mma(gf[i], ones, sum[i]);
        }
      }
      __syncthreads();
    }
    float* part = (float*)a.workspace + ((int64_t)run + e) * size;
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m0 + mw + 16 * i + 4 * g + r;
        if (m >= a.out) continue;
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const int k = k0 + kw + 16 * j + c;
          if (k < a.in) part[(int64_t)m * a.in + k] = acc[i][j][r];
        }
        if (sums && c == 0) part[(int64_t)a.out * a.in + m] = sum[i][r];
      }
  }
}

// dW and db: an expert's parts, in order
__global__ __launch_bounds__(EX_NT) void k_expert_join(ffn_experts a, PlanView v, Shares shares) {
  const int64_t mk = (int64_t)a.out * a.in, size = mk + a.out;
  const int64_t at = (int64_t)blockIdx.x * EX_NT + threadIdx.x;
  if (at >= size) return;
  const int e = blockIdx.y;
  const uint32_t off = a.plan[v.offsets + e], end = off + a.plan[v.counts + e];
  const float* part = (const float*)a.workspace + e * size + at;
  float s = 0.f;
  if (off < end) {
    const uint32_t last = (end - 1) / shares.len;
#pragma unroll 8
    for (uint32_t run = off / shares.len; run <= last; ++run) s += part[run * size];
  }
  if (at < mk) {
    if (a.dW) a.dW[e * mk + at] = s;
  } else if (a.db) {
    a.db[(int64_t)e * a.out + at - mk] = s;
  }
}

// Blocks that fill the card: two a CU.  Runs for 384, 512, 768 and 1024 blocks: weight gradient of 500009 rows, 256 x 256 values,
// 240, 204, 227, 217 us; a million rows of 128 x 128 131, 127, 139, 143.  Runs of less than 256 slots gain nothing.
constexpr int64_t FILL = 512;

// A block's part of dW, and the runs
struct WeightGradient {
  int tm, tk, m_tiles, k_tiles;
  Shares shares;
};
static WeightGradient weight_gradient(const ffn_experts& a) {
  WeightGradient w;
  // Tiles of 128 read dy and x half as often, if there is work for enough of them (64 / 128, us: a million rows of 128 x 128
  // values 268 / 125, 65536 rows 20 / 27; 16384 rows of 256 x 256 24 / 28); float is bound by its products, not by reads.
  const int64_t large = (int64_t)((a.out + 127) / 128) * ((a.in + 127) / 128);
  const bool many = a.dtype != FFN_F32 && a.n / 1024 * large >= FILL / 2;
  w.tm = many && a.out > 64 ? 128 : 64;
  w.tk = many && a.in > 64 ? 128 : 64;
  w.m_tiles = (a.out + w.tm - 1) / w.tm;
  w.k_tiles = (a.in + w.tk - 1) / w.tk;
  const int64_t tiles = (int64_t)w.m_tiles * w.k_tiles, n = a.n;
  int64_t groups = FILL / tiles;
  groups = groups < n / 256 ? groups : n / 256;
  groups = groups < 1 ? 1 : groups;
  w.shares.len = (uint32_t)(((n + groups - 1) / groups + 63) / 64 * 64);
  w.shares.groups = n ? (uint32_t)((n + w.shares.len - 1) / w.shares.len) : 0;
  if (!n) w.shares.len = 64;
  return w;
}

uint64_t expert_workspace(const ffn_experts& a) {
  if (!a.dW && !a.db) return 0;
  return ((uint64_t)weight_gradient(a).shares.groups + a.n_experts) * ((uint64_t)a.out * a.in + a.out) * sizeof(float);
}

template <typename T, bool BACK, int NB>
static void product(const ffn_experts& a, const PlanView& v, hipStream_t st) {
  const int width = BACK ? a.in : a.out, cols = (width + 16 * NB - 1) / (16 * NB);
  const int64_t total = (int64_t)v.n_tiles * cols;
  k_expert<T, BACK, NB><<<grid_of((total + 7) / 8 * 8), EX_NT, 0, st>>>(a, v, total, cols);
}
// Columns a block: all of a row's, so that x is read once, but narrower ones while that leaves CUs without work.  64 / 128 /
// 256 columns a block, us, forward in bf16: 300000 rows, 256 x 256 values 146 / 121 / 118 (dx 168 / 117 / 104); 65536 rows
// 34 / 29 / 41; 4096 rows 8 / 11 / 18; 128 x 128 values, a million rows 171 / 150 / 219, 65536 rows 16 / 14 / 26, 4096 rows
// 6 / 9 / 13; 64 x 64 values, a million rows 66 / 85 / 150.
template <typename T, bool BACK>
static void product(const ffn_experts& a, const PlanView& v, hipStream_t st) {
  const int width = BACK ? a.in : a.out;
  const int64_t tiles = v.n_tiles;
  if (width <= 64 || tiles * ((width + 127) / 128) < FILL) product<T, BACK, 4>(a, v, st);
  else if (width <= 128 || sizeof(T) == 4 || tiles * ((width + 255) / 256) < 2 * FILL) product<T, BACK, 8>(a, v, st);
  else if constexpr (sizeof(T) == 2) product<T, BACK, 16>(a, v, st);  // float: 16 would not fit the registers
}

template <typename T, int TM, int TK>
static void parts(const ffn_experts& a, const PlanView& v, const WeightGradient& w, hipStream_t st) {
  const int64_t total = (int64_t)w.shares.groups * w.m_tiles * w.k_tiles;
  if (total)
    k_expert_dw<T, TM, TK><<<(unsigned)((total + 7) / 8 * 8), EX_NT, 0, st>>>(a, v, total, w.m_tiles, w.k_tiles, w.shares);
}

template <typename T>
static hipError_t run(const ffn_experts& a, bool backward, hipStream_t st) {
  const PlanView v = plan_view(a.n, a.n_experts);
  if (!backward) {
    product<T, false>(a, v, st);
    return hipGetLastError();
  }
  if (a.dx && a.n) product<T, true>(a, v, st);
  if (a.dW || a.db) {
    const WeightGradient w = weight_gradient(a);
    if constexpr (sizeof(T) == 4) {
      parts<T, 64, 64>(a, v, w, st);
    } else {
      if (w.tm == 128 && w.tk == 128) parts<T, 128, 128>(a, v, w, st);
      else if (w.tm == 128) parts<T, 128, 64>(a, v, w, st);
      else if (w.tk == 128) parts<T, 64, 128>(a, v, w, st);
      else parts<T, 64, 64>(a, v, w, st);
    }
    const int64_t size = (int64_t)a.out * a.in + a.out;
    k_expert_join<<<dim3((unsigned)((size + EX_NT - 1) / EX_NT), a.n_experts), EX_NT, 0, st>>>(a, v, w.shares);
  }
  return hipGetLastError();
}

hipError_t launch_experts(const ffn_experts& a, bool backward, hipStream_t st) {
  if (a.dtype == FFN_BF16) return run<__bf16>(a, backward, st);
  if (a.dtype == FFN_F16) return run<_Float16>(a, backward, st);
  return run<float>(a, backward, st);
}

}  // namespace ffn
