// Entry points of the product with bias, activation and residual and of its backward pass, and their kernels beside
// the tiled product of vq_linear.h: the product of a few rows, the join of a split sum, the activation's gradient and
// column sums.
#include <algorithm>

#include "vq_linear.h"

namespace {

// ------------------------------------------------------------------------------ a few rows
// Up to 16 rows: the product is bound by reading W once.  A workgroup owns 16 output channels, its waves share out the
// sum; a wave reads W straight into the fragments of a 16x16 product (lane l: channel l % 16, 16 bytes at piece l / 16
// of a 64-byte step, so consecutive steps of one channel are consecutive lines), eight steps in flight, with x, which
// stays in the L2, in the other operand.  The waves' partial products are added in LDS in wave order.  8 rows, 4096 -> 4096 bf16:
// 8.6 us with W in the caches, 9.9 without (an empty launch takes 2.6, the 34 MB 5.3 at 6.3 TB/s), with gelu and a residual 10.2;
// 1 row, 256 -> 1024: 2.7, with bias and silu 3.5.
// W past the caches gains nothing: 10.1, and 9.4 instead of 9.1 where 100 MB of weights take turns.
constexpr int ROWS_MAX = 16;
constexpr int ROWS_UNROLL = 8;

template <typename T>
__device__ __forceinline__ f32x4 rows_mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (__is_same(T, VqBf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[e], fb[e], c, 0, 0, 0);
    return c;
  }
}

// One element of the epilogue (vql_finish does 16 bytes of them).
template <typename T>
__device__ __forceinline__ void epilogue_one(const VqLinearArgs& a, int64_t i, int j, float c) {
  if (a.bias) c += VqElem<T>::to(reinterpret_cast<const T*>(a.bias)[j]);
  const int kind = vql_kind(a.act);
  if (a.pre) {
    typedef typename VqKept<T, VQL_SIGMOID>::type Kept;
    if (kind == VQL_THRESHOLD) reinterpret_cast<T*>(a.pre)[i * a.J + j] = vql_keep<T, VQL_THRESHOLD>(c, a.act);
    else reinterpret_cast<Kept*>(a.pre)[i * a.J + j] = vql_keep<T, VQL_SIGMOID>(c, a.act);
  }
  c = kind == VQL_THRESHOLD ? vql_act_of<VQL_THRESHOLD, sizeof(T) == 2>(c, a.act)
      : kind == VQL_SIGMOID ? vql_act_of<VQL_SIGMOID, sizeof(T) == 2>(c, a.act)
                            : vql_act_of<VQL_NORMAL, sizeof(T) == 2>(c, a.act);
  if (a.res) c += VqElem<T>::to(reinterpret_cast<const T*>(a.res + i * a.ldr)[j]);
  reinterpret_cast<T*>(a.out)[i * a.J + j] = VqElem<T>::from(c);
}

template <typename T>
__global__ __launch_bounds__(1024) void vql_rows_kernel(VqLinearArgs a) {
  constexpr int E = 16 / sizeof(T), KS = 4 * E;   // elements of the sum per step
  __shared__ float part[16][16 * 20];             // [wave][row][channel, padded]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int sub = lane & 15, piece = lane >> 4;
  const int64_t n = n0 + sub < a.J ? n0 + sub : a.J - 1;
  const int64_t m = sub < a.I ? sub : a.I - 1;    // rows and channels that do not exist repeat the last one, unstored
  const char* wp = a.B + n * a.ldb + piece * 16;
  const char* xp = a.A + m * a.lda + piece * 16;
  const int64_t steps = (a.R + KS - 1) / KS, full = a.R / KS;
  const int64_t per = (steps + waves - 1) / waves;   // this wave's range of the sum
  int64_t s = wave * per;
  const int64_t s1 = s + per < steps ? s + per : steps;
  const int64_t sf = s1 < full ? s1 : full;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (; s + ROWS_UNROLL <= sf; s += ROWS_UNROLL) {
    u32x4 w[ROWS_UNROLL], x[ROWS_UNROLL];
#pragma unroll
    for (int u = 0; u < ROWS_UNROLL; ++u) w[u] = vql_load16<T>(wp + (s + u) * 64);
#pragma unroll
    for (int u = 0; u < ROWS_UNROLL; ++u) x[u] = vql_load16<T>(xp + (s + u) * 64);
#pragma unroll
    for (int u = 0; u < ROWS_UNROLL; ++u) acc = rows_mma<T>(w[u], x[u], acc);
  }
  for (; s < s1; ++s) {
    const int64_t valid = a.R - s * KS - piece * E;
    acc = rows_mma<T>(vql_load16_part<T>(wp + s * 64, valid), vql_load16_part<T>(xp + s * 64, valid), acc);
  }
  *reinterpret_cast<vql_f32x4*>(&part[wave][sub * 20 + 4 * piece]) = acc;   // row `sub`, channels 4 piece ..
  __syncthreads();
  for (int t = threadIdx.x; t < 256; t += blockDim.x) {
    const int row = t >> 4, col = t & 15;
    if (row >= a.I || n0 + col >= a.J) continue;
    float c = 0.0f;
    for (int w = 0; w < waves; ++w) c += part[w][row * 20 + col];
    epilogue_one<T>(a, row, (int)(n0 + col), c);
  }
}

// ------------------------------------------------------------------------------ join of a split sum
// Sums of `parts` rows of n values, for 64 of them at a time from `first` on: wave k takes the rows k, k + 4, .., then the
// four sums are added in order.  All 256 threads of a workgroup call it.
template <typename T>
__device__ __forceinline__ void join_rows(const float* part, int parts, int64_t n, T* out, int64_t first, int64_t step, float (&s)[4][64]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t at = first; at < n; at += step) {
    const int64_t i = at + lane;
    float c = 0.0f;
    if (i < n) {
#pragma unroll 8
      for (int k = wave; k < parts; k += 4) c += part[k * n + i];
    }
    s[wave][lane] = c;
    __syncthreads();
    if (wave == 0 && i < n) out[i] = VqElem<T>::from(((s[0][lane] + s[1][lane]) + s[2][lane]) + s[3][lane]);
    __syncthreads();
  }
}
// Adds the partial sums and applies the epilogue: a workgroup per 32x32 tile, a lane per 16 values of a row as in the
// product kernel; wave k adds the splits k, k + 4, .., then the four sums are added in order (the same bits on every run).
// 256 x 1024 in 32 splits, 34 MB out of the last-level cache: 10.7 us; sixteen waves a tile made it 20.
template <typename T>
__global__ __launch_bounds__(256) void vql_join_kernel(VqLinearArgs a, int tile, int waves_j, int tiles_u, int tiles_v) {
  __shared__ f32x4 sums[3][4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (a.asum) {   // weight gradient: the bias gradient's partial sums too
    __shared__ float rows[4][64];
    join_rows<T>(a.asum, a.sum_parts, a.I, reinterpret_cast<T*>(a.gbias), (int64_t)blockIdx.x * 64, (int64_t)gridDim.x * 64, rows);
  }
  const int per_block = tile * tile / 1024;                 // 32x32 tiles of a block
  const int64_t block = blockIdx.x / per_block, blocks = a.tiles_i * a.tiles_j;
  const int sub = blockIdx.x % per_block;
  const int w = sub / (tiles_u * tiles_v), u = sub / tiles_v % tiles_u, v = sub % tiles_v;
  const int64_t r = block / a.tiles_j * tile + ((w / waves_j) * tiles_u + u) * 32 + (lane & 31);
  const int64_t cv = block % a.tiles_j * tile + ((w % waves_j) * tiles_v + v) * 32;
  f32x4 c[4] = {};
  const float* p = a.part + (block * per_block + sub) * 1024 + lane * 4;
  for (int s = wave; s < a.splits; s += 4)
#pragma unroll
    for (int g = 0; g < 4; ++g) c[g] += *reinterpret_cast<const vql_f32x4*>(p + s * blocks * per_block * 1024 + g * 256);
  if (wave > 0)
#pragma unroll
    for (int g = 0; g < 4; ++g) sums[wave - 1][g][lane] = c[g];
  __syncthreads();
  if (wave > 0) return;
  float all[16];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const f32x4 t = ((c[g] + sums[0][g][lane]) + sums[1][g][lane]) + sums[2][g][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) all[4 * g + e] = t[e];
  }
  const int kind = vql_kind(a.act);
  if (kind == VQL_THRESHOLD) vql_write_lane<T, VQL_THRESHOLD>(a, r, cv, lane >> 5, all);
  else if (kind == VQL_SIGMOID) vql_write_lane<T, VQL_SIGMOID>(a, r, cv, lane >> 5, all);
  else vql_write_lane<T, VQL_NORMAL>(a, r, cv, lane >> 5, all);
}
template <typename T>
__global__ __launch_bounds__(256) void vql_join_sums_kernel(const float* part, int parts, int64_t n, T* out) {
  __shared__ float rows[4][64];
  join_rows<T>(part, parts, n, out, (int64_t)blockIdx.x * 64, n, rows);
}

// ------------------------------------------------------------------------------ activation's gradient
// dp = gy * act'(pre), rounded to T: the operand of both products of the backward pass, whose matrix instructions take T.
// What is read passes the caches by, so that dp, which is read next, stays there (64 Ki x 1024 bf16 and the weight gradient
// behind it 132 -> 121 us).
// pre: T by its size; what it is, vql_kept knows
template <typename T>
__global__ __launch_bounds__(256) void vql_act_grad_kernel(const T* gy, const T* pre, int act, int64_t count, T* dp) {
  constexpr int E = 16 / sizeof(T);
  const int64_t vecs = count / E, stride = (int64_t)gridDim.x * 256;
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < vecs; v += stride) {
    const VqChunk<T> g = __builtin_bit_cast(VqChunk<T>, vql_once16<T>(reinterpret_cast<const char*>(gy + v * E)));
    const VqChunk<T> p = __builtin_bit_cast(VqChunk<T>, vql_once16<T>(reinterpret_cast<const char*>(pre + v * E)));
    VqChunk<T> d;
#pragma unroll
    for (int e = 0; e < E; ++e)
      d.e[e] = VqElem<T>::from(VqElem<T>::to(g.e[e]) * vql_act_slope<sizeof(T) == 2>(vql_kept(p.e[e], act), act));
    vql_store16<T>(dp + v * E, __builtin_bit_cast(u32x4, d));
  }
  const int64_t at = vecs * E + (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at < count)
    dp[at] = VqElem<T>::from(VqElem<T>::to(gy[at]) * vql_act_slope<sizeof(T) == 2>(vql_kept(pre[at], act), act));
}

// The same with the bias gradient: the sums over the rows, of dp before it is rounded (sums of the rounded values are off by
// 1.5 to 2.5 times as much).  A thread keeps the columns of one 16-byte piece and takes every so many-th row, two of them in flight;
// the rows that a workgroup takes at a time are added in LDS at the end.  64 Ki x 1024 bf16: 69 us, 5.9 TB/s.  Before the loads
// passed the caches by, 82; four rows in flight 87, a workgroup's rows next to each other 89.
constexpr int SUMS_NT = 1024, SUMS_WGS = 256;
template <typename T>
__global__ __launch_bounds__(SUMS_NT) void vql_act_grad_sums_kernel(const T* gy, const T* pre, int act, int64_t M, int N, int lanes,
                                                                   T* dp, float* part) {
  constexpr int E = 16 / sizeof(T), U = 2;
  __shared__ float s[SUMS_NT * E];
  const int rows = SUMS_NT / lanes, row = threadIdx.x / lanes, lane = threadIdx.x - row * lanes;
  const int64_t col = ((int64_t)blockIdx.x * lanes + lane) * E, valid = N - col;
  const int64_t stride = (int64_t)gridDim.y * rows;
  float sum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[e] = 0.0f;
  auto one = [&](int64_t m, u32x4 gv, u32x4 pv) {
    const VqChunk<T> g = __builtin_bit_cast(VqChunk<T>, gv), p = __builtin_bit_cast(VqChunk<T>, pv);
    VqChunk<T> d;
#pragma unroll
    for (int e = 0; e < E; ++e) {   // elements behind the row's end are zero: g is
      const float v = VqElem<T>::to(g.e[e]) * vql_act_slope<sizeof(T) == 2>(vql_kept(p.e[e], act), act);
      sum[e] += v;
      d.e[e] = VqElem<T>::from(v);
    }
    vql_store16_part<T>(reinterpret_cast<char*>(dp + m * N + col), __builtin_bit_cast(u32x4, d), valid);
  };
  auto load = [&](const T* from, int64_t m) {
    const char* q = reinterpret_cast<const char*>(from + m * N + col);
    return valid >= E ? vql_once16<T>(q) : vql_load16_part<T>(q, valid);
  };
  if (row < rows && valid > 0) {
    int64_t m = (int64_t)blockIdx.y * rows + row;
    for (; m + (U - 1) * stride < M; m += U * stride) {
      u32x4 g[U], p[U];
#pragma unroll
      for (int u = 0; u < U; ++u) g[u] = load(gy, m + u * stride);
#pragma unroll
      for (int u = 0; u < U; ++u) p[u] = load(pre, m + u * stride);
#pragma unroll
      for (int u = 0; u < U; ++u) one(m + u * stride, g[u], p[u]);
    }
    for (; m < M; m += stride) one(m, load(gy, m), load(pre, m));
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s[threadIdx.x * E + e] = sum[e];
  __syncthreads();
  for (int c = threadIdx.x; c < lanes * E; c += SUMS_NT) {
    const int64_t at = (int64_t)blockIdx.x * lanes * E + c;
    if (at >= N) continue;
    float v = 0.0f;
    for (int r = 0; r < rows; ++r) v += s[r * lanes * E + c];
    part[blockIdx.y * (int64_t)N + at] = v;
  }
}

// ------------------------------------------------------------------------------ column sums
// The bias gradient where no weight gradient is wanted (which carries it along): 64 columns and a range of rows per
// workgroup, four rows at a time.
template <typename T>
__global__ __launch_bounds__(256) void vql_colsum_kernel(const T* g, int64_t M, int N, int64_t rows_per, float* part) {
  __shared__ float s[4][64];
  const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
  const int64_t col = (int64_t)blockIdx.x * 64 + c;
  const int64_t m0 = blockIdx.y * rows_per, m1 = m0 + rows_per < M ? m0 + rows_per : M;
  float sum = 0.0f;
  if (col < N)
    for (int64_t m = m0 + r; m < m1; m += 4) sum += VqElem<T>::to(g[m * N + col]);
  s[r][c] = sum;
  __syncthreads();
  if (r == 0 && col < N) part[(int64_t)blockIdx.y * N + col] = (s[0][c] + s[1][c]) + (s[2][c] + s[3][c]);
}

// ------------------------------------------------------------------------------ choice of tile and split
struct Plan {
  bool rows;       // the few-rows kernel
  int config;
  int splits;
  int64_t steps_per_split;
  int64_t tiles_i;
  int tiles_j;
  int workgroups;
};

constexpr int CUS = 256;

size_t elem_size(int dtype) { return dtype == VQ_F32 ? 4 : 2; }

// What a block of each tile costs: microseconds of a 128-byte step of the sum with 1, 2, 3 workgroups on a CU, and what a
// workgroup pays once (start, first tiles, epilogue); 16-bit and 32-bit types, tiles filled by DMA and through registers.
// Measured on an MI355X, 256 workgroups for each one on a CU, sums of 8 and of 32 steps.
struct Cost {
  int tile, per_cu;
  struct { float step[3], once; } of[2][2];   // [dma][32 bits]
};
const Cost COST[VQL_CONFIGS] = {
    {64, 3, {{{{0.90f, 1.17f, 1.38f}, 4.2f}, {{1.17f, 1.65f, 2.05f}, 6.0f}},
             {{{0.32f, 0.45f, 0.60f}, 4.4f}, {{0.65f, 1.07f, 1.45f}, 6.5f}}}},
    {128, 2, {{{{1.70f, 2.05f}, 8.0f}, {{2.95f, 4.60f}, 12.0f}}, {{{0.72f, 0.95f}, 6.5f}, {{1.97f, 3.69f}, 13.5f}}}},
    {256, 1, {{}, {{{1.55f}, 12.5f}, {{7.15f}, 27.0f}}}},
};
// How the operands' rows lie: 16-bit ones at odd addresses, on 4 bytes at least, on 16 (and so filled by DMA).
enum { ROWS_ODD = 0, ROWS_WORDS = 1, ROWS_DMA = 2 };
// The cheapest tile with its best split of the sum: rounds of workgroups x (steps x time of a step + once), the last round
// with as many on a CU as are left, and the join of a split sum (a launch, the partial sums written and read at 6.5 TB/s:
// they stay in the last-level cache).  Over 36 random products of 17 to 65536 rows and 64 to 4096 channels, every layout, the
// choice took 1.03 times as long on average as the best of all tiles and of 1, 2, 4 .. 32 splits, 1.19 times at worst (5.1 us instead of
// 4.3), 1.15 among those over 10 us.
Plan make_plan(int layout, int64_t I, int J, int64_t R, int dtype, int lie) {
  const size_t es = elem_size(dtype);
  const bool dma = lie == ROWS_DMA;
  Plan best{};
  const int64_t steps = (R * es + 127) / 128;
  double best_t = 1e300;
  // Few rows: the kernel that reads W once, 16 channels to a workgroup whose waves share the sum.  Its time goes by the bytes of a
  // channel and the rows, as measured from 12 to 64 KiB a channel and 128 to 8192 channels; long sums over few channels leave
  // most of the device idle there, and the tiled kernel splits them (us, rows kernel and tiled one: 8 rows, 4096 -> 4096 bf16 9.1 and
  // 13.7, 16 rows, 8192 -> 512 16.7 and 11.9, 1 row, 16384 -> 2048 20.4 and 18.1, -> 4096 23.2 and 26.7; at odd
  // addresses 8 rows, 4097 -> 512 22.8 and 12.3, 1025 -> 512 8.2 and 11.1).
  if (layout == 0 && I <= ROWS_MAX) {
    best.rows = true;
    best.splits = 1;
    const double kib = lie == ROWS_ODD ? 1.75 + 0.085 * I : 0.54 + 0.0225 * I;
    best_t = 2.4 + R * es / 1024.0 * kib * std::max(1.0, (J + 15) / 16 / (double)CUS);
  }
  for (int c = 0; c < VQL_CONFIGS; ++c) {
    const Cost& cost = COST[c];
    const auto& of = cost.of[dma][es == 4];
    if (of.once == 0.0f) continue;
    const int64_t ti = (I + cost.tile - 1) / cost.tile, tj = (J + cost.tile - 1) / cost.tile;
    const int64_t slots = (int64_t)CUS * cost.per_cu;
    const int64_t most = std::max<int64_t>(1, std::min<int64_t>(steps / 4, 2 * slots / std::max<int64_t>(1, ti * tj)));
    for (int64_t s = 1; s <= most; s = s < 8 ? s + 1 : s + s / 8) {
      const int64_t per = (steps + s - 1) / s, sp = steps ? (steps + per - 1) / per : 1;
      const int64_t blocks = ti * tj * sp, rounds = blocks / slots, rest = blocks % slots;
      double t = rounds * (per * of.step[cost.per_cu - 1] + of.once);
      if (rest) t += per * of.step[(rest - 1) / CUS] + of.once;
      if (sp > 1) t += 3.0 + (double)ti * tj * cost.tile * cost.tile * 8 * sp / 6.5e6;
      if (t < best_t) {
        best_t = t;
        best.rows = false;
        best.config = c;
        best.splits = (int)sp;
        best.steps_per_split = per;
        best.tiles_i = ti;
        best.tiles_j = (int)tj;
        best.workgroups = (int)slots;
      }
    }
  }
  return best;
}

int64_t part_bytes(const Plan& p) {
  return p.splits > 1 ? p.splits * p.tiles_i * p.tiles_j * COST[p.config].tile * COST[p.config].tile * 4 : 0;
}
// row slabs of vql_colsum_kernel
int64_t colsum_slabs(int64_t M, int N) {
  const int64_t groups = (N + 63) / 64;
  return std::max<int64_t>(1, std::min<int64_t>((M + 63) / 64, std::max<int64_t>(1, 4 * CUS / groups)));
}

// how vql_act_grad_sums_kernel cuts its matrix: column groups of `lanes` 16-byte pieces, and `slabs` workgroups for the rows
// of each, one to a CU in all, so that the sums to be joined stay few
struct SumsPlan { int groups, lanes, slabs; };
SumsPlan sums_plan(int64_t M, int N, int dtype) {
  const int E = (int)(16 / elem_size(dtype)), pieces = (N + E - 1) / E;
  SumsPlan p;
  p.groups = (pieces + SUMS_NT / 4 - 1) / (SUMS_NT / 4);
  p.lanes = (pieces + p.groups - 1) / p.groups;
  const int64_t rows = SUMS_NT / p.lanes, most = std::max(1, SUMS_WGS / p.groups);
  p.slabs = (int)std::max<int64_t>(1, std::min<int64_t>(most, (M + rows - 1) / rows));
  return p;
}
int64_t sums_bytes(int64_t M, int N, int dtype) { return ((int64_t)sums_plan(M, N, dtype).slabs * N * 4 + 255) & ~(int64_t)255; }

// the activation's gradient, at the head of the backward pass's workspace
int64_t dp_bytes(int64_t M, int N, int dtype) { return (M * N * (int64_t)elem_size(dtype) + 255) & ~(int64_t)255; }

bool bad_sizes(int64_t M, int K, int N) { return M < 0 || K <= 0 || N <= 0; }
bool known(int dtype) { return dtype == VQ_F32 || dtype == VQ_BF16 || dtype == VQ_F16; }
constexpr int MAX_DIM = 1 << 20;
constexpr int64_t MAX_ROWS = (int64_t)1 << 31;
// The product kernel counts its blocks in 32 bits, one round of workgroups beyond the last.  No output that fits the memory has as
// many: 2^30 tiles of 64 x 64 from 64 columns on, and MAX_ROWS / 64 = 2^25 tiles for each 64 columns below.
constexpr int64_t MAX_BLOCKS = (int64_t)1 << 30;
bool pitch_too_wide(int64_t ld, size_t es) { return ld * (int64_t)es > 0x7fffffff / 256 - 128; }

int product(const VqLinearArgs& a, int layout, int dtype, int config, bool dma, hipStream_t s) {
  if (dtype == VQ_F32) return vql_product_f32(a, layout, config, dma, s);
  if (dtype == VQ_BF16) return vql_product_bf16(a, layout, config, dma, s);
  return vql_product_f16(a, layout, config, dma, s);
}

template <template <typename> class F, typename... Args>
int by_type(int dtype, Args&&... args) {
  if (dtype == VQ_F32) return F<float>::run(args...);
  if (dtype == VQ_BF16) return F<VqBf16>::run(args...);
  return F<_Float16>::run(args...);
}
template <typename T> struct RunRows {
  static int run(const VqLinearArgs& a, hipStream_t s) {
    const int64_t steps = (a.R * (int64_t)sizeof(T) + 63) / 64;
    int waves = 1;
    while (waves < 16 && waves * 2 < steps) waves *= 2;   // two steps or more a wave
    if (waves < 4) waves = 4;                             // four waves write the 256 results
    hipLaunchKernelGGL(vql_rows_kernel<T>, dim3((unsigned)((a.J + 15) / 16)), dim3(waves * 64), 0, s, a);
    return vq_hip_status(hipGetLastError());
  }
};
template <typename T> struct RunJoin {
  static int run(const VqLinearArgs& a, int config, hipStream_t s) {
    const int tile = COST[config].tile, waves_j = config == VQL_C256 ? 4 : 2;
    const int tiles_u = config == VQL_C256 ? 4 : tile / 64, tiles_v = config == VQL_C256 ? 2 : tile / 64;
    const int64_t blocks = a.tiles_i * a.tiles_j * tile * tile / 1024;
    hipLaunchKernelGGL(vql_join_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, a, tile, waves_j, tiles_u, tiles_v);
    return vq_hip_status(hipGetLastError());
  }
};
template <typename T> struct RunJoinSums {
  static int run(const float* part, int parts, int64_t n, void* out, hipStream_t s) {
    hipLaunchKernelGGL(vql_join_sums_kernel<T>, dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s, part, parts, n,
                       reinterpret_cast<T*>(out));
    return vq_hip_status(hipGetLastError());
  }
};
template <typename T> struct RunActGrad {
  static int run(const void* gy, const void* pre, int act, int64_t count, void* dp, hipStream_t s) {
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((count / (16 / sizeof(T)) + 255) / 256, 16384));
    hipLaunchKernelGGL(vql_act_grad_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, reinterpret_cast<const T*>(gy),
                       reinterpret_cast<const T*>(pre), act, count, reinterpret_cast<T*>(dp));
    return vq_hip_status(hipGetLastError());
  }
};
template <typename T> struct RunActGradSums {
  static int run(const void* gy, const void* pre, int act, int64_t M, int N, const SumsPlan& p, void* dp, float* part, hipStream_t s) {
    hipLaunchKernelGGL(vql_act_grad_sums_kernel<T>, dim3((unsigned)p.groups, (unsigned)p.slabs), dim3(SUMS_NT), 0, s,
                       reinterpret_cast<const T*>(gy), reinterpret_cast<const T*>(pre), act, M, N, p.lanes,
                       reinterpret_cast<T*>(dp), part);
    return vq_hip_status(hipGetLastError());
  }
};
template <typename T> struct RunColsum {
  static int run(const void* g, int64_t M, int N, int64_t slabs, float* part, hipStream_t s) {
    const int64_t per = (M + slabs - 1) / slabs;
    hipLaunchKernelGGL(vql_colsum_kernel<T>, dim3((unsigned)((N + 63) / 64), (unsigned)slabs), dim3(256), 0, s,
                       reinterpret_cast<const T*>(g), M, N, per, part);
    return vq_hip_status(hipGetLastError());
  }
};

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Runs one of the three products with its epilogue; `gbias` (weight gradient) receives the sums of A, or of the `sum_parts`
// rows of `sums` where the caller has those.
int run_product(int layout, VqLinearArgs a, int dtype, void* gbias, const float* sums, int sum_parts, void* work, hipStream_t s) {
  const int64_t es = (int64_t)elem_size(dtype);
  const int E = (int)(16 / es);
  bool dma = aligned16(a.A) && aligned16(a.B) && a.lda % 16 == 0 && a.ldb % 16 == 0;
  if (layout == 1 && a.J % E) dma = false;                 // a piece of an m-major operand must not pass its row's end
  if (layout == 2 && (a.I % E || a.J % E)) dma = false;
  const bool odd = ((reinterpret_cast<uintptr_t>(a.A) | reinterpret_cast<uintptr_t>(a.B) | a.lda | a.ldb) & 3) != 0;
  const Plan p = make_plan(layout, a.I, a.J, a.R, dtype, dma ? ROWS_DMA : odd ? ROWS_ODD : ROWS_WORDS);
  a.splits = p.splits;
  a.steps_per_split = (int)p.steps_per_split;
  a.tiles_i = p.tiles_i;
  a.tiles_j = p.tiles_j;
  a.workgroups = p.workgroups;
  if (p.splits > 1) {
    if (!work || !aligned16(work)) return VQ_ERR_INVALID_ARG;
    a.part = reinterpret_cast<float*>(work);
  }
  if (p.rows) return by_type<RunRows>(dtype, a, s);
  if (p.tiles_i * p.tiles_j * p.splits > MAX_BLOCKS) return VQ_ERR_UNSUPPORTED;
  if (!sums) a.gbias = gbias;
  if (gbias && !sums && p.splits > 1) a.asum = reinterpret_cast<float*>(reinterpret_cast<char*>(work) + part_bytes(p));
  int rc = product(a, layout, dtype, p.config, dma, s);
  if (rc != VQ_OK) return rc;
  if (p.splits > 1) {
    a.gbias = gbias;
    a.sum_parts = p.splits;
    if (gbias && sums) {
      a.asum = const_cast<float*>(sums);
      a.sum_parts = sum_parts;
    }
    return by_type<RunJoin>(dtype, a, p.config, s);
  }
  return gbias && sums ? by_type<RunJoinSums>(dtype, sums, sum_parts, a.I, gbias, s) : VQ_OK;
}

int64_t product_work(int layout, int64_t I, int J, int64_t R, int dtype, bool sums) {
  int64_t bytes = 0;
  for (int lie = ROWS_ODD; lie <= ROWS_DMA; ++lie) {
    const Plan p = make_plan(layout, I, J, R, dtype, lie);
    bytes = std::max(bytes, part_bytes(p) + (sums && p.splits > 1 ? (int64_t)p.splits * I * 4 : 0));
  }
  return bytes;
}

}  // namespace

extern "C" int64_t vq_linear_work_bytes(int pass, int64_t M, int K, int N, int dtype) {
  if (bad_sizes(M, K, N) || K > MAX_DIM || N > MAX_DIM || M > MAX_ROWS || !known(dtype)) return 0;
  if (pass < VQ_LINEAR_FORWARD || pass > VQ_LINEAR_BACKWARD) return 0;
  if (pass == VQ_LINEAR_BACKWARD)
    return dp_bytes(M, N, dtype) + sums_bytes(M, N, dtype) + std::max(vq_linear_work_bytes(VQ_LINEAR_DGRAD, M, K, N, dtype),
                                            vq_linear_work_bytes(VQ_LINEAR_WGRAD, M, K, N, dtype));
  if (pass == VQ_LINEAR_FORWARD) return product_work(0, M, N, K, dtype, false);
  if (pass == VQ_LINEAR_DGRAD) return product_work(1, M, K, N, dtype, false);
  return std::max(product_work(2, N, K, M, dtype, true), colsum_slabs(M, N) * N * 4);
}

extern "C" int vq_linear(const void* x, int64_t ldx, const void* W, int64_t ldw, const void* bias, const void* residual,
                         int64_t ldr, int dtype, int act, int64_t M, int K, int N, void* y, void* pre, void* work,
                         void* stream) {
  if (bad_sizes(M, K, N) || !known(dtype) || act < VQ_ACT_NONE || act > VQ_ACT_GELU_TANH) return VQ_ERR_INVALID_ARG;
  if (ldx < K || ldw < K || (residual && ldr < N)) return VQ_ERR_INVALID_ARG;
  if (M == 0) return VQ_OK;
  if (!x || !W || !y) return VQ_ERR_INVALID_ARG;
  const size_t es = elem_size(dtype);
  if (K > MAX_DIM || N > MAX_DIM || M > MAX_ROWS || pitch_too_wide(ldx, es) || pitch_too_wide(ldw, es) ||
      (residual && pitch_too_wide(ldr, es)))
    return VQ_ERR_UNSUPPORTED;
  VqLinearArgs a{};
  a.A = reinterpret_cast<const char*>(x);
  a.B = reinterpret_cast<const char*>(W);
  a.lda = ldx * es;
  a.ldb = ldw * es;
  a.I = M;
  a.J = N;
  a.R = K;
  a.out = y;
  a.pre = pre;
  a.bias = bias;
  a.res = reinterpret_cast<const char*>(residual);
  a.ldr = ldr * es;
  a.act = act;
  return run_product(0, a, dtype, nullptr, nullptr, 0, work, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int vq_linear_act_grad(const void* gy, const void* pre, int dtype, int act, int64_t count, void* dp, void* stream) {
  if (count < 0 || !known(dtype) || act <= VQ_ACT_NONE || act > VQ_ACT_GELU_TANH) return VQ_ERR_INVALID_ARG;
  if (count == 0) return VQ_OK;
  if (!gy || !pre || !dp) return VQ_ERR_INVALID_ARG;
  return by_type<RunActGrad>(dtype, gy, pre, act, count, dp, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int vq_linear_dgrad(const void* dp, const void* W, int64_t ldw, int dtype, int64_t M, int K, int N, void* gx,
                               void* work, void* stream) {
  if (bad_sizes(M, K, N) || !known(dtype) || ldw < K) return VQ_ERR_INVALID_ARG;
  if (M == 0) return VQ_OK;
  if (!dp || !W || !gx) return VQ_ERR_INVALID_ARG;
  const size_t es = elem_size(dtype);
  if (K > MAX_DIM || N > MAX_DIM || M > MAX_ROWS || pitch_too_wide(N, es) || pitch_too_wide(ldw, es)) return VQ_ERR_UNSUPPORTED;
  VqLinearArgs a{};
  a.A = reinterpret_cast<const char*>(dp);
  a.B = reinterpret_cast<const char*>(W);
  a.lda = N * es;
  a.ldb = ldw * es;
  a.I = M;
  a.J = K;
  a.R = N;
  a.out = gx;
  return run_product(1, a, dtype, nullptr, nullptr, 0, work, reinterpret_cast<hipStream_t>(stream));
}

namespace {
// sums: `parts` rows whose sum is the bias gradient, or null: it is the column sums of dp then
int weight_gradients(const void* dp, const void* x, int64_t ldx, int dtype, int64_t M, int K, int N, void* gW, void* gbias,
                     const float* sums, int parts, void* work, void* stream) {
  if (bad_sizes(M, K, N) || !known(dtype) || ldx < K || (!gW && !gbias)) return VQ_ERR_INVALID_ARG;
  if (M > 0 && (!dp || (gW && !x))) return VQ_ERR_INVALID_ARG;
  const size_t es = elem_size(dtype);
  if (K > MAX_DIM || N > MAX_DIM || M > MAX_ROWS || pitch_too_wide(N, es) || pitch_too_wide(ldx, es)) return VQ_ERR_UNSUPPORTED;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (!gW) {
    if (sums) return by_type<RunJoinSums>(dtype, sums, parts, (int64_t)N, gbias, s);
    if (!work) return VQ_ERR_INVALID_ARG;
    const int64_t slabs = colsum_slabs(M, N);
    float* part = reinterpret_cast<float*>(work);
    const int rc = by_type<RunColsum>(dtype, dp, M, N, slabs, part, s);
    return rc != VQ_OK ? rc : by_type<RunJoinSums>(dtype, (const float*)part, (int)slabs, (int64_t)N, gbias, s);
  }
  VqLinearArgs a{};
  a.A = reinterpret_cast<const char*>(dp);
  a.B = reinterpret_cast<const char*>(x);
  a.lda = N * es;
  a.ldb = ldx * es;
  a.I = N;
  a.J = K;
  a.R = M;
  a.out = gW;
  return run_product(2, a, dtype, gbias, sums, parts, work, s);
}
}  // namespace

extern "C" int vq_linear_wgrad(const void* dp, const void* x, int64_t ldx, int dtype, int64_t M, int K, int N, void* gW,
                               void* gbias, void* work, void* stream) {
  return weight_gradients(dp, x, ldx, dtype, M, K, N, gW, gbias, nullptr, 0, work, stream);
}

extern "C" int vq_linear_backward(const void* gy, const void* pre, const void* x, int64_t ldx, const void* W, int64_t ldw,
                                  int dtype, int act, int64_t M, int K, int N, void* gx, void* gW, void* gbias, void* work,
                                  void* stream) {
  if (bad_sizes(M, K, N) || !known(dtype) || act < VQ_ACT_NONE || act > VQ_ACT_GELU_TANH) return VQ_ERR_INVALID_ARG;
  // everything the three calls would refuse, before the first of them has launched anything
  if (M > 0 && (!gy || (act != VQ_ACT_NONE && !pre))) return VQ_ERR_INVALID_ARG;
  if ((gx && (!W || ldw < K)) || (gW && ((M > 0 && !x) || ldx < K))) return VQ_ERR_INVALID_ARG;
  if (vq_linear_work_bytes(VQ_LINEAR_BACKWARD, M, K, N, dtype) > 0 && (!work || !aligned16(work))) return VQ_ERR_INVALID_ARG;
  const size_t es = elem_size(dtype);
  if (K > MAX_DIM || N > MAX_DIM || M > MAX_ROWS || pitch_too_wide(N, es) || (gx && pitch_too_wide(ldw, es)) ||
      (gW && pitch_too_wide(ldx, es)))
    return VQ_ERR_UNSUPPORTED;
  const void* dp = gy;
  const float* sums = nullptr;
  int parts = 0;
  if (act != VQ_ACT_NONE && M > 0) {
    char* const after = reinterpret_cast<char*>(work) + dp_bytes(M, N, dtype);
    int rc;
    if (gbias) {
      const SumsPlan p = sums_plan(M, N, dtype);
      sums = reinterpret_cast<const float*>(after);
      parts = p.slabs;
      rc = by_type<RunActGradSums>(dtype, gy, pre, act, M, N, p, work, reinterpret_cast<float*>(after),
                                   reinterpret_cast<hipStream_t>(stream));
    } else {
      rc = vq_linear_act_grad(gy, pre, dtype, act, M * N, work, stream);
    }
    if (rc != VQ_OK) return rc;
    dp = work;
    work = after + sums_bytes(M, N, dtype);
  }
  if (gx) {
    const int rc = vq_linear_dgrad(dp, W, ldw, dtype, M, K, N, gx, work, stream);
    if (rc != VQ_OK) return rc;
  }
  if (gW || gbias) return weight_gradients(dp, x, ldx, dtype, M, K, N, gW, gbias, sums, parts, work, stream);
  return VQ_OK;
}
