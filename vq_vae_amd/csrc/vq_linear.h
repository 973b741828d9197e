// Matrix product with bias, activation and residual in its epilogue, and the products of its backward
// pass (gfx950): shared device code of vq_linear_{f32,bf16,f16}.hip and vq_linear.hip.
//
// All three products are   C[i][j] = sum_r A(i, r) B(j, r)   with fp32 accumulation:
//     forward          i = row, j = output channel, r = input channel    A = x,  B = W      both with r contiguous
//     input gradient   i = row, j = input channel,  r = output channel   A = dp, B = W      B with j contiguous
//     weight gradient  i = output channel, j = input channel, r = row    A = dp, B = x      both with i / j contiguous
// An operand whose reduction index is contiguous is called r-major here, the other kind m-major.
#pragma once
#include "vq_common.h"

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct VqBf16 { uint16_t v; };   // element types of the templates: float, VqBf16, _Float16

// tiles of the product kernel
enum { VQL_C64 = 0, VQL_C128 = 1, VQL_C256 = 2, VQL_CONFIGS = 3 };

struct VqLinearArgs {
  const char* A;
  const char* B;
  int64_t lda, ldb;          // bytes between rows of the operand as it lies in memory
  int64_t I;                 // rows of C
  int J;                     // columns of C
  int64_t R;                 // length of the sum
  int steps_per_split;       // 128-byte steps of the sum that one workgroup takes
  int splits;
  int workgroups;            // that fit the device at a time (a multiple of 8): each takes every so many-th block
  int64_t tiles_i;
  int tiles_j;
  void* out;                 // [I][J]
  void* pre;                 // [I][J] or null: C + bias as VqKept, what the activation's gradient needs
  const void* bias;          // [J] or null
  const char* res;           // [I][J] or null
  int64_t ldr;               // bytes between rows of res
  int act;
  float* part;               // splits > 1: the partial sums, as the product kernel's registers lie
  float* asum;               // weight gradient: the sums of A over r (the bias gradient) of a split sum, [splits][I], or null
  int sum_parts;             // rows of asum, for the join
  void* gbias;               // the same in T, where the sum is not split, and for the join
};

// -------------------------------------------------------------------------------- element conversions
template <typename T> struct VqElem;
template <> struct VqElem<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct VqElem<VqBf16> {
  static __device__ __forceinline__ float to(VqBf16 v) { return __uint_as_float((uint32_t)v.v << 16); }
  static __device__ __forceinline__ VqBf16 from(float f) {
    // the compiler's conversion: round to nearest, ties to even, NaN stays NaN (one instruction per pair)
    return {__builtin_bit_cast(uint16_t, (__bf16)f)};
  }
};
template <> struct VqElem<_Float16> {
  static __device__ __forceinline__ float to(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 from(float f) { return (_Float16)f; }
};

// 16 bytes of T at any element-aligned address (the hardware takes unaligned 16-byte accesses)
template <typename T>
struct alignas(sizeof(T)) VqChunk {
  T e[16 / sizeof(T)];
};
typedef u32x4 vql_u32x4_a2 __attribute__((aligned(2), may_alias));
typedef u32x4 vql_u32x4_a4 __attribute__((aligned(4), may_alias));
typedef u32x4 vql_u32x4_a16 __attribute__((may_alias));
typedef f32x4 vql_f32x4 __attribute__((may_alias));
#define VQL_LDS __attribute__((address_space(3)))
#define VQL_GLOBAL __attribute__((address_space(1)))
typedef uint32_t vql_u32 __attribute__((may_alias));
typedef uint16_t vql_u16 __attribute__((may_alias));
template <typename T>
__device__ __forceinline__ u32x4 vql_load16(const char* p) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const vql_u32x4_a4*>(p);
  else return *reinterpret_cast<const vql_u32x4_a2*>(p);
}
template <typename T>
__device__ __forceinline__ u32x4 vql_once16(const char* p) {   // of what is not read again: past the caches
  if constexpr (sizeof(T) == 4) return __builtin_nontemporal_load(reinterpret_cast<const vql_u32x4_a4*>(p));
  else return __builtin_nontemporal_load(reinterpret_cast<const vql_u32x4_a2*>(p));
}
template <typename T>
__device__ __forceinline__ void vql_store16(void* p, u32x4 v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<vql_u32x4_a4*>(p) = v;
  else *reinterpret_cast<vql_u32x4_a2*>(p) = v;
}
// The same, and past the caches if STREAM: outputs of the product are not read again by it, and keep its operands out of the
// L2 otherwise (operands and outputs out of the caches, bf16: 64 Ki x 256 -> 1024 79 -> 55 us, 64 Ki x 1024 -> 256 49 -> 45).
// Only for accesses that fill 64-byte runs: with rows of 6766 bytes, whose runs straddle the lines, the same kernel took
// 103 us instead of 64.  And only for 16-bit types: fp32 products, bound by the matrix cores, gain nothing (16384 x 1024 -> 4096
// 1002 us without, 1007 with).  A template argument, because the compiler makes one ordinary store of a branch's two.
template <typename T, bool STREAM>
__device__ __forceinline__ void vql_stream16(void* p, u32x4 v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<vql_u32x4_a2*>(p));
  else vql_store16<T>(p, v);
}
// `valid` of the 16 / sizeof(T) elements at p, the others zero
template <typename T>
__device__ __forceinline__ u32x4 vql_load16_part(const char* p, int64_t valid) {
  constexpr int E = 16 / sizeof(T);
  if (valid >= E) return vql_load16<T>(p);
  u32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < E - 1; ++e)
    if (e < valid) {
      if constexpr (sizeof(T) == 4)
        v[e] = *reinterpret_cast<const vql_u32*>(p + 4 * e);
      else
        v[e / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(p + 2 * e) << (16 * (e & 1));
    }
  return v;
}

// v moved down by `by` elements (0 .. all of them), zeros behind
template <typename T>
__device__ __forceinline__ u32x4 vql_shift(u32x4 v, int by) {
  if constexpr (sizeof(T) == 2) {
    if (by & 1) v = u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
    by >>= 1;
  }
  if (by & 1) v = u32x4{v[1], v[2], v[3], 0};
  if (by & 2) v = u32x4{v[2], v[3], 0, 0};
  if (by & 4) v = u32x4{0, 0, 0, 0};
  return v;
}

template <typename T>
__device__ __forceinline__ void vql_store16_part(char* p, u32x4 v, int64_t valid) {
  constexpr int E = 16 / sizeof(T);
  if (valid >= E) {
    vql_store16<T>(p, v);
  } else {
    const VqChunk<T> c = __builtin_bit_cast(VqChunk<T>, v);
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (e < valid) reinterpret_cast<T*>(p)[e] = c.e[e];
  }
}

// -------------------------------------------------------------------------------- activations
// erfc(z) for z >= 0: the Chebyshev fit of Numerical Recipes' erfcc (W. H. Press), itself off by less than 1.2e-7 of the
// value everywhere, and a dozen instructions without a branch.  Their roundings come on top (vql_cdf).
__device__ __forceinline__ float vql_erfc_pos(float z) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.5f, z, 1.0f));
  float q = 0.17087277f;
  q = __builtin_fmaf(q, t, -0.82215223f);
  q = __builtin_fmaf(q, t, 1.48851587f);
  q = __builtin_fmaf(q, t, -1.13520398f);
  q = __builtin_fmaf(q, t, 0.27886807f);
  q = __builtin_fmaf(q, t, -0.18628806f);
  q = __builtin_fmaf(q, t, 0.09678418f);
  q = __builtin_fmaf(q, t, 0.37409196f);
  q = __builtin_fmaf(q, t, 1.00002368f);
  q = __builtin_fmaf(q, t, -1.26551223f);
  return t * __expf(__builtin_fmaf(-z, z, q));
}
// FAST: 16-bit results. 1-ulp reciprocal and the hardware exponential, errors of some 1e-7 against a rounding of
// 2^-9 or 2^-12; the sigmoid and the normal density of fp32 results take the library's functions and true divisions.
template <bool FAST>
__device__ __forceinline__ float vql_sigmoid(float p) {
  if constexpr (FAST) return __builtin_amdgcn_rcpf(1.0f + __expf(-p));
  return 1.0f / (1.0f + expf(-p));
}
// Phi(p), for every type, fp32 too: the library's erfcf takes the branches of all its ranges in a wave with mixed arguments.
// p Phi(p) is off by up to 7.1 * 2^-24 (1 + p^2 / 2) of the value below zero and 7 * 2^-24 above (largest over 2e6 arguments in each
// of nine ranges of -13 .. 8): 2 for the fit, the rest for the fit's own steps, its reciprocal and, in the tail, the exponent's
// rounding.  (0.5 (1 + erf) in fp32 would lose the tail altogether.)
__device__ __forceinline__ float vql_cdf(float p) {
  const float half = 0.5f * vql_erfc_pos(fabsf(p) * 0.70710678f);
  return p < 0.0f ? half : 1.0f - half;
}
// The epilogues of the product kernel, one to a kernel: the epilogue is unrolled over a wave's accumulators, and with all
// activations in it the code outgrows the instruction cache (operands in the caches: 64 Ki x 256 -> 1024 bf16 with gelu_tanh 72 us
// instead of 60; 8192 x 4096 x 4096 with a residual 238 instead of 220).
enum { VQL_PLAIN = 0,     // no bias, activation or residual: the products of the backward pass
       VQL_THRESHOLD = 1, // none and relu
       VQL_SIGMOID = 2,   // silu and gelu_tanh: p sigmoid(p) and p sigmoid(2u)
       VQL_NORMAL = 3 };  // gelu
__host__ __device__ inline int vql_kind(int act) {
  return act == VQ_ACT_SILU || act == VQ_ACT_GELU_TANH ? VQL_SIGMOID : act == VQ_ACT_GELU ? VQL_NORMAL : VQL_THRESHOLD;
}
template <int KIND, bool FAST>
__device__ __forceinline__ float vql_act_of(float p, int act) {
  if constexpr (KIND == VQL_THRESHOLD) {
    const float floor = act == VQ_ACT_RELU ? 0.0f : -__builtin_inff();
    return p < floor ? floor : p;
  } else if constexpr (KIND == VQL_SIGMOID) {
    // silu's b is 2^-100, not zero, which times infinity would be NaN: a + b p^2 is one up to |p| = 2^37, where the sigmoid has
    // long been 0 or 1.  Choosing the argument instead costs an instruction an element (64 Ki x 256 -> 1024 bf16 62.3 -> 63.9 us).
    const float a = act == VQ_ACT_SILU ? 1.0f : 1.5957691216f, b = act == VQ_ACT_SILU ? 0x1p-100f : 0.0713548163f;
    return p * vql_sigmoid<FAST>(p * __builtin_fmaf(b * p, p, a));
  } else {
    return p * vql_cdf(p);
  }
}
// As what p is kept for the activation's gradient.  fp16 for both 16-bit types: its rounding shifts act' by an eighth of what that of
// bf16 does (gradients off by 1.43 instead of 1.5 times the last rounding), and what it takes for infinite lies far beyond where
// act' has its limit.  But relu's needs the sign of the smallest p: bf16 has it.
template <typename T, int KIND> struct VqKept { typedef _Float16 type; };
template <int KIND> struct VqKept<float, KIND> { typedef float type; };
template <> struct VqKept<VqBf16, VQL_THRESHOLD> { typedef VqBf16 type; };
// Rounded as it is kept.  A layer of fp16 keeps relu's p in fp16 too: what is above zero stays there.
template <typename T, int KIND>
__device__ __forceinline__ typename VqKept<T, KIND>::type vql_keep(float p, int act) {
  if constexpr (__is_same(T, _Float16) && KIND == VQL_THRESHOLD) {
    const float least = act == VQ_ACT_RELU ? 0x1p-24f : 0.0f;
    p = p > 0.0f && p < least ? least : p;
  }
  return VqElem<typename VqKept<T, KIND>::type>::from(p);
}
__device__ __forceinline__ float vql_kept(float p, int) { return p; }
__device__ __forceinline__ float vql_kept(_Float16 p, int) { return (float)p; }
__device__ __forceinline__ float vql_kept(VqBf16 p, int act) {
  return act == VQ_ACT_RELU ? VqElem<VqBf16>::to(p) : (float)__builtin_bit_cast(_Float16, p.v);
}
// act'(p).  Beyond |p| = 100 every derivative has its limit, 0 or 1; the clamp keeps inf * 0 out of it.
template <bool FAST>
__device__ __forceinline__ float vql_act_slope(float p0, int act) {
  float p = p0 > 100.0f ? 100.0f : p0;
  p = p < -100.0f ? -100.0f : p;   // NaN passes both
  switch (act) {
    case VQ_ACT_RELU: return p <= 0.0f ? 0.0f : 1.0f;
    case VQ_ACT_SILU: {
      const float s = vql_sigmoid<FAST>(p);
      return s * __builtin_fmaf(p, 1.0f - s, 1.0f);
    }
    case VQ_ACT_GELU: {
      const float g = FAST ? __expf(-0.5f * p * p) : expf(-0.5f * p * p);
      return __builtin_fmaf(p * 0.3989422804f, g, vql_cdf(p));
    }
    case VQ_ACT_GELU_TANH: {
      const float p2 = p * p;
      const float s = vql_sigmoid<FAST>(1.5957691216f * p * __builtin_fmaf(0.044715f, p2, 1.0f));
      const float du2 = 1.5957691216f * __builtin_fmaf(0.134145f, p2, 1.0f);
      return __builtin_fmaf(p * s * (1.0f - s), du2, s);
    }
    default: return 1.0f;
  }
}

// -------------------------------------------------------------------------------- matrix core
// One 16-byte fragment per lane of each operand.  16-bit types: lane l holds index l % 32, r = 8 (l / 32) + 0..7, one
// 32x32x16 product.  fp32: r = 4 (l / 32) + 0..3, four 32x32x2 products (each pairs r = e with r = 4 + e, the same for
// both operands).  D: lane l holds column l % 32 (of `b`), register g row 8 (g / 4) + 4 (l / 32) + g % 4 (of `a`).
template <typename T>
__device__ __forceinline__ f32x16 vql_mma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (__is_same(T, VqBf16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (__is_same(T, _Float16)) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    const f32x4 fa = __builtin_bit_cast(f32x4, a), fb = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[e], fb[e], c, 0, 0, 0);
    return c;
  }
}
template <typename T>
__device__ __forceinline__ float vql_sum16(u32x4 v) {   // sum of the fragment's elements
  float s = 0.0f;
  if constexpr (sizeof(T) == 4) {
    const f32x4 f = __builtin_bit_cast(f32x4, v);
    s = (f[0] + f[1]) + (f[2] + f[3]);
  } else {
    const VqChunk<T> c = __builtin_bit_cast(VqChunk<T>, v);
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = VqElem<T>::to(c.e[e]);
    s = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
  }
  return s;
}

// -------------------------------------------------------------------------------- operand tiles in LDS
// One step of the sum covers 128 bytes of r: 64 elements of 16 bits, 32 of 32 bits.
// r-major tile of `B` indexes: B rows of 128 bytes, 16-byte piece c of row m in slot c ^ (bits 1-3 of m): the 16 rows that a
//   fragment read touches at a time fall on all banks evenly.
// m-major tile: one row of B elements per r, 16-byte piece c of row r in slot c ^ vql_mswz<T>(r): the rows that one
//   transposing read (16 bits: r = 8h + 4t + 0..3 for both halves h) or one fp32 read (r = e and 4 + e) touches lie in
//   different 64- or 128-byte segments.
// The permutation is applied to the source address, so that the DMA, which writes LDS in lane order, needs no more.
template <typename T>
__device__ __forceinline__ int vql_mswz(int r) {
  if constexpr (sizeof(T) == 2) return ((r & 3) | ((r >> 1) & 4)) << 2;
  return ((r >> 2) & 1) << 3;
}

// Which index of a 32-block the lanes of the `b`-side operand hold: the matrix instruction leaves a lane the rows 8g + 4h + r
// (g, r = 0..3) of its column, h = lane / 32; with this order they are the indexes 16 (g / 2) + 8h + 4 (g % 2) + r: two runs
// of eight, one for each half of the 32, in which the lanes of the two halves take turns.
__device__ __forceinline__ int vql_order(int rho) { return (rho & 19) | ((rho & 4) << 1) | ((rho & 8) >> 1); }

template <typename T, bool MMAJOR, int B, int NT, bool DMA, bool ORDERED>
struct VqOperand {
  static constexpr int ES = sizeof(T), E = 16 / ES, BK = 128 / ES;
  static constexpr int BYTES = B * 128;
  static constexpr int CPR = MMAJOR ? B / E : 8;       // 16-byte pieces per row of the tile
  static constexpr int PER = BYTES / 16 / NT;          // pieces per thread
  static constexpr int SWZ = MMAJOR ? CPR - 1 : 7;
  static constexpr bool SUMS = MMAJOR;                 // only the weight gradient's A operand is summed
  const char* base;      // m-major: column m0 of row 0; r-major: row m0
  int64_t ld;            // bytes
  int64_t M, total;      // indexes that exist from m0 on, and altogether
  uint32_t off[PER];     // this lane's byte offsets of a full step

  __device__ __forceinline__ static void where(int n, int wave, int lane, int& row, int& piece) {
    const int p = (wave * PER + n) * 64 + lane;
    row = p / CPR;
    piece = (p % CPR) ^ ((MMAJOR ? vql_mswz<T>(row) : (row >> 1)) & SWZ);
  }
  __device__ __forceinline__ void init(const char* src, int64_t ld_, int64_t m0, int64_t all, int wave, int lane) {
    ld = ld_;
    total = all;
    M = all - m0;
    base = MMAJOR ? src + m0 * ES : src + m0 * ld_;
    if constexpr (DMA) {
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        int row, piece;
        where(n, wave, lane, row, piece);
        if constexpr (MMAJOR) {   // pieces behind the last index repeat the last one: those outputs are not stored
          const int last = (int)(M < B ? M : B) / E - 1;
          off[n] = (uint32_t)(row * ld) + (piece < last ? piece : last) * 16;
        } else {
          const int last = (int)(M < B ? M : B) - 1;
          off[n] = (uint32_t)((row < last ? row : last) * ld) + piece * 16;
        }
      }
    }
  }
  // a whole step (all BK values of r exist), straight into LDS: piece n of this thread's PER
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(int step) const {
    const char* p = MMAJOR ? base + step * (BK * ld) : base + step * (int64_t)128;
    return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7fffffff, 0x00020000);
  }
  __device__ __forceinline__ void dma_piece(__amdgpu_buffer_rsrc_t rs, int n, VQL_LDS char* lds, int wave) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (VQL_LDS void*)(lds + (wave * PER + n) * 1024), 16, off[n], 0, 0, 0);
  }
  __device__ __forceinline__ void dma(int step, VQL_LDS char* lds, int wave) const {
    const __amdgpu_buffer_rsrc_t rs = source(step);
#pragma unroll
    for (int n = 0; n < PER; ++n) dma_piece(rs, n, lds, wave);
  }
  // Any step, by way of registers.  All loads are 16 bytes and unconditional wherever the row has 16 bytes at all, so that
  // they are on their way together: rows that do not exist read the last one instead, a piece that passes the end of its
  // row is read from the row's last 16 bytes and shifted.  What must read as zero does (r behind the end); indexes that do
  // not exist may hold anything finite or not: they reach only outputs that are not stored.
  __device__ __forceinline__ void fetch(int step, int64_t R, int wave, int lane, u32x4 (&v)[PER]) const {
    const int64_t r0 = (int64_t)step * BK;
    const char* const tile = MMAJOR ? base + r0 * ld : base + r0 * ES;
    const int rs = (int)(R - r0 < BK ? R - r0 : BK), ms = (int)(M < B ? M : B);      // r and indexes that exist in the tile
    const int pitch = (int)ld;
    if (rs == BK && (!MMAJOR || ms == B)) {
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        int row, piece;
        where(n, wave, lane, row, piece);
        if (!MMAJOR) row = row < ms ? row : ms - 1;
        v[n] = vql_load16<T>(tile + (uint32_t)(row * pitch + piece * 16));
      }
    } else if ((MMAJOR ? total : R) >= E) {
      // a piece that passes the end of its row: from where the row's last 16 bytes start
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        int row, piece;
        where(n, wave, lane, row, piece);
        const int last = (MMAJOR ? ms : rs) - E, at = piece * E < last ? piece * E : last;
        row = row < (MMAJOR ? rs : ms) ? row : (MMAJOR ? rs : ms) - 1;
        v[n] = vql_load16<T>(tile + (row * pitch + at * ES));
      }
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        int row, piece;
        where(n, wave, lane, row, piece);
        const int over = piece * E - (MMAJOR ? ms : rs) + E;
        v[n] = vql_shift<T>(v[n], (MMAJOR && row >= rs) || over > E ? E : over > 0 ? over : 0);
      }
    } else {   // rows of less than 16 bytes
#pragma unroll
      for (int n = 0; n < PER; ++n) {
        int row, piece;
        where(n, wave, lane, row, piece);
        v[n] = fetch_part(tile, row, piece, rs, ms);
      }
    }
  }
  // one piece, element by element
  __device__ __forceinline__ u32x4 fetch_part(const char* tile, int row, int piece, int rs, int ms) const {
    const bool exists = row < (MMAJOR ? rs : ms);
    const int have = exists ? (MMAJOR ? ms : rs) - piece * E : 0;
    const char* p = tile + (uint32_t)(exists ? row * (int)ld + piece * 16 : 0);
    u32x4 v = {0, 0, 0, 0};
#pragma unroll 1
    for (int e = (have < E ? have : E) - 1; e >= 0; --e) {   // from the last element on, each moving the others up
      if constexpr (ES == 4) {
        v = u32x4{*reinterpret_cast<const vql_u32*>(p + 4 * e), v[0], v[1], v[2]};
      } else {
        const uint32_t x = *reinterpret_cast<const vql_u16*>(p + 2 * e);
        v = u32x4{v[0] << 16 | x, v[1] << 16 | v[0] >> 16, v[2] << 16 | v[1] >> 16, v[3] << 16 | v[2] >> 16};
      }
    }
    return v;
  }
  // a step that is not a whole one, into LDS piece by piece: once in a sum, and with few registers
  __device__ __forceinline__ void fill_part(int step, int64_t R, VQL_LDS char* lds, int wave, int lane) const {
    const int64_t r0 = (int64_t)step * BK;
    const char* const tile = MMAJOR ? base + r0 * ld : base + r0 * ES;
    const int rs = (int)(R - r0 < BK ? R - r0 : BK), ms = (int)(M < B ? M : B);
#pragma unroll 1
    for (int n = 0; n < PER; ++n) {
      int row, piece;
      where(n, wave, lane, row, piece);
      const int have = row < (MMAJOR ? rs : ms) ? (MMAJOR ? ms : rs) - piece * E : 0;
      u32x4 v;
      if (have >= E) v = vql_load16<T>(tile + (uint32_t)(row * (int)ld + piece * 16));
      else v = fetch_part(tile, row, piece, rs, ms);
      *reinterpret_cast<VQL_LDS vql_u32x4_a16*>(lds + ((wave * PER + n) * 64 + lane) * 16) = v;
    }
  }
  __device__ __forceinline__ void commit(VQL_LDS char* lds, int wave, int lane, const u32x4 (&v)[PER]) const {
#pragma unroll
    for (int n = 0; n < PER; ++n) *reinterpret_cast<VQL_LDS vql_u32x4_a16*>(lds + ((wave * PER + n) * 64 + lane) * 16) = v[n];
  }
  // fragment of indexes m .. m + 31 for the q-th quarter of the step
  __device__ __forceinline__ static u32x4 frag(const VQL_LDS char* lds, int m, int q, int lane) {
    const int h = lane >> 5;
    if constexpr (!MMAJOR) {
      const int rho = lane & 31, row = m + (ORDERED ? vql_order(rho) : rho);
      return *reinterpret_cast<const VQL_LDS vql_u32x4_a16*>(lds + row * 128 + (((2 * q + h) ^ ((row >> 1) & 7)) * 16));
    } else if constexpr (ES == 2) {
      // transposing read: each group of 16 lanes names 4 rows (r) of 16 consecutive indexes, 8 bytes a lane, and lane i
      // of the group receives index i of the four rows
      const int s = lane & 15, rho = (lane & 16) + (s & 3) * 4, col = m + (ORDERED ? vql_order(rho) : rho);
      s16x4 half[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 16 * q + 8 * h + 4 * t + (s >> 2);
        const int at = r * (B * 2) + ((((col >> 3) ^ (vql_mswz<T>(r) & SWZ)) * 16) | ((col & 4) * 2));
        half[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((VQL_LDS s16x4*)(lds + at));
      }
      typedef short s16x8 __attribute__((ext_vector_type(8)));
      return __builtin_bit_cast(u32x4, (s16x8)__builtin_shufflevector(half[0], half[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      u32x4 v;
      const int rho = lane & 31, col = m + (ORDERED ? vql_order(rho) : rho);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 8 * q + 4 * h + e;
        v[e] = *reinterpret_cast<const VQL_LDS vql_u32*>(lds + r * (B * 4) + ((((col >> 2) ^ (vql_mswz<T>(r) & SWZ)) * 16) | ((col & 3) * 4)));
      }
      return v;
    }
  }
};

// -------------------------------------------------------------------------------- epilogue
// out = act(c + bias) + residual, rounded once, for 16 / sizeof(T) columns; pre = c + bias (kept for the activation's
// gradient); res: the residual's 16 bytes.
template <typename T, int KIND>
__device__ __forceinline__ void vql_finish(const VqLinearArgs& a, const float* c, const float* bias, u32x4 res, u32x4& out, u32x4& pre) {
  constexpr int E = 16 / sizeof(T);
  typedef typename VqKept<T, KIND>::type Kept;
  float p[E];
  VqChunk<T> y;
  VqChunk<Kept> kept;
  if constexpr (KIND == VQL_PLAIN) {
#pragma unroll
    for (int e = 0; e < E; ++e) y.e[e] = VqElem<T>::from(c[e]);
    out = __builtin_bit_cast(u32x4, y);
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) p[e] = c[e] + bias[e];
  if (a.pre) {
#pragma unroll
    for (int e = 0; e < E; ++e) kept.e[e] = vql_keep<T, KIND>(p[e], a.act);
    pre = __builtin_bit_cast(u32x4, kept);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) p[e] = vql_act_of<KIND, sizeof(T) == 2>(p[e], a.act);
  if (a.res) {
    const VqChunk<T> r = __builtin_bit_cast(VqChunk<T>, res);
#pragma unroll
    for (int e = 0; e < E; ++e) p[e] += VqElem<T>::to(r.e[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) y.e[e] = VqElem<T>::from(p[e]);
  out = __builtin_bit_cast(u32x4, y);
}
// bias[j .. j + W), zero where there is none
template <typename T, int W>
__device__ __forceinline__ void vql_bias(const VqLinearArgs& a, int64_t j, float (&bias)[W]) {
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int e = 0; e < W; ++e) bias[e] = 0.0f;
  if (a.bias) {
#pragma unroll
    for (int k = 0; k < W / E; ++k) {
      const VqChunk<T> b = __builtin_bit_cast(
          VqChunk<T>, vql_load16_part<T>(reinterpret_cast<const char*>(a.bias) + (j + k * E) * (int64_t)sizeof(T), a.J - j - k * E));
#pragma unroll
      for (int e = 0; e < E; ++e) bias[k * E + e] = VqElem<T>::to(b.e[e]);
    }
  }
}
// First column, within a 32x32 tile, of the k-th 16 bytes that a lane of half h holds of its row (see vql_order).
template <typename T>
__device__ __forceinline__ int vql_piece(int k, int h) {
  return sizeof(T) == 2 ? 16 * k + 8 * h : 16 * (k >> 1) + 8 * h + 4 * (k & 1);
}
// The epilogue of what one lane holds of one tile: row r, the columns of its pieces from cv on.  What does not exist is
// left out.
template <typename T, int KIND, typename C>
__device__ __forceinline__ void vql_write_lane(const VqLinearArgs& a, int64_t r, int64_t cv, int h, const C& c) {
  constexpr int ES = sizeof(T), E = 16 / ES;
#pragma unroll
  for (int k = 0; k < 16 / E; ++k) {
    const int64_t col = cv + vql_piece<T>(k, h), left = a.J - col, at = (r * a.J + col) * ES;
    if (r >= a.I || left <= 0) continue;
    float bias[E], v[E];
    if (KIND != VQL_PLAIN) vql_bias<T, E>(a, col, bias);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = c[k * E + e];
    u32x4 res = {0, 0, 0, 0}, y, pre;
    if (KIND != VQL_PLAIN && a.res) res = vql_load16_part<T>(a.res + r * a.ldr + col * ES, left);
    vql_finish<T, KIND>(a, v, bias, res, y, pre);
    vql_store16_part<T>(reinterpret_cast<char*>(a.out) + at, y, left);
    if (KIND != VQL_PLAIN && a.pre) vql_store16_part<T>(reinterpret_cast<char*>(a.pre) + at, pre, left);
  }
}
// Exchanges 16-lane rows: a lane with bit 4 clear keeps p and gets its neighbour's (lane + 16) p as q, one with bit 4 set keeps
// q and gets its neighbour's q as p.  Its own inverse.
__device__ __forceinline__ void vql_swap16(u32x4& p, u32x4& q) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto both = __builtin_amdgcn_permlane16_swap(p[e], q[e], false, false);
    p[e] = both[0];
    q[e] = both[1];
  }
}
// The bias of a wave's part of a block as vql_write takes it, zero where there is none; asked for early, since nothing else of
// the epilogue waits for memory.
template <typename T, int TJ>
__device__ __forceinline__ void vql_ask_bias(const VqLinearArgs& a, int64_t j, int h, u32x4 (&bias_of)[TJ][16 * sizeof(T) / 16]) {
  const char* p = reinterpret_cast<const char*>(a.bias) + j * (int64_t)sizeof(T);
#pragma unroll
  for (int v = 0; v < TJ; ++v)
#pragma unroll
    for (int k = 0; k < (int)(16 * sizeof(T) / 16); ++k)
      bias_of[v][k] = a.bias ? vql_load16<T>(p + (v * 32 + vql_piece<T>(k, h)) * (int)sizeof(T)) : u32x4{0, 0, 0, 0};
}
// The epilogue of a wave's part of a block: rows i .. i + 32 TI, columns j .. j + 32 TJ, all of which exist.  A lane holds 32
// or 64 bytes of one row in pieces of 16; exchanging every other piece with the lane 16 away makes one access of the wave 64
// consecutive bytes of 16 rows instead of twice 16 bytes of 32 rows (64 Ki x 256 -> 1024 bf16: 52 instead of 59 us: the L2 takes
// a request per line and instruction).  The residual of the next tile is on its way while this one is worked on.  Past the caches
// the tiles of a column of them follow each other; in the caches those of a row, so that runs which straddle lines meet again soon
// (64 Ki x 256 -> 1000 bf16 with p kept: 118 instead of 154 us; past the caches 77 and 78).
template <typename T, int KIND, bool STREAM, int TI, int TJ>
__device__ __forceinline__ void vql_write(const VqLinearArgs& a, int64_t i, int64_t j, int lane, const u32x4 (&bias_of)[TJ][16 * sizeof(T) / 16],
                                          const f32x16 (&acc)[TI][TJ]) {
  constexpr int ES = sizeof(T), E = 16 / ES, PV = 16 / E;
  const int h = lane >> 5;
  // One wave-uniform address per tensor and one 32-bit offset per lane: row lane % 16, and the first or second piece of a pair.
  const int64_t pitch = (int64_t)a.J * ES, origin = i * pitch + j * ES;
  char* const yb = reinterpret_cast<char*>(a.out) + origin;
  char* const pb = reinterpret_cast<char*>(a.pre) + origin;
  const char* const rb = a.res + i * a.ldr + j * ES;
  const int lc = vql_piece<T>((lane >> 4) & 1, h) * ES;
  const uint32_t yo = (uint32_t)((lane & 15) * (int)pitch + lc), ro = (uint32_t)((lane & 15) * (int)a.ldr + lc);
  constexpr auto row_of = [](int t) constexpr { return STREAM ? t % TI : t / TJ; };
  constexpr auto col_of = [](int t) constexpr { return STREAM ? t / TI : t % TJ; };
  u32x4 res[2][PV];
  auto load = [&](int t, u32x4 (&to)[PV]) {
#pragma unroll
    for (int k = 0; k < PV; k += 2) {
      const char* p = rb + (int64_t)row_of(t) * 32 * a.ldr + (col_of(t) * 32 + 8 * k) * ES + ro;
      to[k] = vql_load16<T>(p);
      to[k + 1] = vql_load16<T>(p + 16 * a.ldr);
    }
  };
  if (KIND != VQL_PLAIN && a.res) load(0, res[0]);
#pragma unroll
  for (int t = 0; t < TI * TJ; ++t) {
    const int u = row_of(t), v = col_of(t);
    if (KIND != VQL_PLAIN && a.res && t + 1 < TI * TJ) load(t + 1, res[(t + 1) & 1]);
#pragma unroll
    for (int k = 0; k < PV; k += 2) {
      u32x4 y[2], pre[2];
      if (KIND != VQL_PLAIN && a.res) vql_swap16(res[t & 1][k], res[t & 1][k + 1]);
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        float c[E], bias[E];
        const VqChunk<T> b = __builtin_bit_cast(VqChunk<T>, bias_of[v][k + w]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          c[e] = acc[u][v][(k + w) * E + e];
          bias[e] = KIND == VQL_PLAIN ? 0.0f : VqElem<T>::to(b.e[e]);
        }
        vql_finish<T, KIND>(a, c, bias, res[t & 1][k + w], y[w], pre[w]);
      }
      const int64_t step = (int64_t)u * 32 * pitch + (v * 32 + 8 * k) * ES;
      vql_swap16(y[0], y[1]);
      vql_stream16<T, STREAM>(yb + step + yo, y[0]);
      vql_stream16<T, STREAM>(yb + step + 16 * pitch + yo, y[1]);
      if (KIND != VQL_PLAIN && a.pre) {
        vql_swap16(pre[0], pre[1]);
        vql_stream16<T, STREAM>(pb + step + yo, pre[0]);
        vql_stream16<T, STREAM>(pb + step + 16 * pitch + yo, pre[1]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

// -------------------------------------------------------------------------------- one step
// The lane number as a value that the compiler knows nothing about: what is computed from it inside a loop stays there,
// instead of taking up registers all through the kernel.
__device__ __forceinline__ int vql_fresh(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}
template <int TI, int TJ>
struct VqFrags {
  u32x4 a[TI], b[TJ];
};
template <typename OA, typename OB, int TI, int TJ>
__device__ __forceinline__ void vql_read(VqFrags<TI, TJ>& f, const VQL_LDS char* tile, int q, int wi, int wj, int lane) {
#pragma unroll
  for (int u = 0; u < TI; ++u) f.a[u] = OA::frag(tile, (wi * TI + u) * 32, q, lane);
#pragma unroll
  for (int v = 0; v < TJ; ++v) f.b[v] = OB::frag(tile + OA::BYTES, (wj * TJ + v) * 32, q, lane);
}
template <typename T, bool SUMS, int TI, int TJ>
__device__ __forceinline__ void vql_add(const VqFrags<TI, TJ>& f, bool want_sum, float (&asum)[TI]) {
  if (SUMS && want_sum) {
#pragma unroll
    for (int u = 0; u < TI; ++u) asum[u] += vql_sum16<T>(f.a[u]);
  }
}
template <typename T, bool SUMS, int TI, int TJ>
__device__ __forceinline__ void vql_mul(const VqFrags<TI, TJ>& f, bool want_sum, f32x16 (&acc)[TI][TJ], float (&asum)[TI]) {
#pragma unroll
  for (int u = 0; u < TI; ++u)
#pragma unroll
    for (int v = 0; v < TJ; ++v) acc[u][v] = vql_mma<T>(f.b[v], f.a[u], acc[u][v]);
  vql_add<T, SUMS, TI, TJ>(f, want_sum, asum);
}
// Waits until this wave's LDS accesses are done and at most N of its DMA instructions are in flight (`counted`; else
// none), then for the other waves.  A bare barrier: nothing else has to have landed.
template <int N>
__device__ __forceinline__ void vql_publish(bool counted) {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xC07F);                                        // lgkmcnt(0)
  if (N > 0 && counted) __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));   // vmcnt(N)
  else __builtin_amdgcn_s_waitcnt(0x0F70);                                   // vmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// The same behind an epilogue, whose stores are younger than the DMA of the next block's first tiles: `young` of them
// need not have landed either (0, S, 2 S or P; vmcnt counts to 63).
template <int N, int S, int P>
__device__ __forceinline__ void vql_publish_young(bool counted, int young) {
  constexpr auto code = [](int n) constexpr { return 0x0F70 | ((n < 63 ? n : 63) & 15) | (((n < 63 ? n : 63) >> 4) << 14); };
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xC07F);
  if (!counted) __builtin_amdgcn_s_waitcnt(0x0F70);
  else if (young == S) __builtin_amdgcn_s_waitcnt(code(N + S));
  else if (young == 2 * S) __builtin_amdgcn_s_waitcnt(code(N + 2 * S));
  else if (young == P) __builtin_amdgcn_s_waitcnt(code(N + P));
  else __builtin_amdgcn_s_waitcnt(code(N));
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// the same for waves that fill LDS through registers: loads may be in flight
__device__ __forceinline__ void vql_publish_lds() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xC07F);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// One step of the sum: the tiles of this step at from + cur, those of the next at from + nxt.  In registers there are two
// sets of fragments, one read while the other is multiplied, so that neither the LDS reads nor the barrier of a step leave
// the matrix cores idle:
//     q0 | read q1, multiply q0 | read q2, multiply q1 | read q3, multiply q2 | barrier, fill, read the next q0, multiply q3
// `counted`: FLYING of this wave's DMA instructions, those behind the next step's, may still be in flight.  `into` and `from`
// are the same memory; __restrict__ tells the compiler that a fragment read need not wait for the DMA in flight: the
// barriers and the counted waits see to that.
template <typename T, typename OA, typename OB, int TI, int TJ, int FLYING, int S, int P>
__device__ __forceinline__ void vql_step(const OA& oa, const OB& ob, int dma_step, bool dma, bool pending, bool more, bool counted,
                                         int young,
                                         VQL_LDS char* __restrict__ into, const VQL_LDS char* __restrict__ from, int cur, int nxt, int prev,
                                         int wi, int wj, int wave, int lane, bool want_sum, VqFrags<TI, TJ> (&f)[2],
                                         f32x16 (&acc)[TI][TJ], float (&asum)[TI]) {
  constexpr int PIECES = OA::PER + OB::PER, FIRST = PIECES / 2, PROD = TI * TJ;
  auto piece = [&](__amdgpu_buffer_rsrc_t ra, __amdgpu_buffer_rsrc_t rb, int k, VQL_LDS char* to) {
    if (k < OA::PER) oa.dma_piece(ra, k, to, wave);
    else ob.dma_piece(rb, k - OA::PER, to + OA::BYTES, wave);
  };
  {
    vql_read<OA, OB, TI, TJ>(f[1], from + cur, 1, wi, wj, lane);
    __builtin_amdgcn_sched_barrier(0);
    const __amdgpu_buffer_rsrc_t ra = oa.source(dma_step - 1), rb = ob.source(dma_step - 1);
    constexpr int N = PIECES - FIRST, EACH = (N + PROD - 1) / PROD;
#pragma unroll
    for (int m = 0; m < PROD; ++m) {
      acc[m / TJ][m % TJ] = vql_mma<T>(f[0].b[m % TJ], f[0].a[m / TJ], acc[m / TJ][m % TJ]);
      if (pending && m * EACH < N) {
#pragma unroll
        for (int k = m * EACH; k < (m + 1) * EACH && k < N; ++k) piece(ra, rb, FIRST + k, into + prev);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    vql_add<T, OA::SUMS, TI, TJ>(f[0], want_sum, asum);
  }
#pragma unroll
  for (int q = 1; q < 3; ++q) {
    vql_read<OA, OB, TI, TJ>(f[(q + 1) & 1], from + cur, q + 1, wi, wj, lane);
    __builtin_amdgcn_sched_barrier(0);
    vql_mul<T, OA::SUMS, TI, TJ>(f[q & 1], want_sum, acc, asum);
    __builtin_amdgcn_sched_barrier(0);
  }
  vql_publish_young<FLYING, S, P>(counted, young);
  if (more) vql_read<OA, OB, TI, TJ>(f[0], from + nxt, 0, wi, wj, lane);
  __builtin_amdgcn_sched_barrier(0);
  // the DMA instructions one by one between the products
  const __amdgpu_buffer_rsrc_t ra = oa.source(dma_step), rb = ob.source(dma_step);
  constexpr int EACH = (FIRST + PROD - 1) / PROD;
#pragma unroll
  for (int m = 0; m < TI * TJ; ++m) {
    acc[m / TJ][m % TJ] = vql_mma<T>(f[1].b[m % TJ], f[1].a[m / TJ], acc[m / TJ][m % TJ]);
    if (dma && m * EACH < FIRST) {
#pragma unroll
      for (int k = m * EACH; k < (m + 1) * EACH && k < FIRST; ++k) piece(ra, rb, k, into + cur);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  vql_add<T, OA::SUMS, TI, TJ>(f[1], want_sum, asum);
}

// The same for the 128x128 tile, whose quarters have four products a wave (128 cycles, less than the latency of an LDS read under
// load): fragments are read two quarters ahead, and the barrier lies in the middle of a step, with two quarters to multiply
// behind it.  f[0] and f[1] hold the step's first two quarters on entry, and the next step's on return.  Against one quarter ahead,
// one workgroup on a CU: forward 0.72 -> 0.69 us a step, weight gradient 0.85 -> 0.78 (64 Ki x 1024 x 256 bf16 68 -> 65 us), input gradient
// 0.72 -> 0.76; fp32 2.02 -> 1.97.  The 256 tile has no registers for it.
template <typename T, typename OA, typename OB, int TI, int TJ, int FLYING, int S, int P>
__device__ __forceinline__ void vql_step_ahead(const OA& oa, const OB& ob, int dma_step, bool dma, bool more, bool counted, int young,
                                               VQL_LDS char* __restrict__ into, const VQL_LDS char* __restrict__ from, int cur, int nxt,
                                               int wi, int wj, int wave, int lane, bool want_sum, VqFrags<TI, TJ> (&f)[4],
                                               f32x16 (&acc)[TI][TJ], float (&asum)[TI]) {
  constexpr int PIECES = OA::PER + OB::PER, PROD = TI * TJ, EACH = (PIECES + 2 * PROD - 1) / (2 * PROD);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    vql_read<OA, OB, TI, TJ>(f[q + 2], from + cur, q + 2, wi, wj, lane);
    __builtin_amdgcn_sched_barrier(0);
    vql_mul<T, OA::SUMS, TI, TJ>(f[q], want_sum, acc, asum);
    __builtin_amdgcn_sched_barrier(0);
  }
  vql_publish_young<FLYING, S, P>(counted, young);
  const __amdgpu_buffer_rsrc_t ra = oa.source(dma_step), rb = ob.source(dma_step);
#pragma unroll
  for (int q = 2; q < 4; ++q) {
    if (more) vql_read<OA, OB, TI, TJ>(f[q - 2], from + nxt, q - 2, wi, wj, lane);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < PROD; ++m) {
      acc[m / TJ][m % TJ] = vql_mma<T>(f[q].b[m % TJ], f[q].a[m / TJ], acc[m / TJ][m % TJ]);
      if (dma) {
#pragma unroll
        for (int k = ((q - 2) * PROD + m) * EACH; k < ((q - 2) * PROD + m + 1) * EACH && k < PIECES; ++k) {
          if (k < OA::PER) oa.dma_piece(ra, k, into + cur, wave);
          else ob.dma_piece(rb, k - OA::PER, into + cur + OA::BYTES, wave);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    vql_add<T, OA::SUMS, TI, TJ>(f[q], want_sum, asum);
  }
}

// Two steps of the sum for the 64x64 tile, whose quarters have one product a wave (32 cycles, the latency of an LDS read is
// some 150): the fragments of the whole next step are read while this one is multiplied.  A step takes 0.30 us instead of
// 0.34 with one workgroup on a CU; with four products a quarter (tile 128) it takes 0.80 instead of 0.72, the reads delaying
// the first product.  f[0] holds step s on entry, and step s + 2 on return.
template <typename T, typename OA, typename OB, int TI, int TJ, int NS>
__device__ __forceinline__ void vql_two_steps(const OA& oa, const OB& ob, int s, int s1, int last_dma, int64_t R,
                                              VQL_LDS char* __restrict__ into, const VQL_LDS char* __restrict__ from, int& at,
                                              int wi, int wj, int wave, int lane, bool want_sum, VqFrags<TI, TJ> (&f)[2][4],
                                              f32x16 (&acc)[TI][TJ], float (&asum)[TI]) {
  constexpr int PIECES = OA::PER + OB::PER, STAGE = OA::BYTES + OB::BYTES;
#pragma unroll
  for (int half = 0; half < 2; ++half, ++s) {
    if (s >= s1) break;
    const int cur = at * STAGE;
    at = at + 1 == NS ? 0 : at + 1;
    vql_publish<(NS - 2) * PIECES>(s + NS <= last_dma);   // all of the steps on their way (to s + NS - 1) but those behind s + 1
    if (s + 1 < s1) {
#pragma unroll
      for (int q = 0; q < 4; ++q) vql_read<OA, OB, TI, TJ>(f[half ^ 1][q], from + at * STAGE, q, wi, wj, lane);
    }
    __builtin_amdgcn_sched_barrier(0);
    const bool dma = s + NS < last_dma;
    const __amdgpu_buffer_rsrc_t ra = oa.source(s + NS), rb = ob.source(s + NS);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      vql_mul<T, OA::SUMS, TI, TJ>(f[half][q], want_sum, acc, asum);
      if (dma) {   // a quarter of the DMA instructions behind each quarter's products
#pragma unroll
        for (int k = q * PIECES / 4; k < (q + 1) * PIECES / 4; ++k) {
          if (k < OA::PER) oa.dma_piece(ra, k, into + cur, wave);
          else ob.dma_piece(rb, k - OA::PER, into + cur + OA::BYTES, wave);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!dma && s + NS < s1) {   // a step that is not a whole one
      const int l = vql_fresh(lane);
      oa.fill_part(s + NS, R, into + cur, wave, l);
      ob.fill_part(s + NS, R, into + cur + OA::BYTES, wave, l);
    }
  }
}

// -------------------------------------------------------------------------------- the product
namespace {   // the kernels of a translation unit are its own
// A workgroup of WI x WJ waves owns a BI x BJ block of C (and, with splits, a range of the sum); a wave owns
// (BI / WI) x (BJ / WJ) of it in 32x32 accumulator tiles.  DMA: rows start on 16 bytes, so that the tiles go straight into
// LDS; otherwise they go through registers.
// What bounds it (operands out of the caches): 8192 x 4096 -> 4096 bf16 with residual 242 us, 1.14 PFLOP/s, the matrix cores at the
// clock they hold; 64 Ki x 256 -> 1024 bf16 54 us, 3.1 TB/s, with gelu_tanh 63: products, stores and the activation one
// after the other in part; 16384 x 2048 -> 1024 fp32 480 us, 143 TFLOP/s, the matrix cores.
template <typename T, bool AMM, bool BMM, int KIND, int BI, int BJ, int WI, int WJ, int NS, bool DMA>
__global__ __launch_bounds__(WI * WJ * 64, 2) void vql_product_kernel(VqLinearArgs a) {
  constexpr int NT = WI * WJ * 64;
  constexpr int TI = BI / WI / 32, TJ = BJ / WJ / 32;
  constexpr int STAGE = (BI + BJ) * 128;
  typedef VqOperand<T, AMM, BI, NT, DMA, false> OA;
  typedef VqOperand<T, BMM, BJ, NT, DMA, true> OB;
  extern __shared__ __attribute__((aligned(16))) char vql_lds[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave / WJ, wj = wave % WJ;

  const int tiles_i = (int)a.tiles_i, per_split = tiles_i * a.tiles_j, total = per_split * a.splits;   // at most MAX_BLOCKS
  const int steps = (int)((a.R + OA::BK - 1) / OA::BK), full = (int)(a.R / OA::BK);
  VQL_LDS char* lds = (VQL_LDS char*)vql_lds;
  OA oa;
  OB ob;
  int split = 0, tj0 = 0;
  int64_t i0 = 0, j0 = 0;
  int s0 = 0, s1 = 0;

  // Consecutive workgroups go to the 8 dies in turn: give each die a contiguous range of blocks, and walk the range in
  // groups of 8 block rows, so that the blocks in flight on a die share their operands in its L2.
  auto choose = [&](int n) {
    const int q8 = total >> 3, r8 = total & 7, x8 = n & 7;
    int id = x8 * q8 + (x8 < r8 ? x8 : r8) + (n >> 3);
    split = a.splits == 1 ? 0 : id / per_split;
    id -= split * per_split;
    const int group = id / (8 * a.tiles_j), first = group * 8;
    const int gsz = tiles_i - first < 8 ? tiles_i - first : 8;
    id -= first * a.tiles_j;
    tj0 = gsz == 8 ? id >> 3 : id / gsz;
    i0 = (int64_t)(first + id - tj0 * gsz) * BI;
    j0 = (int64_t)tj0 * BJ;
    s0 = split * a.steps_per_split;
    s1 = steps - s0 < a.steps_per_split ? steps : s0 + a.steps_per_split;
    const int l = vql_fresh(lane);
    oa.init(a.A, a.lda, i0, a.I, wave, l);
    ob.init(a.B, a.ldb, j0, a.J, wave, l);
  };
  auto by_registers = [&](int s, int at) {
    const int l = vql_fresh(lane);
    oa.fill_part(s, a.R, lds + at, wave, l);
    ob.fill_part(s, a.R, lds + at + OA::BYTES, wave, l);
  };
  // NS tile pairs lie in LDS; the one that a step has used up is filled for the step NS later, by DMA where that step is a
  // whole one, through registers otherwise.  The first NS steps: the whole ones early (under the epilogue of the block
  // before, whose accumulators leave no registers for the others), the rest late.
  auto begin_early = [&]() {
    if constexpr (DMA) {
#pragma unroll
      for (int k = 0; k < NS; ++k)
        if (s0 + k < s1 && s0 + k < full) {
          oa.dma(s0 + k, lds + k * STAGE, wave);
          ob.dma(s0 + k, lds + k * STAGE + OA::BYTES, wave);
        }
    }
  };
  auto begin_late = [&]() {
    if constexpr (DMA) {
#pragma unroll 1
      for (int k = 0; k < NS; ++k)
        if (s0 + k < s1 && s0 + k >= full) by_registers(s0 + k, k * STAGE);
    }
  };

  // stores of a wave's epilogue: of one tensor, where the whole block exists, and of a partial sum
  constexpr int S = TI * TJ * (16 * (int)sizeof(T) / 16), P = TI * TJ * 4;
  int young = 0;
  int n = blockIdx.x;
  choose(n);
  begin_early();
  for (;;) {
    begin_late();
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int u = 0; u < TI; ++u)
#pragma unroll
      for (int v = 0; v < TJ; ++v)
#pragma unroll
        for (int g = 0; g < 16; ++g) acc[u][v][g] = 0.0f;
    const bool want_sum = AMM && (a.asum || a.gbias) && tj0 == 0 && wj == 0;
    float asum[TI];
#pragma unroll
    for (int u = 0; u < TI; ++u) asum[u] = 0.0f;

    if (s0 < s1) {
      if constexpr (DMA) {
        const int last_dma = s1 < full ? s1 : full;      // steps from here on are filled through registers
        vql_publish_young<(NS - 1) * (OA::PER + OB::PER), S, P>(s0 + NS <= last_dma, young);
        int at = 0;
        if constexpr (TI * TJ == 1) {
          VqFrags<TI, TJ> f[2][4];
#pragma unroll
          for (int q = 0; q < 4; ++q) vql_read<OA, OB, TI, TJ>(f[0][q], lds, q, wi, wj, lane);
          for (int s = s0; s < s1; s += 2)
            vql_two_steps<T, OA, OB, TI, TJ, NS>(oa, ob, s, s1, last_dma, a.R, lds, lds, at, wi, wj, wave, lane, want_sum, f, acc, asum);
        } else if constexpr (TI * TJ == 4) {
          VqFrags<TI, TJ> f[4];
#pragma unroll
          for (int q = 0; q < 2; ++q) vql_read<OA, OB, TI, TJ>(f[q], lds, q, wi, wj, vql_fresh(lane));
          for (int s = s0; s < s1; ++s) {
            const int cur = at * STAGE;
            at = at + 1 == NS ? 0 : at + 1;
            vql_step_ahead<T, OA, OB, TI, TJ, (NS - 2) * (OA::PER + OB::PER), S, P>(
                oa, ob, s + NS, s + NS < last_dma, s + 1 < s1, s + NS - 1 < last_dma, s == s0 ? young : 0, lds, lds, cur, at * STAGE,
                wi, wj, wave, lane, want_sum, f, acc, asum);
            if (s + NS < s1 && s + NS >= last_dma) by_registers(s + NS, cur);
          }
        } else {
          VqFrags<TI, TJ> f[2];
          vql_read<OA, OB, TI, TJ>(f[0], lds, 0, wi, wj, vql_fresh(lane));
          for (int s = s0; s < s1; ++s) {
            const int cur = at * STAGE, prev = at == 0 ? (NS - 1) * STAGE : cur - STAGE;
            at = at + 1 == NS ? 0 : at + 1;
            vql_step<T, OA, OB, TI, TJ, (NS - 2) * (OA::PER + OB::PER), S, P>(
                oa, ob, s + NS, s + NS < last_dma, s > s0 && s + NS - 1 < last_dma, s + 1 < s1, s + NS - 1 < last_dma,
                s == s0 ? young : 0, lds, lds,
                cur, at * STAGE, prev, wi, wj, wave, lane, want_sum, f, acc, asum);
            if (s + NS < s1 && s + NS >= last_dma) by_registers(s + NS, cur);
          }
        }
      } else {
        // the same steps with two buffers; the tiles of the next step wait in registers while this one is worked on
        VqFrags<TI, TJ> f[2];
        u32x4 va[OA::PER], vb[OB::PER];
        auto fetch = [&](int s) {
          const int l = vql_fresh(lane);
          oa.fetch(s, a.R, wave, l, va);
          ob.fetch(s, a.R, wave, l, vb);
        };
        fetch(s0);
        oa.commit(lds, wave, lane, va);
        ob.commit(lds + OA::BYTES, wave, lane, vb);
        if (s0 + 1 < s1) fetch(s0 + 1);
        vql_publish_lds();
        vql_read<OA, OB, TI, TJ>(f[0], lds, 0, wi, wj, lane);
        int cur = 0;
        for (int s = s0; s < s1; ++s) {
#pragma unroll
          for (int q = 0; q < 3; ++q) {
            vql_read<OA, OB, TI, TJ>(f[(q + 1) & 1], lds + cur, q + 1, wi, wj, lane);
            __builtin_amdgcn_sched_barrier(0);
            vql_mul<T, OA::SUMS, TI, TJ>(f[q & 1], want_sum, acc, asum);
            __builtin_amdgcn_sched_barrier(0);
          }
          cur ^= STAGE;
          if (s + 1 < s1) {
            oa.commit(lds + cur, wave, lane, va);
            ob.commit(lds + cur + OA::BYTES, wave, lane, vb);
          }
          vql_publish_lds();
          if (s + 2 < s1) fetch(s + 2);
          if (s + 1 < s1) vql_read<OA, OB, TI, TJ>(f[0], lds + cur, 0, wi, wj, lane);
          __builtin_amdgcn_sched_barrier(0);
          vql_mul<T, OA::SUMS, TI, TJ>(f[1], want_sum, acc, asum);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }

    // What this block needs from here on; its LDS buffers are free (every wave has passed the last step's barrier), so that
    // the next block's first tiles are on their way under the epilogue.
    const int64_t iw = i0 + wi * TI * 32, jw = j0 + wj * TJ * 32;
    const bool inside = i0 + BI <= a.I && j0 + BJ <= a.J;
    const int64_t this_split = split, this_block = i0 / BI * a.tiles_j + tj0;
    n += gridDim.x;
    const bool more = n < total;
    u32x4 bias_of[TJ][16 * sizeof(T) / 16];
    if (KIND != VQL_PLAIN && inside && a.splits == 1) vql_ask_bias<T, TJ>(a, jw, vql_fresh(lane) >> 5, bias_of);
    if (more) {
      choose(n);
      begin_early();
    }

    if (AMM && want_sum) {
#pragma unroll
      for (int u = 0; u < TI; ++u) {
        const float s = asum[u] + __shfl_xor(asum[u], 32);
        const int64_t i = iw + u * 32 + (lane & 31);
        if (lane < 32 && i < a.I) {
          if (a.splits > 1) ((VQL_GLOBAL float*)a.asum)[this_split * a.I + i] = s;
          else if constexpr (sizeof(T) == 4) ((VQL_GLOBAL float*)a.gbias)[i] = s;   // the two may become one store: to a global address
          else reinterpret_cast<T*>(a.gbias)[i] = VqElem<T>::from(s);
        }
      }
    }
    if (a.splits > 1) {
      // as the registers lie, 1 KiB an instruction: [split][block][wave][32x32 tile][4 groups of 4 columns][lane][4]
      float* to = a.part + ((this_split * per_split + this_block) * WI * WJ + wave) * (TI * TJ * 1024) + vql_fresh(lane) * 4;
#pragma unroll
      for (int u = 0; u < TI; ++u)
#pragma unroll
        for (int v = 0; v < TJ; ++v)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 w = {acc[u][v][4 * g], acc[u][v][4 * g + 1], acc[u][v][4 * g + 2], acc[u][v][4 * g + 3]};
            *reinterpret_cast<vql_f32x4*>(to + ((u * TJ + v) * 4 + g) * 256) = w;
          }
    } else if (inside) {
      const uintptr_t runs = reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.pre) | (a.J * sizeof(T));
      if (sizeof(T) == 2 && (runs & 63) == 0) {
        asm volatile("; a block that starts unlike the other: else what both begin with is kept in registers, which spill");
        vql_write<T, KIND, true, TI, TJ>(a, iw, jw, vql_fresh(lane), bias_of, acc);
      } else {
        vql_write<T, KIND, false, TI, TJ>(a, iw, jw, vql_fresh(lane), bias_of, acc);
      }
    } else {
      const int l = vql_fresh(lane);
#pragma unroll
      for (int u = 0; u < TI; ++u)
#pragma unroll
        for (int v = 0; v < TJ; ++v) vql_write_lane<T, KIND>(a, iw + u * 32 + (l & 31), jw + v * 32, l >> 5, acc[u][v]);
    }
    young = a.splits > 1 ? P : inside ? (KIND != VQL_PLAIN && a.pre ? 2 * S : S) : 0;
    if (!more) break;
  }
}

}  // namespace

// Launches the product of one element type: layout 0 = forward, 1 = input gradient, 2 = weight gradient.
int vql_product_f32(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s);
int vql_product_bf16(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s);
int vql_product_f16(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s);

namespace {
// One kernel of the family: its entry in the table of kernels with large LDS, and its launch.
template <typename T, bool AMM, bool BMM, int KIND, int BI, int BJ, int WI, int WJ, int NS, bool DMA>
struct VqProduct {
  static constexpr int LDS = NS * (BI + BJ) * 128;
  static const void* address() { return reinterpret_cast<const void*>(&vql_product_kernel<T, AMM, BMM, KIND, BI, BJ, WI, WJ, NS, DMA>); }
  static inline VqLdsRegistrar registrar{address(), LDS};
  static int launch(const VqLinearArgs& a, hipStream_t s) {
    (void)&registrar;
    const int rc = vq_lds_ensure(address(), LDS, nullptr);
    if (rc != VQ_OK) return rc;
    const int64_t total = a.tiles_i * a.tiles_j * a.splits;
    const int64_t blocks = total < a.workgroups ? total : a.workgroups;
    hipLaunchKernelGGL((vql_product_kernel<T, AMM, BMM, KIND, BI, BJ, WI, WJ, NS, DMA>), dim3((unsigned)blocks), dim3(WI * WJ * 64), LDS, s, a);
    return vq_hip_status(hipGetLastError());
  }
};
template <typename T, bool AMM, bool BMM, int KIND>
int vql_launch_layout(const VqLinearArgs& a, int config, bool dma, hipStream_t s) {
  if (config == VQL_C256) return dma ? VqProduct<T, AMM, BMM, KIND, 256, 256, 2, 4, 2, true>::launch(a, s) : VQ_ERR_INVALID_ARG;
  if (config == VQL_C128)
    return dma ? VqProduct<T, AMM, BMM, KIND, 128, 128, 2, 2, 2, true>::launch(a, s) : VqProduct<T, AMM, BMM, KIND, 128, 128, 2, 2, 2, false>::launch(a, s);
  return dma ? VqProduct<T, AMM, BMM, KIND, 64, 64, 2, 2, 3, true>::launch(a, s) : VqProduct<T, AMM, BMM, KIND, 64, 64, 2, 2, 2, false>::launch(a, s);
}
template <typename T>
int vql_product(const VqLinearArgs& a, int layout, int config, bool dma, hipStream_t s) {
  if (layout == 1) return vql_launch_layout<T, false, true, VQL_PLAIN>(a, config, dma, s);
  if (layout == 2) return vql_launch_layout<T, true, true, VQL_PLAIN>(a, config, dma, s);
  // a split sum's epilogue is the join's
  const int kind = a.splits > 1 ? VQL_THRESHOLD : vql_kind(a.act);
  if (kind == VQL_SIGMOID) return vql_launch_layout<T, false, false, VQL_SIGMOID>(a, config, dma, s);
  if (kind == VQL_NORMAL) return vql_launch_layout<T, false, false, VQL_NORMAL>(a, config, dma, s);
  return vql_launch_layout<T, false, false, VQL_THRESHOLD>(a, config, dma, s);
}
}  // namespace

// The kernels of one element type (the compiler's host pass leaves kernels out that it meets only through VqProduct).
#define VQL_KERNELS_OF(T, AMM, BMM, KIND)                                                       \
  template __global__ void vql_product_kernel<T, AMM, BMM, KIND, 256, 256, 2, 4, 2, true>(VqLinearArgs);  \
  template __global__ void vql_product_kernel<T, AMM, BMM, KIND, 128, 128, 2, 2, 2, true>(VqLinearArgs);  \
  template __global__ void vql_product_kernel<T, AMM, BMM, KIND, 128, 128, 2, 2, 2, false>(VqLinearArgs); \
  template __global__ void vql_product_kernel<T, AMM, BMM, KIND, 64, 64, 2, 2, 3, true>(VqLinearArgs);    \
  template __global__ void vql_product_kernel<T, AMM, BMM, KIND, 64, 64, 2, 2, 2, false>(VqLinearArgs);
#define VQL_KERNELS(T)                              \
  namespace {                                       \
  VQL_KERNELS_OF(T, false, false, VQL_THRESHOLD)    \
  VQL_KERNELS_OF(T, false, false, VQL_SIGMOID)      \
  VQL_KERNELS_OF(T, false, false, VQL_NORMAL)       \
  VQL_KERNELS_OF(T, false, true, VQL_PLAIN)         \
  VQL_KERNELS_OF(T, true, true, VQL_PLAIN)          \
  }
