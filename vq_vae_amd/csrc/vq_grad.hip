// Global gradient norm over many tensors and clipping by it (gfx950).
//
//     norm = (sum over all tensors |g|^p)^(1/p), p = 1, 2, inf        c = min(1, max_norm / (norm + 1e-6))
//     out = round(g c)
//
// Both are streams: 2 operations per element against 2 or 4 bytes.  What costs here is launches (a model has hundreds
// of tensors, most of them small) and, for clipping, that the gradients are read twice, since no element can be scaled
// before the last one is summed.
//   * The tensors' addresses and sizes travel in the kernel arguments, up to 136 tensors a launch: nothing is copied to
//     the device, and a captured launch holds its own table.
//   * The tensors are cut into chunks of 32 KiB; a workgroup takes a contiguous run of chunks, so it searches the table
//     once and then walks it.
//   * Squares are summed in 64 bits: their range (1e-38 squared to 1e38 squared) and a sum over 1e9 elements are outside
//     what 32 bits hold, and the stream leaves the time (v_fma_f64 runs at half the fp32 rate).
//   * Every workgroup writes one partial sum; the readers add them all in a fixed order.  No atomics, no counter that
//     would have to be cleared, the same bits on every run.
// 792 MB of fp32 gradients: norm 126 us, 6.3 TB/s; 528 MB bf16 clipped into 1056 MB fp32: 360 us, 5.9 TB/s of the 2.1 GB.
// Chunks dealt out in turn instead of in runs: norm 123, clipping 370.
#include <algorithm>
#include <new>

#include "vq_linear.h"

namespace {

constexpr int GT = 136;               // tensors of one launch: 136 x 29 bytes of the 4 KiB of kernel arguments
constexpr int G_CHUNK = 32768;        // bytes of a gradient per chunk
constexpr int G_WGS = 2048;           // workgroups of all launches of a pass, 8 per CU
constexpr int G_MAX_TENSORS = 1 << 16;

struct GradTable {
  const char* src[GT];
  char* dst[GT];
  int64_t numel[GT];
  uint32_t chunk_end[GT];   // chunks of this launch up to and including tensor i
  uint8_t type[GT];         // source type | destination type << 4
  int n;
  int wgs;
};

__device__ __forceinline__ int table_find(const GradTable& t, uint32_t chunk) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (chunk < t.chunk_end[mid]) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Calls f(tensor, first element, elements) for every chunk of this workgroup's run; backwards: last chunk first.
template <bool BACKWARDS, typename F>
__device__ __forceinline__ void for_chunks(const GradTable& t, F f) {
  const uint32_t total = t.chunk_end[t.n - 1];
  uint32_t c0 = (uint32_t)((uint64_t)total * blockIdx.x / t.wgs), c1 = (uint32_t)((uint64_t)total * (blockIdx.x + 1) / t.wgs);
  if (c0 >= c1) return;
  int i = table_find(t, BACKWARDS ? c1 - 1 : c0);
  for (uint32_t k = c0; k < c1; ++k) {
    const uint32_t c = BACKWARDS ? c1 - 1 - (k - c0) : k;
    if (BACKWARDS) {
      while (i > 0 && c < t.chunk_end[i - 1]) --i;
    } else {
      while (c >= t.chunk_end[i]) ++i;
    }
    const uint32_t first = i > 0 ? t.chunk_end[i - 1] : 0;
    const int64_t per = G_CHUNK / ((t.type[i] & 15) == VQ_F32 ? 4 : 2);
    const int64_t at = (int64_t)(c - first) * per;
    f(i, at, t.numel[i] - at < per ? t.numel[i] - at : per);
  }
}

__device__ __forceinline__ double norm_add(double acc, float v, int kind) {
  if (kind == VQ_NORM_2) return __builtin_fma((double)v, (double)v, acc);
  if (kind == VQ_NORM_1) return acc + (double)fabsf(v);
  const double d = (double)fabsf(v);
  return (d > acc || d != d) ? d : acc;              // a NaN stays: no comparison with it holds
}
__device__ __forceinline__ double norm_merge(double a, double b, int kind) {
  if (kind != VQ_NORM_INF) return a + b;
  if (a != a) return a;
  return (b > a || b != b) ? b : a;
}

// ONCE: nobody reads the gradients again, so they pass the caches by (792 MB fp32 141 -> 126 us, 66 MB 16.8 -> 15.2); where they
// are clipped next they stay (360 us instead of 387).
template <typename T, bool ONCE>
__device__ __forceinline__ void norm_chunk(const char* src, int64_t at, int64_t count, int kind, double (&acc)[2]) {
  constexpr int E = 16 / sizeof(T), U = G_CHUNK / 16 / 256;
  const char* p = src + at * (int64_t)sizeof(T);
  if (count == G_CHUNK / (int64_t)sizeof(T)) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const char* at_u = p + (u * 256 + threadIdx.x) * 16;
      v[u] = ONCE ? vql_once16<T>(at_u) : vql_load16<T>(at_u);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const VqChunk<T> c = __builtin_bit_cast(VqChunk<T>, v[u]);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e & 1] = norm_add(acc[e & 1], VqElem<T>::to(c.e[e]), kind);
    }
  } else {
    for (int64_t v = threadIdx.x; v * E < count; v += 256) {
      const VqChunk<T> c = __builtin_bit_cast(VqChunk<T>, vql_load16_part<T>(p + v * 16, count - v * E));   // zeros add nothing
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e & 1] = norm_add(acc[e & 1], VqElem<T>::to(c.e[e]), kind);
    }
  }
}

// All 256 threads' values merged; the result in every thread.
__device__ __forceinline__ double block_merge(double v, int kind, double* s) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = norm_merge(v, __shfl_xor(v, off), kind);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = norm_merge(norm_merge(s[0], s[1], kind), norm_merge(s[2], s[3], kind), kind);
  __syncthreads();
  return v;
}

template <int KIND, bool ONCE>
__global__ __launch_bounds__(256) void vqg_partial_kernel(GradTable t, double* part) {
  __shared__ double s[4];
  double acc[2] = {0.0, 0.0};
  for_chunks<false>(t, [&](int i, int64_t at, int64_t count) {
    const int type = t.type[i] & 15;
    if (type == VQ_F32) norm_chunk<float, ONCE>(t.src[i], at, count, KIND, acc);
    else if (type == VQ_BF16) norm_chunk<VqBf16, ONCE>(t.src[i], at, count, KIND, acc);
    else norm_chunk<_Float16, ONCE>(t.src[i], at, count, KIND, acc);
  });
  const double v = block_merge(norm_merge(acc[0], acc[1], KIND), KIND, s);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// The norm from all partial sums, the same order in every workgroup.
__device__ __forceinline__ double whole_norm(const double* part, int n, int kind, double* s) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) v = norm_merge(v, part[i], kind);
  v = block_merge(v, kind, s);
  return kind == VQ_NORM_2 ? __builtin_sqrt(v) : v;
}

__global__ __launch_bounds__(256) void vqg_finish_kernel(const double* part, int n, int kind, float* norm) {
  __shared__ double s[4];
  const double v = whole_norm(part, n, kind, s);
  if (threadIdx.x == 0) *norm = (float)v;
}

// Loads and stores past the caches: the gradients of the norm pass stay there, to be found by this one, instead of making room
// for results (528 MB bf16 into fp32 422 -> 360 us, 264 MB fp32 into fp32 163 -> 129, 33 MB in place 22.8 -> 22.6; with somebody
// who reads the result next 605 -> 539, 210 -> 181, 30.2 -> 30.4).  One access is 16 bytes of the result a lane, so that a wave
// fills whole lines also where 16-bit gradients become fp32 (two stores of 16 bytes at 32-byte distance made it 650).
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 vqg_u32x2_a2 __attribute__((aligned(2), may_alias));
template <typename S, int W>
struct alignas(sizeof(S)) VqRun {
  S e[W];
};
template <typename S, int W>
__device__ __forceinline__ VqRun<S, W> load_run(const char* p) {
  if constexpr (W * sizeof(S) == 8) {
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const vqg_u32x2_a2*>(p));
    return __builtin_bit_cast(VqRun<S, W>, v);
  } else {
    return __builtin_bit_cast(VqRun<S, W>, vql_once16<S>(p));
  }
}
template <typename S, typename D>
__device__ __forceinline__ void scale_chunk(const char* src, char* dst, int64_t at, int64_t count, float c) {
  constexpr int W = 16 / sizeof(D), U = G_CHUNK / (W * sizeof(S)) / 256;
  const char* p = src + at * (int64_t)sizeof(S);
  D* q = reinterpret_cast<D*>(dst) + at;
  auto one = [&](const VqRun<S, W>& g, int64_t first) {
    VqChunk<D> o;
#pragma unroll
    for (int e = 0; e < W; ++e) o.e[e] = VqElem<D>::from(VqElem<S>::to(g.e[e]) * c);
    const u32x4 w = __builtin_bit_cast(u32x4, o);
    if constexpr (sizeof(D) == 4) __builtin_nontemporal_store(w, reinterpret_cast<vql_u32x4_a4*>(q + first));
    else __builtin_nontemporal_store(w, reinterpret_cast<vql_u32x4_a2*>(q + first));
  };
  if (count == G_CHUNK / (int64_t)sizeof(S)) {
    VqRun<S, W> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_run<S, W>(p + (u * 256 + threadIdx.x) * (int)(W * sizeof(S)));
#pragma unroll
    for (int u = 0; u < U; ++u) one(v[u], (int64_t)(u * 256 + threadIdx.x) * W);
  } else {
    for (int64_t v = threadIdx.x; v * W < count; v += 256) {
      if (count - v * W >= W) {
        one(load_run<S, W>(p + v * (int64_t)(W * sizeof(S))), v * W);
      } else {
        for (int64_t i = v * W; i < count; ++i) q[i] = VqElem<D>::from(VqElem<S>::to(reinterpret_cast<const S*>(p)[i]) * c);
      }
    }
  }
}

// Every workgroup adds the partial sums itself (16 KiB out of the L2) rather than waiting for another launch to do it.
// Tensors scaled in place are left alone where c is 1.  The run is walked backwards: what the norm pass read last is
// what the caches still hold.
__global__ __launch_bounds__(256) void vqg_scale_kernel(GradTable t, const double* part, int n_part, int kind, float max_norm,
                                                        float* norm) {
  __shared__ double s[4];
  const double total = whole_norm(part, n_part, kind, s);
  const float rounded = (float)total;                // c goes by the norm that is returned: infinite beyond fp32, and then zero
  double cd = (double)max_norm / ((double)rounded + 1e-6);
  cd = cd > 1.0 ? 1.0 : cd;                          // NaN passes
  const float c = (float)cd;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = rounded;
  for_chunks<true>(t, [&](int i, int64_t at, int64_t count) {
    if (c == 1.0f && t.src[i] == t.dst[i]) return;
    switch (t.type[i]) {
      case VQ_F32 | VQ_F32 << 4: scale_chunk<float, float>(t.src[i], t.dst[i], at, count, c); break;
      case VQ_BF16 | VQ_BF16 << 4: scale_chunk<VqBf16, VqBf16>(t.src[i], t.dst[i], at, count, c); break;
      case VQ_F16 | VQ_F16 << 4: scale_chunk<_Float16, _Float16>(t.src[i], t.dst[i], at, count, c); break;
      case VQ_BF16 | VQ_F32 << 4: scale_chunk<VqBf16, float>(t.src[i], t.dst[i], at, count, c); break;
      default: scale_chunk<_Float16, float>(t.src[i], t.dst[i], at, count, c); break;
    }
  });
}

int64_t chunks_of(const vq_tensor_ref& r) {
  const int64_t per = G_CHUNK / (r.src_type == VQ_F32 ? 4 : 2);
  return (r.numel + per - 1) / per;
}
int launches_of(int n) { return (n + GT - 1) / GT; }

// Checks the list; total chunks out.
int check_refs(const vq_tensor_ref* refs, int n, bool scale, int64_t* chunks) {
  if (n < 0 || (n > 0 && !refs)) return VQ_ERR_INVALID_ARG;
  if (n > G_MAX_TENSORS) return VQ_ERR_TOO_LARGE;
  *chunks = 0;
  for (int i = 0; i < n; ++i) {
    const vq_tensor_ref& r = refs[i];
    if (r.numel < 0 || r.src_type < VQ_F32 || r.src_type > VQ_F16) return VQ_ERR_INVALID_ARG;
    if (r.numel > 0 && !r.src) return VQ_ERR_INVALID_ARG;
    if (scale) {
      if (r.numel > 0 && !r.dst) return VQ_ERR_INVALID_ARG;
      if (r.dst_type != r.src_type && r.dst_type != VQ_F32) return VQ_ERR_INVALID_ARG;
    }
    *chunks += chunks_of(r);
  }
  return *chunks > (int64_t)0x7fffffff ? VQ_ERR_UNSUPPORTED : VQ_OK;
}

// Calls f(table, workgroups) for every launch of a pass over the list; the workgroups of all launches are shared out by
// their chunks.
template <typename F>
int for_tables(const vq_tensor_ref* refs, int n, bool scale, int64_t chunks, F f) {
  for (int i = 0; i < n;) {
    GradTable t;
    t.n = 0;
    uint32_t mine = 0;
    for (; i < n && t.n < GT; ++i) {
      const vq_tensor_ref& r = refs[i];
      if (r.numel == 0) continue;
      t.src[t.n] = reinterpret_cast<const char*>(r.src);
      t.dst[t.n] = reinterpret_cast<char*>(r.dst);
      t.numel[t.n] = r.numel;
      t.type[t.n] = (uint8_t)(r.src_type | (scale ? r.dst_type : 0) << 4);
      mine += (uint32_t)chunks_of(r);
      t.chunk_end[t.n++] = mine;
    }
    if (t.n == 0) continue;
    t.wgs = (int)std::min<int64_t>(mine, std::max<int64_t>(1, (int64_t)G_WGS * mine / chunks));
    const int rc = f(t);
    if (rc != VQ_OK) return rc;
  }
  return VQ_OK;
}

template <int KIND>
void launch_partials(const GradTable& t, bool once, double* at, hipStream_t s) {
  if (once) hipLaunchKernelGGL((vqg_partial_kernel<KIND, true>), dim3(t.wgs), dim3(256), 0, s, t, at);
  else hipLaunchKernelGGL((vqg_partial_kernel<KIND, false>), dim3(t.wgs), dim3(256), 0, s, t, at);
}
int run_partials(const vq_tensor_ref* refs, int n, int kind, bool once, int64_t chunks, double* part, int* n_part, hipStream_t s) {
  *n_part = 0;
  return for_tables(refs, n, false, chunks, [&](const GradTable& t) {
    double* at = part + *n_part;
    if (kind == VQ_NORM_2) launch_partials<VQ_NORM_2>(t, once, at, s);
    else if (kind == VQ_NORM_1) launch_partials<VQ_NORM_1>(t, once, at, s);
    else launch_partials<VQ_NORM_INF>(t, once, at, s);
    *n_part += t.wgs;
    return vq_hip_status(hipGetLastError());
  });
}

}  // namespace

extern "C" int vq_tensor_refs_overlap(const vq_tensor_ref* refs, int n) {
  if (n <= 0 || !refs) return 0;
  struct Run { uintptr_t at, end; };
  Run few[256];
  Run* runs = n <= 128 ? few : new (std::nothrow) Run[2 * (size_t)n];
  if (!runs) return 1;
  size_t k = 0;
  for (int i = 0; i < n; ++i) {
    const vq_tensor_ref& r = refs[i];
    if (r.numel <= 0) continue;
    const uintptr_t s = reinterpret_cast<uintptr_t>(r.src), d = reinterpret_cast<uintptr_t>(r.dst);
    runs[k++] = {d, d + (uintptr_t)r.numel * (r.dst_type == VQ_F32 ? 4 : 2)};
    if (s != d || r.src_type != r.dst_type) runs[k++] = {s, s + (uintptr_t)r.numel * (r.src_type == VQ_F32 ? 4 : 2)};
  }
  std::sort(runs, runs + k, [](const Run& a, const Run& b) { return a.at < b.at; });
  int found = 0;
  for (size_t i = 1; i < k; ++i) found |= runs[i].at < runs[i - 1].end;
  if (runs != few) delete[] runs;
  return found;
}

extern "C" int64_t vq_grad_norm_work_bytes(int n) { return n < 0 ? 0 : ((int64_t)G_WGS + launches_of(n)) * 8; }

extern "C" int vq_grad_norm(const vq_tensor_ref* refs, int n, int kind, float* norm, void* work, void* stream) {
  int64_t chunks = 0;
  const int ok = check_refs(refs, n, false, &chunks);
  if (ok != VQ_OK) return ok;
  if (kind < VQ_NORM_INF || kind > VQ_NORM_2 || !norm || !work || (reinterpret_cast<uintptr_t>(work) & 7)) return VQ_ERR_INVALID_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* part = reinterpret_cast<double*>(work);
  int n_part = 0;
  const int rc = run_partials(refs, n, kind, true, chunks, part, &n_part, s);
  if (rc != VQ_OK) return rc;
  hipLaunchKernelGGL(vqg_finish_kernel, dim3(1), dim3(256), 0, s, part, n_part, kind, norm);
  return vq_hip_status(hipGetLastError());
}

extern "C" int vq_clip_grads(const vq_tensor_ref* refs, int n, int kind, float max_norm, float* norm, void* work, void* stream) {
  int64_t chunks = 0;
  const int ok = check_refs(refs, n, true, &chunks);
  if (ok != VQ_OK) return ok;
  if (kind < VQ_NORM_INF || kind > VQ_NORM_2 || !norm || !work || (reinterpret_cast<uintptr_t>(work) & 7) || !(max_norm >= 0.0f))
    return VQ_ERR_INVALID_ARG;
  if (vq_tensor_refs_overlap(refs, n)) return VQ_ERR_INVALID_ARG;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  double* part = reinterpret_cast<double*>(work);
  int n_part = 0;
  int rc = run_partials(refs, n, kind, false, chunks, part, &n_part, s);
  if (rc != VQ_OK) return rc;
  if (n_part == 0) {   // no elements: the norm is zero
    hipLaunchKernelGGL(vqg_finish_kernel, dim3(1), dim3(256), 0, s, part, 0, kind, norm);
    return vq_hip_status(hipGetLastError());
  }
  return for_tables(refs, n, true, chunks, [&](const GradTable& t) {
    hipLaunchKernelGGL(vqg_scale_kernel, dim3(t.wgs), dim3(256), 0, s, t, (const double*)part, n_part, kind, max_norm, norm);
    norm = nullptr;
    return vq_hip_status(hipGetLastError());
  });
}
