// fb_clip.cu -- the global norm of many gradient tensors, and clipping.
//
//   norm = sqrt(sum g^2),  c = min(1, max_norm / (norm + eps)),  out = c g
//
// Two kernels, whatever the tensors' number and types.  All tensors' elements are cut into chunks of
// kChunkBytes, the table of tensors travels in the kernel's parameters (kTensors to a launch; more take
// more launches), and CTA b of a launch takes chunks b, b + grid, ...:
//
//   clip_sum    each CTA's sum of squares: fp32 for the 16 or 32 squares of a thread and chunk, fp64 beyond
//   clip_scale  each CTA adds all CTAs' sums, in order, to the norm (the same bits everywhere and every time),
//               and scales its chunks; in place with c = 1 there is nothing to do.  It takes the chunks from the
//               last to the first: what clip_sum read last is still in L2.
//
// Both are bound by HBM bandwidth for many elements; for few by the two launches, the second of which is
// under way while the first runs.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "fb_common.cuh"

namespace fb {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;                                // 16-byte loads a thread has under way
constexpr int kChunkBytes = kThreads * kUnroll * 16;      // 16 KB
constexpr int kTensors = 96;                              // per launch: the table stays under 4 KB
constexpr int kCtasPerSm = 6;

struct Tensor {
  const void* g;
  void* out;
  int64_t n;
  uint32_t chunk0;    // its first chunk in the launch
  uint8_t dtype, out_dtype;
};

struct ClipParams {
  Tensor t[kTensors];
  int count;
  uint32_t chunks;    // of the launch
  double* part;       // clip_sum: this launch's sums; clip_scale: all launches'
  int parts;          // clip_scale
  float max_norm, eps;
  float* norm;        // clip_scale: where its first launch writes the norm
  bool in_place;      // all of them
};
static_assert(sizeof(ClipParams) <= 4096, "kernel parameters");

// Elements of a chunk: vectors of N elements of memory from the 16-byte boundary at or before the tensor, so that
// every load is aligned; the tensor's first and last vector may be partly its own.
template <typename T, int N> struct Span {
  using W = typename std::conditional<N * sizeof(T) == 16, uint4, uint2>::type;
  static constexpr int kVectors = kChunkBytes / sizeof(W), kEach = kVectors / kThreads;  // of a chunk, of a thread
  const T* base;
  int64_t lo, hi;  // the tensor's elements from there
  int64_t v0;      // the thread's first vector
  bool full;       // the whole chunk is the tensor's
  __device__ Span(const Tensor& t, uint32_t chunk) {
    const int shift = (int)((reinterpret_cast<uintptr_t>(t.g) & 15) / sizeof(T));
    base = static_cast<const T*>(t.g) - shift;
    lo = shift;
    hi = shift + t.n;
    v0 = (int64_t)(chunk - t.chunk0) * kVectors;
    full = v0 * N >= lo && (v0 + kVectors) * N <= hi;
    v0 += threadIdx.x;
  }
  __device__ const W* at(int i) const { return reinterpret_cast<const W*>(base) + v0 + i * kThreads; }
  __device__ bool has(int64_t element) const { return element >= lo && element < hi; }
  // the thread's vectors as floats, 0 where the tensor has none
  __device__ void load(float (&f)[kEach][N]) const {
    W w[kEach];
    if (full) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) w[i] = *at(i);
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int64_t e0 = (v0 + i * kThreads) * N;
        if (has(e0) && has(e0 + N - 1)) {
          w[i] = *at(i);
        } else {
          w[i] = W{};
          T* e = reinterpret_cast<T*>(&w[i]);
#pragma unroll
          for (int x = 0; x < N; ++x)
            if (has(e0 + x)) e[x] = base[e0 + x];
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const T* e = reinterpret_cast<const T*>(&w[i]);
#pragma unroll
      for (int x = 0; x < N; ++x) f[i][x] = to_f32(e[x]);
    }
  }
};

// The tensor that holds a chunk, searched from the one that held an earlier (or, DOWN, a later) chunk
template <bool DOWN>
__device__ __forceinline__ int tensor_of(const ClipParams& p, uint32_t chunk, int from) {
  if (DOWN) {
    while (p.t[from].chunk0 > chunk) --from;
  } else {
    while (from + 1 < p.count && p.t[from + 1].chunk0 <= chunk) ++from;
  }
  return from;
}

template <typename T>
__device__ __forceinline__ float squares(const Tensor& t, uint32_t chunk) {
  constexpr int N = 16 / sizeof(T);
  using S = Span<T, N>;
  const S s(t, chunk);
  float f[S::kEach][N], sum = 0.f;
  s.load(f);
#pragma unroll
  for (int i = 0; i < S::kEach; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) sum = fmaf(f[i][e], f[i][e], sum);
  return sum;
}

// The sum over the block, in every thread
__device__ __forceinline__ double block_sum(double d) {
  __shared__ double sh[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = d;
  __syncthreads();
  d = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) d += sh[w];
  return d;
}

__global__ void __launch_bounds__(kThreads, kCtasPerSm) clip_sum(const __grid_constant__ ClipParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  double sum = 0.0;
  int at = 0;
  for (uint32_t chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
    at = tensor_of<false>(p, chunk, at);
    const Tensor& t = p.t[at];
    if (t.dtype == FB_F32) sum += squares<float>(t, chunk);
    else if (t.dtype == FB_BF16) sum += squares<__nv_bfloat16>(t, chunk);
    else sum += squares<__half>(t, chunk);
  }
  const double d = block_sum(sum);
  if (threadIdx.x == 0) p.part[blockIdx.x] = d;
}

// 16 bytes stored per thread and vector, neighbours next to one another: 16-bit gradients on their way to fp32 are
// taken 8 bytes at a time (with 16, a warp's stores left every other 16 bytes for the next: 54 us against 41)
template <typename T, typename U>
__device__ __forceinline__ void scale(const Tensor& t, uint32_t chunk, float c) {
  constexpr int N = 16 / sizeof(U);
  using S = Span<T, N>;
  const S s(t, chunk);
  U* out = static_cast<U*>(t.out) - s.lo;  // element i of the span goes to out[i]
  const bool aligned = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  float f[S::kEach][N];
  s.load(f);
#pragma unroll
  for (int i = 0; i < S::kEach; ++i) {
    const int64_t e0 = (s.v0 + i * kThreads) * N;
    uint4 w;
    U* e = reinterpret_cast<U*>(&w);
#pragma unroll
    for (int x = 0; x < N; ++x) e[x] = from_f32<U>(f[i][x] * c);
    if (aligned && (s.full || (s.has(e0) && s.has(e0 + N - 1)))) {
      *reinterpret_cast<uint4*>(out + e0) = w;
    } else {
#pragma unroll
      for (int x = 0; x < N; ++x)
        if (s.has(e0 + x)) out[e0 + x] = e[x];
    }
  }
}

__global__ void __launch_bounds__(kThreads, kCtasPerSm) clip_scale(const __grid_constant__ ClipParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  double d = 0.0;
  for (int i = threadIdx.x; i < p.parts; i += kThreads) d += p.part[i];
  const float norm = (float)sqrt(block_sum(d));
  if (p.norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.norm = norm;
  float c = p.max_norm / (norm + p.eps);
  if (c >= 1.f) c = 1.f;  // a NaN norm stays NaN
  if (c == 1.f && p.in_place) return;
  int at = p.count - 1;
  for (uint32_t i = blockIdx.x; i < p.chunks; i += gridDim.x) {
    const uint32_t chunk = p.chunks - 1 - i;
    at = tensor_of<true>(p, chunk, at);
    const Tensor& t = p.t[at];
    if (t.dtype == FB_F32) scale<float, float>(t, chunk, c);
    else if (t.dtype == FB_BF16 && t.out_dtype == FB_BF16) scale<__nv_bfloat16, __nv_bfloat16>(t, chunk, c);
    else if (t.dtype == FB_BF16) scale<__nv_bfloat16, float>(t, chunk, c);
    else if (t.out_dtype == FB_F16) scale<__half, __half>(t, chunk, c);
    else scale<__half, float>(t, chunk, c);
  }
}

int sm_count() {
  static int count[64];  // per device; 0: not asked yet (two threads that ask write the same)
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (count[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    count[dev] = n;
  }
  return count[dev];
}

bool bad_dtype(int d) { return d != FB_F32 && d != FB_F16 && d != FB_BF16; }
int size_of(int dtype) { return dtype == FB_F32 ? 4 : 2; }

uint64_t chunks_of(const void* g, int64_t n, int dtype) {
  if (n == 0) return 0;
  const uint64_t bytes = (uint64_t)n * size_of(dtype) + (reinterpret_cast<uintptr_t>(g) & 15);
  return (bytes + kChunkBytes - 1) / kChunkBytes;
}

// Every launch leaves at most kCtasPerSm sums per SM
size_t workspace_size(const fb_clip_args* a) {
  const size_t launches = (size_t)std::max(1, (a->count + kTensors - 1) / kTensors);
  return launches * kCtasPerSm * sm_count() * sizeof(double);
}

int check(const fb_clip_args* a) {
  if (a == nullptr || a->norm == nullptr) return FB_ERR_ARG;
  if (a->count < 0) return FB_ERR_SHAPE;
  if (a->count > 0 && (a->grads == nullptr || a->numel == nullptr || a->dtype == nullptr)) return FB_ERR_ARG;
  if (a->out != nullptr && (!(a->max_norm >= 0.f) || !(a->eps >= 0.f))) return FB_ERR_ARG;
  for (int i = 0; i < a->count; ++i) {
    if (a->numel[i] < 0 || a->numel[i] > (1ll << 36)) return FB_ERR_SHAPE;  // a launch's chunks count in 32 bits
    if (bad_dtype(a->dtype[i])) return FB_ERR_DTYPE;
    if (a->out != nullptr && a->out_dtype != nullptr && a->out_dtype[i] != a->dtype[i] && a->out_dtype[i] != FB_F32)
      return FB_ERR_DTYPE;
    if (a->numel[i] == 0) continue;
    if (a->grads[i] == nullptr || (a->out != nullptr && a->out[i] == nullptr)) return FB_ERR_ARG;
    const int out_size = a->out_dtype != nullptr ? size_of(a->out_dtype[i]) : size_of(a->dtype[i]);
    if (reinterpret_cast<uintptr_t>(a->grads[i]) % size_of(a->dtype[i]) != 0 ||
        (a->out != nullptr && reinterpret_cast<uintptr_t>(a->out[i]) % out_size != 0))
      return FB_ERR_ALIGN;
  }
  if (a->workspace == nullptr || a->workspace_bytes < workspace_size(a)) return FB_ERR_WORKSPACE;
  return FB_OK;
}

// The launch's table: tensors [i0, i1)
void fill(ClipParams* p, const fb_clip_args* a, int i0, int i1) {
  p->count = 0;
  p->chunks = 0;
  p->in_place = true;
  for (int i = i0; i < i1; ++i) {
    const uint64_t n = chunks_of(a->grads[i], a->numel[i], a->dtype[i]);
    if (n == 0) continue;
    Tensor& t = p->t[p->count++];
    t.g = a->grads[i];
    t.out = a->out != nullptr ? a->out[i] : nullptr;
    p->in_place = p->in_place && t.out == t.g;
    t.n = a->numel[i];
    t.chunk0 = p->chunks;
    t.dtype = (uint8_t)a->dtype[i];
    t.out_dtype = (uint8_t)(a->out_dtype != nullptr ? a->out_dtype[i] : a->dtype[i]);
    p->chunks += (uint32_t)n;
  }
}

int clip(const fb_clip_args* a, cudaStream_t s) {
  const int rc = check(a);
  if (rc != FB_OK) return rc;
  const int most = kCtasPerSm * sm_count(), launches = std::max(1, (a->count + kTensors - 1) / kTensors);
  ClipParams p{};
  p.max_norm = a->max_norm;
  p.eps = a->eps;
  double* sums = static_cast<double*>(a->workspace);
  int parts = 0;
  cudaError_t e = cudaSuccess;
  for (int l = 0; l < launches && e == cudaSuccess; ++l) {
    fill(&p, a, l * kTensors, std::min(a->count, (l + 1) * kTensors));
    const int grid = (int)std::max<uint32_t>(1, std::min<uint32_t>(p.chunks, most));
    p.part = sums + parts;
    parts += grid;
    clip_sum<<<grid, kThreads, 0, s>>>(p);
    e = cudaGetLastError();
  }
  // one launch: its table still is in p
  p.part = sums;
  p.parts = parts;
  int n = launches;
  for (int l = 0; l < (a->out != nullptr ? launches : 1) && e == cudaSuccess; ++l, ++n) {
    if (launches > 1) fill(&p, a, l * kTensors, std::min(a->count, (l + 1) * kTensors));
    p.norm = l == 0 ? a->norm : nullptr;
    if (a->out == nullptr) p.chunks = 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(std::max<uint32_t>(1, std::min<uint32_t>(p.chunks, most)));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, clip_scale, p);
  }
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return FB_ERR_LAUNCH;
  }
  set_last_launch_count(n);
  return FB_OK;
}

}  // namespace
}  // namespace fb

extern "C" {

size_t fb_clip_workspace_size(const fb_clip_args* args) { return args ? fb::workspace_size(args) : 0; }
int fb_clip_grad_norm(const fb_clip_args* args, void* stream) {
  return fb::clip(args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
