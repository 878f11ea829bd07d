// fb_clip.cu -- the global norm of many gradient tensors, and clipping.
//
//   norm = sqrt(sum g^2),  c = min(1, max_norm / (norm + eps)),  out = c g
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "fb_common.cuh"

namespace fb {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocks = 64;  // per tensor

template <typename T>
__global__ void __launch_bounds__(kThreads) clip_sum_simple(const T* g, int64_t n, double* part) {
  float s = 0.f;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)kBlocks * kThreads) {
    const float x = to_f32(g[i]);
    s += x * x;
  }
  double d = s;
  for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  __shared__ double sh[kThreads / 32];
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    d = 0.0;
    for (int i = 0; i < kThreads / 32; ++i) d += sh[i];
    part[blockIdx.x] = d;
  }
}

__global__ void clip_norm_simple(const double* part, int n, float* norm) {
  double d = 0.0;
  for (int i = 0; i < n; ++i) d += part[i];
  *norm = (float)sqrt(d);
}

__device__ __forceinline__ float clip_factor(float norm, float max_norm, float eps) {
  const float c = max_norm / (norm + eps);
  return c >= 1.f ? 1.f : c;  // a NaN norm stays NaN
}

template <typename T, typename U>
__global__ void __launch_bounds__(kThreads) clip_scale_simple(const T* g, U* out, int64_t n, const float* norm,
                                                              float max_norm, float eps) {
  const float c = clip_factor(*norm, max_norm, eps);
  if (c == 1.f && static_cast<const void*>(g) == static_cast<const void*>(out)) return;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)kBlocks * kThreads)
    out[i] = from_f32<U>(to_f32(g[i]) * c);
}

template <typename T, typename U>
void scale_one(const fb_clip_args* a, int i, cudaStream_t s) {
  clip_scale_simple<T, U><<<kBlocks, kThreads, 0, s>>>(static_cast<const T*>(a->grads[i]), static_cast<U*>(a->out[i]),
                                                       a->numel[i], a->norm, a->max_norm, a->eps);
}

bool bad_dtype(int d) { return d != FB_F32 && d != FB_F16 && d != FB_BF16; }

size_t workspace_size(const fb_clip_args* a) { return (size_t)std::max(a->count, 1) * kBlocks * sizeof(double); }

int clip(const fb_clip_args* a, cudaStream_t s) {
  if (a == nullptr || a->norm == nullptr) return FB_ERR_ARG;
  if (a->count < 0) return FB_ERR_SHAPE;
  if (a->count > 0 && (a->grads == nullptr || a->numel == nullptr || a->dtype == nullptr)) return FB_ERR_ARG;
  if (a->out != nullptr && (!(a->max_norm >= 0.f) || !(a->eps >= 0.f))) return FB_ERR_ARG;
  for (int i = 0; i < a->count; ++i) {
    if (a->numel[i] < 0) return FB_ERR_SHAPE;
    if (bad_dtype(a->dtype[i])) return FB_ERR_DTYPE;
    if (a->out != nullptr && a->out_dtype != nullptr && a->out_dtype[i] != a->dtype[i] && a->out_dtype[i] != FB_F32)
      return FB_ERR_DTYPE;
    if (a->numel[i] > 0 && (a->grads[i] == nullptr || (a->out != nullptr && a->out[i] == nullptr))) return FB_ERR_ARG;
  }
  if (a->workspace == nullptr || a->workspace_bytes < workspace_size(a)) return FB_ERR_WORKSPACE;
  double* part = static_cast<double*>(a->workspace);
  int launches = 1;
  for (int i = 0; i < a->count; ++i, ++launches) {
    double* to = part + (size_t)i * kBlocks;
    if (a->dtype[i] == FB_F32)
      clip_sum_simple<float><<<kBlocks, kThreads, 0, s>>>(static_cast<const float*>(a->grads[i]), a->numel[i], to);
    else if (a->dtype[i] == FB_F16)
      clip_sum_simple<__half><<<kBlocks, kThreads, 0, s>>>(static_cast<const __half*>(a->grads[i]), a->numel[i], to);
    else
      clip_sum_simple<__nv_bfloat16>
          <<<kBlocks, kThreads, 0, s>>>(static_cast<const __nv_bfloat16*>(a->grads[i]), a->numel[i], to);
  }
  clip_norm_simple<<<1, 1, 0, s>>>(part, a->count * kBlocks, a->norm);
  for (int i = 0; a->out != nullptr && i < a->count; ++i, ++launches) {
    const int in = a->dtype[i], to = a->out_dtype != nullptr ? a->out_dtype[i] : in;
    if (in == FB_F32) scale_one<float, float>(a, i, s);
    else if (in == FB_F16 && to == FB_F16) scale_one<__half, __half>(a, i, s);
    else if (in == FB_F16) scale_one<__half, float>(a, i, s);
    else if (to == FB_BF16) scale_one<__nv_bfloat16, __nv_bfloat16>(a, i, s);
    else scale_one<__nv_bfloat16, float>(a, i, s);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return FB_ERR_LAUNCH;
  }
  set_last_launch_count(launches);
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
