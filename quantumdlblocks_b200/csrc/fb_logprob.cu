// fb_logprob.cu -- log probabilities of given tokens, with entropy and the top alternatives of each row.
//
//   forward   lse = log sum exp x, logp = x_t - lse, entropy = lse - sum p x, the top_k largest x
//   backward  grad = g_logp ([c = t] - p) + sum_i g_top_i ([c = top_i] - p) - g_entropy p (log p + entropy)
#include <cuda_runtime.h>

#include <cmath>

#include "fb_common.cuh"

namespace fb {
namespace {

constexpr int kThreads = 256;

struct LogprobParams {
  int64_t rows;
  int V, K;
  const void* x;
  int64_t ld;
  const int64_t* targets;
  float* logp;
  float* entropy;
  float* lse;
  float* top_logp;
  int64_t* top_index;
  const float* g_logp;
  const float* g_entropy;
  const float* g_top;
  void* grad;
  int64_t grad_ld;
};

__device__ __forceinline__ float block_max(float v, float* sh) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int i = 1; i < kThreads / 32; ++i) v = fmaxf(v, sh[i]);
  return v;
}

__device__ __forceinline__ float block_sum(float v, float* sh) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int i = 1; i < kThreads / 32; ++i) v += sh[i];
  return v;
}

// 32 bits that order as the float does, NaN above everything, -0 and 0 alike
__device__ __forceinline__ uint32_t ordered(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// (value, column) as one number: greater value first, then the lower column
__device__ __forceinline__ uint64_t order_key(float x, int c) {
  return (uint64_t)ordered(x) << 32 | (uint32_t)~c;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_fwd_simple(const LogprobParams p) {
  __shared__ float sh[kThreads / 32];
  __shared__ uint64_t best;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  float m = -INFINITY;
  for (int c = threadIdx.x; c < p.V; c += kThreads) m = fmaxf(m, to_f32(x[c]));
  m = block_max(m, sh);
  float s = 0.f, u = 0.f;
  for (int c = threadIdx.x; c < p.V; c += kThreads) {
    const float d = to_f32(x[c]) - m, e = expf(d);
    s += e;
    u += e * fmaxf(d, -1e30f);  // a column at -inf adds 0, not 0 * inf
  }
  s = block_sum(s, sh);
  u = block_sum(u, sh);
  const float lse = m + logf(s);
  if (threadIdx.x == 0) {
    const int64_t t = p.targets[row];
    p.lse[row] = lse;
    p.logp[row] = (t >= 0 && t < p.V) ? (to_f32(x[t]) - m) - logf(s) : NAN;
    p.entropy[row] = logf(s) - u / s;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < p.K; ++i) {  // the largest below the last one taken
    uint64_t k = 0;
    for (int c = threadIdx.x; c < p.V; c += kThreads) {
      const uint64_t o = order_key(to_f32(x[c]), c);
      if (o < last && o > k) k = o;
    }
    if (threadIdx.x == 0) best = 0;
    __syncthreads();
    atomicMax(reinterpret_cast<unsigned long long*>(&best), (unsigned long long)k);
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) {
      const int c = (int)~(uint32_t)last;
      p.top_index[row * p.K + i] = c;
      p.top_logp[row * p.K + i] = (to_f32(x[c]) - m) - logf(s);
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_bwd_simple(const LogprobParams p) {
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.ld;
  T* dx = static_cast<T*>(p.grad) + row * p.grad_ld;
  const float lse = p.lse[row], h = p.entropy[row];
  const int64_t t = p.targets[row];
  const float g = p.g_logp ? p.g_logp[row] : 0.f, gh = p.g_entropy ? p.g_entropy[row] : 0.f;
  float a = (t >= 0 && t < p.V) || g == 0.f ? g : NAN;
  if (p.g_top)
    for (int i = 0; i < p.K; ++i) a += p.g_top[row * p.K + i];
  for (int c = threadIdx.x; c < p.V; c += kThreads) {
    float lp = to_f32(x[c]) - lse;
    lp = lp < -200.f ? -200.f : lp;  // p is 0 there, and -inf must not meet it; a NaN stays
    float d = -expf(lp) * (a + gh * (lp + h));
    if (c == t) d += g;
    if (p.g_top)
      for (int i = 0; i < p.K; ++i)
        if (p.top_index[row * p.K + i] == c) d += p.g_top[row * p.K + i];
    dx[c] = from_f32<T>(d);
  }
}

int logprob(const fb_logprob_args* a, void* stream, bool backward) {
  if (a == nullptr) return FB_ERR_ARG;
  if (a->rows < 0 || a->rows > 0x7FFFFFFF || a->vocab < 1 || a->ld < a->vocab || a->top_k < 0 ||
      a->top_k > FB_MAX_TOP_K || a->top_k > a->vocab)
    return FB_ERR_SHAPE;
  if (a->dtype != FB_F32 && a->dtype != FB_F16 && a->dtype != FB_BF16) return FB_ERR_DTYPE;
  if (backward && a->grad_ld < a->vocab) return FB_ERR_SHAPE;
  if (a->rows == 0) {
    set_last_launch_count(0);
    return FB_OK;
  }
  if (a->logits == nullptr || a->targets == nullptr || a->lse == nullptr || a->entropy == nullptr) return FB_ERR_ARG;
  if (!backward && a->logp == nullptr) return FB_ERR_ARG;
  if (!backward && a->top_k > 0 && (a->top_logp == nullptr || a->top_index == nullptr)) return FB_ERR_ARG;
  if (backward && a->grad == nullptr) return FB_ERR_ARG;
  if (backward && a->top_k > 0 && a->g_top != nullptr && a->top_index == nullptr) return FB_ERR_ARG;
  LogprobParams p{a->rows, a->vocab, a->top_k, a->logits, a->ld, a->targets, a->logp, a->entropy, a->lse, a->top_logp,
                  a->top_index, a->g_logp, a->g_entropy, a->top_k > 0 ? a->g_top : nullptr, a->grad, a->grad_ld};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned n = (unsigned)a->rows;
  if (backward) {
    if (a->dtype == FB_F32) logprob_bwd_simple<float><<<n, kThreads, 0, s>>>(p);
    else if (a->dtype == FB_F16) logprob_bwd_simple<__half><<<n, kThreads, 0, s>>>(p);
    else logprob_bwd_simple<__nv_bfloat16><<<n, kThreads, 0, s>>>(p);
  } else {
    if (a->dtype == FB_F32) logprob_fwd_simple<float><<<n, kThreads, 0, s>>>(p);
    else if (a->dtype == FB_F16) logprob_fwd_simple<__half><<<n, kThreads, 0, s>>>(p);
    else logprob_fwd_simple<__nv_bfloat16><<<n, kThreads, 0, s>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return FB_ERR_LAUNCH;
  }
  set_last_launch_count(1);
  return FB_OK;
}

}  // namespace
}  // namespace fb

extern "C" {

int fb_logprob_fwd(const fb_logprob_args* args, void* stream) { return fb::logprob(args, stream, false); }
int fb_logprob_bwd(const fb_logprob_args* args, void* stream) { return fb::logprob(args, stream, true); }

}  // extern "C"
