// fb_paged.cu -- generating from a trained flash-Born GPT: Born attention of one new token per
// sequence over a paged key-value cache, and the kernel that fills that cache.
//
//   paged_born_fwd   a_j = relu(scale_h <q, k_j>), p_j = a_j^2, out = (sum_j p_j v_j) / (sum_j p_j + eps)
//   paged_qkv_write  Q, K = l2n(rope(.)), V; K and V rows into their pages' slots
#include <cuda_runtime.h>

#include "fb_common.cuh"

namespace fb {
namespace {

struct PagedParams {
  int S, H, Hkv, G, D;
  int page, pages, width;  // page rows, pages, table columns
  int window;
  float eps, scale_value;
  const float* scale;
  int scale_per_head;
  const void* q;
  int64_t qs[3];
  const void* k;
  int64_t ks[4];
  const void* v;
  int64_t vs[4];
  void* out;
  int64_t os[3];
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The keys [lo, hi) of one sequence: what the length, the table's capacity and the window leave.
__device__ __forceinline__ void key_range(const PagedParams& p, int s, int& lo, int& hi) {
  const int64_t cap = (int64_t)p.page * p.width;
  hi = max(p.lens[s], 0);
  if (hi > cap) hi = (int)cap;
  lo = p.window > 0 ? max(hi - p.window, 0) : 0;
}

// relu that keeps a NaN
__device__ __forceinline__ float relu(float x) { return x <= 0.f ? 0.f : x; }

constexpr int kWarps = 4;

// One CTA per (sequence, query head), one key per warp at a time, up to 8 elements per lane.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) paged_born_simple(const PagedParams p) {
  const int s = blockIdx.x, h = blockIdx.y, kvh = h / p.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int lo, hi;
  key_range(p, s, lo, hi);
  const float sc = p.scale ? p.scale[p.scale_per_head ? h : 0] : p.scale_value;
  const T* q = static_cast<const T*>(p.q) + s * p.qs[0] + h * p.qs[1];
  float qr[8], acc[8], z = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    qr[i] = d < p.D ? to_f32(q[d * p.qs[2]]) : 0.f;
    acc[i] = 0.f;
  }
  for (int j = lo + warp; j < hi; j += kWarps) {
    const int pg = p.table[s * p.table_stride + j / p.page], row = j % p.page;
    if (pg < 0 || pg >= p.pages) continue;
    const T* k = static_cast<const T*>(p.k) + pg * p.ks[0] + kvh * p.ks[1] + row * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + pg * p.vs[0] + kvh * p.vs[1] + row * p.vs[2];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d < p.D) dot += qr[i] * to_f32(k[d]);
    }
    const float a = relu(warp_sum(dot) * sc);
    const float w = a * a;
    z += w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d < p.D) acc[i] += w * to_f32(v[d]);
    }
  }
  __shared__ float so[kWarps][256], sz[kWarps];
#pragma unroll
  for (int i = 0; i < 8; ++i) so[warp][lane + 32 * i] = acc[i];
  if (lane == 0) sz[warp] = z;
  __syncthreads();
  z = 0.f;
  for (int w = 0; w < kWarps; ++w) z += sz[w];
  T* out = static_cast<T*>(p.out) + s * p.os[0] + h * p.os[1];
  for (int d = threadIdx.x; d < p.D; d += kWarps * 32) {
    float o = 0.f;
    for (int w = 0; w < kWarps; ++w) o += so[w][d];
    out[d * p.os[2]] = from_f32<T>(z == 0.f ? 0.f : o / (z + p.eps));
  }
}

struct WriteParams {
  int64_t N;
  int H, Hkv, D, page, pages, rope_rows;
  float eps;
  const void* qkv;
  int64_t ld;
  const float* cos;
  const float* sin;
  const int64_t* positions;
  const int64_t* slots;
  void* k;
  int64_t ks[4];
  void* v;
  int64_t vs[4];
  void* q;
  void* k_out;
  void* v_out;
};

// One warp per (token, head).
template <typename T>
__global__ void __launch_bounds__(256) paged_write_simple(const WriteParams p) {
  const int heads = p.H + 2 * p.Hkv;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= p.N * heads) return;
  const int64_t n = item / heads;
  const int h = (int)(item % heads), lane = threadIdx.x & 31, half = p.D / 2;
  const T* x = static_cast<const T*>(p.qkv) + n * p.ld + (int64_t)h * p.D;
  const int64_t slot = p.slots[n], pos = p.positions[n];
  const bool stored = slot >= 0 && slot < (int64_t)p.pages * p.page;
  const int64_t pg = stored ? slot / p.page : 0;
  const int row = stored ? (int)(slot % p.page) : 0;
  if (h >= p.H + p.Hkv) {  // V
    const int kvh = h - p.H - p.Hkv;
    T* to = static_cast<T*>(p.v) + pg * p.vs[0] + kvh * p.vs[1] + row * p.vs[2];
    T* copy = p.v_out ? static_cast<T*>(p.v_out) + (n * p.Hkv + kvh) * p.D : nullptr;
    for (int d = lane; d < p.D; d += 32) {
      if (stored) to[d] = x[d];
      if (copy) copy[d] = x[d];
    }
    return;
  }
  const bool known = pos >= 0 && pos < p.rope_rows;
  float a[4], b[4], ss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    if (d >= half) continue;
    const float c = known ? p.cos[pos * half + d] : NAN, sn = known ? p.sin[pos * half + d] : NAN;
    const float x1 = to_f32(x[d]), x2 = to_f32(x[d + half]);
    a[i] = x1 * c - x2 * sn;
    b[i] = x1 * sn + x2 * c;
    ss += a[i] * a[i] + b[i] * b[i];
  }
  const float r = rsqrtf(warp_sum(ss) + p.eps);
  T *to, *copy = nullptr;
  bool put = true;
  if (h < p.H) {
    to = static_cast<T*>(p.q) + (n * p.H + h) * p.D;
  } else {
    const int kvh = h - p.H;
    to = static_cast<T*>(p.k) + pg * p.ks[0] + kvh * p.ks[1] + row * p.ks[2];
    put = stored;
    if (p.k_out) copy = static_cast<T*>(p.k_out) + (n * p.Hkv + kvh) * p.D;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 32 * i;
    if (d >= half) continue;
    const T lo = from_f32<T>(a[i] * r), hi = from_f32<T>(b[i] * r);
    if (put) to[d] = lo, to[d + half] = hi;
    if (copy) copy[d] = lo, copy[d + half] = hi;
  }
}

int launched(int n) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return FB_ERR_LAUNCH;
  }
  set_last_launch_count(n);
  return FB_OK;
}

bool bad_dtype(int d) { return d != FB_F32 && d != FB_F16 && d != FB_BF16; }

bool bad_strides(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0) return true;
  return s[n - 1] != 1;
}

int paged_fwd(const fb_paged_args* a, cudaStream_t st) {
  if (a == nullptr) return FB_ERR_ARG;
  if (a->seqs < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65535 ||
      a->head_dim < 1 || a->head_dim > 256 || a->page_size < 1 || a->num_pages < 0 || a->max_pages < 0 ||
      (int64_t)a->page_size * a->max_pages > 0x7FFFFFFF)
    return FB_ERR_SHAPE;
  if (bad_dtype(a->dtype)) return FB_ERR_DTYPE;
  if (a->window_size < 0 || !(a->eps >= 0.f)) return FB_ERR_ARG;
  if (a->scale != nullptr && a->scale_numel != 1 && a->scale_numel != a->heads) return FB_ERR_ARG;
  if (a->seqs == 0) {
    set_last_launch_count(0);
    return FB_OK;
  }
  const bool keys = a->num_pages > 0 && a->max_pages > 0;
  if (a->q == nullptr || a->out == nullptr || a->lens == nullptr) return FB_ERR_ARG;
  if (keys && (a->k == nullptr || a->v == nullptr || a->table == nullptr)) return FB_ERR_ARG;
  if (bad_strides(a->k_stride, 4) || bad_strides(a->v_stride, 4) || bad_strides(a->q_stride, 3) ||
      bad_strides(a->out_stride, 3) || a->table_stride < 0)
    return FB_ERR_ALIGN;
  PagedParams p{};
  p.S = a->seqs; p.H = a->heads; p.Hkv = a->kv_heads; p.G = a->heads / a->kv_heads; p.D = a->head_dim;
  p.page = a->page_size; p.pages = a->num_pages; p.width = keys ? a->max_pages : 0;
  p.window = a->window_size; p.eps = a->eps; p.scale_value = a->scale_value;
  p.scale = a->scale; p.scale_per_head = a->scale_numel > 1;
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
  for (int i = 0; i < 3; ++i) p.qs[i] = a->q_stride[i], p.os[i] = a->out_stride[i];
  for (int i = 0; i < 4; ++i) p.ks[i] = a->k_stride[i], p.vs[i] = a->v_stride[i];
  p.table = a->table; p.table_stride = a->table_stride; p.lens = a->lens;
  const dim3 grid(p.S, p.H);
  if (a->dtype == FB_F32) paged_born_simple<float><<<grid, kWarps * 32, 0, st>>>(p);
  else if (a->dtype == FB_F16) paged_born_simple<__half><<<grid, kWarps * 32, 0, st>>>(p);
  else paged_born_simple<__nv_bfloat16><<<grid, kWarps * 32, 0, st>>>(p);
  return launched(1);
}

int paged_write(const fb_paged_write_args* a, cudaStream_t st) {
  if (a == nullptr) return FB_ERR_ARG;
  if (a->tokens < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65535 ||
      a->head_dim < 2 || a->head_dim > 256 || a->head_dim % 2 != 0 || a->page_size < 1 || a->num_pages < 0 ||
      a->rope_rows < 0)
    return FB_ERR_SHAPE;
  if (bad_dtype(a->dtype)) return FB_ERR_DTYPE;
  if (a->tokens == 0) {
    set_last_launch_count(0);
    return FB_OK;
  }
  if (a->qkv == nullptr || a->cos == nullptr || a->sin == nullptr || a->positions == nullptr || a->slots == nullptr ||
      a->q == nullptr || (a->k_out == nullptr) != (a->v_out == nullptr) || !(a->eps >= 0.f) ||
      (a->num_pages > 0 && (a->k == nullptr || a->v == nullptr)))
    return FB_ERR_ARG;
  if (bad_strides(a->k_stride, 4) || bad_strides(a->v_stride, 4) || a->qkv_stride < 0) return FB_ERR_ALIGN;
  WriteParams p{};
  p.N = a->tokens; p.H = a->heads; p.Hkv = a->kv_heads; p.D = a->head_dim;
  p.page = a->page_size; p.pages = a->num_pages; p.rope_rows = a->rope_rows; p.eps = a->eps;
  p.qkv = a->qkv; p.ld = a->qkv_stride; p.cos = a->cos; p.sin = a->sin;
  p.positions = a->positions; p.slots = a->slots; p.k = a->k; p.v = a->v; p.q = a->q;
  p.k_out = a->k_out; p.v_out = a->v_out;
  for (int i = 0; i < 4; ++i) p.ks[i] = a->k_stride[i], p.vs[i] = a->v_stride[i];
  const int64_t blocks = (p.N * (p.H + 2 * p.Hkv) + 7) / 8;
  if (blocks > 0x7FFFFFFF) return FB_ERR_SHAPE;
  if (a->dtype == FB_F32) paged_write_simple<float><<<(unsigned)blocks, 256, 0, st>>>(p);
  else if (a->dtype == FB_F16) paged_write_simple<__half><<<(unsigned)blocks, 256, 0, st>>>(p);
  else paged_write_simple<__nv_bfloat16><<<(unsigned)blocks, 256, 0, st>>>(p);
  return launched(1);
}

}  // namespace
}  // namespace fb

extern "C" {

size_t fb_paged_workspace_size(const fb_paged_args*) { return 0; }
int fb_paged_born_fwd(const fb_paged_args* args, void* stream) {
  return fb::paged_fwd(args, static_cast<cudaStream_t>(stream));
}
int fb_paged_qkv_write(const fb_paged_write_args* args, void* stream) {
  return fb::paged_write(args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
