// fb_paged.cu -- generating from a trained flash-Born GPT: Born attention of one new token per
// sequence over a paged key-value cache, and the kernel that fills that cache.
//
//   paged_born_fwd   a_j = relu(scale_h <q, k_j>), p_j = a_j^2, out = (sum_j p_j v_j) / (sum_j p_j + eps)
//   paged_qkv_write  Q, K = l2n(rope(.)), V; K and V rows into their pages' slots
//
// The attention reads every key and value once and does 4 operations per element and query head:
// HBM bandwidth bounds it.  Born weights need no running maximum, so a sequence's keys can be cut
// anywhere and the pieces' (sum p v, sum p) just add.  The work is cut evenly whatever the lengths:
// a unit is (sequence, kv head, up to HU query heads), its keys are tiles of kTile, all units' tiles
// form one line, and CTA c of C takes the c-th C-th of it.  Lengths are read on the device (the host
// knows only the table's width), so a call needs no synchronisation and replays from a graph.  A unit
// inside one CTA's share is finished there; pieces of a unit that spans shares go to the workspace,
// two slots per CTA, and a second kernel adds them in share order (the same bits every time).
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "fb_common.cuh"

namespace fb {
namespace {

constexpr int kWarps = 4;             // per CTA
constexpr int kSub = 16;              // keys a warp takes at a time
constexpr int kTile = kWarps * kSub;  // keys a CTA takes at a time
constexpr int kJoinThreads = 256;

struct PagedParams {
  int S, H, Hkv, G, D;
  int page, pages, width;  // page rows, pages, table columns
  int page_shift;          // log2 of page where it is a power of two, else -1
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
  int HU, chunks, U;  // query heads per unit, units per kv head, units per sequence
  int C;              // CTAs that share the tiles
  float* part;        // [C][2][HU][D] sums of p v, then [C][2][HU] sums of p
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The keys [lo, hi) of one sequence: what the length, the table's capacity and the window leave; and
// the tiles they take, counted from a multiple of kSub so that a warp's keys do not straddle pages
// whose size is a multiple of it.  A sequence without keys has one (empty) tile: its zeros get written.
struct Keys {
  int lo, hi, base, tiles;
};
__device__ __forceinline__ Keys keys_of(const PagedParams& p, int s) {
  Keys k;
  k.hi = min(max(p.lens[s], 0), p.page * p.width);
  k.lo = p.window > 0 ? max(k.hi - p.window, 0) : 0;
  k.base = k.lo & ~(kSub - 1);
  k.tiles = max((k.hi - k.base + kTile - 1) / kTile, 1);
  return k;
}

// relu that keeps a NaN
__device__ __forceinline__ float relu(float x) { return x <= 0.f ? 0.f : x; }

// The tiles of the sequences before `stop` (or of all: stop = S), summed by a whole block.  Per
// sequence, to be multiplied by the units.
template <int THREADS>
__device__ int64_t tiles_before(const PagedParams& p, int stop, int64_t* sh) {
  int64_t n = 0;
  for (int s = threadIdx.x; s < stop; s += THREADS) n += keys_of(p, s).tiles;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) n += sh[w];
  return n;
}

// The sequence that holds tile t (in tiles per sequence, t below the total) and the tiles before it,
// searched by the whole block, THREADS sequences at a time.
template <int THREADS>
__device__ void find_sequence(const PagedParams& p, int64_t t, int64_t* sh, int& seq, int64_t& before) {
  __shared__ int found;
  __shared__ int64_t found_before;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) found = -1;
  int64_t start = 0;
  for (int s0 = 0; s0 < p.S; s0 += THREADS) {
    const int s = s0 + threadIdx.x;
    const int64_t n = s < p.S ? keys_of(p, s).tiles : 0;
    int64_t incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = incl;
    __syncthreads();
    int64_t all = start;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) incl += sh[w];
      all += sh[w];
    }
    incl += start;
    if (t < incl && t >= incl - n) {
      found = s;
      found_before = incl - n;
    }
    start = all;
    if (t < all) break;  // the same for every thread
  }
  __syncthreads();
  seq = found;
  before = found_before;
}

// Where a piece's sums go: the result when it is the whole unit, else the CTA's slot in the workspace
// (slot 1: the unit begins here and goes on in the next CTA; slot 0: it began before).  red holds each
// warp's [HU][D + 4] sums of p v and rz its HU sums of p.
template <typename T>
__device__ void finish_piece(const PagedParams& p, const float* red, int red_warp, const float* rz, int s, int unit,
                             bool whole, bool begins) {
  const int kvh = unit / p.chunks, h0 = unit % p.chunks * p.HU, nh = min(p.HU, p.G - h0);
  const int ld = p.D + 4;
  const int64_t slot = (int64_t)blockIdx.x * 2 + (begins ? 1 : 0);
  for (int i = threadIdx.x; i < nh * p.D; i += kWarps * 32) {
    const int h = i / p.D, d = i % p.D;
    float o = 0.f, z = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      o += red[w * red_warp + h * ld + d];
      z += rz[w * p.HU + h];
    }
    if (whole) {
      T* out = static_cast<T*>(p.out) + s * p.os[0] + (int64_t)(kvh * p.G + h0 + h) * p.os[1];
      out[d] = from_f32<T>(z == 0.f ? 0.f : o / (z + p.eps));
    } else {
      p.part[(slot * p.HU + h) * p.D + d] = o;
      if (d == 0) p.part[(int64_t)p.C * 2 * p.HU * p.D + slot * p.HU + h] = z;
    }
  }
}

// Walks the CTA's share of the tiles: piece(s, keys, unit, first tile, last tile + 1, whole, begins).
template <typename F>
__device__ __forceinline__ void walk_share(const PagedParams& p, int64_t* sh, F&& piece) {
  const int64_t total = tiles_before<kWarps * 32>(p, p.S, sh) * p.U;
  const int64_t C = min((int64_t)p.C, total);  // no empty shares
  if (blockIdx.x >= C) return;
  const int64_t t0 = total * blockIdx.x / C, t1 = total * (blockIdx.x + 1) / C;
  int s;
  int64_t first;
  find_sequence<kWarps * 32>(p, t0 / p.U, sh, s, first);
  first *= p.U;
  Keys k = keys_of(p, s);
  for (int64_t t = t0; t < t1;) {
    while (t >= first + (int64_t)k.tiles * p.U) {
      first += (int64_t)k.tiles * p.U;
      k = keys_of(p, ++s);
    }
    const int unit = (int)((t - first) / k.tiles), a = (int)((t - first) % k.tiles);
    const int b = (int)min((int64_t)k.tiles, a + (t1 - t));
    piece(s, k, unit, a, b, a == 0 && b == k.tiles, a == 0);
    t += b - a;
  }
}

// Page and row of a key; false where the table holds no page for it.
__device__ __forceinline__ bool find_page(const PagedParams& p, const int32_t* table, int key, int& pg, int& row) {
  const int i = p.page_shift >= 0 ? key >> p.page_shift : key / p.page;
  pg = table[i];
  row = key - i * p.page;
  return pg >= 0 && pg < p.pages;
}

// ------------------------------------------------------------------------------------------
// Tensor-core kernel: bf16 or fp16, D = 64 or 128, rows on 16-byte boundaries
// ------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_1688_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint32_t f2_to_bf2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xFFFFu))); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }

template <int D> struct TcShape {
  static constexpr int kStageBytes = 2 * kSub * D * 2;  // per warp: kSub keys, then their values
  static constexpr int kStages = D == 64 ? 4 : 3;
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  static constexpr int kCtasPerSm = D == 64 ? 3 : 2;
};

// Rows of the matrix instructions are the unit's query heads (up to 16), so a key is read once for all
// of them.  Lane (r = lane / 4, c = lane % 4) of a warp needs, of kSub keys,
//   S = Q K^T  (B = K^T):  keys r and r + 8, and of them any dimensions as long as Q's fragment has
//              the same: it takes the 16-byte pieces at 32 j + 8 c
//   O = P V    (B = V):  keys 2c, 2c + 1, 2c + 8, 2c + 9; column r of instruction (jj, e) is dimension
//              64 jj + 8 r + e, so it takes the 16-byte pieces at 64 jj + 8 r and pairs two keys' words
// and S's accumulator has P's operand layout: no transposing load, no exchange between lanes.  Each warp
// has a ring of kStages x kSub keys and values of its own in shared memory and no barrier with the others.
// Its copies take whole rows by neighbouring lanes (copied in the lanes' own order instead, a sector crossed
// from L2 twice: 1.94 GB for 0.97 GB of keys).  Piece i of row t lies at i ^ 4 (t & 1) for keys, i ^ 2 ((t / 2) & 3)
// for values: eight lanes' reads then fall on eight different bank groups.
template <typename T, int D>
__global__ void __launch_bounds__(kWarps * 32, TcShape<D>::kCtasPerSm) paged_born_tc(const PagedParams p) {
  using Sh = TcShape<D>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t sh[kWarps];
  __shared__ float rz[kWarps * 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * Sh::kStages * Sh::kStageBytes;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
  constexpr int kRow = 2 * D;          // bytes
  constexpr int kPieces = D / 8;       // per row
  constexpr int kRows = 32 / kPieces;  // that one copy instruction takes
  const int cp_row = lane / kPieces, cp_piece = lane % kPieces;
  float* red = reinterpret_cast<float*>(smem);
  constexpr int kRedWarp = Sh::kStages * Sh::kStageBytes / 4;
  static_assert(16 * (D + 4) <= kRedWarp, "a warp's sums fit its ring");
  const bool page_uniform = p.page % kSub == 0;  // a warp's keys are rows of one page

  asm volatile("griddepcontrol.launch_dependents;");
  walk_share(p, sh, [&](int s, const Keys& kk, int unit, int ta, int tb, bool whole, bool begins) {
    const int kvh = unit / p.chunks, h0 = unit % p.chunks * p.HU, nh = min(p.HU, p.G - h0);
    const int32_t* table = p.table + s * p.table_stride;
    const T* kbase = static_cast<const T*>(p.k) + kvh * p.ks[1];
    const T* vbase = static_cast<const T*>(p.v) + kvh * p.vs[1];
    const int first = kk.base + ta * kTile + warp * kSub;  // this warp's first key
    const int n = kk.hi > first ? min(tb - ta, (kk.hi - first + kTile - 1) / kTile) : 0;  // its steps

    // page of the step's first key (page_uniform) or of key lane & 15
    auto lookup = [&](int i) -> int {
      const int key = first + i * kTile + (page_uniform ? 0 : lane & 15);
      if (i >= n || key >= kk.hi || (!page_uniform && key < kk.lo)) return -1;
      return table[p.page_shift >= 0 ? key >> p.page_shift : key / p.page];
    };
    auto issue = [&](int i, int pg) {
      const int key0 = first + i * kTile;
      if (i < n) {
        const uint32_t to = ring_s + (i % Sh::kStages) * Sh::kStageBytes;
        const bool have = pg >= 0 && pg < p.pages;
        int row0 = 0;
        const T *ksrc = kbase + 8 * cp_piece, *vsrc = vbase + 8 * cp_piece;
        if (page_uniform) {
          row0 = p.page_shift >= 0 ? key0 & (p.page - 1) : key0 % p.page;
          if (have) {
            ksrc += pg * p.ks[0] + (row0 + cp_row) * p.ks[2];
            vsrc += pg * p.vs[0] + (row0 + cp_row) * p.vs[2];
          }
        } else {
          row0 = (key0 + (lane & 15)) % p.page;
        }
        const int packed = have ? pg : -1;
#pragma unroll
        for (int x = 0; x < kSub / kRows; ++x) {
          const int t = x * kRows + cp_row;
          const T *kx = ksrc, *vx = vsrc;
          bool ok = have;
          if (page_uniform) {
            ok = ok && key0 + t >= kk.lo && key0 + t < kk.hi;
            if (ok) kx += x * kRows * p.ks[2], vx += x * kRows * p.vs[2];
          } else {
            const int g = __shfl_sync(0xffffffffu, packed, t), w = __shfl_sync(0xffffffffu, row0, t);
            ok = g >= 0;
            if (ok) kx += g * p.ks[0] + w * p.ks[2], vx += g * p.vs[0] + w * p.vs[2];
          }
          copy16(to + t * kRow + (cp_piece ^ 4 * (t & 1)) * 16, kx, ok);
          copy16(to + kSub * kRow + t * kRow + (cp_piece ^ 2 * (t >> 1 & 3)) * 16, vx, ok);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    // Q: heads r and r + 8 of the unit, zero where it has fewer
    uint32_t qf[D / 16][4];
    float sc[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int h = r + 8 * x;
      const int head = kvh * p.G + h0 + h;
      const T* q = static_cast<const T*>(p.q) + s * p.qs[0] + head * p.qs[1];
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (h < nh) w = *reinterpret_cast<const uint4*>(q + 32 * j + 8 * c);
        qf[2 * j][x] = w.x;
        qf[2 * j][2 + x] = w.y;
        qf[2 * j + 1][x] = w.z;
        qf[2 * j + 1][2 + x] = w.w;
      }
      sc[x] = h < nh ? (p.scale ? p.scale[p.scale_per_head ? head : 0] : p.scale_value) : 0.f;
    }
    float o[D / 8][4], z[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    {
      int pg[Sh::kStages - 1];
#pragma unroll
      for (int i = 0; i < Sh::kStages - 1; ++i) pg[i] = lookup(i);
#pragma unroll
      for (int i = 0; i < Sh::kStages - 1; ++i) issue(i, pg[i]);
    }
    int next = lookup(Sh::kStages - 1);
    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Sh::kStages - 2) : "memory");
      __syncwarp();  // the other lanes' copies have landed too
      const uint8_t* stage = ring + (i % Sh::kStages) * Sh::kStageBytes;
      const uint8_t* kst = stage + r * kRow + c * 16;
      const uint8_t* vst = stage + (kSub + 2 * c) * kRow + (r ^ 2 * c) * 16;
      float sacc[2][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sacc[x][e] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint4 w = *reinterpret_cast<const uint4*>(kst + 8 * x * kRow + 64 * (j ^ (r & 1)));
          mma_16816<T>(sacc[x], qf[2 * j], w.x, w.y);
          mma_16816<T>(sacc[x], qf[2 * j + 1], w.z, w.w);
        }
      }
      // sacc[x][e]: head r + 8 (e / 2), key 8 x + 2 c + e % 2.  A key that does not count has K and V of
      // zero; its weight is set to 0 as well, for a Q that is not finite.
      float w[2][4];
      const int key0 = first + i * kTile;
      const bool edge = key0 < kk.lo || key0 + kSub > kk.hi;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float a = relu(sacc[x][e] * sc[e >> 1]);
          w[x][e] = a * a;
          const int key = key0 + 8 * x + 2 * c + (e & 1);
          if (edge && (key < kk.lo || key >= kk.hi)) w[x][e] = 0.f;
        }
      if constexpr (!kHalf) {
        // P goes into the product as the sum of two bf16 numbers, 16 bits of it: one alone would add as much
        // error as the rounding of the result does (measured: 2.3e-3 of the result against 1.6e-3)
        uint32_t pf[4], pl[4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float w0 = w[x][2 * y], w1 = w[x][2 * y + 1];
            const uint32_t b = f2_to_bf2(w0, w1);
            pf[2 * x + y] = b;
            pl[2 * x + y] = f2_to_bf2(w0 - __uint_as_float(b << 16), w1 - __uint_as_float(b & 0xFFFF0000u));
            z[y] += w0 + w1;
          }
#pragma unroll
        for (int jj = 0; jj < D / 64; ++jj) {
          uint4 v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            v[x] = *reinterpret_cast<const uint4*>(vst + ((x & 1) + 8 * (x >> 1)) * kRow + 128 * jj);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v0 = (&v[0].x)[e], v1 = (&v[1].x)[e], v2 = (&v[2].x)[e], v3 = (&v[3].x)[e];
            const uint32_t even0 = __byte_perm(v0, v1, 0x5410), even1 = __byte_perm(v2, v3, 0x5410);
            const uint32_t odd0 = __byte_perm(v0, v1, 0x7632), odd1 = __byte_perm(v2, v3, 0x7632);
            mma_16816<T>(o[8 * jj + 2 * e], pf, even0, even1);
            mma_16816<T>(o[8 * jj + 2 * e + 1], pf, odd0, odd1);
            mma_16816<T>(o[8 * jj + 2 * e], pl, even0, even1);
            mma_16816<T>(o[8 * jj + 2 * e + 1], pl, odd0, odd1);
          }
        }
      } else {
        // fp16 cannot hold p = a^2 (a > 256 overflows it): P goes through TF32, fp16's 11 bits with fp32's
        // range, in which V's values are exact.  Instruction x takes key 8 x + 2 c as its column c and
        // 8 x + 2 c + 1 as c + 4.
        uint32_t pf[2][4];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t b;
            asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(b) : "f"(w[x][e]));
            pf[x][(e >> 1) + 2 * (e & 1)] = b;
            z[e >> 1] += __uint_as_float(b);
          }
#pragma unroll
        for (int jj = 0; jj < D / 64; ++jj) {
          uint4 v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            v[x] = *reinterpret_cast<const uint4*>(vst + ((x & 1) + 8 * (x >> 1)) * kRow + 128 * jj);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t va = (&v[2 * x].x)[e], vb = (&v[2 * x + 1].x)[e];
              mma_1688_tf32(o[8 * jj + 2 * e], pf[x], __float_as_uint(half_lo(va)), __float_as_uint(half_lo(vb)));
              mma_1688_tf32(o[8 * jj + 2 * e + 1], pf[x], __float_as_uint(half_hi(va)), __float_as_uint(half_hi(vb)));
            }
        }
      }
      __syncwarp();
      issue(i + Sh::kStages - 1, next);  // over the stage that every lane read in the previous step
      next = lookup(i + Sh::kStages);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();  // every lane has read its last stage before the sums go over the ring

    // o[8 jj + e][.]: heads r, r + 8; dimensions 64 jj + 16 c + e and + 8.  Sums over the warps.
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      z[y] += __shfl_xor_sync(0xffffffffu, z[y], 1);
      z[y] += __shfl_xor_sync(0xffffffffu, z[y], 2);
      const int h = r + 8 * y;
      if (h < nh) {
        if (c == 0) rz[warp * p.HU + h] = z[y];
        float* to = red + warp * kRedWarp + h * (D + 4) + 16 * c;
#pragma unroll
        for (int jj = 0; jj < D / 64; ++jj)
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 8; e += 4)
              *reinterpret_cast<float4*>(to + 64 * jj + 8 * half + e) =
                  make_float4(o[8 * jj + e][2 * y + half], o[8 * jj + e + 1][2 * y + half],
                              o[8 * jj + e + 2][2 * y + half], o[8 * jj + e + 3][2 * y + half]);
      }
    }
    __syncthreads();
    finish_piece<T>(p, red, kRedWarp, rz, s, unit, whole, begins);
    __syncthreads();  // the sums are read before the ring and rz are written again
  });
}

// ------------------------------------------------------------------------------------------
// CUDA-core kernel: every other type, head dimension and alignment, fp32 arithmetic
// ------------------------------------------------------------------------------------------
template <typename T, int VEC> struct Piece;  // VEC elements of one load, as floats
template <typename T> struct Piece<T, 1> {
  __device__ static void load(const T* p, float (&f)[1]) { f[0] = to_f32(*p); }
};
template <> struct Piece<float, 4> {
  __device__ static void load(const float* p, float (&f)[4]) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    f[0] = w.x, f[1] = w.y, f[2] = w.z, f[3] = w.w;
  }
};
template <> struct Piece<__nv_bfloat16, 8> {
  __device__ static void load(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float((&w.x)[i] << 16);
      f[2 * i + 1] = __uint_as_float((&w.x)[i] & 0xFFFF0000u);
    }
  }
};
template <> struct Piece<__half, 8> {
  __device__ static void load(const __half* p, float (&f)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = half_lo((&w.x)[i]), f[2 * i + 1] = half_hi((&w.x)[i]);
  }
};

// Lane (r, c) takes key r of 8 and the pieces c, c + 4, ... of its row (VEC elements each, E = NI VEC of
// them, E at least D / 4): a dot product is finished by two shuffles among four lanes, the four have the
// weight, and each adds it times its own part of the value row.  The eight keys' sums meet at the end of the
// piece.  HU query heads share a read of the row; a kv head with more is several units.
template <typename T, int VEC, int NI, int HU>
__global__ void __launch_bounds__(kWarps * 32) paged_born_general(const PagedParams p) {
  constexpr int E = NI * VEC;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t sh[kWarps];
  __shared__ float rz[kWarps * HU];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  float* red = reinterpret_cast<float*>(smem);
  const int red_warp = HU * (p.D + 4);
  float* qsm = red + kWarps * red_warp;  // [HU][4 E] scaled queries, piece i of lane c at (i * 4 + c) VEC

  asm volatile("griddepcontrol.launch_dependents;");
  walk_share(p, sh, [&](int s, const Keys& kk, int unit, int ta, int tb, bool whole, bool begins) {
    const int kvh = unit / p.chunks, h0 = unit % p.chunks * p.HU, nh = min(p.HU, p.G - h0);
    const int32_t* table = p.table + s * p.table_stride;
    const T* kbase = static_cast<const T*>(p.k) + kvh * p.ks[1];
    const T* vbase = static_cast<const T*>(p.v) + kvh * p.vs[1];
    for (int i = threadIdx.x; i < HU * 4 * E; i += kWarps * 32) {
      const int h = i / (4 * E), d = i % (4 * E), head = kvh * p.G + h0 + h;
      float x = 0.f;
      if (h < nh && d < p.D)
        x = to_f32(static_cast<const T*>(p.q)[s * p.qs[0] + head * p.qs[1] + d]);
      qsm[i] = x;
    }
    float sc[HU];
#pragma unroll
    for (int h = 0; h < HU; ++h)
      sc[h] = h < nh ? (p.scale ? p.scale[p.scale_per_head ? kvh * p.G + h0 + h : 0] : p.scale_value) : 0.f;
    __syncthreads();
    float o[HU][E], z[HU];
#pragma unroll
    for (int h = 0; h < HU; ++h) {
      z[h] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) o[h][e] = 0.f;
    }
    const int end = min(kk.hi, kk.base + tb * kTile);
    for (int key0 = kk.base + ta * kTile + warp * 8; key0 < end; key0 += kWarps * 8) {
      const int key = key0 + r;
      int pg = 0, row = 0;
      const bool counts = key >= kk.lo && key < end && find_page(p, table, key, pg, row);
      const T* k = kbase + pg * p.ks[0] + row * p.ks[2];
      const T* v = vbase + pg * p.vs[0] + row * p.vs[2];
      float kf[NI][VEC], vf[NI][VEC];
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int d = (i * 4 + c) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) kf[i][e] = vf[i][e] = 0.f;
        if (counts && d < p.D) {
          Piece<T, VEC>::load(k + d, kf[i]);
          Piece<T, VEC>::load(v + d, vf[i]);
        }
      }
#pragma unroll
      for (int h = 0; h < HU; ++h) {
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) dot = fmaf(qsm[h * 4 * E + (i * 4 + c) * VEC + e], kf[i][e], dot);
        dot += __shfl_xor_sync(0xffffffffu, dot, 1);
        dot += __shfl_xor_sync(0xffffffffu, dot, 2);
        const float a = relu(dot * sc[h]);
        const float w = counts ? a * a : 0.f;
        z[h] += w;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[h][i * VEC + e] = fmaf(w, vf[i][e], o[h][i * VEC + e]);
      }
    }
#pragma unroll
    for (int h = 0; h < HU; ++h) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) z[h] += __shfl_xor_sync(0xffffffffu, z[h], x);
      if (lane == 0) rz[warp * HU + h] = z[h];
#pragma unroll
      for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) o[h][e] += __shfl_xor_sync(0xffffffffu, o[h][e], x);
        const int d = (e / VEC * 4 + c) * VEC + e % VEC;
        if (r == 0 && d < p.D) red[warp * red_warp + h * (p.D + 4) + d] = o[h][e];
      }
    }
    __syncthreads();
    finish_piece<T>(p, red, red_warp, rz, s, unit, whole, begins);
    __syncthreads();
  });
}

// ------------------------------------------------------------------------------------------
// The pieces of units that span several CTAs' shares, added in share order: one CTA per query head,
// kJoinThreads / D' threads (D' = D rounded up to a power of two) on each dimension.
// ------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_join(const PagedParams p) {
  __shared__ int64_t sh[kJoinThreads / 32];
  __shared__ float so[kJoinThreads], sz[kJoinThreads];
  const int s = blockIdx.x / p.H, head = blockIdx.x % p.H;
  const int kvh = head / p.G, chunk = head % p.G / p.HU, h = head % p.G % p.HU;
  const int64_t total = tiles_before<kJoinThreads>(p, p.S, sh) * p.U;
  const int64_t before = tiles_before<kJoinThreads>(p, s, sh) * p.U;
  const int n = keys_of(p, s).tiles;
  const int64_t t0 = before + (int64_t)(kvh * p.chunks + chunk) * n;
  // CTA of tile t: the last one whose share starts at or before it
  const int64_t C = min((int64_t)p.C, total);
  const int c0 = (int)(((t0 + 1) * C - 1) / total), c1 = (int)(((t0 + n) * C - 1) / total);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1) return;  // finished by that CTA
  int width = 1;
  while (width < p.D) width <<= 1;
  const int ways = kJoinThreads / width, way = threadIdx.x / width, d = threadIdx.x % width;
  const float* zs = p.part + (int64_t)p.C * 2 * p.HU * p.D;
  float o = 0.f, z = 0.f;
  if (d < p.D) {
#pragma unroll 4
    for (int c = c0 + way; c <= c1; c += ways) {
      const int64_t slot = (int64_t)c * 2 + (c == c0 ? 1 : 0);
      o += p.part[(slot * p.HU + h) * p.D + d];
      z += zs[slot * p.HU + h];
    }
  }
  so[threadIdx.x] = o;
  sz[threadIdx.x] = z;
  __syncthreads();
  if (way == 0 && d < p.D) {
    for (int w = 1; w < ways; ++w) {
      o += so[w * width + d];
      z += sz[w * width + d];
    }
    T* out = static_cast<T*>(p.out) + s * p.os[0] + head * p.os[1];
    out[d] = from_f32<T>(z == 0.f ? 0.f : o / (z + p.eps));
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

bool aligned16(const void* p, const int64_t* s, int n, int size) {
  bool ok = (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  for (int i = 0; i < n; ++i) ok = ok && s[i] * size % 16 == 0;
  return ok;
}

// What a call launches, from sizes, types and alignment alone.
struct PagedPlan {
  bool tc;        // the tensor-core kernel
  int vec;        // CUDA-core kernel: elements per load
  int size_class; // ... and 0, 1, 2: D up to 64, 128, 256
  bool join;
  int HU, chunks, C;
  size_t workspace;
};

PagedPlan plan_paged(const fb_paged_args* a) {
  PagedPlan pl{};
  const int G = a->heads / a->kv_heads, size = a->dtype == FB_F32 ? 4 : 2;
  const bool rows16 = a->head_dim * size % 16 == 0 && aligned16(a->k, a->k_stride, 3, size) &&
                      aligned16(a->v, a->v_stride, 3, size);
  pl.tc = size == 2 && (a->head_dim == 64 || a->head_dim == 128) && rows16 && aligned16(a->q, a->q_stride, 2, size);
  pl.vec = rows16 ? 16 / size : 1;
  pl.size_class = a->head_dim <= 64 ? 0 : a->head_dim <= 128 ? 1 : 2;
  const int hu = pl.tc ? 16 : 4 >> pl.size_class;
  pl.HU = hu;
  pl.chunks = (G + hu - 1) / hu;
  // The most tiles that the lengths can give: the table's capacity, or the window and what it straddles
  int64_t cap = (int64_t)a->page_size * a->max_pages;
  if (a->window_size > 0) cap = std::min<int64_t>(cap, (int64_t)a->window_size + kSub);
  const int64_t per_unit = std::max<int64_t>((cap + kTile - 1) / kTile, 1);
  const int64_t units = (int64_t)a->seqs * a->kv_heads * pl.chunks;
  const int per_sm = pl.tc ? (a->head_dim == 64 ? TcShape<64>::kCtasPerSm : TcShape<128>::kCtasPerSm) : 4;
  // units of one tile cannot be cut: one CTA each, nothing to join
  pl.join = per_unit > 1;
  pl.C = (int)std::min<int64_t>(units * per_unit, pl.join ? (int64_t)per_sm * sm_count() : 0x7FFFFFFF);
  pl.workspace = pl.join ? (size_t)pl.C * 2 * pl.HU * (a->head_dim + 1) * sizeof(float) : 0;
  return pl;
}

int check_paged(const fb_paged_args* a) {
  if (a == nullptr) return FB_ERR_ARG;
  if (a->seqs < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65535 ||
      a->head_dim < 1 || a->head_dim > 256 || a->page_size < 1 || a->num_pages < 0 || a->max_pages < 0 ||
      (int64_t)a->page_size * a->max_pages > 0x7FFFFFFF - 2 * kTile || (int64_t)a->seqs * a->heads > 0x7FFFFFFF)
    return FB_ERR_SHAPE;
  if (bad_dtype(a->dtype)) return FB_ERR_DTYPE;
  if (a->window_size < 0 || !(a->eps >= 0.f)) return FB_ERR_ARG;
  if (a->scale != nullptr && a->scale_numel != 1 && a->scale_numel != a->heads) return FB_ERR_ARG;
  if (a->seqs == 0) return FB_OK;
  const bool keys = a->num_pages > 0 && a->max_pages > 0;
  if (a->q == nullptr || a->out == nullptr || a->lens == nullptr) return FB_ERR_ARG;
  if (keys && (a->k == nullptr || a->v == nullptr || a->table == nullptr)) return FB_ERR_ARG;
  if (bad_strides(a->k_stride, 4) || bad_strides(a->v_stride, 4) || bad_strides(a->q_stride, 3) ||
      bad_strides(a->out_stride, 3) || a->table_stride < 0)
    return FB_ERR_ALIGN;
  return FB_OK;
}

template <typename T>
cudaError_t launch_general(const PagedParams& p, const PagedPlan& pl, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int smem = (kWarps * p.HU * (p.D + 4) + p.HU * (256 >> (2 - pl.size_class))) * (int)sizeof(float);
  const dim3 grid(p.C), block(kWarps * 32);
  if (pl.vec > 1) {
    if (pl.size_class == 0) paged_born_general<T, V, 16 / V, 4><<<grid, block, smem, st>>>(p);
    else if (pl.size_class == 1) paged_born_general<T, V, 32 / V, 2><<<grid, block, smem, st>>>(p);
    else paged_born_general<T, V, 64 / V, 1><<<grid, block, smem, st>>>(p);
  } else {
    if (pl.size_class == 0) paged_born_general<T, 1, 16, 4><<<grid, block, smem, st>>>(p);
    else if (pl.size_class == 1) paged_born_general<T, 1, 32, 2><<<grid, block, smem, st>>>(p);
    else paged_born_general<T, 1, 64, 1><<<grid, block, smem, st>>>(p);
  }
  return cudaGetLastError();
}

template <typename T, int D>
cudaError_t launch_tc(const PagedParams& p, cudaStream_t st) {
  const cudaError_t e = set_smem_limit_once(reinterpret_cast<const void*>(&paged_born_tc<T, D>), TcShape<D>::kSmem);
  if (e != cudaSuccess) return e;
  paged_born_tc<T, D><<<p.C, kWarps * 32, TcShape<D>::kSmem, st>>>(p);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_paged(const PagedParams& p, const PagedPlan& pl, cudaStream_t st) {
  cudaError_t e;
  if constexpr (sizeof(T) == 2) {
    e = !pl.tc ? launch_general<T>(p, pl, st) : p.D == 64 ? launch_tc<T, 64>(p, st) : launch_tc<T, 128>(p, st);
  } else {
    e = launch_general<T>(p, pl, st);
  }
  if (e != cudaSuccess || !pl.join) return e;
  // the join's CTAs start while the last shares still run (their count is read meanwhile) and wait for them
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(p.S * p.H));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join<T>, p);
}

int paged_fwd(const fb_paged_args* a, cudaStream_t st) {
  const int rc = check_paged(a);
  if (rc != FB_OK) return rc;
  if (a->seqs == 0) {
    set_last_launch_count(0);
    return FB_OK;
  }
  const PagedPlan pl = plan_paged(a);
  if (pl.workspace > 0 && (a->workspace == nullptr || a->workspace_bytes < pl.workspace)) return FB_ERR_WORKSPACE;
  PagedParams p{};
  p.S = a->seqs; p.H = a->heads; p.Hkv = a->kv_heads; p.G = a->heads / a->kv_heads; p.D = a->head_dim;
  p.page = a->page_size; p.pages = a->num_pages;
  p.width = a->num_pages > 0 ? a->max_pages : 0;
  p.page_shift = -1;
  if ((p.page & (p.page - 1)) == 0)
    for (p.page_shift = 0; (1 << p.page_shift) < p.page;) ++p.page_shift;
  p.window = a->window_size; p.eps = a->eps; p.scale_value = a->scale_value;
  p.scale = a->scale; p.scale_per_head = a->scale_numel > 1;
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
  for (int i = 0; i < 3; ++i) p.qs[i] = a->q_stride[i], p.os[i] = a->out_stride[i];
  for (int i = 0; i < 4; ++i) p.ks[i] = a->k_stride[i], p.vs[i] = a->v_stride[i];
  p.table = a->table; p.table_stride = a->table_stride; p.lens = a->lens;
  p.HU = pl.HU; p.chunks = pl.chunks; p.U = p.Hkv * p.chunks; p.C = pl.C;
  p.part = static_cast<float*>(a->workspace);
  cudaError_t e;
  if (a->dtype == FB_F32) e = launch_paged<float>(p, pl, st);
  else if (a->dtype == FB_F16) e = launch_paged<__half>(p, pl, st);
  else e = launch_paged<__nv_bfloat16>(p, pl, st);
  if (e != cudaSuccess) {
    record_cuda_error(e);
    return FB_ERR_LAUNCH;
  }
  set_last_launch_count(pl.join ? 2 : 1);
  return FB_OK;
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

size_t fb_paged_workspace_size(const fb_paged_args* args) {
  return fb::check_paged(args) == FB_OK && args->seqs > 0 ? fb::plan_paged(args).workspace : 0;
}
int fb_paged_born_fwd(const fb_paged_args* args, void* stream) {
  return fb::paged_fwd(args, static_cast<cudaStream_t>(stream));
}
int fb_paged_qkv_write(const fb_paged_write_args* args, void* stream) {
  return fb::paged_write(args, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
