// Rotary positions, and rotated rows written to the pages of a latent cache.
//
//   y[c]     = (x[c] cos - x[c'] sin) amplitude
//   y[c']    = (x[c'] cos + x[c] sin) amplitude      angle = position * freqs[i]
//
// for the pairs (c, c') of the `rot` channels from `offset` on: (2i, 2i + 1) in
// the interleaved layout, (i, i + rot/2) in the half layout; the other channels
// pass through bit for bit.  The inverse rotates by -angle: with the same
// amplitude it is the transposed map, so it is also the gradient's.
//
// Angles: position * freqs[i] is formed and reduced to a fraction of a turn in
// 64 bits (at position 10^6 a 32-bit product is off by 0.03 rad), the fraction
// (|f| <= 1/2, so within 2^-26 turns after rounding) goes to sincospif, and the
// rotation runs in 32 bits with one rounding at the end.
//
// Both kernels are bound by HBM: every channel is read and written once (only
// the rotated ones when x is rotated in place).  A thread has several units' loads in
// flight before it waits for any (x may be y, so the compiler cannot do it), and ahead
// of the angles.  Measured: 4099 tokens x 64 heads x 512 in bf16 (537 MB) 96 us, 5.6
// TB/s, 0.86 of the copy rate (one unit at a time behind the angles: 155 us); 32771
// cache rows (67 MB) 13.5 us, 5.0 TB/s; 64 rows 2.1 us, 64 tokens' queries 4.1 us,
// which is launch and latency.
#include <limits.h>
#include <string.h>

#include "kernels.cuh"

namespace dsv4 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V elements moved as one access: 16 bytes, or one element where alignment allows no more.
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T v[V];
};

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  if constexpr (V * sizeof(T) == 16) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    memcpy(&r, &w, 16);
  } else {
    r.v[0] = *p;
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& r) {
  if constexpr (V * sizeof(T) == 16) {
    uint4 w;
    memcpy(&w, &r, 16);
    *reinterpret_cast<uint4*>(p) = w;
  } else {
    *p = r.v[0];
  }
}

// An index tensor of either width.  Values that do not fit 32 bits come back as
// INT_MIN / INT_MAX, which every range check refuses.
__device__ __forceinline__ int load_index(const void* p, int is64, long long i) {
  if (!is64) return __ldg(static_cast<const int*>(p) + i);
  const long long v = __ldg(static_cast<const long long*>(p) + i);
  return v > INT_MAX ? INT_MAX : v < INT_MIN ? INT_MIN : static_cast<int>(v);
}

__device__ __forceinline__ float2 rotary_cos_sin(long long position, double freq, float amplitude, bool inverse) {
  const double turns = static_cast<double>(position) * freq * 0.15915494309189533577;  // 1 / (2 pi)
  const float f = static_cast<float>(turns - rint(turns));
  float s, c;
  sincospif(2.0f * f, &s, &c);
  return make_float2(c * amplitude, (inverse ? -s : s) * amplitude);
}

// Rotary geometry of one head of D channels, cut into units of one thread's work.
struct RotaryShape {
  int D, rot, offset, interleaved;
};

// Units that rotate (first) and all units of a head.  V = 1: a rotating unit is
// one pair; else one pack of V/2 interleaved pairs, or two packs of V half-layout pairs.
template <int V>
__host__ __device__ __forceinline__ int rotary_units(const RotaryShape& r) {
  return V == 1 ? r.rot / 2 : r.interleaved ? r.rot / V : r.rot / 2 / V;
}
template <int V>
__host__ __device__ __forceinline__ int head_units(const RotaryShape& r) {
  return rotary_units<V>(r) + (r.D - r.rot) / V;
}

// One unit of one head, loaded, turned and stored in three steps so that a thread has
// the loads of several units in flight (x and y may be the same memory, so the
// compiler cannot move a load above a store).  x, y are the head's channel 0.
template <typename T, int V, bool kInter>
struct RotaryUnit {
  static constexpr bool kTwo = V == 1 || !kInter;  // a rotating unit has two packs
  Pack<T, V> p, q;
  int ca, cb;

  __device__ __forceinline__ void load(const T* x, int u, int n_rot, const RotaryShape& r) {
    if (u >= n_rot) {  // a pass-through pack, before or behind the rotated channels
      ca = (u - n_rot) * V;
      if (ca >= r.offset) ca += r.rot;
    } else if (kTwo) {
      ca = r.offset + (kInter ? 2 * u : u * V);
      cb = kInter ? ca + 1 : ca + r.rot / 2;
      q = load_pack<T, V>(x + cb);
    } else {
      ca = r.offset + u * V;
    }
    p = load_pack<T, V>(x + ca);
  }

  __device__ __forceinline__ void turn_and_store(T* y, int u, int n_rot, const float2* cs) {
    if (u < n_rot) {
      if constexpr (kTwo) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 t = cs[u * V + i];
          const float a = to_f32(p.v[i]), b = to_f32(q.v[i]);
          p.v[i] = from_f32<T>(a * t.x - b * t.y);
          q.v[i] = from_f32<T>(b * t.x + a * t.y);
        }
        store_pack<T, V>(y + cb, q);
      } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float2 t = cs[u * (V / 2) + i];
          const float a = to_f32(p.v[2 * i]), b = to_f32(p.v[2 * i + 1]);
          p.v[2 * i] = from_f32<T>(a * t.x - b * t.y);
          p.v[2 * i + 1] = from_f32<T>(b * t.x + a * t.y);
        }
      }
    }
    store_pack<T, V>(y + ca, p);
  }
};

// n / d for n < 2^15 by a multiplication: ceil(2^32 / d) is off by less than d, which
// moves the product by less than n d / 2^32 < 1 / 4 of a step while d < 2^15.
struct FastDiv {
  unsigned d, m;
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)__umulhi((unsigned)n, m); }
};
static FastDiv fast_div(int d) { return FastDiv{(unsigned)d, d > 1 ? (unsigned)(((1ull << 32) + d - 1) / d) : 0u}; }

struct RotaryArgs {
  const void* x;
  void* y;
  const void* positions;  // [B,S], int32 or int64
  const double* freqs;    // [rot / 2] radians per position
  long long xs[3], ys[3];  // strides of (b, s, h) in elements
  int pos64, S, H, tokens;
  int tile_tokens, tile_heads, head_tiles;  // one CTA: tile_tokens tokens x tile_heads heads
  FastDiv by_head;                          // units per head
  int in_place, inverse;
  float amplitude;
  RotaryShape r;
};

constexpr int kRotThreads = 256;
constexpr int kRotMax = 4096;     // rotated channels per head
constexpr int kRotMaxDim = 32760;  // channels per head (FastDiv)
constexpr int kRotTable = 2048;   // cosine / sine pairs a CTA keeps (16 KB)
constexpr int kRotPacks = 4;      // packs per thread, their loads in flight together
constexpr int kRotTokens = 64;    // tokens a CTA takes at most

// One CTA takes a tile of tokens x heads.  Every thread has its first units on the
// way before the tokens' cosines and sines are worked out for all heads.
template <typename T, int V, bool kInter>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  __shared__ float2 cs[kRotTable];
  const int tok0 = (int)(blockIdx.x / a.head_tiles) * a.tile_tokens;
  const int h0 = (blockIdx.x % a.head_tiles) * a.tile_heads;
  const int n_tok = min(a.tile_tokens, a.tokens - tok0);
  const int n_head = min(a.tile_heads, a.H - h0);
  const int pairs = a.r.rot / 2;
  const int n_rot = rotary_units<V>(a.r);
  const int per_head = (int)a.by_head.d, total = n_tok * n_head * per_head;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);

  constexpr int kRotBatch = RotaryUnit<T, V, kInter>::kTwo ? kRotPacks / 2 : kRotPacks;
  constexpr int kRotUnits = kRotThreads * kRotBatch;
  RotaryUnit<T, V, kInter> unit[kRotBatch];
  int at[kRotBatch], un[kRotBatch];  // token within the tile, unit of the head
  long long to[kRotBatch];           // where the head begins in y
  auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < kRotBatch; ++j) {
      const int i = base + j * kRotThreads;
      if (i >= total) continue;
      const int th = a.by_head.div(i);  // token and head
      un[j] = i - th * per_head;
      at[j] = n_tok == 1 ? 0 : th / n_head;
      const int h = h0 + th - at[j] * n_head;
      int s = tok0 + at[j], b = 0;
      if (a.S != a.tokens) {
        b = s / a.S;
        s -= b * a.S;
      }
      to[j] = b * a.ys[0] + s * a.ys[1] + h * a.ys[2];
      unit[j].load(x + b * a.xs[0] + s * a.xs[1] + h * a.xs[2], un[j], n_rot, a.r);
    }
  };
  load(threadIdx.x);
  for (int i = threadIdx.x; i < n_tok * pairs; i += kRotThreads) {
    const long long tok = tok0 + i / pairs;
    const long long pos = a.pos64 ? __ldg(static_cast<const long long*>(a.positions) + tok)
                                  : (long long)__ldg(static_cast<const int*>(a.positions) + tok);
    cs[i] = rotary_cos_sin(pos, __ldg(a.freqs + i % pairs), a.amplitude, a.inverse != 0);
  }
  __syncthreads();
  for (int base = threadIdx.x; base < total; base += kRotUnits) {
    if (base >= kRotUnits) load(base);
#pragma unroll
    for (int j = 0; j < kRotBatch; ++j)
      if (base + j * kRotThreads < total) unit[j].turn_and_store(y + to[j], un[j], n_rot, cs + at[j] * pairs);
  }
}

struct AppendArgs {
  const void* rows;       // [T, D], stride row_stride
  void* pages;            // [P][page][D], page_stride apart
  const int* table;       // [n_seqs][max_pages]
  const void* seq_ids;    // [T]
  const void* positions;  // [T]
  const double* freqs;    // [rot / 2], or NULL with rot = 0
  long long row_stride, page_stride;
  int T, idx64, n_seqs, max_pages, n_pages, page_size;
  float amplitude;
  RotaryShape r;
};

constexpr int kAppendRows = 8;    // one warp per row
constexpr int kAppendPairs = 256;  // rot <= 512

// One warp per row: its pairs' cosines and sines by its lanes, then units of 16
// bytes from the row to its page.  Rows with a negative sequence or position are
// padding and are skipped; others out of range, or on no page, are reported.
template <typename T, int V, bool kInter>
__global__ void __launch_bounds__(32 * kAppendRows) cache_append_kernel(const AppendArgs a) {
  __shared__ float2 cs_all[kAppendRows][kAppendPairs];
  constexpr int kBatch = 2;  // units in flight per lane: a row of 512 channels
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kAppendRows + w;
  if (t >= a.T) return;
  const int s = a.seq_ids ? load_index(a.seq_ids, a.idx64, t) : (int)t;
  const int pos = load_index(a.positions, a.idx64, t);
  const T* x = static_cast<const T*>(a.rows) + t * a.row_stride;
  const int n_rot = rotary_units<V>(a.r), n = head_units<V>(a.r);
  // the row's first units are on their way while the page is looked up
  RotaryUnit<T, V, kInter> unit[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; ++j)
    if (lane + 32 * j < n) unit[j].load(x, lane + 32 * j, n_rot, a.r);
  if (s < 0 || pos < 0) return;
  const int slot = pos / a.page_size;
  int page = -1;
  if (s < a.n_seqs && slot < a.max_pages) page = __ldg(a.table + (long long)s * a.max_pages + slot);
  float2* cs = cs_all[w];
  for (int i = lane; i < a.r.rot / 2; i += 32) cs[i] = rotary_cos_sin(pos, __ldg(a.freqs + i), a.amplitude, false);
  __syncwarp();
  if (page < 0 || page >= a.n_pages) {
    if (lane == 0) record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return;
  }
  T* y = static_cast<T*>(a.pages) + page * a.page_stride + (long long)(pos - slot * a.page_size) * a.r.D;
  for (int u = lane; u < n; u += 32 * kBatch) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (u > lane && u + 32 * j < n) unit[j].load(x, u + 32 * j, n_rot, a.r);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (u + 32 * j < n) unit[j].turn_and_store(y, u + 32 * j, n_rot, cs);
  }
}

// Whether 16-byte packs of V elements never straddle a border.
static bool packs_ok(const RotaryShape& r, int V) {
  return r.D % V == 0 && r.offset % V == 0 && r.rot % V == 0 && (r.interleaved || (r.rot / 2) % V == 0);
}

template <typename T>
static int launch_rotary_t(RotaryArgs a, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  bool vec = packs_ok(a.r, V) && !((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) & 15);
  for (int i = 0; i < 3; ++i) vec = vec && a.xs[i] % V == 0 && a.ys[i] % V == 0;
  const int n_rot = vec ? rotary_units<V>(a.r) : rotary_units<1>(a.r);
  const int per_head = a.in_place ? n_rot : vec ? head_units<V>(a.r) : head_units<1>(a.r);
  if (per_head == 0) return DSV4_OK;
  // heads of a token first, then more tokens, up to a batch of units per thread
  const int kRotUnits = kRotThreads * (vec && a.r.interleaved ? kRotPacks : kRotPacks / 2);
  a.tile_heads = kRotUnits / per_head < 1 ? 1 : kRotUnits / per_head;
  if (a.tile_heads > a.H) a.tile_heads = a.H;
  a.head_tiles = (a.H + a.tile_heads - 1) / a.tile_heads;
  int tt = kRotUnits / (per_head * a.tile_heads);
  const int by_table = a.r.rot ? kRotTable / (a.r.rot / 2) : kRotTokens;
  if (tt > by_table) tt = by_table;
  if (tt > kRotTokens) tt = kRotTokens;
  if (tt < 1) tt = 1;
  a.tile_tokens = tt;
  a.by_head = fast_div(per_head);
  const long long grid = ((long long)a.tokens + tt - 1) / tt * a.head_tiles;
  if (grid > INT_MAX) return DSV4_ERR_UNSUPPORTED;
  auto kernel = vec ? (a.r.interleaved ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>)
                    : (a.r.interleaved ? rotary_kernel<T, 1, true> : rotary_kernel<T, 1, false>);
  launch_k(kernel, (unsigned)grid, kRotThreads, 0, st, a);
  return cudaGetLastError() == cudaSuccess ? DSV4_OK : DSV4_ERR_CUDA;
}

int launch_rotary(const void* x, void* y, int dtype, const void* positions, int pos64, const double* freqs, int B,
                  int S, int H, int D, int rot, int offset, int interleaved, int inverse, float amplitude,
                  const long long* xs, const long long* ys, cudaStream_t st) {
  RotaryArgs a{};
  a.x = x;
  a.y = y;
  a.positions = positions;
  a.freqs = freqs;
  for (int i = 0; i < 3; ++i) {
    a.xs[i] = xs[i];
    a.ys[i] = ys[i];
  }
  a.pos64 = pos64;
  a.S = S;
  a.H = H;
  if ((long long)B * S > INT_MAX) return DSV4_ERR_UNSUPPORTED;
  a.tokens = B * S;
  // batches that follow each other like positions do are one run of positions
  if (B == 1 || (xs[0] == S * xs[1] && ys[0] == S * ys[1])) a.S = a.tokens;
  a.in_place = x == y;
  a.inverse = inverse;
  a.amplitude = amplitude;
  a.r = RotaryShape{D, rot, offset, interleaved};
  if (dtype == DSV4_DTYPE_BF16) return launch_rotary_t<__nv_bfloat16>(a, st);
  if (dtype == DSV4_DTYPE_FP16) return launch_rotary_t<__half>(a, st);
  return launch_rotary_t<float>(a, st);
}

template <typename T>
static int launch_cache_append_t(const AppendArgs& a, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  const bool vec = packs_ok(a.r, V) && a.row_stride % V == 0 && !(reinterpret_cast<uintptr_t>(a.rows) & 15);
  const unsigned grid = (unsigned)((a.T + kAppendRows - 1) / kAppendRows);
  auto kernel = vec ? (a.r.interleaved ? cache_append_kernel<T, V, true> : cache_append_kernel<T, V, false>)
                    : (a.r.interleaved ? cache_append_kernel<T, 1, true> : cache_append_kernel<T, 1, false>);
  launch_k(kernel, grid, 32 * kAppendRows, 0, st, a);
  return cudaGetLastError() == cudaSuccess ? DSV4_OK : DSV4_ERR_CUDA;
}

int launch_cache_append(const void* rows, long long row_stride, int dtype, int T, int D, void* pages, int n_pages,
                        int page_size, long long page_stride, const int* table, int n_seqs, int max_pages,
                        const void* seq_ids, const void* positions, int idx64, const double* freqs, int rot, int offset,
                        int interleaved, float amplitude, cudaStream_t st) {
  AppendArgs a{};
  a.rows = rows;
  a.pages = pages;
  a.table = table;
  a.seq_ids = seq_ids;
  a.positions = positions;
  a.freqs = freqs;
  a.row_stride = row_stride;
  a.page_stride = page_stride;
  a.T = T;
  a.idx64 = idx64;
  a.n_seqs = n_seqs;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  a.page_size = page_size;
  a.amplitude = amplitude;
  a.r = RotaryShape{D, rot, offset, interleaved};
  return dtype == DSV4_DTYPE_BF16 ? launch_cache_append_t<__nv_bfloat16>(a, st) : launch_cache_append_t<__half>(a, st);
}

}  // namespace dsv4
