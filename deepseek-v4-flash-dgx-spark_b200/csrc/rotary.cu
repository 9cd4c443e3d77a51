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
// the rotated ones when x is rotated in place).
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

// One unit of one head: x, y are the head's channel 0; cs the pairs' cosines and sines.
template <typename T, int V>
__device__ __forceinline__ void rotary_unit(const T* x, T* y, int u, int n_rot, const RotaryShape& r, const float2* cs) {
  using P = Pack<T, V>;
  if (u >= n_rot) {  // a pass-through pack, before or behind the rotated channels
    int c = (u - n_rot) * V;
    if (c >= r.offset) c += r.rot;
    store_pack<T, V>(y + c, load_pack<T, V>(x + c));
    return;
  }
  if (r.interleaved && V > 1) {
    const int c = r.offset + u * V;
    P p = load_pack<T, V>(x + c);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 t = cs[u * (V / 2) + i];
      const float a = to_f32(p.v[2 * i]), b = to_f32(p.v[2 * i + 1]);
      p.v[2 * i] = from_f32<T>(a * t.x - b * t.y);
      p.v[2 * i + 1] = from_f32<T>(b * t.x + a * t.y);
    }
    store_pack<T, V>(y + c, p);
    return;
  }
  const int ca = r.offset + (r.interleaved ? 2 * u : u * V);
  const int cb = r.interleaved ? ca + 1 : ca + r.rot / 2;
  P p = load_pack<T, V>(x + ca), q = load_pack<T, V>(x + cb);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 t = cs[u * V + i];
    const float a = to_f32(p.v[i]), b = to_f32(q.v[i]);
    p.v[i] = from_f32<T>(a * t.x - b * t.y);
    q.v[i] = from_f32<T>(b * t.x + a * t.y);
  }
  store_pack<T, V>(y + ca, p);
  store_pack<T, V>(y + cb, q);
}

struct RotaryArgs {
  const void* x;
  void* y;
  const void* positions;  // [B,S], int32 or int64
  const double* freqs;    // [rot / 2] radians per position
  long long xs[3], ys[3];  // strides of (b, s, h) in elements
  int pos64, S, H;
  long long tokens;
  int tile_tokens, tile_heads, head_tiles;  // one CTA: tile_tokens tokens x tile_heads heads
  int in_place, inverse;
  float amplitude;
  RotaryShape r;
};

constexpr int kRotThreads = 256;
constexpr int kRotMax = 4096;     // rotated channels per head
constexpr int kRotTable = 2048;   // cosine / sine pairs a CTA keeps (16 KB)
constexpr int kRotUnits = 1024;   // units a CTA takes: four per thread

// One CTA takes a tile of tokens x heads: the tokens' cosines and sines go to
// shared memory once, then every thread moves units of 16 bytes.
template <typename T, int V>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotaryArgs a) {
  __shared__ float2 cs[kRotTable];
  const long long tok0 = (long long)(blockIdx.x / a.head_tiles) * a.tile_tokens;
  const int h0 = (blockIdx.x % a.head_tiles) * a.tile_heads;
  const int n_tok = (int)min((long long)a.tile_tokens, a.tokens - tok0);
  const int n_head = min(a.tile_heads, a.H - h0);
  const int pairs = a.r.rot / 2;
  for (int i = threadIdx.x; i < n_tok * pairs; i += kRotThreads) {
    const long long tok = tok0 + i / pairs;
    const long long pos = a.pos64 ? __ldg(static_cast<const long long*>(a.positions) + tok)
                                  : (long long)__ldg(static_cast<const int*>(a.positions) + tok);
    cs[i] = rotary_cos_sin(pos, __ldg(a.freqs + i % pairs), a.amplitude, a.inverse != 0);
  }
  __syncthreads();
  const int n_rot = rotary_units<V>(a.r);
  const int per_head = a.in_place ? n_rot : head_units<V>(a.r);
  const int per_tok = n_head * per_head;
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
#pragma unroll 4
  for (int i = threadIdx.x; i < n_tok * per_tok; i += kRotThreads) {
    const int t = i / per_tok, j = i - t * per_tok;
    const int h = j / per_head, u = j - h * per_head;
    const long long tok = tok0 + t, b = tok / a.S, s = tok - b * a.S;
    rotary_unit<T, V>(x + b * a.xs[0] + s * a.xs[1] + (long long)(h0 + h) * a.xs[2],
                      y + b * a.ys[0] + s * a.ys[1] + (long long)(h0 + h) * a.ys[2], u, n_rot, a.r, cs + t * pairs);
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
template <typename T, int V>
__global__ void __launch_bounds__(32 * kAppendRows) cache_append_kernel(const AppendArgs a) {
  __shared__ float2 cs_all[kAppendRows][kAppendPairs];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = (long long)blockIdx.x * kAppendRows + w;
  if (t >= a.T) return;
  const int s = a.seq_ids ? load_index(a.seq_ids, a.idx64, t) : (int)t;
  const int pos = load_index(a.positions, a.idx64, t);
  if (s < 0 || pos < 0) return;
  const int slot = pos / a.page_size;
  int page = -1;
  if (s < a.n_seqs && slot < a.max_pages) page = __ldg(a.table + (long long)s * a.max_pages + slot);
  if (page < 0 || page >= a.n_pages) {
    if (lane == 0) record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return;
  }
  float2* cs = cs_all[w];
  for (int i = lane; i < a.r.rot / 2; i += 32) cs[i] = rotary_cos_sin(pos, __ldg(a.freqs + i), a.amplitude, false);
  __syncwarp();
  const T* x = static_cast<const T*>(a.rows) + t * a.row_stride;
  T* y = static_cast<T*>(a.pages) + page * a.page_stride + (long long)(pos % a.page_size) * a.r.D;
  const int n_rot = rotary_units<V>(a.r), n = head_units<V>(a.r);
#pragma unroll 2
  for (int u = lane; u < n; u += 32) rotary_unit<T, V>(x, y, u, n_rot, a.r, cs);
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
  // heads of a token first, then more tokens, up to kRotUnits units per CTA
  a.tile_heads = kRotUnits / per_head < 1 ? 1 : kRotUnits / per_head;
  if (a.tile_heads > a.H) a.tile_heads = a.H;
  a.head_tiles = (a.H + a.tile_heads - 1) / a.tile_heads;
  int tt = kRotUnits / (per_head * a.tile_heads);
  const int by_table = a.r.rot ? kRotTable / (a.r.rot / 2) : 64;
  if (tt > by_table) tt = by_table;
  if (tt < 1) tt = 1;
  a.tile_tokens = tt;
  const long long grid = (a.tokens + tt - 1) / tt * a.head_tiles;
  if (grid > INT_MAX) return DSV4_ERR_UNSUPPORTED;
  if (vec)
    launch_k(rotary_kernel<T, V>, (unsigned)grid, kRotThreads, 0, st, a);
  else
    launch_k(rotary_kernel<T, 1>, (unsigned)grid, kRotThreads, 0, st, a);
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
  a.tokens = (long long)B * S;
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
  if (vec)
    launch_k(cache_append_kernel<T, V>, grid, 32 * kAppendRows, 0, st, a);
  else
    launch_k(cache_append_kernel<T, 1>, grid, 32 * kAppendRows, 0, st, a);
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
