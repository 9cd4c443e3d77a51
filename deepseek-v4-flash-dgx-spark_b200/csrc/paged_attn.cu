// Attention of single tokens over the pages of a latent cache, on the tensor core.
//
//   out[t,h] = sum_j p[h,j] kv[j]      over the visible keys j of row t's sequence,
//   p[h,j] = exp(z[h,j] - m[h]) / (sum_j exp(z - m) + exp(sink[h] - m)),
//   z[h,j] = scale * q[t,h] . kv[j],   m[h] = max(max_j z[h,j], sink[h]).
//
// Row t stands at position p of sequence s and sees the keys j <= p, with a
// window only those above p - window and the first `first` ones.  Key j is row
// j % page_size of page page_table[s][j / page_size]; one cache row is key and
// value of every head.  A row with nothing visible gives zeros; scores of NaN or
// infinities give what the formula does, whether one CTA holds the row or several.
//
// Per chunk of 64 keys two products on tcgen05 (kind::f16, fp32 accumulators in TMEM):
//   S[h,j]   = Q[h,:] . C[j,:]      M = 64 heads, N = 64 keys, K = D
//   O^T[d,h] += C^T[d,j] . P[h,j]   M = 128 of D, N = heads, K = 64 keys
// The second reads the same shared memory as an MN-major operand, so a key's row
// is loaded once and never transposed.  With S's rows on heads a thread keeps two
// heads' running max and sum in registers and takes their scores from one
// tcgen05.ld.16x256b (M = 64 fills 16 lanes of each TMEM quarter).
//
// Bound: a row of D = 512 is 1 KB from HBM and 131 kFLOP with 64 heads.  Issued from
// warp-uniform code the two products cost 36 and 51 cycles per instruction (measured),
// 1970 cycles per chunk, against 2840 at which an SM's share of HBM delivers the chunk's
// 64 KB.  What is left is the ring: shared memory holds Q (64 KB) and 2.25 chunks, and a
// stage comes back only after its load (about 2000 cycles), its chunk's softmax (1250)
// and both products, a period of 2850 to 3000 cycles.  Shared memory is not far from its
// own rate either: a chunk moves about 296 KB through it (Q 64, the keys 64 for each
// product, the weights 4 x 8, the load 64, the weights' stores 8), 2310 cycles at 128
// bytes each.  Measured over whole calls, 16 rows of 40000, 60000 and 80000 keys: 138,
// 194 and 254 us, 4.75, 5.05 and 5.15 TB/s (0.73 to 0.80 of the copy rate), of which
// about 20 us are start, output and join.  Chunks of 128 keys cost fewer tensor cycles
// per key but hold all of the ring until their softmax is done, and the loads stand
// still for half of the time (16 rows of up to 131072 keys: 353 against 291 us at that
// step).
//
// Work split: the visible keys of all rows, in boxes of up to 64 keys on one page,
// form one list, and the list is cut into equal shares, one per CTA (one CTA per
// SM).  Every CTA finds its share from the lengths on the device, so ragged
// batches fill the SMs, nothing is read back and a captured graph follows the
// lengths of each replay.  A row that crosses a border leaves fp32 partials (max,
// sum, O) that paged_attn_join_kernel merges; every CTA has at most two such pieces.
//
// Warp roles (352 threads): warp 0 loads Q and the pages by TMA into a ring of
// stages (64 keys x 128 channels, 16 KB), warp 1 issues the score products as the
// stages arrive, up to a chunk ahead of warp 2, which issues the output products
// when their weights are there and gives the stages back one by one.  Warps 3-10 do
// the softmax: warp w takes the heads of TMEM quarter w % 4 and half of the chunk's
// keys, and at the end the channels of that quarter and half of the heads.  (One
// warp for both products spends 4000 cycles a chunk on issuing and polling.)
#include <limits.h>

#include <type_traits>

#include "kernels.cuh"

namespace dsv4 {

constexpr int kPaChunk = 64;                      // keys per chunk
constexpr int kPaThreads = 352;
constexpr int kPaSoft = 256;                      // softmax threads: warps 3-10
constexpr int kPaTile = kPaChunk * 128;           // 8 KB: 64 keys x 64 channels, 128-byte swizzled
constexpr int kPaStage = 2 * kPaTile;             // 16 KB: 64 keys x 128 channels
constexpr int kPaMaxStages = 12;
constexpr int kPaCtrl = 2048;
constexpr int kPaSmemMax = 232448;                // shared memory a CTA may use
constexpr int kPaMaxGrid = 1024;                  // CTAs (one per SM)
constexpr int kPaTmemCols = 512;                  // S: two buffers of 64 columns; O^T at 256
constexpr int kPaMinChunks = 1;                   // least chunks per CTA
constexpr int kPaSnapChunks = 3;                  // a border moves so far to a row's begin or end
constexpr float kPaNoMax = -3.402823466e38f;      // running max of a piece before its first finite score
constexpr float kLog2e = 1.4426950408889634f;

// Weights are 2^(score - m), scores in base 2.  m is set to `lift` below the largest
// score so far, and again only once a score passes m by lift + headroom, so the largest
// weight of a row lies between 2^lift and 2^(lift + headroom).  bf16 has fp32's range
// and needs no lift.  fp16 ends at 2^16 and counts in steps of 2^-24 below 2^-14: with
// the lift a key keeps all bits of its weight down to 2^-23 of the largest one and some
// down to 2^-34, which counts where one dominating key of small values stands before
// many others.  A lift of 12 and 3 of headroom would keep three more bits, but the
// output is rescaled more often (64 ragged rows of 64 fp16 heads 84.0 us at lift 5, 84.8
// at 9, 87.8 at 12).
template <typename T>
struct PaWeight {
  static constexpr float lift = 0.f, headroom = 10.f;
};
template <>
struct PaWeight<__half> {
  static constexpr float lift = 9.f, headroom = 6.f;
};

struct PaArgs {
  void* out;              // [T, H, D]
  const int* table;       // [n_seqs][max_pages]
  const void* seq_ids;    // [T] or NULL (row t reads sequence t)
  const void* positions;  // [T]
  const float* sink;      // [H] or NULL
  float* part_o;          // [grid][2][N][D]
  float* part_ml;         // [grid][2][N][2]: max (base 2; -inf: no key seen), sum
  int4* plan;             // [grid]: row, head group, boxes of the row before this CTA's border, boxes of the row
  int* share;             // [1] boxes from border to border
  int T, H, D, groups;
  int n_seqs, max_pages, n_pages, page_log, box_log;
  int idx64, window, first, stages, min_share, snap;
  float scale;
};

// What row t sees: keys [w_lo, p] and [0, f), in n boxes of 1 << box_log keys; box b
// covers the keys from (b < nfb ? b : b - nfb + wbb) << box_log.
struct PaRow {
  int s, p, w_lo, f, nfb, wbb, n;
};

// Sequence and position of row t (negative: padding).
__device__ __forceinline__ int2 pa_index(const PaArgs& a, int t) {
  if (t >= a.T) return make_int2(-1, -1);
  return make_int2(a.seq_ids ? load_index(a.seq_ids, a.idx64, t) : t, load_index(a.positions, a.idx64, t));
}

__device__ __forceinline__ PaRow pa_row(const PaArgs& a, int2 sp) {
  PaRow r{};
  r.s = sp.x;
  r.p = sp.y;
  if (r.s < 0 || r.p < 0) return r;
  if (r.s >= a.n_seqs || (r.p >> a.page_log) >= a.max_pages) {
    record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return r;
  }
  r.w_lo = a.window > 0 ? max(0, r.p - a.window + 1) : 0;
  r.f = min(a.first, r.w_lo);
  r.wbb = r.w_lo >> a.box_log;
  r.nfb = min((r.f + (1 << a.box_log) - 1) >> a.box_log, r.wbb);
  r.n = r.nfb + (r.p >> a.box_log) + 1 - r.wbb;
  return r;
}
__device__ __forceinline__ int pa_box_key(const PaArgs& a, const PaRow& r, int b) {
  return (b < r.nfb ? b : b - r.nfb + r.wbb) << a.box_log;
}

// The list of `total` boxes is cut at every `share` boxes.  A border that falls less
// than `snap` boxes from the begin or end of a row moves there: a piece of a row
// costs its fp32 partials (256 KB written and read at 64 heads x 512), as much as
// some chunks of keys.
__device__ __forceinline__ int pa_share(int total, int ctas, int min_share) {
  return max(total / ctas + (total % ctas != 0), min_share);
}
__device__ __forceinline__ int pa_snap(int o, int n, int snap) {
  if (o <= 0) return 0;
  if (o >= n) return n;
  if (min(o, n - o) > snap) return o;
  return o <= n - o ? 0 : n;
}

struct PaShared {
  uint64_t full[kPaMaxStages], empty[kPaMaxStages];
  uint64_t q_full[4], q_empty, s_full[2], s_free[2], p_ready[2], pv_done[2], last[2];
  uint32_t tmem;
  int abort;
  int t0, g0, i0;           // this CTA's first row, head group and box
  int begin, end;           // its boxes of the list
  int scan[kPaThreads / 32];
  float red[2 * 64];        // one value per key half and head
  float m[64], f[64];       // max, factor per head
};
static_assert(sizeof(PaShared) <= kPaCtrl, "control block too small");

__device__ __forceinline__ bool pa_aborted(PaShared& sh) { return *reinterpret_cast<volatile int*>(&sh.abort) != 0; }

// A bounded wait.  Once any wait of the CTA has run out, every wait returns at
// once: the roles run through their loops without waiting (loading and issuing
// nothing more), so no barrier is left with a missing thread.
__device__ __forceinline__ bool pa_wait(PaShared& sh, uint64_t* bar, uint32_t parity, int err) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (!pa_aborted(sh)) {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (globaltimer() - t0 > kWaitTimeoutNs) {
      record_error(err);
      *reinterpret_cast<volatile int*>(&sh.abort) = 1;
    }
  }
  return false;
}

__device__ __forceinline__ void soft_sync() { asm volatile("barrier.cta.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool soft_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The sink's weight against the max (1 where it is the max, also an infinite one).
__device__ __forceinline__ float pa_sink(float sink, float mx) { return sink == mx ? 1.f : ex2(sink - mx); }

// n consecutive fp32 columns of this thread's TMEM lane, n = 8, 16 or 32.
template <int n>
__device__ __forceinline__ void tmem_ldn(uint32_t taddr, float (&v)[n]) {
  if constexpr (n == 32) {
    tmem_ld32_wait(taddr, v);
  } else if constexpr (n == 16) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
  } else {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
  }
}
template <int n>
__device__ __forceinline__ void tmem_stn(uint32_t taddr, const float (&v)[n]) {
  if constexpr (n == 32) {
    tmem_st32(taddr, v);
  } else {
#pragma unroll
    for (int i = 0; i < n; i += 8)
      asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr + i),
                   "r"(__float_as_uint(v[i])), "r"(__float_as_uint(v[i + 1])), "r"(__float_as_uint(v[i + 2])),
                   "r"(__float_as_uint(v[i + 3])), "r"(__float_as_uint(v[i + 4])), "r"(__float_as_uint(v[i + 5])),
                   "r"(__float_as_uint(v[i + 6])), "r"(__float_as_uint(v[i + 7]))
                   : "memory");
  }
}

// 32 columns of 16 TMEM lanes: v[4c + 0, 1] are columns 8c + 2 (lane % 4) + 0, 1 of TMEM
// lane lane / 4, v[4c + 2, 3] the same columns eight lanes further.
__device__ __forceinline__ void tmem_ld_16x32(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
               "tcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// kind::f16 instruction descriptor: A and B both fp16 or both bf16, fp32 D.
template <typename T>
__host__ __device__ constexpr uint32_t pa_idesc(uint32_t m, uint32_t n, uint32_t a_mn) {
  const uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn << 15) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// Rows of both maps are split into 64-channel tiles: coordinates (0, row, tile, page or token).
__device__ __forceinline__ void tma_load_tiles(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int row, int tile,
                                               int z) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(0), "r"(row), "r"(tile), "r"(z)
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const T a = from_f32<T>(lo), b = from_f32<T>(hi);
  uint16_t x, y;
  memcpy(&x, &a, 2);
  memcpy(&y, &b, 2);
  return (uint32_t)x | ((uint32_t)y << 16);
}

// The sum of two packed values in 32 bits.
template <typename T>
__device__ __forceinline__ float sum2(uint32_t v) {
  if constexpr (std::is_same<T, __half>::value) {
    __half2 h;
    memcpy(&h, &v, 4);
    const float2 f = __half22float2(h);
    return f.x + f.y;
  } else {
    return __uint_as_float(v << 16) + __uint_as_float(v & 0xffff0000u);
  }
}

// Lane l of four holds column l of four rows; it gets row l % 4 of the four columns.
__device__ __forceinline__ float4 transpose4(float a0, float a1, float a2, float a3, int lane) {
  const bool o1 = lane & 1, o2 = lane & 2;
  const float r0 = __shfl_xor_sync(0xffffffffu, o1 ? a0 : a1, 1);
  const float r1 = __shfl_xor_sync(0xffffffffu, o1 ? a2 : a3, 1);
  if (o1) {
    a0 = r0;
    a2 = r1;
  } else {
    a1 = r0;
    a3 = r1;
  }
  const float s0 = __shfl_xor_sync(0xffffffffu, o2 ? a0 : a2, 2);
  const float s1 = __shfl_xor_sync(0xffffffffu, o2 ? a1 : a3, 2);
  return o2 ? make_float4(s0, s1, a2, a3) : make_float4(a0, a1, s0, s1);
}

// N: heads per group, padded to 16, 32 or 64 (rows past H load as zeros).  The score
// product always takes 64 rows of Q: with N < 64 those past N are whatever follows
// in shared memory, and no one reads their scores.
template <typename T, int N>
__global__ void __launch_bounds__(kPaThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map,
                      const PaArgs a) {
  constexpr int HPT = N / 2;  // heads per thread of the output
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int DT = a.D / 128, NST = a.stages;
  uint8_t* sQ = smem;                               // 2 DT tiles of [N heads][128 B]
  uint8_t* ring = sQ + DT * 2 * N * 128;            // NST stages of two tiles [64 keys][128 B]
  uint8_t* sP = ring + NST * kPaStage;              // 2 buffers of [N heads][64 keys]
  PaShared& sh = *reinterpret_cast<PaShared*>(sP + 2 * N * 128);
  const int nsub = kPaChunk >> a.box_log;           // boxes per chunk

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  // ---- this CTA's share of the box list -------------------------------------
  const int per = (a.T + kPaThreads - 1) / kPaThreads;
  const int r0 = min(a.T, tid * per), r1 = min(a.T, r0 + per);
  int mine = 0, n_r0 = 0;  // boxes of this thread's rows, and of the first
  for (int t = r0; t < r1; ++t) {
    const int n = pa_row(a, pa_index(a, t)).n;
    if (t == r0) n_r0 = n;
    mine += n * a.groups;
  }
  if (warp == 0) {
    if (lane < NST) {
      mbar_init(&sh.full[lane], 1);
      mbar_init(&sh.empty[lane], 1);
    }
    if (lane < 4) mbar_init(&sh.q_full[lane], 1);
    if (lane < 2) {
      mbar_init(&sh.s_full[lane], 1);
      mbar_init(&sh.s_free[lane], kPaSoft / 32);
      mbar_init(&sh.p_ready[lane], kPaSoft / 32);
      mbar_init(&sh.pv_done[lane], 1);
      mbar_init(&sh.last[lane], 1);
    }
    if (lane == 0) {
      mbar_init(&sh.q_empty, 1);
      sh.abort = 0;
      sh.begin = sh.end = 0;
      tma_prefetch_desc(&q_map);
      tma_prefetch_desc(&kv_map);
    }
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&sh.tmem, kPaTmemCols);
    tmem_relinquish();
  }
  {
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sh.scan[warp] = inc;
    __syncthreads();
    const int of_warp = lane < kPaThreads / 32 ? sh.scan[lane] : 0;
    const int total = __reduce_add_sync(0xffffffffu, of_warp);
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0);
    const int share = pa_share(total, (int)gridDim.x, a.min_share);
    // borders blockIdx.x and blockIdx.x + 1 (past the list: its end)
    const int at0 = before + inc - mine;
#pragma unroll 1
    for (int x = 0; x < 2; ++x) {
      const int border = (int)min((long long)share * ((int)blockIdx.x + x), (long long)total);
      if (border == total && tid == 0) {
        if (x) sh.end = total;
        if (!x) sh.begin = total;
        if (!x) a.plan[blockIdx.x] = make_int4(-1, 0, 0, 0);
      }
      if (border == total || border < at0 || border >= at0 + mine) continue;
      int at = at0, t = r0, n = n_r0;  // the row that holds it
      while (border >= at + n * a.groups) {
        at += n * a.groups;
        ++t;
        n = pa_row(a, pa_index(a, t)).n;
      }
      int g = 0, o = border - at;
      while (o >= n) {
        o -= n;
        ++g;
      }
      const int on = pa_snap(o, n, min(a.snap, share >> 1));
      if (x) {
        sh.end = border - o + on;
      } else {
        sh.begin = border - o + on;
        sh.t0 = t;
        sh.g0 = g;
        sh.i0 = on;
        a.plan[blockIdx.x] = make_int4(t, g, o, n);
      }
    }
    if (tid == 0 && blockIdx.x == 0) *a.share = share;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t t_s = __shfl_sync(0xffffffffu, sh.tmem, 0), t_o = t_s + 256;
  int left = __shfl_sync(0xffffffffu, sh.end - sh.begin, 0);
  int t = __shfl_sync(0xffffffffu, sh.t0, 0), g = __shfl_sync(0xffffffffu, sh.g0, 0);
  int i = __shfl_sync(0xffffffffu, sh.i0, 0);
  int2 sp = left > 0 ? pa_index(a, t) : make_int2(-1, -1);  // the row at hand; the next one's is loaded early

  if (warp == 0) {
    // ------------------------------------------------------------- loads
    int slot = 0, issued = 0;
    uint32_t phase = 0, q_phase = 0;
    bool ok = true, q_issued = false;
    while (left > 0 && ok && t < a.T) {
      const PaRow r = pa_row(a, sp);
      const int2 sp_next = pa_index(a, t + 1);
      const int i1 = min(r.n, i + left);
      if (i < i1) {
        const int* row = a.table + (long long)r.s * a.max_pages;
        left -= i1 - i;
        // lane b loads box b of the chunk; hidden keys and keys on no page are left out
        auto page_at = [&](int b) -> int {
          if (lane >= nsub || b >= i1) return -1;
          const int page = __ldg(row + (pa_box_key(a, r, b) >> a.page_log));
          return page < a.n_pages ? page : -1;
        };
        auto load_q = [&]() {
          ok = __all_sync(0xffffffffu, pa_wait(sh, &sh.q_empty, q_phase ^ 1, DSV4_DEVERR_TIMEOUT_PRODUCER));
          if (!ok) return;
          q_phase ^= 1;
          q_issued = true;
          if (lane < DT) {
            mbar_arrive_expect_tx(&sh.q_full[lane], 2 * N * 128);
            tma_load_tiles(smem_u32(sQ + 2 * lane * N * 128), &q_map, &sh.q_full[lane], 64 * g, 2 * lane, t);
          }
          __syncwarp();
        };
        // the first piece takes Q first; later ones a chunk of keys first, while the
        // score products of the piece before may still read Q
        bool q_due = true;
        if (!q_issued) {
          load_q();
          q_due = false;
        }
        int page = page_at(i + lane);
        for (; i < i1 && ok; i += nsub) {
          const int key = pa_box_key(a, r, i + lane);
          const bool on = page >= 0;
          const int page_now = page;
          page = page_at(i + nsub + lane);
          const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, on)) * (256u << a.box_log);
          for (int dt = 0; dt < DT; ++dt) {
            ok = __all_sync(0xffffffffu, pa_wait(sh, &sh.empty[slot], phase ^ 1, DSV4_DEVERR_TIMEOUT_PRODUCER));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], bytes);
            __syncwarp();
            if (on) {
              const uint32_t dst = smem_u32(ring + slot * kPaStage) + (lane << (a.box_log + 7));
              const int y = key & ((1 << a.page_log) - 1);
              tma_load_tiles(dst, &kv_map, &sh.full[slot], y, 2 * dt, page_now);
              if (nsub > 1) tma_load_tiles(dst + kPaTile, &kv_map, &sh.full[slot], y, 2 * dt + 1, page_now);
            }
            ++issued;
            if (++slot == NST) {
              slot = 0;
              phase ^= 1;
            }
          }
          if (q_due && ok) {
            load_q();
            q_due = false;
          }
        }
      }
      i = 0;
      if (++g >= a.groups) {
        g = 0;
        ++t;
        sp = sp_next;
      }
    }
    // the join may be launched once every CTA is here: its start then overlaps the last
    // chunks (any earlier, its CTAs crowd the SMs that this grid leaves free)
    if (lane == 0) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // every copy has landed before the CTA can exit, also when a wait ran out
    for (int k = 0; k < min(issued, NST); ++k) {
      if (slot == 0) {
        slot = NST;
        phase ^= 1;
      }
      --slot;
      mbar_wait(&sh.full[slot], phase, DSV4_DEVERR_TIMEOUT_PRODUCER);
    }
    if (q_issued)
      for (int k = 0; k < DT; ++k) mbar_wait(&sh.q_full[k], q_phase ^ 1, DSV4_DEVERR_TIMEOUT_PRODUCER);
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------- score products
    // All lanes run the loops, so that descriptors stay in uniform registers; one issues.
    const bool el = elect_one();
    constexpr uint32_t id = pa_idesc<T>(64, kPaChunk, 0);
    // descriptors of the first tile; an address moves the low field by bytes / 16
    const uint64_t dq = sdesc_k_sw128(smem_u32(sQ)), dk = sdesc_k_sw128(smem_u32(ring));
    bool ok = true;
    uint32_t k = 0;  // chunks so far
    int slot = 0;
    uint32_t phase = 0, q_phase = 0;
    while (left > 0 && ok && t < a.T) {
      const int n = pa_row(a, sp).n;
      const int2 sp_next = pa_index(a, t + 1);
      const int i1 = min(n, i + left);
      if (i < i1) {
        left -= i1 - i;
        bool begin = true;
        for (; i < i1 && ok; i += nsub, ++k) {
          const uint32_t b = __shfl_sync(0xffffffffu, k & 1, 0);
          const uint32_t d = __shfl_sync(0xffffffffu, t_s, 0) + 64 * b;
          const int slot0 = __shfl_sync(0xffffffffu, slot, 0);
          ok = pa_wait(sh, &sh.s_free[b], ((k >> 1) & 1) ^ 1, DSV4_DEVERR_TIMEOUT_MMA);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            if (dt >= DT) break;
            if (begin) ok = ok && pa_wait(sh, &sh.q_full[dt], q_phase, DSV4_DEVERR_TIMEOUT_MMA);
            int su = slot0 + dt;
            uint32_t ph = phase;
            if (su >= NST) {
              su -= NST;
              ph ^= 1;
            }
            ok = ok && pa_wait(sh, &sh.full[su], ph, DSV4_DEVERR_TIMEOUT_MMA);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if (el) {
              const uint64_t ad = dq + dt * (2 * N * 128 / 16), bd = dk + su * (kPaStage / 16);
#pragma unroll
              for (int kk = 0; kk < 8; ++kk)
                tc_mma_f16(d, ad + (kk >> 2) * (N * 128 / 16) + 2 * (kk & 3),
                           bd + (kk >> 2) * (kPaTile / 16) + 2 * (kk & 3), id, (dt || kk) ? 1u : 0u);
            }
          }
          if (ok && el) {
            tc_commit(&sh.s_full[b]);
            if (i + nsub >= i1) tc_commit(&sh.q_empty);  // the piece's last use of Q
          }
          begin = false;
          slot += DT;
          if (slot >= NST) {
            slot -= NST;
            phase ^= 1;
          }
        }
        q_phase ^= 1;
      }
      i = 0;
      if (++g >= a.groups) {
        g = 0;
        ++t;
        sp = sp_next;
      }
    }
    // every product of this warp is done before TMEM is released
    if (el) tc_commit(&sh.last[0]);
    mbar_wait(&sh.last[0], 0, DSV4_DEVERR_TIMEOUT_MMA);
    __syncwarp();
  } else if (warp == 2) {
    // --------------------------------------------------- output products
    const bool el = elect_one();
    constexpr uint32_t id = pa_idesc<T>(128, N, 1);
    const uint64_t dm = sdesc_mn_sw128(smem_u32(ring), kPaTile), dp = sdesc_k_sw128(smem_u32(sP));
    bool ok = true;
    uint32_t k = 0;
    int slot = 0;
    while (left > 0 && ok && t < a.T) {
      const int n = pa_row(a, sp).n;
      const int2 sp_next = pa_index(a, t + 1);
      const int i1 = min(n, i + left);
      if (i < i1) {
        left -= i1 - i;
        bool begin = true;  // the piece's output starts anew
        for (; i < i1 && ok; i += nsub, ++k) {
          const uint32_t b = __shfl_sync(0xffffffffu, k & 1, 0);
          const uint32_t d = __shfl_sync(0xffffffffu, t_o, 0);
          const int slot0 = __shfl_sync(0xffffffffu, slot, 0);
          const uint32_t more = __shfl_sync(0xffffffffu, begin ? 0 : 1, 0);
          ok = __all_sync(0xffffffffu, pa_wait(sh, &sh.p_ready[b], (k >> 1) & 1, DSV4_DEVERR_TIMEOUT_MMA));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            if (dt >= DT) break;
            const int su = slot0 + dt >= NST ? slot0 + dt - NST : slot0 + dt;
            if (el) {
              const uint64_t ad = dm + su * (kPaStage / 16), bd = dp + b * (N * 128 / 16);
#pragma unroll
              for (int kk = 0; kk < kPaChunk / 16; ++kk)
                tc_mma_f16(d + N * dt, ad + kk * (16 * 128 / 16), bd + 2 * kk, id, kk ? 1u : more);
              tc_commit(&sh.empty[su]);
            }
          }
          if (el) tc_commit(&sh.pv_done[b]);
          begin = false;
          slot += DT;
          if (slot >= NST) slot -= NST;
        }
      }
      i = 0;
      if (++g >= a.groups) {
        g = 0;
        ++t;
        sp = sp_next;
      }
    }
    if (el) tc_commit(&sh.last[1]);
    mbar_wait(&sh.last[1], 0, DSV4_DEVERR_TIMEOUT_MMA);
    __syncwarp();
  } else {
    // ----------------------------------------------------------- softmax
    const int st = tid - 96;                  // 0 .. 255
    const int wi = warp - 3;                  // 0 .. 7
    const int q4 = warp & 3, half = wi >> 2;  // TMEM lane quarter; key half, then head half
    const int ha = 16 * q4 + (lane >> 2);     // this thread's heads: ha and ha + 8
    const bool active = 16 * q4 < N;          // quarters past N hold no heads
    const int c0 = 32 * half + 2 * (lane & 3);  // its keys: c0 + 8c and c0 + 8c + 1, c = 0 .. 3
    const int row = q4 * 32 + lane, h0 = half * HPT;  // output: channel of a 128-channel block, heads
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    const float scale2 = a.scale * kLog2e;
    T* out = static_cast<T*>(a.out);

    // rows that see nothing
    for (int z = blockIdx.x; z < a.T; z += gridDim.x) {
      if (pa_row(a, pa_index(a, z)).n) continue;
      uint4* o = reinterpret_cast<uint4*>(out + (size_t)z * a.H * a.D);
      for (int u = st; u < a.H * a.D / 8; u += kPaSoft) o[u] = make_uint4(0, 0, 0, 0);
    }

    uint32_t k = 0;     // chunks so far
    int slot = 0;       // ring position of this chunk's first stage
    while (left > 0 && t < a.T) {
      const PaRow r = pa_row(a, sp);
      const int2 sp_next = pa_index(a, t + 1);
      const int i_begin = i, i1 = min(r.n, i + left);
      if (i < i1) {
        const int* pages = a.table + (long long)r.s * a.max_pages;
        left -= i1 - i;
        // Whether key slot x of the chunk from box b on is visible, and its page there.
        auto seen = [&](int b, int x) -> bool {
          b += x >> a.box_log;
          if (b >= i1) return false;
          const int key = pa_box_key(a, r, b) + (x & ((1 << a.box_log) - 1));
          if (key > r.p || (key < r.w_lo && key >= r.f)) return false;
          const int p = __ldg(pages + (key >> a.page_log));
          if (p >= 0 && p < a.n_pages) return true;
          record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
          return false;
        };
        float m_a = kPaNoMax, m_b = kPaNoMax, l_a = 0.f, l_b = 0.f;
        bool any_seen = false;  // of the piece's keys
        bool see0 = seen(i, lane), see1 = seen(i, lane + 32);
        for (; i < i1; i += nsub, ++k) {
          const uint32_t lo = __ballot_sync(0xffffffffu, see0), hi = __ballot_sync(0xffffffffu, see1);
          any_seen |= (lo | hi) != 0;
          if (i + nsub < i1) {
            see0 = seen(i + nsub, lane);
            see1 = seen(i + nsub, lane + 32);
          }
          const uint32_t b = k & 1, u = (k >> 1) & 1;
          pa_wait(sh, &sh.s_full[b], u, DSV4_DEVERR_TIMEOUT_EPILOGUE);
          tc_fence_after();
          float z[16];
          float top_a = -INFINITY, top_b = -INFINITY;
          if (active) {
            tmem_ld_16x32(t_s + 64 * b + 32 * half + lane_base, z);
            tc_fence_before();
#pragma unroll
            for (int x = 0; x < 16; ++x) z[x] *= scale2;
            const uint32_t mask = (half ? hi : lo) >> (2 * (lane & 3));
            if (mask != (0xffffffffu >> (2 * (lane & 3)))) {
#pragma unroll
              for (int x = 0; x < 16; ++x)
                if (!(mask >> (8 * (x >> 2) + (x & 1)) & 1)) z[x] = -INFINITY;
            }
#pragma unroll
            for (int x = 0; x < 16; x += 4) {
              top_a = fmaxf(top_a, fmaxf(z[x], z[x + 1]));
              top_b = fmaxf(top_b, fmaxf(z[x + 2], z[x + 3]));
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.s_free[b]);
          constexpr float kLift = PaWeight<T>::lift, kRaise = kLift + PaWeight<T>::headroom;
          if (soft_or(top_a > m_a + kRaise || top_b > m_b + kRaise)) {
            // raise every head's max to its largest score so far (less the lift), over both key halves
            if (active) {
              top_a = fmaxf(top_a, __shfl_xor_sync(0xffffffffu, top_a, 1));
              top_b = fmaxf(top_b, __shfl_xor_sync(0xffffffffu, top_b, 1));
              top_a = fmaxf(top_a, __shfl_xor_sync(0xffffffffu, top_a, 2));
              top_b = fmaxf(top_b, __shfl_xor_sync(0xffffffffu, top_b, 2));
              if ((lane & 3) == 0) {
                sh.red[64 * half + ha] = top_a;
                sh.red[64 * half + ha + 8] = top_b;
              }
            }
            soft_sync();
            if (active) {
              const float n_a = fmaxf(m_a, fmaxf(sh.red[ha], sh.red[64 + ha]) - kLift);
              const float n_b = fmaxf(m_b, fmaxf(sh.red[ha + 8], sh.red[64 + ha + 8]) - kLift);
              const float f_a = ex2(m_a - n_a), f_b = ex2(m_b - n_b);
              m_a = n_a;
              m_b = n_b;
              l_a *= f_a;
              l_b *= f_b;
              if ((lane & 3) == 0 && half == 0) {
                sh.f[ha] = f_a;
                sh.f[ha + 8] = f_b;
              }
            }
            if (i > i_begin) {
              pa_wait(sh, &sh.pv_done[b ^ 1], ((k - 1) >> 1) & 1, DSV4_DEVERR_TIMEOUT_EPILOGUE);
              soft_sync();
              tc_fence_after();
              for (int dt = 0; dt < DT; ++dt) {
                float o[HPT];
                tmem_ldn<HPT>(t_o + N * dt + h0 + lane_base, o);
#pragma unroll
                for (int x = 0; x < HPT; ++x) o[x] *= sh.f[h0 + x];
                tmem_stn<HPT>(t_o + N * dt + h0 + lane_base, o);
              }
              tmem_wait_st();
            }
            soft_sync();  // sh.red and sh.f are read before they are written again
          }
          // the output product of two chunks ago has read this buffer of P
          if (k > 1) pa_wait(sh, &sh.pv_done[b], u ^ 1, DSV4_DEVERR_TIMEOUT_EPILOGUE);
          if ((lo & hi) != 0xffffffffu) {
            // whatever lies in a hidden row must not reach the output product (0 x NaN)
            for (int x = wi; x < kPaChunk; x += 8) {
              if ((x < 32 ? lo >> x : hi >> (x - 32)) & 1) continue;
              for (int y = lane; y < 16 * DT; y += 32) {
                int s = slot + (y >> 4);
                if (s >= NST) s -= NST;
                *reinterpret_cast<uint4*>(ring + s * kPaStage + ((y >> 3) & 1) * kPaTile + x * 128 + (y & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
              }
            }
          }
          if (active) {
            // weights, rounded to the cache's type as the product takes them, and summed as
            // rounded: the error of a weight that dominates its row then cancels in the quotient
            uint8_t* p0 = sP + b * (N * 128) + ha * 128 + 4 * (lane & 3);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t w_a = pack2<T>(ex2(z[4 * c] - m_a), ex2(z[4 * c + 1] - m_a));
              const uint32_t w_b = pack2<T>(ex2(z[4 * c + 2] - m_b), ex2(z[4 * c + 3] - m_b));
              l_a += sum2<T>(w_a);
              l_b += sum2<T>(w_b);
              const int unit = ((4 * half + c) ^ (ha & 7)) << 4;  // rows ha and ha + 8 swizzle alike
              *reinterpret_cast<uint32_t*>(p0 + unit) = w_a;
              *reinterpret_cast<uint32_t*>(p0 + 8 * 128 + unit) = w_b;
            }
          }
          fence_proxy_async_shared();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_ready[b]);
          slot += DT;
          if (slot >= NST) slot -= NST;
        }
        // ---- the piece's output: O^T columns times a factor per head
        if (active) {
#pragma unroll
          for (int o = 1; o < 4; o <<= 1) {
            l_a += __shfl_xor_sync(0xffffffffu, l_a, o);
            l_b += __shfl_xor_sync(0xffffffffu, l_b, o);
          }
          if ((lane & 3) == 0) {
            sh.red[64 * half + ha] = l_a;
            sh.red[64 * half + ha + 8] = l_b;
            if (half == 0) {
              // no key at all is told apart from scores that raised no max (NaN, -inf)
              sh.m[ha] = any_seen ? m_a : -INFINITY;
              sh.m[ha + 8] = any_seen ? m_b : -INFINITY;
            }
          }
        }
        pa_wait(sh, &sh.pv_done[(k - 1) & 1], ((k - 1) >> 1) & 1, DSV4_DEVERR_TIMEOUT_EPILOGUE);
        tc_fence_after();
        soft_sync();
        const bool whole = i_begin == 0 && i1 == r.n;
        const size_t piece = (size_t)blockIdx.x * 2 + (i_begin == 0);
        const int heads = min(N, a.H - 64 * g);
        if (st < N) {
          const float l = sh.red[st] + sh.red[64 + st], m = sh.m[st];
          if (whole) {
            const float sk = a.sink && st < heads ? __ldg(a.sink + 64 * g + st) * kLog2e : -INFINITY;
            const float mx = fmaxf(m, sk);
            const float den = l * ex2(m - mx) + pa_sink(sk, mx);
            sh.f[st] = m == -INFINITY ? 0.f : ex2(m - mx) / den;
          } else {
            a.part_ml[(piece * N + st) * 2] = m;
            a.part_ml[(piece * N + st) * 2 + 1] = l;
          }
        }
        soft_sync();
        for (int dt = 0; dt < DT; ++dt) {
          float o[HPT];
          tmem_ldn<HPT>(t_o + N * dt + h0 + lane_base, o);
          const int d = 128 * dt + row;
          if (whole) {
            // four lanes exchange four heads each, so that a thread has four channels of
            // one head: 8-byte stores instead of 2-byte ones, which take 4 cycles each
#pragma unroll
            for (int x = 0; x < HPT; x += 4) {
              const float4 v = transpose4(o[x], o[x + 1], o[x + 2], o[x + 3], lane);
              const int h = h0 + x + (lane & 3);
              const float f = sh.f[h];
              if (h < heads)
                *reinterpret_cast<uint2*>(out + ((size_t)t * a.H + 64 * g + h) * a.D + (d & ~3)) =
                    make_uint2(pack2<T>(v.x * f, v.y * f), pack2<T>(v.z * f, v.w * f));
            }
          } else {
            float* dst = a.part_o + (piece * N + h0) * a.D + d;
#pragma unroll
            for (int x = 0; x < HPT; ++x) dst[(size_t)x * a.D] = o[x];
          }
        }
        tc_fence_before();  // before the next piece's first output product (ordered by p_ready)
        soft_sync();        // sh.m, sh.f and sh.red are reused
      }
      i = 0;
      if (++g >= a.groups) {
        g = 0;
        ++t;
        sp = sp_next;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sh.tmem, kPaTmemCols);
  }
}

// Join the pieces of the rows that cross CTA borders.  Border c is a row's first if it
// lies inside the row and the border before does not; the row's pieces are then CTA
// c - 1's second kind (the one that holds its begin) and the first kind of CTAs c,
// c + 1, ...  Every CTA lists those rows from the plan, and the work units (row, head)
// go round the warps of the grid: one warp per unit, or all eight of a CTA, each on
// every eighth piece, where the units are few.
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kJoinSpread = 120 * 1024;  // shared memory that keeps a second CTA off the SM
constexpr int kJoinAhead = 4;  // pieces whose loads are in flight together

template <typename T, int N>
__global__ void __launch_bounds__(kJoinThreads) paged_attn_join_kernel(const PaArgs a, int n_plan) {
  __shared__ int4 rows[kPaMaxGrid];   // row, head group, first piece's CTA, pieces
  __shared__ int count[kJoinWarps];
  __shared__ float4 red[kJoinWarps][4][32];
  __shared__ float den_of[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, DT = a.D / 128;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // all of the attention's stores
  const int share = *a.share, snap = min(a.snap, share / 2);
  int n_rows = 0;  // in border order, so that every CTA has the same list
  for (int base = 1; base < n_plan; base += kJoinThreads) {
    const int c = base + threadIdx.x;
    int4 pl = make_int4(-1, 0, 0, 0);
    if (c < n_plan) pl = a.plan[c];
    auto inside = [&](int o) { return o > 0 && o < pl.w && pa_snap(o, pl.w, snap) == o; };
    const bool on = pl.x >= 0 && inside(pl.z) && !inside(pl.z - share);
    const unsigned vote = __ballot_sync(0xffffffffu, on);
    if (lane == 0) count[warp] = __popc(vote);
    __syncthreads();
    int at = n_rows;
    for (int w = 0; w < kJoinWarps; ++w) {
      if (w < warp) at += count[w];
      n_rows += count[w];
    }
    if (on) {
      int more = (pl.w - pl.z - 1) / share;  // borders of the row behind this one
      if (more && !inside(pl.z + more * share)) --more;
      rows[at + __popc(vote & ((1u << lane) - 1))] = make_int4(pl.x, pl.y, c - 1, 2 + more);
    }
    __syncthreads();
  }
  const int units = n_rows * N;
  const bool together = units <= (int)gridDim.x;
  const int first = together ? blockIdx.x : blockIdx.x * kJoinWarps + warp;
  const int step = together ? gridDim.x : gridDim.x * kJoinWarps;
  for (int u = first; u < units; u += step) {
    const int h = u % N;
    const int4 r = rows[u / N];
    const int head = 64 * r.y + h;
    if (head >= a.H) continue;
    auto piece = [&](int i) { return ((size_t)r.z * 2 + (i == 0 ? 1 : 2 * i)) * N + h; };
    // each lane holds the maxima of pieces lane, lane + 32, ...
    const float sk = a.sink ? __ldg(a.sink + head) * kLog2e : -INFINITY;
    const int p0 = together ? warp : 0, ps = together ? kJoinWarps : 1;
    float4 o[kJoinAhead][4];
    float2 ml[kJoinAhead];
    auto load = [&](int i0) {
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const int i = i0 + j * ps;
        if (i >= r.w) continue;
        const size_t at = piece(i);
        ml[j] = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (x < DT) o[j][x] = *reinterpret_cast<const float4*>(a.part_o + at * a.D + 128 * x + 4 * lane);
      }
    };
    load(p0);  // on the way while the maxima are compared
    float top = -INFINITY;
    for (int i = lane; i < r.w; i += 32) top = fmaxf(top, a.part_ml[piece(i) * 2]);
#pragma unroll
    for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const bool any_seen = top > -INFINITY;
    const float mx = fmaxf(top, sk);
    float den = 0.f;
    float4 acc[4] = {};
    for (int i0 = p0; i0 < r.w; i0 += ps * kJoinAhead) {
      if (i0 != p0) load(i0);
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        // only a piece that saw no key is left out: NaN and infinities reach the sum
        if (i0 + j * ps >= r.w || ml[j].x == -INFINITY) continue;
        const float f = ex2(ml[j].x - mx);
        den += ml[j].y * f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (x >= DT) break;
          acc[x].x += o[j][x].x * f;
          acc[x].y += o[j][x].y * f;
          acc[x].z += o[j][x].z * f;
          acc[x].w += o[j][x].w * f;
        }
      }
    }
    if (together) {
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (x < DT) red[warp][x][lane] = acc[x];
      if (lane == 0) den_of[warp] = den;
      __syncthreads();
      if (warp >= DT) continue;
      // warp x adds up channels 128 x .. +127
      den = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < kJoinWarps; ++w) {
        den += den_of[w];
        const float4 v = red[w][warp][lane];
        sum.x += v.x;
        sum.y += v.y;
        sum.z += v.z;
        sum.w += v.w;
      }
      acc[0] = sum;
    }
    den += pa_sink(sk, mx);
    const float inv = any_seen ? 1.f / den : 0.f;
    T* dst = static_cast<T*>(a.out) + ((size_t)r.x * a.H + head) * a.D + (together ? 128 * warp : 0) + 4 * lane;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (x >= (together ? 1 : DT)) break;
      *reinterpret_cast<uint2*>(dst + 128 * x) =
          make_uint2(pack2<T>(acc[x].x * inv, acc[x].y * inv), pack2<T>(acc[x].z * inv, acc[x].w * inv));
    }
  }
}

// ---------------------------------------------------------------- host side
struct PaShape {
  int N, groups, stages, grid, join_grid;
  size_t smem;
};

// Heads come in groups of 64 (the cache rows of a further group are read again,
// from L2 when it follows closely); fewer heads take the next of 16, 32, 64.
static PaShape pa_shape(int T, int H, int D, long long max_keys, int num_sms) {
  PaShape s;
  s.N = H > 32 ? 64 : H > 16 ? 32 : 16;
  s.groups = (H + 63) / 64;
  const int fixed = 1024 + (D / 64) * s.N * 128 + 2 * s.N * 128 + kPaCtrl;
  s.stages = (kPaSmemMax - fixed) / kPaStage;
  if (s.stages > kPaMaxStages) s.stages = kPaMaxStages;
  s.smem = (size_t)fixed + (size_t)s.stages * kPaStage;
  const long long most = (long long)T * s.groups * ((max_keys + kPaChunk - 1) / kPaChunk);
  if (num_sms > kPaMaxGrid) num_sms = kPaMaxGrid;
  s.grid = (int)(most < num_sms ? (most < 1 ? 1 : most) : num_sms);
  // a CTA for every head of a row that may be split, up to four per SM
  const long long split = s.grid - 1 < (long long)T * s.groups ? s.grid - 1 : (long long)T * s.groups;
  const long long units = split * s.N;
  s.join_grid = (int)(units < 4LL * num_sms ? (units < 1 ? 1 : units) : 4LL * num_sms);
  return s;
}

static long long pa_pieces_bytes(const PaShape& s, int D) { return (long long)s.grid * 2 * s.N * (D + 2) * 4; }

long long paged_attn_workspace(int T, int H, int D, long long max_keys, int num_sms) {
  const PaShape s = pa_shape(T, H, D, max_keys, num_sms);
  return pa_pieces_bytes(s, D) + (long long)s.grid * 16 + 16;
}

// 16-bit rows as {64 channels, rows, 64-channel tiles, z}: a box of `tiles` tiles x
// box_rows rows lands as [tile][row][64 channels], 128-byte swizzled.
static int make_tmap_tiles16(CUtensorMap* m, bool fp16, const void* base, int channels, int rows, long long row_stride,
                             int z, long long z_stride, int box_rows, int tiles) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return DSV4_ERR_CUDA;
  cuuint64_t dims[4] = {64, (cuuint64_t)rows, (cuuint64_t)(channels / 64), (cuuint64_t)z};
  cuuint64_t strides[3] = {(cuuint64_t)row_stride * 2, 128, (cuuint64_t)z_stride * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)tiles, 1};
  cuuint32_t es[4] = {1, 1, 1, 1};
  const CUresult r = enc(m, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? DSV4_OK : DSV4_ERR_CUDA;
}

template <typename T, int N>
static int launch_paged_attn_t(const PaShape& s, const CUtensorMap& qm, const CUtensorMap& kvm, const PaArgs& a,
                               int num_sms, cudaStream_t st) {
  if (ensure_smem_attr(reinterpret_cast<const void*>(paged_attn_kernel<T, N>), (int)s.smem)) return DSV4_ERR_CUDA;
  launch_k(paged_attn_kernel<T, N>, s.grid, kPaThreads, s.smem, st, qm, kvm, a);
  if (s.grid > 1) {
    // launched while the attention ends: its CTAs take the SMs' places as they get free
    // and wait there for the whole grid (griddepcontrol.wait); few CTAs get an SM each
    const size_t spread = s.join_grid <= num_sms ? kJoinSpread : 0;
    if (spread && ensure_smem_attr(reinterpret_cast<const void*>(paged_attn_join_kernel<T, N>), (int)spread))
      return DSV4_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)s.join_grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cfg.dynamicSmemBytes = spread;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    count_launch();
    if (cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<T, N>, a, s.grid) != cudaSuccess) {
      cudaGetLastError();
      return DSV4_ERR_CUDA;
    }
  }
  return cudaGetLastError() == cudaSuccess ? DSV4_OK : DSV4_ERR_CUDA;
}

int launch_paged_attn(const void* q, bool fp16, int T, int H, int D, long long q_stride_t, long long q_stride_h,
                      const void* pages, int n_pages, int page_size, long long page_stride, const int* table,
                      int n_seqs, int max_pages, const void* seq_ids, const void* positions, int idx64,
                      const float* sink, float scale, int window, int first, void* out, void* ws, long long ws_bytes,
                      int num_sms, cudaStream_t st) {
  const long long max_keys = (long long)max_pages * page_size;
  if (paged_attn_workspace(T, H, D, max_keys, num_sms) > ws_bytes || !ws) return DSV4_ERR_WORKSPACE;
  const PaShape s = pa_shape(T, H, D, max_keys, num_sms);
  // the kernel counts boxes (page_size rows, at most 64) of all rows in 32 bits
  const int box = page_size < kPaChunk ? page_size : kPaChunk;
  if ((long long)T * s.groups * (max_keys / box + 1) > INT_MAX) return DSV4_ERR_UNSUPPORTED;
  CUtensorMap qm, kvm;
  int rc = make_tmap_tiles16(&qm, fp16, q, D, H, q_stride_h, T, q_stride_t, s.N, 2);
  if (rc == DSV4_OK)
    rc = make_tmap_tiles16(&kvm, fp16, pages, D, page_size, D, n_pages, page_stride, box, box == kPaChunk ? 2 : 1);
  if (rc != DSV4_OK) return rc;
  PaArgs a{};
  a.out = out;
  a.table = table;
  a.seq_ids = seq_ids;
  a.positions = positions;
  a.sink = sink;
  a.part_o = static_cast<float*>(ws);
  a.part_ml = a.part_o + (size_t)s.grid * 2 * s.N * D;
  a.plan = reinterpret_cast<int4*>(static_cast<char*>(ws) + pa_pieces_bytes(s, D));
  a.share = reinterpret_cast<int*>(a.plan + s.grid);
  a.T = T;
  a.H = H;
  a.D = D;
  a.groups = s.groups;
  a.n_seqs = n_seqs;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  while (1 << a.page_log < page_size) ++a.page_log;
  a.box_log = a.page_log < 6 ? a.page_log : 6;
  a.idx64 = idx64;
  a.window = window;
  a.first = first;
  a.stages = s.stages;
  a.min_share = kPaMinChunks * (kPaChunk >> a.box_log);
  a.snap = kPaSnapChunks * (kPaChunk >> a.box_log);
  a.scale = scale;
  if (fp16) {
    if (s.N == 64) return launch_paged_attn_t<__half, 64>(s, qm, kvm, a, num_sms, st);
    if (s.N == 32) return launch_paged_attn_t<__half, 32>(s, qm, kvm, a, num_sms, st);
    return launch_paged_attn_t<__half, 16>(s, qm, kvm, a, num_sms, st);
  }
  if (s.N == 64) return launch_paged_attn_t<__nv_bfloat16, 64>(s, qm, kvm, a, num_sms, st);
  if (s.N == 32) return launch_paged_attn_t<__nv_bfloat16, 32>(s, qm, kvm, a, num_sms, st);
  return launch_paged_attn_t<__nv_bfloat16, 16>(s, qm, kvm, a, num_sms, st);
}

}  // namespace dsv4
