// Attention of single tokens over the pages of a latent cache, on the tensor core.
//
//   out[t,h] = sum_j p[h,j] kv[j]      over the visible keys j of row t's sequence,
//   p[h,j] = exp(z[h,j] - m[h]) / (sum_j exp(z - m) + exp(sink[h] - m)),
//   z[h,j] = scale * q[t,h] . kv[j],   m[h] = max(max_j z[h,j], sink[h]).
//
// Row t stands at position p of sequence s and sees the keys j <= p, with a
// window only those above p - window and the first `first` ones.  Key j is row
// j % page_size of page page_table[s][j / page_size]; one cache row is key and
// value of every head.  A row with nothing visible gives zeros.
//
// As in sparse_attn.cu the two products put the cache rows on the M side:
//   S^T[j,h] = C[j,:] . Q[h,:]     M = 128 rows, N = heads, K = D
//   O^T[d,h] += C^T[d,j] . P[h,j]  M = 128 of D, N = heads, K = 128 rows
// and the second product reads the same shared memory as an MN-major operand.
//
// Bound: a row of D = 512 is 1 KB from HBM and 131 kFLOP with 64 heads, so the
// cache streams at the HBM rate if the tensor core sustains 830 TFLOP/s.
//
// Work split: the visible chunks of 128 keys of all rows form one list, and the
// list is cut into equal shares, one per CTA (at most one CTA per SM).  Every CTA
// finds its share from the lengths on the device, so ragged batches fill the SMs,
// nothing is read back and a captured graph follows the lengths of each replay.
// A row that crosses a border leaves fp32 partials (max, sum, O) that
// paged_attn_join_kernel merges; every CTA has at most two such pieces.
//
// Warp roles (320 threads): warp 0 loads Q and the pages by TMA into a ring of
// [128 rows][64 channels] tiles, warp 1 issues the products, warps 2-9 do the
// softmax: warp w reads TMEM lane quarter w % 4 (lane = cache row in the scores,
// = channel in the output) and half of the heads.  A tile goes back to the ring
// as soon as the output product that reads it last is done.
#include <limits.h>

#include <type_traits>

#include "kernels.cuh"

namespace dsv4 {

constexpr int kPaChunk = 128;
constexpr int kPaThreads = 320;
constexpr int kPaSoft = 256;                      // softmax threads: warps 2-9
constexpr int kPaTile = kPaChunk * 128;           // 16 KB: 128 rows x 64 channels
constexpr int kPaMaxStages = 12;
constexpr int kPaCtrl = 2048;
constexpr int kPaSmemMax = 232448;                // shared memory a CTA may use
constexpr int kPaMaxGrid = 1024;                  // CTAs (one per SM)
constexpr int kPaTmemCols = 512;                  // S: two buffers of 64 columns; O^T at 256
constexpr float kPaRescaleLog2 = 10.0f;           // headroom of the running max, base 2
constexpr float kPaNoMax = -3.402823466e38f;      // running max of a piece before its first key
constexpr float kLog2e = 1.4426950408889634f;

struct PaArgs {
  void* out;              // [T, H, D]
  const int* table;       // [n_seqs][max_pages]
  const void* seq_ids;    // [T] or NULL (row t reads sequence t)
  const void* positions;  // [T]
  const float* sink;      // [H] or NULL
  float* part_o;          // [grid][2][N][D]
  float* part_ml;         // [grid][2][N][2]: max, sum
  int4* plan;             // [grid]: row, head group, chunks of the row before this CTA, chunks of the row
  int* share;             // [1] chunks per CTA
  int T, H, D, groups;
  int n_seqs, max_pages, n_pages, page_size;
  int idx64, window, first, stages, min_share;
  float scale;
};

// What row t sees: keys [w_lo, p] and [0, f).  Chunk i of its n covers the keys
// from 128 * (i < nf ? i : i - nf + wb).
struct PaRow {
  int s, p, w_lo, f, nf, wb, n;
};

__device__ __forceinline__ PaRow pa_row(const PaArgs& a, int t) {
  PaRow r{};
  r.s = a.seq_ids ? load_index(a.seq_ids, a.idx64, t) : t;
  r.p = load_index(a.positions, a.idx64, t);
  if (r.s < 0 || r.p < 0) return r;
  if (r.s >= a.n_seqs || r.p / a.page_size >= a.max_pages) {
    record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return r;
  }
  r.w_lo = a.window > 0 ? max(0, r.p - a.window + 1) : 0;
  r.f = min(a.first, r.w_lo);
  r.wb = r.w_lo / kPaChunk;
  r.nf = min((r.f + kPaChunk - 1) / kPaChunk, r.wb);
  r.n = r.nf + r.p / kPaChunk + 1 - r.wb;
  return r;
}
__device__ __forceinline__ int pa_key0(const PaRow& r, int i) { return kPaChunk * (i < r.nf ? i : i - r.nf + r.wb); }

struct PaShared {
  uint64_t full[kPaMaxStages], empty[kPaMaxStages];
  uint64_t q_full, q_empty, s_full[2], s_free[2], p_ready, pv_done, last;
  uint32_t tmem;
  int abort;
  int t0, g0, i0;           // this CTA's first row, head group and chunk
  long long left;           // chunks of its share
  long long scan[kPaThreads / 32 + 1];
  float red[4 * 64];        // one value per lane quarter and head
  float m[64], f[64];       // running max, factor
};
static_assert(sizeof(PaShared) <= kPaCtrl, "control block too small");

// A bounded wait.  Once any wait of the CTA has run out, every wait returns at
// once: the roles run through their loops without waiting (loading and issuing
// nothing more), so no barrier is left with a missing thread.
__device__ __forceinline__ bool pa_wait(PaShared& sh, uint64_t* bar, uint32_t parity, int err) {
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  while (*reinterpret_cast<volatile int*>(&sh.abort) == 0) {
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

// Reduce n values per lane over the warp's 32 lanes (max, or sum): whole
// exchanges while a lane's half would be empty, then recursive halving.  Lane l
// gets the reduction of value l % n.
template <int n, bool kSum>
__device__ __forceinline__ float warp_reduce_n(float (&v)[n], int lane) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    if (o >= n) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float r = __shfl_xor_sync(0xffffffffu, v[i], o);
        v[i] = kSum ? v[i] + r : fmaxf(v[i], r);
      }
    } else {
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < o; ++i) {
        const float send = up ? v[i] : v[i + o];
        const float keep = up ? v[i + o] : v[i];
        const float r = __shfl_xor_sync(0xffffffffu, send, o);
        v[i] = kSum ? keep + r : fmaxf(keep, r);
      }
    }
  }
  return v[0];
}

// kind::f16 instruction descriptor: A and B both fp16 or both bf16, fp32 D, M = 128.
template <typename T>
__host__ __device__ constexpr uint32_t pa_idesc(uint32_t n, uint32_t a_mn, uint32_t b_mn) {
  const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn << 15) | (b_mn << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void tma_load_3d_at(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// N: heads per group, padded to 16, 32 or 64 (rows past H load as zeros).
template <typename T, int N>
__global__ void __launch_bounds__(kPaThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map,
                      const PaArgs a) {
  constexpr int HPT = N / 2;  // heads per softmax thread
  const float scale2 = a.scale * kLog2e;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int KT = a.D / 64, DT = a.D / 128, NST = a.stages;
  uint8_t* ring = smem;                             // NST tiles of [128 rows][128 B]
  uint8_t* sQ = ring + NST * kPaTile;               // KT tiles of [N heads][128 B]
  uint8_t* sP = sQ + KT * N * 128;                  // 2 tiles of [N heads][128 B]
  PaShared& sh = *reinterpret_cast<PaShared*>(sP + 2 * N * 128);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], 1);
    }
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_free[i], kPaSoft / 32);
    }
    mbar_init(&sh.p_ready, kPaSoft / 32);
    mbar_init(&sh.pv_done, 1);
    mbar_init(&sh.last, 1);
    fence_barrier_init();
    sh.abort = 0;
    sh.left = 0;
  }
  if (warp == 1) {
    tmem_alloc(&sh.tmem, kPaTmemCols);
    tmem_relinquish();
  }

  // ---- this CTA's share of the chunk list -----------------------------------
  {
    const int per = (a.T + kPaThreads - 1) / kPaThreads;
    const int r0 = min(a.T, tid * per), r1 = min(a.T, r0 + per);
    long long mine = 0;
    for (int t = r0; t < r1; ++t) mine += (long long)pa_row(a, t).n * a.groups;
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sh.scan[warp] = inc;
    __syncthreads();
    if (tid == 0) {
      long long run = 0;
      for (int i = 0; i < kPaThreads / 32; ++i) {
        const long long v = sh.scan[i];
        sh.scan[i] = run;
        run += v;
      }
      sh.scan[kPaThreads / 32] = run;
    }
    __syncthreads();
    const long long total = sh.scan[kPaThreads / 32];
    long long share = (total + gridDim.x - 1) / gridDim.x;
    if (share < a.min_share) share = a.min_share;
    const long long begin = share * blockIdx.x, end = min(total, begin + share);
    long long at = sh.scan[warp] + inc - mine;
    if (begin < end && at <= begin && begin < at + mine) {
      for (int t = r0; t < r1; ++t) {
        const int n = pa_row(a, t).n;
        if (begin < at + (long long)n * a.groups) {
          sh.t0 = t;
          sh.g0 = (int)((begin - at) / n);
          sh.i0 = (int)((begin - at) % n);
          sh.left = end - begin;
          a.plan[blockIdx.x] = make_int4(t, sh.g0, sh.i0, n);
          break;
        }
        at += (long long)n * a.groups;
      }
    }
    if (tid == 0) {
      if (begin >= end) a.plan[blockIdx.x] = make_int4(-1, 0, 0, 0);
      if (blockIdx.x == 0) *a.share = (int)min(share, (long long)INT_MAX);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t t_s = sh.tmem, t_o = sh.tmem + 256;

  if (warp == 0) {
    // ------------------------------------------------------------- loads
    const int rb = min(a.page_size, kPaChunk), nsub = kPaChunk / rb;  // rows per box, boxes per tile
    long long left = sh.left;
    int t = sh.t0, g = sh.g0, i = sh.i0;
    int slot = 0, issued = 0;
    uint32_t phase = 0, q_phase = 0;
    bool ok = true, q_issued = false;
    while (left > 0 && ok && t < a.T) {
      const PaRow r = pa_row(a, t);
      const int i1 = (int)min((long long)r.n, i + left);
      if (i < i1) {
        ok = __all_sync(0xffffffffu, pa_wait(sh, &sh.q_empty, q_phase ^ 1, DSV4_DEVERR_TIMEOUT_PRODUCER));
        if (!ok) break;
        q_phase ^= 1;
        q_issued = true;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sh.q_full, KT * N * 128);
          for (int kt = 0; kt < KT; ++kt)
            tma_load_3d_at(smem_u32(sQ + kt * N * 128), &q_map, &sh.q_full, 64 * kt, 64 * g, t);
        }
        const int* row = a.table + (long long)r.s * a.max_pages;
        left -= i1 - i;
        for (; i < i1 && ok; ++i) {
          // lane b loads box b of every tile: rows key .. key + rb - 1, on one page
          const int key = pa_key0(r, i) + lane * rb;
          int page = -1;
          if (lane < nsub && key <= r.p) page = __ldg(row + key / a.page_size);
          const bool on = page >= 0 && page < a.n_pages;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, on)) * rb * 128;
          for (int kt = 0; kt < KT; ++kt) {
            ok = __all_sync(0xffffffffu, pa_wait(sh, &sh.empty[slot], phase ^ 1, DSV4_DEVERR_TIMEOUT_PRODUCER));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&sh.full[slot], bytes);
            __syncwarp();
            if (on)
              tma_load_3d_at(smem_u32(ring + slot * kPaTile) + lane * rb * 128, &kv_map, &sh.full[slot], 64 * kt,
                             key % a.page_size, page);
            ++issued;
            if (++slot == NST) {
              slot = 0;
              phase ^= 1;
            }
          }
        }
      }
      i = 0;
      if (++g >= a.groups) {
        g = 0;
        ++t;
      }
    }
    // every copy has landed before the CTA can exit, also when a wait ran out
    for (int k = 0; k < min(issued, NST); ++k) {
      if (slot == 0) {
        slot = NST;
        phase ^= 1;
      }
      --slot;
      mbar_wait(&sh.full[slot], phase, DSV4_DEVERR_TIMEOUT_PRODUCER);
    }
    if (q_issued) mbar_wait(&sh.q_full, q_phase ^ 1, DSV4_DEVERR_TIMEOUT_PRODUCER);
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------- products
    if (lane == 0) {
      constexpr uint32_t id_qk = pa_idesc<T>(N, 0, 0), id_pv = pa_idesc<T>(N, 1, N == 64);
      // descriptors of the first tile; an address moves the low field by bytes / 16
      const uint64_t dk = sdesc_k_sw128(smem_u32(ring)), dm = sdesc_mn_sw128(smem_u32(ring), kPaTile);
      const uint64_t dq = sdesc_k_sw128(smem_u32(sQ));
      const uint64_t dp = N == 64 ? sdesc_mn_sw128(smem_u32(sP), kPaTile) : sdesc_k_sw128(smem_u32(sP));
      long long left = sh.left;
      const long long chunks = left;
      // with room for two chunks the next chunk's scores are issued before this one's output
      const bool ahead = NST >= 2 * KT;
      int t = sh.t0, g = sh.g0, i = sh.i0, n = 0;  // walk of the score products
      int i1 = 0;
      bool fresh_q = false;
      int slot = 0, pv_slot = 0;
      uint32_t phase = 0, q_phase = 0;
      long long qk_done = 0;
      bool ok = true;
      // the first chunk of a row (or of this share) starts its output anew
      uint64_t begins = 0;  // bit k % 64: chunk k begins a piece
      auto scores = [&]() {
        while (i >= i1) {  // next piece
          if (n) {
            i = 0;
            if (++g >= a.groups) {
              g = 0;
              ++t;
            }
          }
          if (t >= a.T) {
            ok = false;
            return;
          }
          n = pa_row(a, t).n;
          i1 = (int)min((long long)n, i + left);
          if (n == 0) {
            g = a.groups - 1;
            n = 1;
            i = i1 = 0;
          } else {
            fresh_q = true;
          }
        }
        const int b = (int)(qk_done & 1);
        const uint32_t u = (uint32_t)(qk_done >> 1) & 1;
        if (fresh_q) {
          ok = ok && pa_wait(sh, &sh.q_full, q_phase, DSV4_DEVERR_TIMEOUT_MMA);
          q_phase ^= 1;
        }
        ok = ok && pa_wait(sh, &sh.s_free[b], u ^ 1, DSV4_DEVERR_TIMEOUT_MMA);
        tc_fence_after();
        for (int kt = 0; kt < KT && ok; ++kt) {
          ok = pa_wait(sh, &sh.full[slot], phase, DSV4_DEVERR_TIMEOUT_MMA);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = dk + slot * (kPaTile / 16), bd = dq + kt * (N * 128 / 16);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_f16(t_s + 64 * b, ad + 2 * kk, bd + 2 * kk, id_qk, (kt | kk) ? 1u : 0u);
          if (++slot == NST) {
            slot = 0;
            phase ^= 1;
          }
        }
        if (ok) tc_commit(&sh.s_full[b]);
        begins = fresh_q ? begins | (1ull << (qk_done & 63)) : begins & ~(1ull << (qk_done & 63));
        fresh_q = false;
        ++i;
        --left;
        if (ok && i >= i1) tc_commit(&sh.q_empty);  // the piece's last use of Q
        ++qk_done;
      };
      auto outputs = [&](long long k) {
        ok = ok && pa_wait(sh, &sh.p_ready, (uint32_t)k & 1, DSV4_DEVERR_TIMEOUT_MMA);
        if (!ok) return;
        tc_fence_after();
        const bool begin = (begins >> (k & 63)) & 1;
        for (int dt = 0; dt < DT; ++dt) {
          // channels 128 dt .. +127 are tiles 2 dt and 2 dt + 1 of the chunk, side by
          // side in the ring (its length is even)
          const uint64_t ad = dm + pv_slot * (kPaTile / 16);
#pragma unroll
          for (int kk = 0; kk < kPaChunk / 16; ++kk) {
            const uint64_t bd = N == 64 ? dp + kk * (16 * 128 / 16) : dp + (kk >> 2) * (N * 128 / 16) + 2 * (kk & 3);
            tc_mma_f16(t_o + N * dt, ad + kk * (16 * 128 / 16), bd, id_pv, (!begin || kk) ? 1u : 0u);
          }
          tc_commit(&sh.empty[pv_slot]);
          tc_commit(&sh.empty[pv_slot + 1]);
          pv_slot = pv_slot + 2 == NST ? 0 : pv_slot + 2;
        }
        tc_commit(&sh.pv_done);
      };
      if (ahead && chunks > 0) scores();
      for (long long k = 0; k < chunks; ++k) {
        if (!ahead)
          scores();
        else if (k + 1 < chunks)
          scores();
        outputs(k);
      }
      // every product of this CTA is done before TMEM is released
      tc_commit(&sh.last);
      mbar_wait(&sh.last, 0, DSV4_DEVERR_TIMEOUT_MMA);
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------- softmax
    const int st = tid - 64;                  // 0 .. 255
    const int q4 = warp & 3;                  // TMEM lane quarter
    const int h0 = warp < 6 ? 0 : HPT;        // warps 2-5 the first half of the heads, 6-9 the second
    const int row = q4 * 32 + lane;           // cache row of the chunk; channel of a 128-channel tile
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    T* out = static_cast<T*>(a.out);

    // rows that see nothing
    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
      if (pa_row(a, t).n) continue;
      uint4* o = reinterpret_cast<uint4*>(out + (size_t)t * a.H * a.D);
      for (int u = st; u < a.H * a.D / 8; u += kPaSoft) o[u] = make_uint4(0, 0, 0, 0);
    }

    long long left = sh.left;
    int t = sh.t0, g = sh.g0, i = sh.i0;
    long long k = 0;    // chunks so far
    int slot = 0;       // ring position of this chunk's first tile
    while (left > 0 && t < a.T) {
      const PaRow r = pa_row(a, t);
      const int i_begin = i, i1 = (int)min((long long)r.n, i + left);
      if (i < i1) {
        const int* pages = a.table + (long long)r.s * a.max_pages;
        float l_run[HPT];
#pragma unroll
        for (int x = 0; x < HPT; ++x) l_run[x] = 0.f;
        if (st < N) sh.m[st] = kPaNoMax;
        soft_sync();
        left -= i1 - i;
        auto page_at = [&](int c) -> int {
          const int key = pa_key0(r, c) + row;
          if (key > r.p || (key < r.w_lo && key >= r.f)) return -1;
          const int p = __ldg(pages + key / a.page_size);
          if (p < 0 || p >= a.n_pages) {
            record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
            return -1;
          }
          return p;
        };
        int page_next = page_at(i);
        for (; i < i1; ++i, ++k) {
          const bool valid = page_next >= 0;
          if (i + 1 < i1) page_next = page_at(i + 1);
          const int b = (int)(k & 1);
          pa_wait(sh, &sh.s_full[b], (uint32_t)(k >> 1) & 1, DSV4_DEVERR_TIMEOUT_EPILOGUE);
          tc_fence_after();
          float z[HPT];
          tmem_ldn<HPT>(t_s + 64 * b + lane_base + h0, z);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.s_free[b]);
          float over = -INFINITY;  // how far the scores exceed the running max
          if (valid) {
#pragma unroll
            for (int x = 0; x < HPT; x += 4) {
              const float4 m4 = *reinterpret_cast<const float4*>(&sh.m[h0 + x]);
              over = fmaxf(over, fmaxf(fmaf(z[x], scale2, -m4.x), fmaf(z[x + 1], scale2, -m4.y)));
              over = fmaxf(over, fmaxf(fmaf(z[x + 2], scale2, -m4.z), fmaf(z[x + 3], scale2, -m4.w)));
            }
          }
          if (!valid) {
            // whatever lies in the hidden row must not reach the output product (0 x NaN):
            // this thread clears its half of the row's channels
            int s = slot + (h0 ? KT / 2 : 0);
            for (int kt = 0; kt < KT / 2; ++kt, ++s) {
              uint4* dst = reinterpret_cast<uint4*>(ring + (s >= NST ? s - NST : s) * kPaTile + row * 128);
#pragma unroll
              for (int x = 0; x < 8; ++x) dst[x] = make_uint4(0, 0, 0, 0);
            }
          }
          // the previous chunk's output product has read P and written O
          if (k > 0) pa_wait(sh, &sh.pv_done, (uint32_t)(k - 1) & 1, DSV4_DEVERR_TIMEOUT_EPILOGUE);
          if (soft_or(over > kPaRescaleLog2)) {
            // raise every head's max to its largest score so far
            tc_fence_after();
            float v[HPT];
#pragma unroll
            for (int x = 0; x < HPT; ++x) v[x] = valid ? z[x] * scale2 : -INFINITY;
            const float top = warp_reduce_n<HPT, false>(v, lane);
            if (lane < HPT) sh.red[q4 * 64 + h0 + lane] = top;
            soft_sync();
            if (st < N) {
              const float cm = fmaxf(fmaxf(sh.red[st], sh.red[64 + st]), fmaxf(sh.red[128 + st], sh.red[192 + st]));
              const float mo = sh.m[st], mn = fmaxf(mo, cm);
              sh.f[st] = ex2(mo - mn);
              sh.m[st] = mn;
            }
            soft_sync();
#pragma unroll
            for (int x = 0; x < HPT; ++x) l_run[x] *= sh.f[h0 + x];
            if (i > i_begin) {
              for (int dt = 0; dt < DT; ++dt) {
                float o[HPT];
                tmem_ldn<HPT>(t_o + N * dt + h0 + lane_base, o);
#pragma unroll
                for (int x = 0; x < HPT; ++x) o[x] *= sh.f[h0 + x];
                tmem_stn<HPT>(t_o + N * dt + h0 + lane_base, o);
              }
              tmem_wait_st();
            }
          }
          // weights, rounded to the cache's type as the product takes them; the sum adds
          // them unrounded (their rounding errors average out over the keys)
          if constexpr (N == 64) {
            // P[j][h], heads contiguous: 128-byte rows, 128-byte swizzle (MN-major operand)
            uint8_t* prow = sP + row * 128;
#pragma unroll
            for (int x = 0; x < HPT; x += 8) {
              Pack<T, 8> w;
#pragma unroll
              for (int y = 0; y < 8; y += 4) {
                const float4 m4 = *reinterpret_cast<const float4*>(&sh.m[h0 + x + y]);
                const float mm[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const float e = valid ? ex2(fmaf(z[x + y + c], scale2, -mm[c])) : 0.f;
                  l_run[x + y + c] += e;
                  w.v[y + c] = from_f32<T>(e);
                }
              }
              store_pack<T, 8>(reinterpret_cast<T*>(prow + ((((h0 + x) >> 3) ^ (row & 7)) << 4)), w);
            }
          } else {
            // P[h][j], keys contiguous (K-major operand): 16 or 8 heads per thread
#pragma unroll
            for (int x = 0; x < HPT; ++x) {
              const float e = valid ? ex2(fmaf(z[x], scale2, -sh.m[h0 + x])) : 0.f;
              l_run[x] += e;
              *reinterpret_cast<T*>(sP + sw128_offset(N, h0 + x, row)) = from_f32<T>(e);
            }
          }
          fence_proxy_async_shared();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.p_ready);
          slot += KT;
          if (slot >= NST) slot -= NST;
        }
        // ---- the piece's output: O^T columns times a factor per head
        pa_wait(sh, &sh.pv_done, (uint32_t)(k - 1) & 1, DSV4_DEVERR_TIMEOUT_EPILOGUE);
        tc_fence_after();
        const float sum = warp_reduce_n<HPT, true>(l_run, lane);
        if (lane < HPT) sh.red[q4 * 64 + h0 + lane] = sum;
        soft_sync();
        const bool whole = i_begin == 0 && i1 == r.n;
        const size_t piece = (size_t)blockIdx.x * 2 + (i_begin == 0);
        const int heads = min(N, a.H - 64 * g);
        if (st < N) {
          const float l = (sh.red[st] + sh.red[64 + st]) + (sh.red[128 + st] + sh.red[192 + st]);
          const float m = sh.m[st];
          if (whole) {
            const float sk = a.sink && st < heads ? __ldg(a.sink + 64 * g + st) * kLog2e : -INFINITY;
            const float mx = fmaxf(m, sk);
            const float den = l * ex2(m - mx) + ex2(sk - mx);
            sh.f[st] = m == kPaNoMax ? 0.f : ex2(m - mx) / den;
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
            T* dst = out + ((size_t)t * a.H + 64 * g + h0) * a.D + d;
#pragma unroll
            for (int x = 0; x < HPT; ++x)
              if (h0 + x < heads) dst[(size_t)x * a.D] = from_f32<T>(o[x] * sh.f[h0 + x]);
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

// Join the pieces of the rows that cross CTA borders.  Border c (CTA c begins inside
// a row) is a row's first if the row begins in CTA c - 1; the row's pieces are then
// CTA c - 1's second kind (the one that holds its begin) and the first kind of CTAs
// c, c + 1, ...  Every CTA lists those rows from the plan, and the work units (row,
// head, 128 channels) go round the warps of the grid: one warp per unit, or all
// eight of a CTA, each on every eighth piece, where the units are few (one long row
// left in 65 pieces: 64 heads x 4 units).
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kJoinAhead = 8;  // pieces whose loads are in flight together

template <typename T, int N>
__global__ void __launch_bounds__(kJoinThreads) paged_attn_join_kernel(const PaArgs a, int n_plan) {
  __shared__ int4 rows[kPaMaxGrid];   // row, head group, first piece, pieces
  __shared__ int count[kJoinWarps];
  __shared__ float red[kJoinWarps][32][4];
  __shared__ float den_of[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long share = *a.share;
  int n_rows = 0;  // in border order, so that every CTA has the same list
  for (int base = 1; base < n_plan; base += kJoinThreads) {
    const int c = base + threadIdx.x;
    int4 pl = make_int4(-1, 0, 0, 0);  // row, group, chunks before the border, chunks of the row
    if (c < n_plan) pl = a.plan[c];
    const bool on = pl.x >= 0 && pl.z > 0 && pl.z <= share;
    const unsigned vote = __ballot_sync(0xffffffffu, on);
    if (lane == 0) count[warp] = __popc(vote);
    __syncthreads();
    int at = n_rows;
    for (int w = 0; w < kJoinWarps; ++w) {
      if (w < warp) at += count[w];
      n_rows += count[w];
    }
    if (on) rows[at + __popc(vote & ((1u << lane) - 1))] = make_int4(pl.x, pl.y, c - 1, 2 + (int)((pl.w - pl.z - 1) / share));
    __syncthreads();
  }
  const int slices = a.D / 128;
  const long long units = (long long)n_rows * N * slices;
  const bool together = units * kJoinWarps <= (long long)gridDim.x * kJoinWarps;
  const long long first = together ? blockIdx.x : (long long)blockIdx.x * kJoinWarps + warp;
  const long long step = together ? gridDim.x : (long long)gridDim.x * kJoinWarps;
  for (long long u = first; u < units; u += step) {
    const int slice = (int)(u % slices), h = (int)(u / slices % N);
    const int4 r = rows[u / slices / N];
    const int head = 64 * r.y + h;
    if (head >= a.H) continue;
    auto piece = [&](int i) { return (size_t)r.z * 2 + (i == 0 ? 1 : 2 * i); };
    // each lane holds the maxima and sums of pieces lane, lane + 32, ...
    const float sk = a.sink ? __ldg(a.sink + head) * kLog2e : -INFINITY;
    float mx = sk;
    for (int i = lane; i < r.w; i += 32) mx = fmaxf(mx, a.part_ml[(piece(i) * N + h) * 2]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float den = 0.f, acc[4] = {};
    const int p0 = together ? warp : 0, ps = together ? kJoinWarps : 1;
    for (int i0 = p0; i0 < r.w; i0 += ps * kJoinAhead) {
      float4 o[kJoinAhead];
      float f[kJoinAhead];
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        const int i = i0 + j * ps;
        f[j] = 0.f;
        if (i >= r.w) continue;
        const size_t at = piece(i) * N + h;
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
        o[j] = *reinterpret_cast<const float4*>(a.part_o + at * a.D + 128 * slice + 4 * lane);
        if (ml.x != kPaNoMax) {
          f[j] = ex2(ml.x - mx);
          den += ml.y * f[j];
        }
      }
#pragma unroll
      for (int j = 0; j < kJoinAhead; ++j) {
        if (f[j] == 0.f) continue;
        acc[0] += o[j].x * f[j];
        acc[1] += o[j].y * f[j];
        acc[2] += o[j].z * f[j];
        acc[3] += o[j].w * f[j];
      }
    }
    if (together) {
      __syncthreads();
#pragma unroll
      for (int x = 0; x < 4; ++x) red[warp][lane][x] = acc[x];
      if (lane == 0) den_of[warp] = den;
      __syncthreads();
      if (warp) continue;
      for (int w = 1; w < kJoinWarps; ++w) {
        den += den_of[w];
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[x] += red[w][lane][x];
      }
    }
    const bool any = den > 0.f || den != den;
    den += ex2(sk - mx);
    Pack<T, 4> out;
#pragma unroll
    for (int x = 0; x < 4; ++x) out.v[x] = from_f32<T>(any ? acc[x] / den : 0.f);
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + ((size_t)r.x * a.H + head) * a.D + 128 * slice + 4 * lane) =
        *reinterpret_cast<const uint2*>(&out);
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
  s.stages = (kPaSmemMax - fixed) / kPaTile;
  if (s.stages > kPaMaxStages) s.stages = kPaMaxStages;
  s.stages &= ~1;  // two tiles of one 128-channel output block lie side by side
  s.smem = (size_t)fixed + (size_t)s.stages * kPaTile;
  const long long most = (long long)T * s.groups * ((max_keys + kPaChunk - 1) / kPaChunk);
  if (num_sms > kPaMaxGrid) num_sms = kPaMaxGrid;
  s.grid = (int)(most < num_sms ? (most < 1 ? 1 : most) : num_sms);
  // a unit per warp for every row that may be split, up to eight CTAs per SM
  const long long split = s.grid - 1 < (long long)T * s.groups ? s.grid - 1 : (long long)T * s.groups;
  const long long units = split * s.N * (D / 128);
  s.join_grid = (int)(units < 8LL * num_sms ? (units < 1 ? 1 : units) : 8LL * num_sms);
  return s;
}

static long long pa_pieces_bytes(const PaShape& s, int D) { return (long long)s.grid * 2 * s.N * (D + 2) * 4; }

long long paged_attn_workspace(int T, int H, int D, long long max_keys, int num_sms) {
  const PaShape s = pa_shape(T, H, D, max_keys, num_sms);
  return pa_pieces_bytes(s, D) + (long long)s.grid * 16 + 16;
}

// 16-bit elements [z][y][64-channel tiles], 128-byte swizzled boxes of rows x 64 channels.
static int make_tmap_rows16(CUtensorMap* m, bool fp16, const void* base, int channels, int y, long long y_stride, int z,
                            long long z_stride, int box_rows) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return DSV4_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)y, (cuuint64_t)z};
  cuuint64_t strides[2] = {(cuuint64_t)y_stride * 2, (cuuint64_t)z_stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  cuuint32_t es[3] = {1, 1, 1};
  const CUresult r = enc(m, fp16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                         const_cast<void*>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? DSV4_OK : DSV4_ERR_CUDA;
}

template <typename T, int N>
static int launch_paged_attn_t(const PaShape& s, const CUtensorMap& qm, const CUtensorMap& kvm, const PaArgs& a,
                               cudaStream_t st) {
  if (ensure_smem_attr(reinterpret_cast<const void*>(paged_attn_kernel<T, N>), (int)s.smem)) return DSV4_ERR_CUDA;
  launch_k(paged_attn_kernel<T, N>, s.grid, kPaThreads, s.smem, st, qm, kvm, a);
  if (s.grid > 1) launch_k(paged_attn_join_kernel<T, N>, s.join_grid, kJoinThreads, 0, st, a, s.grid);
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
  CUtensorMap qm, kvm;
  int rc = make_tmap_rows16(&qm, fp16, q, D, H, q_stride_h, T, q_stride_t, s.N);
  if (rc == DSV4_OK)
    rc = make_tmap_rows16(&kvm, fp16, pages, D, page_size, D, n_pages, page_stride,
                          page_size < kPaChunk ? page_size : kPaChunk);
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
  a.page_size = page_size;
  a.idx64 = idx64;
  a.window = window;
  a.first = first;
  a.stages = s.stages;
  a.min_share = 1;
  a.scale = scale;
  if (fp16) {
    if (s.N == 64) return launch_paged_attn_t<__half, 64>(s, qm, kvm, a, st);
    if (s.N == 32) return launch_paged_attn_t<__half, 32>(s, qm, kvm, a, st);
    return launch_paged_attn_t<__half, 16>(s, qm, kvm, a, st);
  }
  if (s.N == 64) return launch_paged_attn_t<__nv_bfloat16, 64>(s, qm, kvm, a, st);
  if (s.N == 32) return launch_paged_attn_t<__nv_bfloat16, 32>(s, qm, kvm, a, st);
  return launch_paged_attn_t<__nv_bfloat16, 16>(s, qm, kvm, a, st);
}

}  // namespace dsv4
