// Pages of a cache and the sequences that hold them.
//
//   pages      [L][P][page_size][D]   the cache rows, in every layer under one page id
//   page_table [S][M] int32           a sequence's pages in order, -1 behind the last
//   seq_lens   [S]    int32           tokens a sequence has room for
//   page_refs  [P]    int32           sequences that hold a page; 0 = free
//
// reserve hands free pages (lowest id first) to sequences that grow, fork lets a
// child share its parent's full pages and copies the part-filled last one, free
// drops a sequence's pages, compact moves the used pages to the lowest ids.  All
// of it happens on the device in stream order, so the operations can be captured
// into a graph and need no copy of the tables on the host.
//
// The bookkeeping is a few hundred KB of integers and bound by latency: one CTA
// of 1024 threads walks the page counts with ballots and one scan per 16384 pages
// (4096 in a small pool), its results are the same in every run (free pages are taken
// in ascending order and counts are integer sums), and the row copies follow as a
// second kernel over all SMs, bound by HBM.  Measured: planning 4.5 us (1024 pages, fork or compact)
// and 11.6 us (255 sequences taking half of 32768 pages); the copies of a compaction
// in 43 layers 166 us for about 1.08 GB, the rate of a plain copy.
#include <limits.h>

#include "kernels.cuh"

namespace dsv4 {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanShared = 2048;  // claims and offsets stay in shared memory up to so many sequences / entries

// Exclusive scan of one int per thread over the CTA; *total gets the sum.
// `scratch` is kPlanWarps + 1 ints of shared memory.
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += n;
  }
  __syncthreads();  // the scratch of an earlier scan has been read
  if (lane == 31) scratch[w] = inc;
  __syncthreads();
  if (w == 0) {
    const int x = scratch[lane];
    int s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += n;
    }
    scratch[lane] = s - x;
    if (lane == 31) scratch[kPlanWarps] = s;
  }
  __syncthreads();
  *total = scratch[kPlanWarps];
  return scratch[w] + inc - v;
}

// Ascending ids p in [begin, end) with (refs[p] > 0) == used: their number, and
// the ids themselves in list[0 .. limit).  Stops once `limit` are found.  kPlanStep
// pages per thread and scan step have their loads in flight together.
template <int kPlanStep>
__device__ __forceinline__ int collect_step(const int* refs, int begin, int end, bool used, int limit, int* list,
                                             int* scratch) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int found = 0;
  for (long long base = begin; base < end && found < limit; base += kPlanThreads * kPlanStep) {
    // warp w takes 32 * kPlanStep consecutive pages, a ballot per 32
    const long long p0 = base + w * 32 * kPlanStep + lane;
    unsigned hit[kPlanStep];
    int mine = 0;
#pragma unroll
    for (int j = 0; j < kPlanStep; ++j) {
      const long long p = p0 + 32 * j;
      hit[j] = __ballot_sync(0xffffffffu, p < end && (refs[p] > 0) == used);
    }
#pragma unroll
    for (int j = 0; j < kPlanStep; ++j) mine += __popc(hit[j]);
    int total;
    int at = found + block_scan(lane == 0 ? mine : 0, scratch, &total);
    at = __shfl_sync(0xffffffffu, at, 0);
#pragma unroll
    for (int j = 0; j < kPlanStep; ++j) {
      if (hit[j] >> lane & 1) {
        const int k = at + __popc(hit[j] & ((1u << lane) - 1));
        if (k < limit) list[k] = (int)(p0 + 32 * j);
      }
      at += __popc(hit[j]);
    }
    found += total;
  }
  __syncthreads();
  return found;
}

__device__ __forceinline__ int collect_pages(const int* refs, int begin, int end, bool used, int limit, int* list,
                                             int* scratch) {
  if (end - begin <= 4 * kPlanThreads) return collect_step<4>(refs, begin, end, used, limit, list, scratch);
  return collect_step<16>(refs, begin, end, used, limit, list, scratch);
}

// owner[s] becomes the first entry that names sequence s (atomicMin over the entries).
__device__ __forceinline__ void init_owners(int* owner, int n_seqs) {
  for (int s = threadIdx.x; s < n_seqs; s += blockDim.x) owner[s] = INT_MAX;
  __syncthreads();
}

struct PageState {
  int* table;
  int* lens;
  int* refs;
  int n_seqs, max_pages, n_pages, page_size;
};

__device__ __forceinline__ int pages_of(int len, int page_size) {
  return len <= 0 ? 0 : (len - 1) / page_size + 1;
}

// Workspace: owner [n_seqs], start [n + 1], picked [n_pages].
__global__ void __launch_bounds__(kPlanThreads) cache_reserve_kernel(const PageState st, const int* seqs,
                                                                     const int* new_lens, int n, int* ws) {
  __shared__ int scratch[kPlanWarps + 1];
  __shared__ int owner_s[kPlanShared], start_s[kPlanShared + 1];
  __shared__ long long row_s[kPlanShared];  // where page k of the call goes in the table, less k
  int* owner = st.n_seqs <= kPlanShared ? owner_s : ws;
  int* start = n <= kPlanShared ? start_s : ws + st.n_seqs;
  int* picked = ws + st.n_seqs + n + 1;
  init_owners(owner, st.n_seqs);
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = seqs[i];
    if (s >= 0 && s < st.n_seqs) atomicMin(owner + s, i);
  }
  __syncthreads();
  long long total = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int s = seqs[i], len = new_lens[i];
      if (s >= 0) {
        const bool ok = s < st.n_seqs && owner[s] == i && len >= 0 && pages_of(len, st.page_size) <= st.max_pages;
        if (ok)
          need = max(0, pages_of(len, st.page_size) - pages_of(st.lens[s], st.page_size));
        else
          record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
      }
    }
    int sum;
    const int at = block_scan(need, scratch, &sum);
    // past n_pages the exact sum no longer matters: the call is refused
    if (i < n) start[i] = (int)min(total + at, (long long)INT_MAX);
    if (i < n && need && i < kPlanShared)
      row_s[i] = (long long)seqs[i] * st.max_pages + pages_of(st.lens[seqs[i]], st.page_size) - start[i];
    total = min(total + sum, (long long)INT_MAX);
  }
  if (threadIdx.x == 0) start[n] = (int)total;
  __syncthreads();
  if (total > st.n_pages || (total > 0 && collect_pages(st.refs, 0, st.n_pages, false, (int)total, picked, scratch) < total)) {
    if (threadIdx.x == 0) record_error(DSV4_DEVERR_NO_PAGES);
    return;
  }
  // a warp per entry, or several where the entries are few; four pages per lane in flight
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int warps = n < kPlanWarps ? kPlanWarps / n : 1;
  for (int e = w; e < n * warps; e += kPlanWarps) {
    const int i = e / warps, from = start[i], to = start[i + 1];
    if (from == to) continue;
    const long long at = i < kPlanShared
                             ? row_s[i]
                             : (long long)seqs[i] * st.max_pages + pages_of(st.lens[seqs[i]], st.page_size) - from;
    for (int k0 = from + (e % warps) * 128 + lane; k0 < to; k0 += 128 * warps) {
      int p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = k0 + 32 * j < to ? picked[k0 + 32 * j] : -1;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (p[j] < 0) continue;
        st.table[at + k0 + 32 * j] = p[j];
        st.refs[p[j]] = 1;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int s = seqs[i], len = new_lens[i];
    if (s >= 0 && s < st.n_seqs && owner[s] == i && len >= 0 && pages_of(len, st.page_size) <= st.max_pages)
      st.lens[s] = max(st.lens[s], len);
  }
}

// One CTA per entry.  Each table entry is claimed by an exchange, so a sequence
// named twice is dropped once.
__global__ void __launch_bounds__(256) cache_free_kernel(const PageState st, const int* seqs) {
  const int s = seqs[blockIdx.x];
  if (s < 0) return;
  if (s >= st.n_seqs) {
    if (threadIdx.x == 0) record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return;
  }
  int* row = st.table + (long long)s * st.max_pages;
  for (int j = threadIdx.x; j < st.max_pages; j += blockDim.x) {
    if (row[j] < 0) continue;
    const int p = atomicExch(row + j, -1);
    if (p < 0) continue;
    if (p < st.n_pages)
      atomicSub(st.refs + p, 1);
    else
      record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
  }
  if (threadIdx.x == 0) st.lens[s] = 0;
}

// Workspace: owner [n_seqs], len [n] (-1 = entry refused), fresh [n] (page for the
// part-filled last page, -1 = none), picked [n].
__global__ void __launch_bounds__(kPlanThreads) cache_fork_plan_kernel(const PageState st, const int* parents,
                                                                       const int* children, const int* fork_lens, int n,
                                                                       int* ws) {
  __shared__ int scratch[kPlanWarps + 1];
  __shared__ int owner_s[kPlanShared];
  int* owner = st.n_seqs <= kPlanShared ? owner_s : ws;
  int* len_of = ws + st.n_seqs;
  int* fresh = len_of + n;
  int* picked = fresh + n;
  init_owners(owner, st.n_seqs);
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    const int c = children[i];
    if (parents[i] >= 0 && c >= 0 && c < st.n_seqs) atomicMin(owner + c, i);
  }
  __syncthreads();
  int total = 0;
  for (int base = 0; base < n; base += kPlanThreads) {
    const int i = base + threadIdx.x;
    int need = 0;
    if (i < n) {
      const int p = parents[i], c = children[i];
      int len = -1;
      if (p >= 0 && c >= 0) {  // a negative id on either side is padding
        bool ok = p < st.n_seqs && c < st.n_seqs && owner[c] == i && st.lens[c] == 0;
        if (ok) {
          len = fork_lens ? fork_lens[i] : st.lens[p];
          ok = len >= 0 && len <= st.lens[p] && pages_of(len, st.page_size) <= st.max_pages;
        }
        if (!ok) {
          len = -1;
          record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
        }
      }
      len_of[i] = len;
      need = len > 0 && len % st.page_size != 0;
    }
    int sum;
    const int at = total + block_scan(need, scratch, &sum);
    if (i < n) fresh[i] = need ? at : -1;  // rank among the fresh pages for now
    total += sum;
  }
  __syncthreads();
  if (total > 0 && collect_pages(st.refs, 0, st.n_pages, false, total, picked, scratch) < total) {
    if (threadIdx.x == 0) record_error(DSV4_DEVERR_NO_PAGES);
    for (int i = threadIdx.x; i < n; i += kPlanThreads) len_of[i] = -1;
    return;
  }
  for (int i = threadIdx.x; i < n; i += kPlanThreads) {
    if (len_of[i] < 0) continue;
    if (fresh[i] >= 0) {
      fresh[i] = picked[fresh[i]];
      st.refs[fresh[i]] = 1;
    }
    st.lens[children[i]] = len_of[i];
  }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 8;  // 16-byte loads in flight per thread

// `n16` units of 16 bytes by the whole CTA.
__device__ __forceinline__ void copy_units(const uint4* src, uint4* dst, int n16) {
  for (int i = threadIdx.x; i < n16; i += kCopyThreads * kCopyUnroll) {
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
      if (i + j * kCopyThreads < n16) v[j] = src[i + j * kCopyThreads];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
      if (i + j * kCopyThreads < n16) dst[i + j * kCopyThreads] = v[j];
  }
}

struct PageRows {
  char* base;
  long long layer_stride, page_stride;  // bytes
  int n_layers, row16;                  // 16-byte units per row
};

// CTA (i, l): the rows of entry i's part-filled page in layer l; layer 0's CTA
// writes the child's table row and counts the shared pages.
__global__ void __launch_bounds__(kCopyThreads) cache_fork_copy_kernel(const PageState st, const PageRows rows,
                                                                       const int* parents, const int* children, int n,
                                                                       const int* ws) {
  const int i = blockIdx.x % n, l = blockIdx.x / n;
  const int* len_of = ws + st.n_seqs;
  const int len = len_of[i];
  if (len <= 0) return;
  const int full = len / st.page_size, rest = len % st.page_size;
  const int* from = st.table + (long long)parents[i] * st.max_pages;
  const int fresh = len_of[n + i];
  if (l == 0) {
    int* to = st.table + (long long)children[i] * st.max_pages;
    for (int j = threadIdx.x; j < full; j += kCopyThreads) {
      const int p = from[j];
      if (p >= 0 && p < st.n_pages) {
        to[j] = p;
        atomicAdd(st.refs + p, 1);
      } else {
        record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
      }
    }
    if (threadIdx.x == 0 && rest) to[full] = fresh;
  }
  if (!rest) return;
  const int p = from[full];
  if (p < 0 || p >= st.n_pages) {
    if (threadIdx.x == 0) record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return;
  }
  char* layer = rows.base + l * rows.layer_stride;
  copy_units(reinterpret_cast<const uint4*>(layer + p * rows.page_stride),
             reinterpret_cast<uint4*>(layer + fresh * rows.page_stride), rest * rows.row16);
}

// The k-th hole below the number of used pages takes the k-th used page above it,
// both ascending, so no page is source and target.  Workspace: n_moves [1],
// src [n_pages / 2], dst [n_pages / 2].
__global__ void __launch_bounds__(kPlanThreads) cache_compact_plan_kernel(const PageState st, int* page_map, int* ws) {
  __shared__ int scratch[kPlanWarps + 1];
  int* src = ws + 1;
  int* dst = src + st.n_pages / 2;
  int mine = 0, used;
  for (int p = threadIdx.x; p < st.n_pages; p += kPlanThreads) {
    const bool u = st.refs[p] > 0;
    mine += u;
    page_map[p] = u ? p : -1;
  }
  block_scan(mine, scratch, &used);
  // as many holes below `used` as used pages above it: at most n_pages / 2
  const int moves = collect_pages(st.refs, 0, used, false, INT_MAX, dst, scratch);
  collect_pages(st.refs, used, st.n_pages, true, moves, src, scratch);
  for (int k = threadIdx.x; k < moves; k += kPlanThreads) {
    page_map[src[k]] = dst[k];
    st.refs[dst[k]] = st.refs[src[k]];
    st.refs[src[k]] = 0;
  }
  if (threadIdx.x == 0) ws[0] = moves;
}

constexpr int kCopyPart = kCopyThreads * kCopyUnroll;  // 16-byte units of one part: 32 KB

// Page copies src[k] -> dst[k] in every layer, in parts of 32 KB spread over the
// grid; first the table entries follow the map.
__global__ void __launch_bounds__(kCopyThreads) cache_compact_copy_kernel(const PageState st, const PageRows rows,
                                                                          const int* page_map, const int* ws) {
  const long long entries = (long long)st.n_seqs * st.max_pages;
  for (long long i = (long long)blockIdx.x * kCopyThreads + threadIdx.x; i < entries; i += (long long)gridDim.x * kCopyThreads) {
    const int p = st.table[i];
    if (p < 0) continue;
    if (p < st.n_pages) {
      const int to = __ldg(page_map + p);
      if (to != p) st.table[i] = to;
    } else {
      record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    }
  }
  const int* src = ws + 1;
  const int* dst = src + st.n_pages / 2;
  const int page16 = st.page_size * rows.row16, parts = (page16 + kCopyPart - 1) / kCopyPart;
  const long long work = (long long)ws[0] * rows.n_layers * parts;
  for (long long w = blockIdx.x; w < work; w += gridDim.x) {
    const int part = (int)(w % parts);
    const long long kl = w / parts;
    const int l = (int)(kl % rows.n_layers), k = (int)(kl / rows.n_layers);
    char* layer = rows.base + l * rows.layer_stride;
    copy_units(reinterpret_cast<const uint4*>(layer + src[k] * rows.page_stride) + part * kCopyPart,
               reinterpret_cast<uint4*>(layer + dst[k] * rows.page_stride) + part * kCopyPart,
               min(kCopyPart, page16 - part * kCopyPart));
  }
}

constexpr int kCopyCtas = 16384;  // CTAs that keep every SM copying to the end

// Pages src[i] -> dst[i] in every layer.  An entry whose target is another
// entry's source, or an earlier entry's target, could not be ordered against it:
// it is reported and skipped.  Each CTA looks through the lists once and copies its
// page in a part of the layers: a CTA per layer read the lists again for each (2000
// pages of 4 KB in 43 layers 317 -> 178 us, 20000 in 8 layers 3245 -> 1103 us, where the
// lists still cost more than the copies; 200 pages of 64 KB in 43 layers 173 us either way).
__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const PageRows rows, int n_pages, int page_size,
                                                                  const int* src, const int* dst, int n, int parts) {
  const int i = blockIdx.x % n;
  const int s = src[i], d = dst[i];
  if (s < 0 || d < 0 || s == d) return;
  bool bad = s >= n_pages || d >= n_pages;
  for (int j = threadIdx.x; j < n && !bad; j += kCopyThreads)
    bad = src[j] >= 0 && dst[j] >= 0 && j != i && (src[j] == d || (j < i && dst[j] == d));
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) record_error(DSV4_DEVERR_BAD_CACHE_INDEX);
    return;
  }
  for (int l = blockIdx.x / n; l < rows.n_layers; l += parts) {
    char* layer = rows.base + l * rows.layer_stride;
    copy_units(reinterpret_cast<const uint4*>(layer + s * rows.page_stride),
               reinterpret_cast<uint4*>(layer + d * rows.page_stride), page_size * rows.row16);
  }
}

static int launched() { return cudaGetLastError() == cudaSuccess ? DSV4_OK : DSV4_ERR_CUDA; }

long long cache_reserve_workspace(int n, int n_seqs, int n_pages) { return 4LL * ((long long)n_seqs + n + 1 + n_pages); }
long long cache_fork_workspace(int n, int n_seqs) { return 4LL * ((long long)n_seqs + 3LL * n); }
long long cache_compact_workspace(int n_pages) { return 4LL * (1 + (long long)n_pages); }

int launch_cache_reserve(int* table, int* lens, int* refs, int n_seqs, int max_pages, int n_pages, int page_size,
                         const int* seqs, const int* new_lens, int n, int* ws, cudaStream_t st) {
  const PageState s{table, lens, refs, n_seqs, max_pages, n_pages, page_size};
  launch_k(cache_reserve_kernel, 1, kPlanThreads, 0, st, s, seqs, new_lens, n, ws);
  return launched();
}

int launch_cache_free(int* table, int* lens, int* refs, int n_seqs, int max_pages, int n_pages, const int* seqs, int n,
                      cudaStream_t st) {
  const PageState s{table, lens, refs, n_seqs, max_pages, n_pages, 1};
  launch_k(cache_free_kernel, (unsigned)n, 256, 0, st, s, seqs);
  return launched();
}

int launch_cache_fork(void* pages, int n_layers, long long layer_stride, long long page_stride, int row_bytes,
                      int* table, int* lens, int* refs, int n_seqs, int max_pages, int n_pages, int page_size,
                      const int* parents, const int* children, const int* fork_lens, int n, int* ws, cudaStream_t st) {
  const PageState s{table, lens, refs, n_seqs, max_pages, n_pages, page_size};
  const PageRows r{static_cast<char*>(pages), layer_stride, page_stride, n_layers, row_bytes / 16};
  if ((long long)n * n_layers > INT_MAX) return DSV4_ERR_UNSUPPORTED;
  launch_k(cache_fork_plan_kernel, 1, kPlanThreads, 0, st, s, parents, children, fork_lens, n, ws);
  launch_k(cache_fork_copy_kernel, (unsigned)n * n_layers, kCopyThreads, 0, st, s, r, parents, children, n,
           (const int*)ws);
  return launched();
}

int launch_cache_compact(void* pages, int n_layers, long long layer_stride, long long page_stride, int row_bytes,
                         int* table, int* refs, int n_seqs, int max_pages, int n_pages, int page_size, int* page_map,
                         int* ws, int num_sms, cudaStream_t st) {
  const PageState s{table, nullptr, refs, n_seqs, max_pages, n_pages, page_size};
  const PageRows r{static_cast<char*>(pages), layer_stride, page_stride, n_layers, row_bytes / 16};
  launch_k(cache_compact_plan_kernel, 1, kPlanThreads, 0, st, s, page_map, ws);
  launch_k(cache_compact_copy_kernel, (unsigned)num_sms * 4, kCopyThreads, 0, st, s, r, (const int*)page_map,
           (const int*)ws);
  return launched();
}

int launch_cache_copy(void* pages, int n_layers, long long layer_stride, long long page_stride, int row_bytes,
                      int n_pages, int page_size, const int* src, const int* dst, int n, cudaStream_t st) {
  const PageRows r{static_cast<char*>(pages), layer_stride, page_stride, n_layers, row_bytes / 16};
  const int share = kCopyCtas / n, parts = share < 1 ? 1 : share > n_layers ? n_layers : share;
  launch_k(cache_copy_kernel, (unsigned)n * parts, kCopyThreads, 0, st, r, n_pages, page_size, src, dst, n,
           parts);
  return launched();
}

}  // namespace dsv4
