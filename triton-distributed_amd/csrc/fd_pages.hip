// Pages of a paged KV cache: copy, reserve, fork, free, compact (gfx950).
//
// The state is on the device: block_table [batch, width] int32 (a row's pages from the front, -1 behind them), kv_lens
// [batch], page_refs [num_pages] (rows that hold a page, 0 = free).  Nothing is read on the host.  Free pages are handed
// out lowest id first and in the order of the requests, so a sequence of calls gives the same tables every time: the scans
// that number free pages run in one workgroup, and what many workgroups do concurrently (reference counts of shared
// pages) are integer additions, whose order does not matter.
// Bound: the bytes of the pages that move (read and written once, 16 bytes a lane), else launch latency -- the scan of a
// pool's reference counts is 4 bytes a page, in 16 KB steps that end as soon as enough free pages are found.  Measured
// on caches of four layers, pages of 16 tokens x 8 heads of 128 in bf16: a copy of 777 of them 81 us = 5.0 TB/s, a compaction
// that moves 442 MB 95 us = 4.6 TB/s (a plain 1 GiB copy: 5.1 TB/s); freeing and forking 64 rows is bound by the host's
// part of two calls (21 us).  The one-workgroup plans grow with what they look at: a reserve that finds nothing free 8 us in
// a pool of 4096 pages, 31 us in 65536, 0.41 ms in 2^20; a fork's plan, which compares every child with those before it,
// 84 us for 1024 forks, 0.9 ms for 4096, 13 ms for 16384 (the most that a call takes).
#include "fd_common.h"

namespace {

constexpr int kScanThreads = 1024;
constexpr int kScanStep = 4 * kScanThreads;   // reference counts per step of a scan

// Inclusive prefix sum over a workgroup of kScanThreads; *total: the sum.  s_wave: [17] ints of LDS.
__device__ __forceinline__ int block_scan(int x, int* s_wave, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int up = __shfl_up(incl, off);
    if (lane >= off) incl += up;
  }
  __syncthreads();                            // s_wave may still be read from the scan before
  if (lane == 63) s_wave[wave] = incl;
  __syncthreads();
  int mine = lane < kScanThreads / 64 ? s_wave[lane] : 0;
#pragma unroll
  for (int off = 1; off < kScanThreads / 64; off <<= 1) {
    const int up = __shfl_up(mine, off);
    if (lane >= off) mine += up;
  }
  *total = __shfl(mine, kScanThreads / 64 - 1);
  return incl + (wave > 0 ? __shfl(mine, wave - 1) : 0);
}

__device__ __forceinline__ i32x4 load_refs(const int32_t* refs, int at, int num_pages) {
  i32x4 r = {-1, -1, -1, -1};                 // pages past the pool are neither free nor live
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at + k < num_pages) r[k] = refs[at + k];
  return r;
}

// visit(rank, page) for the first `wanted` free pages in ascending order; returns how many there were.
template <typename F>
__device__ __forceinline__ int for_free_pages(const int32_t* refs, int num_pages, int wanted, int* s_wave, F visit) {
  int found = 0;
  for (int base = 0; base < num_pages && found < wanted; base += kScanStep) {
    const int at = base + 4 * (int)threadIdx.x;
    const i32x4 r = load_refs(refs, at, num_pages);
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) mine += r[k] == 0 ? 1 : 0;
    int total;
    int rank = found + block_scan(mine, s_wave, &total) - mine;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r[k] == 0) {
        if (rank < wanted) visit(rank, at + k);
        ++rank;
      }
    found += total;
  }
  return min(found, wanted);
}

// ---------------------------------------------------------------- copy

// Workgroups walk the (entry, layer, pool, piece) items of a list of page copies.  count: entries, or count_at: where they
// are counted on the device.
struct CopyJob {
  PagePool pool;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* count_at;
  int32_t count, pieces;
  int64_t piece_bytes;
};

__device__ __forceinline__ void copy_pages(const CopyJob& c, int wg, int wgs) {
  const int n = c.count_at ? *c.count_at : c.count;
  const int64_t per_entry = (int64_t)c.pool.layers * 2 * c.pieces;
  for (int64_t item = wg; item < n * per_entry; item += wgs) {
    const int entry = (int)(item / per_entry);
    int rest = (int)(item - entry * per_entry);
    const int piece = rest % c.pieces;
    rest /= c.pieces;
    const int which = rest & 1, layer = rest >> 1;
    const int s = c.src[entry], d = c.dst[entry];
    if (s < 0 || s >= c.pool.num_pages || d < 0 || d >= c.pool.num_pages || s == d) continue;
    const int64_t bytes = c.pool.page_bytes[which];
    const int64_t first = piece * c.piece_bytes;
    const int64_t last = first + c.piece_bytes < bytes ? first + c.piece_bytes : bytes;
    char* base = c.pool.base[which] + layer * c.pool.layer_stride[which];
    const char* from = base + s * c.pool.page_stride[which];
    char* to = base + d * c.pool.page_stride[which];
    const int64_t step = (int64_t)blockDim.x * 16;
    int64_t at = first + (int64_t)threadIdx.x * 16;
    // four requests in flight per lane; the pages are used once here: past the caches
    for (; at + 3 * step < last; at += 4 * step) {
      u32x4 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = load_stream_b128(from + at + k * step);
#pragma unroll
      for (int k = 0; k < 4; ++k) __builtin_nontemporal_store(x[k], (u32x4*)(to + at + k * step));
    }
    for (; at < last; at += step) __builtin_nontemporal_store(load_stream_b128(from + at), (u32x4*)(to + at));
  }
}

__global__ void __launch_bounds__(256) fd_pages_copy_kernel(const CopyJob c) { copy_pages(c, blockIdx.x, gridDim.x); }

// Piece size: 16 KB (four 128-bit requests per lane of 256), less while the list would not give every CU four workgroups.
void set_pieces(CopyJob* c, int64_t entries) {
  const int64_t page = c->pool.page_bytes[0] > c->pool.page_bytes[1] ? c->pool.page_bytes[0] : c->pool.page_bytes[1];
  int64_t piece = 16384;
  while (piece > 4096 && entries * c->pool.layers * 2 * ((page + piece - 1) / piece) < 1024) piece >>= 1;
  c->piece_bytes = piece;
  c->pieces = (int)((page + piece - 1) / piece);
}

constexpr int64_t kCopyGrid = 4096;   // workgroups that walk a list: 16 per CU

// ---------------------------------------------------------------- reserve

constexpr int kMaxReserveBatch = 4096;
constexpr int kMaxReservePages = 1 << 20;     // of a row and call: 1024 rows' wants fit 32 bits ...
constexpr int kWantedEnough = (1 << 30) - 1;  // ... and sums of more than any pool holds stop here
constexpr int kNothingMissing = 0x7fffffff;

// Whether row b holds the page of its last token, and with it, from the front, those of all `len` (at most width * P): not
// where tokens were counted that no page had been granted for.
__device__ __forceinline__ bool holds_length(const PageTables& t, int b, int len, int P) {
  return len == 0 || t.bt[b * t.sbt + (len - 1) / P] >= 0;
}

__global__ void __launch_bounds__(kScanThreads) fd_pages_reserve_kernel(const PageTables t, int num_pages, int P,
                                                                       const int32_t* __restrict__ new_tokens, int uniform,
                                                                       int32_t* __restrict__ ok) {
  __shared__ int s_wave[17];
  __shared__ int s_end[kMaxReserveBatch];     // pages wanted by rows 0 .. b
  __shared__ int s_at[kMaxReserveBatch];      // first missing entry of row b
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // a wave per row counts the entries that are missing for its tokens to come
  for (int b = wave; b < t.batch; b += kScanThreads / 64) {
    const int len = max(t.kv_lens[b], 0);
    const int64_t grown = (int64_t)len + max(new_tokens ? new_tokens[b] : uniform, 0);
    const int64_t last = (grown + P - 1) / P;
    int missing = -1, first = 0;              // -1: refused, the table has no room or lacks pages that the length counts on
    if (last <= t.width && (grown == len || holds_length(t, b, len, P))) {
      first = (int)(((int64_t)len + P - 1) / P);
      int have = 0;
      for (int j = first + lane; j < (int)last; j += 64) have += t.bt[b * t.sbt + j] >= 0 ? 1 : 0;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) have += __shfl_xor(have, off);
      missing = max((int)last - first - have, 0);
      first = missing > 0 ? first + have : kNothingMissing;
      if (missing > kMaxReservePages) missing = -1;
    }
    if (lane == 0) {
      s_end[b] = missing;
      s_at[b] = first;
    }
  }
  __syncthreads();
  int wanted = 0;
  for (int b0 = 0; b0 < t.batch; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    const int need = b < t.batch ? s_end[b] : 0;
    int total;
    const int incl = block_scan(max(need, 0), s_wave, &total);
    if (b < t.batch) {
      s_end[b] = min(wanted + incl, kWantedEnough);
      if (need < 0) s_at[b] = -1;
    }
    wanted = min(wanted + total, kWantedEnough);
  }
  __syncthreads();
  // how many of them the pool can give is known only when the scan has run; the pages are noted as they are found and a
  // row that does not get all of its pages gets none: the count is taken first
  int found = for_free_pages(t.refs, num_pages, wanted, s_wave, [](int, int) {});
  __syncthreads();
  for_free_pages(t.refs, num_pages, found, s_wave, [&](int rank, int page) {
    int lo = 0, hi = t.batch - 1;             // the row that the rank belongs to: first b with s_end[b] > rank
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > rank) hi = mid; else lo = mid + 1;
    }
    if (s_end[lo] > found) return;
    const int before = lo ? s_end[lo - 1] : 0;
    t.bt[lo * t.sbt + s_at[lo] + (rank - before)] = page;
    t.refs[page] = 1;
  });
  for (int b = threadIdx.x; b < t.batch; b += kScanThreads)
    ok[b] = s_at[b] == kNothingMissing || (s_at[b] >= 0 && s_end[b] <= found) ? 1 : 0;
}

// ---------------------------------------------------------------- fork

// Workspace of a fork, [n] int32 each: parents' lengths (-1: refused) and the fresh pages.
__global__ void __launch_bounds__(kScanThreads) fd_pages_fork_plan_kernel(const PageTables t, int num_pages, int P,
                                                                          const int32_t* __restrict__ parents,
                                                                          const int32_t* __restrict__ children, int n,
                                                                          int32_t* __restrict__ lens,
                                                                          int32_t* __restrict__ fresh,
                                                                          int32_t* __restrict__ ok) {
  __shared__ int s_wave[17];
  int wanted = 0;
  for (int i0 = 0; i0 < n; i0 += kScanThreads) {
    const int i = i0 + threadIdx.x;
    int len = -1;
    if (i < n) {
      const int p = parents[i], c = children[i];
      bool good = p >= 0 && p < t.batch && c >= 0 && c < t.batch && p != c && t.kv_lens[c] == 0 && t.bt[c * t.sbt] < 0;
      for (int j = 0; good && j < i; ++j) good = children[j] != c;    // a row that was named before
      if (good) {
        len = (int)min((int64_t)max(t.kv_lens[p], 0), (int64_t)t.width * P);
        if (!holds_length(t, p, len, P)) len = -1;
      }
    }
    const int need = len > 0 && len % P ? 1 : 0;
    int total;
    const int rank = wanted + block_scan(need, s_wave, &total) - need;
    if (i < n) {
      lens[i] = len;
      fresh[i] = need ? -2 - rank : -1;       // a rank until the scan below has found its page
    }
    wanted += total;
  }
  __syncthreads();
  // rank -> page: the ranks are in list order, so the page of rank r belongs to the r-th entry that needs one; the list of
  // pages goes behind the two arrays
  int32_t* pages = fresh + n;
  const int found = for_free_pages(t.refs, num_pages, wanted, s_wave, [&](int rank, int page) { pages[rank] = page; });
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kScanThreads) {
    int good = lens[i] >= 0 ? 1 : 0;
    const int f = fresh[i];
    if (f <= -2) {
      const int rank = -2 - f;
      if (rank < found) {
        fresh[i] = pages[rank];
      } else {
        lens[i] = -1;
        good = 0;
      }
    }
    ok[i] = good;
  }
}

// Workgroup (i, 0) writes fork i's table row, reference counts and length; (i, 1 + k) copies the last page's tokens in
// pool k & 1 of layer k >> 1.
__global__ void __launch_bounds__(256) fd_pages_fork_kernel(const PagePool pool, const PageTables t,
                                                            const int32_t* __restrict__ parents,
                                                            const int32_t* __restrict__ children,
                                                            const int32_t* __restrict__ lens,
                                                            const int32_t* __restrict__ fresh) {
  const int i = blockIdx.x;
  const int len = lens[i];
  if (len < 0) return;
  const int p = parents[i], c = children[i], page = fresh[i];
  const int whole = len / pool.page_size, part = len - whole * pool.page_size;
  if (blockIdx.y == 0) {
    for (int j = threadIdx.x; j < t.width; j += 256) {
      int e = -1;
      if (j < whole) {
        e = t.bt[p * t.sbt + j];
        if (e >= 0 && e < pool.num_pages) atomicAdd(t.refs + e, 1);
      } else if (j == whole && part) {
        e = page;
        t.refs[page] = 1;
      }
      t.bt[c * t.sbt + j] = e;
    }
    if (threadIdx.x == 0) t.kv_lens[c] = len;
  } else if (part) {
    const int which = (blockIdx.y - 1) & 1, layer = (blockIdx.y - 1) >> 1;
    const int from_page = t.bt[p * t.sbt + whole];
    if (from_page < 0 || from_page >= pool.num_pages) return;
    char* base = pool.base[which] + layer * pool.layer_stride[which];
    const char* from = base + from_page * pool.page_stride[which];
    char* to = base + page * pool.page_stride[which];
    const int64_t bytes = pool.page_bytes[which] / pool.page_size * part;
    for (int64_t at = (int64_t)threadIdx.x * 16; at < bytes; at += 256 * 16) *(u32x4*)(to + at) = *(const u32x4*)(from + at);
  }
}

// ---------------------------------------------------------------- free

// A workgroup per listed row.  An entry is taken out of the table with an exchange, so a row that is listed twice gives its
// pages back once.
__global__ void __launch_bounds__(256) fd_pages_free_kernel(const PageTables t, int num_pages,
                                                            const int32_t* __restrict__ rows) {
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= t.batch) return;
  for (int j = threadIdx.x; j < t.width; j += 256) {
    const int e = atomicExch(t.bt + row * t.sbt + j, -1);
    if (e < 0 || e >= num_pages) continue;
    if (atomicSub(t.refs + e, 1) <= 0) atomicAdd(t.refs + e, 1);   // (a page that nobody held stays free)
  }
  if (threadIdx.x == 0) t.kv_lens[row] = 0;
}

// ---------------------------------------------------------------- compact

// Workspace: count [1] (and 3 words to spare), src [num_pages], dst [num_pages], moved-to [num_pages].
__global__ void __launch_bounds__(kScanThreads) fd_pages_compact_plan_kernel(int32_t* __restrict__ refs, int num_pages,
                                                                             int32_t* __restrict__ live_out,
                                                                             int32_t* __restrict__ count,
                                                                             int32_t* __restrict__ src,
                                                                             int32_t* __restrict__ dst,
                                                                             int32_t* __restrict__ to) {
  __shared__ int s_wave[17];
  int mine = 0;
  for (int at = 4 * (int)threadIdx.x; at < num_pages; at += kScanStep) {
    const i32x4 r = load_refs(refs, at, num_pages);
#pragma unroll
    for (int k = 0; k < 4; ++k) mine += r[k] > 0 ? 1 : 0;
  }
  int live;
  block_scan(mine, s_wave, &live);
  // free pages below `live` take the live pages at or above it, both in ascending order (there are equally many)
  int n_dst = 0, n_src = 0;
  for (int base = 0; base < num_pages; base += kScanStep) {
    const int at = base + 4 * (int)threadIdx.x;
    const i32x4 r = load_refs(refs, at, num_pages);
    int both = 0;                              // holes below `live` in the low half, live pages above in the high half
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (at + k < live) both += r[k] == 0 ? 1 : 0;
      else both += r[k] > 0 ? 1 << 16 : 0;
    }
    int total;
    const int before = block_scan(both, s_wave, &total) - both;
    int kd = n_dst + (before & 0xffff), ks = n_src + (before >> 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (at + k < live) {
        if (r[k] == 0) dst[kd++] = at + k;
      } else if (at + k < num_pages) {
        if (r[k] > 0) src[ks++] = at + k;
        else to[at + k] = at + k;
      }
    }
    n_dst += total & 0xffff;
    n_src += total >> 16;
  }
  __syncthreads();
  const int moves = min(n_dst, n_src);         // (equal, unless a count was negative)
  for (int k = threadIdx.x; k < moves; k += kScanThreads) {
    const int s = src[k], d = dst[k];
    to[s] = d;
    refs[d] = refs[s];
    refs[s] = 0;
  }
  for (int k = moves + threadIdx.x; k < n_src; k += kScanThreads) to[src[k]] = src[k];
  if (threadIdx.x == 0) {
    *count = moves;
    *live_out = live;
  }
}

// The first `table_wgs` workgroups rewrite the table, the others move the pages.
__global__ void __launch_bounds__(256) fd_pages_compact_kernel(const CopyJob c, const PageTables t, int table_wgs,
                                                               const int32_t* __restrict__ live_at,
                                                               const int32_t* __restrict__ to) {
  if ((int)blockIdx.x >= table_wgs) {
    copy_pages(c, blockIdx.x - table_wgs, gridDim.x - table_wgs);
    return;
  }
  const int live = *live_at;
  const int64_t total = (int64_t)t.batch * t.width;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < total; k += (int64_t)table_wgs * 256) {
    const int64_t b = k / t.width;
    int32_t* e = t.bt + b * t.sbt + (k - b * t.width);
    const int page = *e;
    if (page >= live && page < c.pool.num_pages) *e = to[page];
  }
}

int launched() { return hipGetLastError() == hipSuccess ? FD_OK : FD_ERR_LAUNCH; }

}  // namespace

int fd_launch_pages_copy(hipStream_t stream, const PagePool& pool, const int32_t* src, const int32_t* dst, int n) {
  CopyJob c = {};
  c.pool = pool; c.src = src; c.dst = dst; c.count = n;
  set_pieces(&c, n);
  int64_t wgs = (int64_t)n * pool.layers * 2 * c.pieces;
  if (wgs > kCopyGrid) wgs = kCopyGrid;
  hipLaunchKernelGGL(fd_pages_copy_kernel, dim3((unsigned)wgs), dim3(256), 0, stream, c);
  return launched();
}

int fd_launch_pages_reserve(hipStream_t stream, const PageTables& t, int num_pages, int page_size,
                            const int32_t* new_tokens, int uniform, int32_t* ok) {
  if (t.batch > kMaxReserveBatch) return FD_ERR_TOO_LARGE;
  hipLaunchKernelGGL(fd_pages_reserve_kernel, dim3(1), dim3(kScanThreads), 0, stream, t, num_pages, page_size, new_tokens,
                     uniform, ok);
  return launched();
}

int fd_launch_pages_fork(hipStream_t stream, const PagePool& pool, const PageTables& t, const int32_t* parents,
                         const int32_t* children, int n, int32_t* ok, int32_t* ws) {
  if (2 * (int64_t)pool.layers + 1 > 65535) return FD_ERR_TOO_LARGE;
  hipLaunchKernelGGL(fd_pages_fork_plan_kernel, dim3(1), dim3(kScanThreads), 0, stream, t, pool.num_pages, pool.page_size,
                     parents, children, n, ws, ws + n, ok);
  if (int rc = launched()) return rc;
  hipLaunchKernelGGL(fd_pages_fork_kernel, dim3((unsigned)n, (unsigned)(1 + 2 * pool.layers)), dim3(256), 0, stream, pool,
                     t, parents, children, ws, ws + n);
  return launched();
}

int fd_launch_pages_free(hipStream_t stream, const PageTables& t, int num_pages, const int32_t* rows, int n) {
  hipLaunchKernelGGL(fd_pages_free_kernel, dim3((unsigned)n), dim3(256), 0, stream, t, num_pages, rows);
  return launched();
}

int fd_launch_pages_compact(hipStream_t stream, const PagePool& pool, const PageTables& t, int32_t* live, int32_t* ws) {
  const int64_t N = pool.num_pages;
  int32_t *count = ws, *src = ws + 4, *dst = src + N, *to = dst + N;
  hipLaunchKernelGGL(fd_pages_compact_plan_kernel, dim3(1), dim3(kScanThreads), 0, stream, t.refs, pool.num_pages, live,
                     count, src, dst, to);
  if (int rc = launched()) return rc;
  CopyJob c = {};
  c.pool = pool; c.src = src; c.dst = dst; c.count_at = count;
  set_pieces(&c, N / 2 > 0 ? N / 2 : 1);
  int64_t table_wgs = ((int64_t)t.batch * t.width + 1023) / 1024;
  if (table_wgs > 256) table_wgs = 256;
  if (table_wgs < 1) table_wgs = 1;
  hipLaunchKernelGGL(fd_pages_compact_kernel, dim3((unsigned)(table_wgs + kCopyGrid)), dim3(256), 0, stream, c, t,
                     (int)table_wgs, live, to);
  return launched();
}
