// Pages of a paged KV cache that several sequences share, sm_100a.
//
// A block table [rows][cols] holds the page of every `block_size` tokens of a row, -1
// where it has none; refs[p] counts the table entries that hold page p (0: free). The
// cache is one or two planes (rows of values; the fp8 cache's block scales), each
// [layers][pages][page bytes] with any layer stride.
//
//  * pages_fork     — new row i continues row parents[i]: its pages are shared, the old
//                     rows give theirs up; counts move by integer atomics, whose order
//                     does not matter.
//  * pages_reserve  — room for more tokens in every row, from the lowest free pages, and a
//                     private copy of a last page that other rows hold too.
//  * pages_free     — chosen rows give their pages back.
//  * pages_compact  — live pages move to the front: the j-th live page behind the first
//                     `live` ones moves to the j-th free page among them.
//  * pages_copy     — the data movement of all of them: (source, destination) pairs over
//                     every layer and plane.
//
// The index kernels run in one CTA where an order is needed (which row gets which page):
// tables and counts are a few KB, and what they cost is the latency of reading them. The
// copies are bound by memory: bulk copies through shared memory, in pieces of a quarter of
// a page or so, move 400 pages x 27 layers (0.8 GB) at 6.06 TB/s, 94% of the measured copy
// bandwidth; the same copies by 16-byte loads and stores of 2,048 threads per SM reached
// 5.34 TB/s. Three CTAs per SM keep one thread's issue from bounding small pieces: partly
// filled pages of 256 rows 40.6 us, against 47.5 us with two larger rings.
//
// Reference: the page / block-table bookkeeping of the KV arena
// (crates/spark-abi/vendor/sparkpipe/include/sparkpipe/spark_kv_cache.h:227-300); sharing
// between live sequences is this framework's own.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <stdexcept>

#include "common.cuh"
#include "launch.h"
#include "pdl.h"

namespace sp {

namespace {

constexpr int kCopyThreads = 128;
constexpr int kStages = 4, kStageBytes = 18432;  // a copy CTA's ring: 72 KB, three per SM
constexpr int kCopyCtas = 3;
constexpr int kIndexThreads = 1024;
constexpr int kGrants = 4096;   // pages granted in one call that fit in shared memory
constexpr int kNearRefs = 8192; // page counts that do

// Exclusive prefix sum of one value per thread over the CTA; every thread gets the total.
SP_DEVI int block_scan(int v, int* total, int* warp_sums) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto scan = [&](int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const int x = scan(v);
  __syncthreads();  // the previous scan's readers are done with warp_sums
  if (lane == 31) warp_sums[w] = x;
  __syncthreads();
  const int sums = scan(lane < (int)blockDim.x >> 5 ? warp_sums[lane] : 0);  // in every warp
  *total = __shfl_sync(0xffffffffu, sums, 31);
  const int base = __shfl_sync(0xffffffffu, sums, w > 0 ? w - 1 : 0);
  return (w > 0 ? base : 0) + x - v;
}

SP_DEVI int pages_of(int tokens, int block_size) { return tokens <= 0 ? 0 : (tokens - 1) / block_size + 1; }

}  // namespace

// ------------------------------------------------------------------ fork
// CTAs [0, rows): old row b gives its pages up; CTAs [rows, rows + n): new row i.
__global__ void __launch_bounds__(128) pages_fork_kernel(const int* __restrict__ table, int rows, int cols,
                                                         const int* __restrict__ lens, const int* __restrict__ parents,
                                                         int* __restrict__ refs, int pages, int block_size,
                                                         int* __restrict__ new_table, int* __restrict__ new_lens) {
  griddep_wait();
  griddep_launch();
  if (blockIdx.x < rows) {
    const int* t = table + (long long)blockIdx.x * cols;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) {
      const int e = t[c];
      if (e >= 0 && e < pages) atomicSub(refs + e, 1);
    }
    return;
  }
  const int i = blockIdx.x - rows;
  const int p = parents[i];
  const bool there = p >= 0 && p < rows;
  const int len = there ? lens[p] : 0;
  const int held = pages_of(len, block_size);
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const int e = c < held ? table[(long long)p * cols + c] : -1;
    new_table[(long long)i * cols + c] = e;
    if (e >= 0 && e < pages) atomicAdd(refs + e, 1);
  }
  if (threadIdx.x == 0) new_lens[i] = len;
}

void pages_fork(const int* table, int rows, int cols, const int* lens, const int* parents, int n, int* refs, int pages,
                int block_size, int* new_table, int* new_lens, cudaStream_t s) {
  if (rows + n <= 0) return;
  launch_k(pages_fork_kernel, dim3((unsigned)(rows + n)), dim3(128), 0, s, table, rows, cols, lens, parents, refs,
           pages, block_size, new_table, new_lens);
}

// ------------------------------------------------------------------ reserve
// One CTA, a thread per row: what the row needs, its place among the needs of the rows before
// it, the lowest free pages (as many as are needed), the grants. The counts of up to
// kNearRefs pages and up to kGrants granted pages stay in shared memory, so that a beam step
// pays two dependent reads of memory (a row's length, its last page); larger caches read
// refs again, larger grants go through `free_list` [pages]. `work` gets the copy list, (source,
// destination, tokens) records, and `copies` its length. A row whose partly filled last page is
// missing, and with `strict` one whose tokens go past the table's width, cannot be served: it
// stays as it is, a holder of its pages like any idle row.
__global__ void __launch_bounds__(kPagesMaxRows)
    pages_reserve_kernel(int* __restrict__ table, int rows, int cols, const int* __restrict__ lens,
                         const int* __restrict__ row_tokens, int tokens, int strict, int* refs, int pages,
                         int block_size, int* free_list, int* __restrict__ work, int* __restrict__ copies,
                         int* __restrict__ short_by) {
  extern __shared__ int smem[];
  int* grants = smem;           // [kGrants]
  int* near = grants + kGrants; // [min(pages, kNearRefs)]
  __shared__ int tails[kPagesMaxRows];  // last page of a row that may have to leave it, else -1
  __shared__ bool unserved[kPagesMaxRows];
  __shared__ int warp_sums[32];
  __shared__ int s_copies;
  griddep_wait();
  griddep_launch();
  const int b = threadIdx.x;
  const bool in_near = pages <= kNearRefs;
  const int* counts = in_near ? near : refs;  // as they were before the call
  if (b == 0) s_copies = 0;
  int* t = table + (long long)b * cols;
  int len = 0, want = 0, tail = -1, first = 0, last = 0, fresh = 0;
  int lacks = 0;  // pages that the row lacks
  if (b < rows) {
    len = max(lens[b], 0);
    want = row_tokens ? row_tokens[b] : (len > 0 ? tokens : 0);
  }
  if (in_near)
    for (int p = b; p < pages; p += blockDim.x) near[p] = refs[p];
  if (want > 0) {
    if (len % block_size != 0 && len / block_size < cols) {
      tail = t[len / block_size];
      if (tail < 0 || tail >= pages) lacks = 1;
    }
    first = pages_of(len, block_size);
    const long long end = ((long long)len + want - 1) / block_size + 1;
    last = int(min((long long)cols, end));
    for (int c = first; c < last; ++c) fresh += t[c] < 0;
    if (strict && end > cols) lacks += int(min(end - cols, (long long)INT_MAX / 2));
    if (lacks > 0) {
      lacks += fresh;
      tail = -1;
      fresh = 0;
    }
  }
  tails[b] = tail;
  __syncthreads();
  bool leaves = false;
  // before any row's change: in large caches `counts` is refs itself
  const int holders = tail >= 0 ? counts[tail] : 0;
  if (holders > 1) {
    // the rows before this one with the same last page will have left it
    int earlier = 0;
#pragma unroll 8
    for (int q = 0; q < b; ++q) earlier += tails[q] == tail;
    leaves = holders - earlier > 1;
  }
  const int need = fresh + leaves;
  int all, total;
  const int start = block_scan(need, &all, warp_sums);
  // free pages, lowest first
  int* list = all <= kGrants ? grants : free_list;
  int found = 0;
  for (int p0 = 0; p0 < pages && found < all; p0 += blockDim.x) {
    const int p = p0 + b;
    const int is_free = p < pages && counts[p] <= 0;
    const int at = found + block_scan(is_free, &total, warp_sums);
    if (is_free && at < all) list[at] = p;
    found += total;
  }
  const bool served = start + need <= found;
  unserved[b] = need > 0 && !served;
  __syncthreads();
  if (!served) lacks += need;  // of a row that cannot be served need is 0
  if (all > found && need == 0 && holders > 1) {
    // a row that was to keep the page must not write to it while an earlier one is still there
    for (int q = 0; q < b; ++q)
      if (tails[q] == tail && unserved[q]) lacks = 1;
  }
  if (b < rows) {
    short_by[b] = lacks;
    if (served && need > 0) {
      int g = start;
      if (leaves) {  // the shared last page comes first
        const int page = list[g++];
        int* rec = work + 3 * atomicAdd(&s_copies, 1);
        rec[0] = tail;
        rec[1] = page;
        rec[2] = len % block_size;
        atomicSub(refs + tail, 1);
        refs[page] = 1;
        t[len / block_size] = page;
      }
      for (int c = first; c < last && fresh > 0; ++c)
        if (t[c] < 0) {
          const int page = list[g++];
          refs[page] = 1;
          t[c] = page;
        }
    }
  }
  __syncthreads();
  if (b == 0) *copies = s_copies;
}

void pages_reserve(int* table, int rows, int cols, const int* lens, const int* row_tokens, int tokens, bool strict,
                   int* refs, int pages, int block_size, int* free_list, int* work, int* copies, int* short_by,
                   cudaStream_t s) {
  if (rows <= 0) return;
  if (rows > kPagesMaxRows) throw std::runtime_error("pages_reserve: too many rows");
  set_smem_bytes(pages_reserve_kernel, (int)sizeof(int) * (kGrants + kNearRefs));
  launch_k(pages_reserve_kernel, dim3(1), dim3(kPagesMaxRows),
           sizeof(int) * (kGrants + (pages <= kNearRefs ? pages : 0)), s, table, rows, cols, lens, row_tokens, tokens,
           strict ? 1 : 0, refs, pages, block_size, free_list, work, copies, short_by);
}

// ------------------------------------------------------------------ free
__global__ void __launch_bounds__(128) pages_free_kernel(int* __restrict__ table, int cols, int* __restrict__ refs,
                                                         int pages, const int* __restrict__ rows, int n) {
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.x;
  if (rows) {  // a row that is named twice is freed once
    int named = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) named |= rows[i] == b;
    if (!__syncthreads_or(named)) return;
  }
  int* t = table + (long long)b * cols;
  for (int c = threadIdx.x; c < cols; c += blockDim.x) {
    const int e = t[c];
    if (e >= 0 && e < pages) atomicSub(refs + e, 1);
    t[c] = -1;
  }
}

void pages_free(int* table, int rows, int cols, int* refs, int pages, const int* which, int n, cudaStream_t s) {
  if (rows <= 0) return;
  launch_k(pages_free_kernel, dim3((unsigned)rows), dim3(128), 0, s, table, cols, refs, pages, which, n);
}

// ------------------------------------------------------------------ compact
// One CTA: live pages are counted, then the free pages below that count and the live ones
// at or above it are listed in order (equally many) and paired. `work`: [pages] x (source,
// destination, tokens) pairs; `holes` [pages].
__global__ void __launch_bounds__(kIndexThreads)
    pages_compact_kernel(int* __restrict__ refs, int pages, int block_size, int* __restrict__ page_map,
                         int* __restrict__ live_out, int* __restrict__ work, int* __restrict__ holes,
                         int* __restrict__ copies) {
  __shared__ int warp_sums[32];
  griddep_wait();
  griddep_launch();
  int mine = 0, live, total;
  for (int p = threadIdx.x; p < pages; p += blockDim.x) mine += refs[p] > 0;
  block_scan(mine, &live, warp_sums);
  int n_holes = 0;
  for (int p0 = 0; p0 < live; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const int hole = p < live && refs[p] <= 0;
    const int at = n_holes + block_scan(hole, &total, warp_sums);
    if (hole) holes[at] = p;
    if (p < live) page_map[p] = hole ? -1 : p;
    n_holes += total;
  }
  __syncthreads();
  int moved = 0;
  for (int p0 = live; p0 < pages; p0 += blockDim.x) {
    const int p = p0 + threadIdx.x;
    const int r = p < pages ? refs[p] : 0;
    const int moves = r > 0;
    const int at = moved + block_scan(moves, &total, warp_sums);
    if (moves) {
      const int to = holes[at];
      work[3 * at] = p;
      work[3 * at + 1] = to;
      work[3 * at + 2] = block_size;
      page_map[p] = to;
      refs[to] = r;
      refs[p] = 0;
    } else if (p < pages) {
      page_map[p] = -1;
    }
    moved += total;
  }
  if (threadIdx.x == 0) {
    *copies = moved;
    *live_out = live;
  }
}

void pages_compact(int* refs, int pages, int block_size, int* page_map, int* live, int* work, int* holes, int* copies,
                   cudaStream_t s) {
  launch_k(pages_compact_kernel, dim3(1), dim3(kIndexThreads), 0, s, refs, pages, block_size, page_map, live, work,
           holes, copies);
}

// ------------------------------------------------------------------ copy
// Checks a caller's (source, destination) pairs and writes the copy list. A pair with -1,
// or of a page with itself, is skipped. Pairs whose order would matter (a page that is
// the destination of two pairs, or the destination of one and the source of another), and
// pages outside the cache, refuse the whole call: nothing is copied and the status word is
// set. `marks`: a bit per page in shared memory.
__global__ void __launch_bounds__(kIndexThreads)
    pages_pairs_kernel(const int* __restrict__ src, const int* __restrict__ dst, int n, int pages, int block_size,
                       int* __restrict__ work, int* __restrict__ copies, int* err) {
  extern __shared__ int smem[];
  unsigned* marks = reinterpret_cast<unsigned*>(smem);
  __shared__ int s_count;
  griddep_wait();
  griddep_launch();
  for (int i = threadIdx.x; i < (pages + 31) / 32; i += blockDim.x) marks[i] = 0;
  if (threadIdx.x == 0) s_count = 0;
  __syncthreads();
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int a = src[i], b = dst[i];
    if (a == -1 || b == -1) continue;
    if (a < 0 || b < 0 || a >= pages || b >= pages) { bad = 1; continue; }
    if (a == b) continue;
    if (atomicOr(&marks[b >> 5], 1u << (b & 31)) & (1u << (b & 31))) bad = 1;
  }
  bad = __syncthreads_or(bad);
  for (int i = threadIdx.x; i < n && !bad; i += blockDim.x) {
    const int a = src[i], b = dst[i];
    if (a == -1 || b == -1 || a == b) continue;
    if (marks[a >> 5] & (1u << (a & 31))) bad = 1;
    const int at = atomicAdd(&s_count, 1);
    work[3 * at] = a;
    work[3 * at + 1] = b;
    work[3 * at + 2] = block_size;
  }
  bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    *copies = bad ? 0 : s_count;
    if (bad && err) atomicCAS(err, 0, kErrBadIndex);
  }
}

void pages_pairs(const int* src, const int* dst, int n, int pages, int block_size, int* work, int* copies, int* err,
                 cudaStream_t s) {
  if (pages > kPagesMaxMarked) throw std::runtime_error("copy_pages: too many pages");
  const size_t bytes = sizeof(int) * ((pages + 31) / 32);
  set_smem_bytes(pages_pairs_kernel, kPagesMaxMarked / 8);
  launch_k(pages_pairs_kernel, dim3(1), dim3(kIndexThreads), bytes, s, src, dst, n, pages, block_size, work, copies,
           err);
}

// Every thread that runs the small or unaligned part of a copy moves 4-byte words.
struct CopyPlane {
  char* base;
  long long layer_stride;  // bytes
  int page_bytes, token_bytes;
};

SP_DEVI void copy_words(const CopyPlane& p, int layer, int src, int dst, int from, int to, int first, int step) {
  const long long off = layer * p.layer_stride;
  const int* s = reinterpret_cast<const int*>(p.base + off + (long long)src * p.page_bytes);
  int* d = reinterpret_cast<int*>(p.base + off + (long long)dst * p.page_bytes);
  for (int w = from / 4 + first; w < to / 4; w += 4 * step) {
    int v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (w + j * step < to / 4) v[j] = s[w + j * step];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (w + j * step < to / 4) d[w + j * step] = v[j];
  }
}

// A table's entries through the page map of a compaction.
SP_DEVI void remap_table(int* table, long long entries, const int* page_map, int pages) {
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < entries;
       i += (long long)gridDim.x * blockDim.x) {
    const int e = table[i];
    if (e >= 0 && e < pages) table[i] = page_map[e];
  }
}

SP_DEVI void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(src)), "r"(bytes)
               : "memory");
}

// Units are (pair, layer, piece of the first plane), dealt to the CTAs in turn. One thread moves
// them through a ring of shared memory with bulk copies: the load of a unit goes out while the
// one before it is stored. The other warps move the second plane (block scales, a thirtieth
// of the bytes) and what a token count leaves of 16 bytes. Pairs carry a token count because a
// last page is copied as far as its row has tokens.
__global__ void __launch_bounds__(kCopyThreads)
    pages_copy_kernel(const int* __restrict__ work, const int* __restrict__ copies, int layers, CopyPlane a,
                      CopyPlane b, int pieces, int piece_bytes, int* __restrict__ table, long long entries,
                      const int* __restrict__ page_map, int pages, int* err) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kStages];
  __shared__ int s_err;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    s_err = 0;
    fence_mbarrier_init();
  }
  griddep_wait();
  griddep_launch();
  if (table) remap_table(table, entries, page_map, pages);
  const int rows = *copies * layers;  // (pair, layer)
  if (threadIdx.x >= 32) {
    const int lane = threadIdx.x & 31, per_cta = kCopyThreads / 32 - 1;
    for (int q = blockIdx.x * per_cta + (threadIdx.x >> 5) - 1; q < rows; q += gridDim.x * per_cta) {
      const int c = q / layers, layer = q - c * layers;
      const int src = work[3 * c], dst = work[3 * c + 1], tokens = work[3 * c + 2];
      const int end = tokens * a.token_bytes;
      copy_words(a, layer, src, dst, end & ~15, end, lane, 32);
      if (b.base) copy_words(b, layer, src, dst, 0, tokens * b.token_bytes, lane, 32);
    }
    return;
  }
  if (threadIdx.x != 0) return;
  const int units = rows * pieces;
  const int n = units <= (int)blockIdx.x ? 0 : (units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  char* to[kStages];
  int bytes[kStages];
  bool ok = true;
  int issued = 0;
  for (int i0 = 0; i0 < n + 1 && ok; i0 += kStages) {
#pragma unroll
    for (int st = 0; st < kStages; ++st) {
      const int i = i0 + st;
      if (i < n && ok) {
        // the store that last read this stage: all but the youngest kStages - 2 have been read
        if (i >= kStages) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kStages - 2) : "memory");
        const int u = blockIdx.x + i * gridDim.x;
        const int q = u / pieces, at = (u - q * pieces) * piece_bytes;
        const int c = q / layers, layer = q - c * layers;
        const long long off = layer * a.layer_stride + at;
        to[st] = a.base + off + (long long)work[3 * c + 1] * a.page_bytes;
        bytes[st] = max(0, min(piece_bytes, (work[3 * c + 2] * a.token_bytes & ~15) - at));
        mbar_arrive_expect_tx(&full[st], bytes[st]);
        if (bytes[st])
          bulk_load(ring + st * kStageBytes, a.base + off + (long long)work[3 * c] * a.page_bytes, bytes[st], &full[st]);
        issued = i + 1;
      }
      constexpr int kPrev = kStages - 1;
      const int j = i - 1, ps = (st + kPrev) % kStages;
      if (j >= 0 && j < n && ok) {
        ok = mbar_wait(&full[ps], (j / kStages) & 1, &s_err, err, kErrWaitTimeoutProducer);
        if (ok && bytes[ps]) bulk_store(to[ps], ring + ps * kStageBytes, bytes[ps]);
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    }
  }
  // after a wait that gave up: loads in flight land before the CTA gives up its memory
  for (int j = max(0, issued - kStages); j < issued && !ok; ++j) mbar_drain(&full[j % kStages], (j / kStages) & 1);
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// Planes whose pages are not 16-byte aligned: a CTA per (pair, layer).
__global__ void __launch_bounds__(kCopyThreads)
    pages_copy_words_kernel(const int* __restrict__ work, const int* __restrict__ copies, int layers, CopyPlane a,
                            CopyPlane b, int* __restrict__ table, long long entries, const int* __restrict__ page_map,
                            int pages) {
  griddep_wait();
  griddep_launch();
  if (table) remap_table(table, entries, page_map, pages);
  const int rows = *copies * layers;
  for (int q = blockIdx.x; q < rows; q += gridDim.x) {
    const int c = q / layers, layer = q - c * layers;
    const int src = work[3 * c], dst = work[3 * c + 1], tokens = work[3 * c + 2];
    copy_words(a, layer, src, dst, 0, tokens * a.token_bytes, threadIdx.x, kCopyThreads);
    if (b.base) copy_words(b, layer, src, dst, 0, tokens * b.token_bytes, threadIdx.x, kCopyThreads);
  }
}

// Pieces of a first plane's page, about equal ones: a 73,728-byte page in four of a whole stage. A
// plane whose pages are not all 16-byte aligned is copied by words, a page at a time.
static int page_pieces(const PagePlane& p, int block_size) {
  const int page_bytes = p.token_bytes * block_size;
  const bool wide = ((reinterpret_cast<uintptr_t>(p.base) | (uintptr_t)p.layer_stride | (uintptr_t)page_bytes) & 15) == 0;
  return wide ? (page_bytes + kStageBytes - 1) / kStageBytes : 0;
}

bool pages_copy_fits(const PagePlane& a, int layers, int block_size, long long max_copies) {
  return max_copies * layers * std::max(1, page_pieces(a, block_size)) < (1ll << 30);
}

void pages_copy(const PagePlane& a, const PagePlane& b, int layers, int block_size, const int* work, const int* copies,
                long long max_copies, int* table, long long entries, const int* page_map, int pages, int* err,
                int num_sms, cudaStream_t s) {
  auto plane = [&](const PagePlane& p) {
    return CopyPlane{static_cast<char*>(p.base), p.layer_stride, p.token_bytes * block_size, p.token_bytes};
  };
  const CopyPlane ca = plane(a), cb = plane(b);
  const int wide = page_pieces(a, block_size), pieces = std::max(1, wide);
  const int piece_bytes = ((ca.page_bytes + pieces - 1) / pieces + 15) / 16 * 16;
  const long long units = max_copies * layers * pieces;
  const long long want = std::max(units, table ? (entries + kCopyThreads - 1) / kCopyThreads : 0ll);
  if (want <= 0) return;
  if (wide) {
    set_smem_bytes(pages_copy_kernel, kStages * kStageBytes);
    launch_k(pages_copy_kernel, dim3((unsigned)std::min<long long>(want, (long long)kCopyCtas * num_sms)),
             dim3(kCopyThreads), kStages * kStageBytes, s, work, copies, layers, ca, cb, pieces, piece_bytes, table,
             entries, page_map, pages, err);
  } else {
    launch_k(pages_copy_words_kernel, dim3((unsigned)std::min<long long>(want, 8ll * num_sms)), dim3(kCopyThreads), 0,
             s, work, copies, layers, ca, cb, table, entries, page_map, pages);
  }
}

}  // namespace sp
