// pages.cuh -- page management of a K/V cache whose tables live in device memory.
//
// The reference keeps one dense [layer][position][dim] cache per decoder (ane/stories/infer.go:
// 113-114) and has nothing of this kind.  Sequences that start from a common prompt (samples,
// beams, users of one system prompt) hold the prompt's pages in common: refs[p] counts the
// block-table entries that name page p, and a page is free when its count is 0.
//
//   fork     child rows share the parent's complete pages (refs + 1); a partly filled last page
//            is copied, so a page with room left always has one owner and appending never writes
//            into a shared page
//   free     refs - 1 for every entry of the rows; pages that reach 0 are pushed on the free
//            stack in ascending order (the order does not depend on which CTA came first)
//   compact  the L live pages move to ids 0..L-1: the k-th live page at or above L goes to the
//            k-th dead page below L, the fewest moves there are; tables follow
//   copy     listed pages, every layer
//
// Every table is an int32 array on the device, so parents chosen by a kernel (beam search) need
// no host round trip and a step can be captured in a CUDA graph.  What cannot be served writes
// `status`: a fork with any bad request changes nothing; copy, free and compact skip the entries
// that are out of range and do the rest.
#pragma once
#include "common.cuh"

namespace llm {

// Status words of page requests, beside DeviceError's.
enum PageError : int {
  kPageExhausted = 3,   // the free stack holds fewer pages than the request needs
  kPageBadRequest = 4,  // a slot, length or page out of range, or a slot listed twice
};

struct PageTables {
  uint8_t* pool;           // [layers][n_pages][block_bytes]
  int* n_free;
  int* status;
  int* npages;             // [max_seqs]
  int* refs;               // [n_pages]
  int* free_pages;         // [n_pages] stack
  int* table;              // [max_seqs][max_pages]
  int* work;               // PageWork::words() ints, zero between calls except the lists
  int n_layers, n_pages, max_seqs, max_pages;
  int block_bytes;         // n_kv_heads * 2 * 16 * head_dim * 2: one page of one layer
};

// Layout of the work area.  ticket, marks and bits are zero between calls.
struct PageWork {
  enum { kTicket = 0, kValid = 1, kCount = 2, kLive = 3, kMoves = 4, kHeader = 16 };
  static __host__ __device__ size_t marks() { return kHeader; }                                  // [max_seqs]
  static __host__ __device__ size_t first(int seqs) { return marks() + seqs; }                   // [max_seqs]
  static __host__ __device__ size_t bits(int seqs) { return first(seqs) + seqs; }                // [n_pages / 32]
  static __host__ __device__ size_t src(int seqs, int pages) { return bits(seqs) + (pages + 31) / 32; }  // [n_pages]
  static __host__ __device__ size_t dst(int seqs, int pages) { return src(seqs, pages) + pages; }        // [n_pages]
  static __host__ __device__ size_t words(int seqs, int pages) { return dst(seqs, pages) + pages; }
};

constexpr int kPlanThreads = 1024;
constexpr int kFreeThreads = 256;
constexpr int kCopyThreads = 256;
constexpr int kCopyChunk = 4096;  // bytes of a chunk: 16 per thread; a block of any geometry is whole chunks
constexpr int kCopyBatch = 4;     // chunks a CTA has in flight

__device__ __forceinline__ void page_fail(int* status, int code) { atomicCAS(status, 0, code); }

// Exclusive prefix sum over the CTA's values (at most 1024); `total` is their sum.  `s` holds 33 ints.
__device__ __forceinline__ int block_exclusive(int v, int* s, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // s is free again
  if (lane == 31) s[warp] = x;
  __syncthreads();
  if (warp == 0) {
    const int w = lane < static_cast<int>(blockDim.x >> 5) ? s[lane] : 0;
    int y = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) y += z;
    }
    s[lane] = y - w;
    if (lane == 31) s[32] = y;
  }
  __syncthreads();
  total = s[32];
  return s[warp] + x - v;
}

// Copies page src[i] -> dst[i] in every layer, i < n, over the CTAs of the grid.  Moving a page is
// its bytes read and written once, so what counts is bytes in flight in an order that memory likes: a
// CTA takes `turns` runs of kCopyBatch consecutive chunks (16 KB), every load of a run before its
// first store, and the hardware hands out CTAs in order.  Chunks run over (move, layer, offset in the
// block).  2048 pages of 4 x 64 KiB: 167 us (6430 GB/s, 0.98 of a plain copy); CTAs that stay and stride over
// the list 171 to 202 us depending on the stride, bulk copies through shared memory 169 to 222 us.
__device__ __forceinline__ void copy_pages(const uint8_t* from, int from_pages, uint8_t* to, int to_pages, int n_layers,
                                           int block_bytes, const int* src, const int* dst, int n, int turns, int* status) {
  const unsigned chunks = block_bytes / kCopyChunk;
  const long long all = static_cast<long long>(n) * n_layers * chunks;
  for (int turn = 0; turn < turns; ++turn) {
    const long long w = (static_cast<long long>(blockIdx.x) * turns + turn) * kCopyBatch;
    if (w >= all) break;
    const long long blk = w / chunks;
    unsigned chunk = static_cast<unsigned>(w - blk * chunks);
    int i = static_cast<int>(blk / n_layers), layer = static_cast<int>(blk - static_cast<long long>(i) * n_layers);
    uint4 v[kCopyBatch];
    uint8_t* out[kCopyBatch];
#pragma unroll
    for (int u = 0; u < kCopyBatch; ++u) {
      out[u] = nullptr;
      if (w + u < all) {
        const int a = src[i], b = dst[i];
        if (a < 0 || a >= from_pages || b < 0 || b >= to_pages) {
          if (threadIdx.x == 0) page_fail(status, kPageBadRequest);
        } else {
          const size_t at = static_cast<size_t>(chunk) * kCopyChunk + threadIdx.x * 16;
          v[u] = __ldcs(reinterpret_cast<const uint4*>(from + (static_cast<size_t>(layer) * from_pages + a) * block_bytes + at));
          out[u] = to + (static_cast<size_t>(layer) * to_pages + b) * block_bytes + at;
        }
        if (++chunk == chunks) {
          chunk = 0;
          if (++layer == n_layers) layer = 0, ++i;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kCopyBatch; ++u)
      if (out[u]) __stcs(reinterpret_cast<uint4*>(out[u]), v[u]);
  }
}

__global__ void __launch_bounds__(kCopyThreads, 5) pages_copy_kernel(PageTables from, PageTables to, const int* src,
                                                                     const int* dst, int n) {
  copy_pages(from.pool, from.n_pages, to.pool, to.n_pages, from.n_layers, from.block_bytes, src, dst, n, 1, from.status);
}

// ----------------------------------------------------------------------------- fork
struct ForkParams {
  PageTables t;
  const int *parents, *children, *lens, *rooms;
  int n;
};
struct ForkShape {
  int keep, fresh;
  bool grow, tail;
};
// What request i asks for; false when it asks for something that is not there.
__device__ __forceinline__ bool fork_shape(const ForkParams& p, int i, ForkShape& f) {
  const int par = p.parents[i], child = p.children[i], len = p.lens[i], room = p.rooms[i];
  f = {0, 0, par == child, false};
  if (child < 0 || child >= p.t.max_seqs || par < -1 || par >= p.t.max_seqs || room < 0) return false;
  if (room > p.t.max_pages * 16) return false;
  if (f.grow) {
    f.keep = p.t.npages[child];
  } else {
    if (p.t.npages[child] != 0 || len < 0 || len > room) return false;
    if (len > (par < 0 ? 0 : p.t.npages[par] * 16)) return false;
    f.keep = len >> 4;
    f.tail = (len & 15) != 0;
  }
  f.fresh = max(0, (room + 15) / 16 - f.keep);
  return true;
}

// One CTA: checks every request, numbers the new pages (a prefix sum in request order) and takes them
// off the stack.  Bound by latency: three dependent reads and two scans per 1024 requests, 5 us.
// The second launch then copies and fills rows on every SM: 64 beams into 512, 252 MB, 41 us in all
// (a copy's rate would be 38.5; the parents' last pages come from L2 for seven of eight children).
__global__ void __launch_bounds__(kPlanThreads) pages_fork_plan_kernel(ForkParams p) {
  __shared__ int s_scan[33];
  __shared__ int s_bad;
  griddep_launch_dependents();
  griddep_wait();
  int* const work = p.t.work;
  int* const mark = work + PageWork::marks();
  int* const first = work + PageWork::first(p.t.max_seqs);
  int* const src = work + PageWork::src(p.t.max_seqs, p.t.n_pages);
  int* const dst = work + PageWork::dst(p.t.max_seqs, p.t.n_pages);
  const int have = min(*p.t.n_free, p.t.n_pages);
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  int base = 0, moves = 0;
  for (int i0 = 0; i0 < p.n; i0 += kPlanThreads) {
    const int i = i0 + threadIdx.x;
    ForkShape f{0, 0, false, false};
    if (i < p.n) {
      if (!fork_shape(p, i, f)) s_bad = 1;
      else if (atomicExch(mark + p.children[i], 1) != 0) s_bad = 1;
    }
    int total;
    const int off = block_exclusive(f.fresh, s_scan, total);
    if (i < p.n) first[i] = base + off;
    // the copies of partly filled pages; a request that needs one takes a new page, so the list
    // is no longer than the pool when the request is served
    int tails;
    const int at = moves + block_exclusive(f.tail ? 1 : 0, s_scan, tails);
    if (f.tail && base + off < have && at < p.t.n_pages) {
      src[at] = p.t.table[static_cast<size_t>(p.parents[i]) * p.t.max_pages + f.keep];
      dst[at] = p.t.free_pages[have - 1 - base - off];
    }
    moves += tails;
    base += total;
    if (base > p.t.n_pages) break;  // more than the pool has: refused below; also keeps the sum small
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.n; i += kPlanThreads) {
    const int c = p.children[i];
    if (c >= 0 && c < p.t.max_seqs) mark[c] = 0;
  }
  if (threadIdx.x == 0) {
    const bool bad = s_bad != 0, out = base > have;
    if (bad) page_fail(p.t.status, kPageBadRequest);
    else if (out) page_fail(p.t.status, kPageExhausted);
    work[PageWork::kValid] = !bad && !out;
    work[PageWork::kCount] = have;
    work[PageWork::kMoves] = moves;
    if (!bad && !out) *p.t.n_free = have - base;
  }
}

// Rows and reference counts of a checked request, by the first CTAs of the grid, and the pages per
// slot by the last of `waits` CTAs to arrive (0: of those that fill rows): the others still read them.
// *s_last tells the CTA whether it was the last.
__device__ __forceinline__ void fork_rows(const ForkParams& p, const int* first, int top, int* s_last, int waits = 0) {
  const int rows = min(static_cast<int>(min(gridDim.x, 0x7fffffffu)), p.n);
  if (threadIdx.x == 0) *s_last = 0;
  if (waits == 0 && static_cast<int>(blockIdx.x) >= rows) {
    __syncthreads();
    return;
  }
  for (int i = blockIdx.x; i < p.n; i += gridDim.x) {
    ForkShape f;
    fork_shape(p, i, f);
    const int par = p.parents[i];
    int* row = p.t.table + static_cast<size_t>(p.children[i]) * p.t.max_pages;
    const int* old = p.t.table + static_cast<size_t>(par < 0 ? 0 : par) * p.t.max_pages;
    for (int j = threadIdx.x; j < f.keep + f.fresh; j += kCopyThreads) {
      if (j < f.keep) {
        if (f.grow) continue;
        const int e = old[j];
        row[j] = e;
        if (e >= 0 && e < p.t.n_pages) atomicAdd(p.t.refs + e, 1);
        else page_fail(p.t.status, kDevBadPage);
      } else {
        const int e = p.t.free_pages[top - 1 - first[i] - (j - f.keep)];
        row[j] = e;
        if (e >= 0 && e < p.t.n_pages) p.t.refs[e] = 1;
        else page_fail(p.t.status, kDevBadPage);
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    *s_last = atomicAdd(p.t.work + PageWork::kTicket, 1) == (waits ? waits : rows) - 1;
  }
  __syncthreads();
  if (!*s_last) return;
  __threadfence();
  for (int i = threadIdx.x; i < p.n; i += kCopyThreads) {
    const int par = p.parents[i], child = p.children[i];
    const int keep = par == child ? p.t.npages[child] : p.lens[i] >> 4;
    p.t.npages[child] = max(keep, (p.rooms[i] + 15) / 16);
  }
}

// Rows, reference counts and the copies of partly filled pages.  The rows are read while npages
// still holds the old counts; the last CTA stores the new ones.
__global__ void __launch_bounds__(kCopyThreads, 5) pages_fork_kernel(ForkParams p) {
  __shared__ int s_last;
  griddep_wait();
  int* const work = p.t.work;
  if (!work[PageWork::kValid]) return;
  const int* first = work + PageWork::first(p.t.max_seqs);
  const int top = work[PageWork::kCount];  // the stack before this call
  copy_pages(p.t.pool, p.t.n_pages, p.t.pool, p.t.n_pages, p.t.n_layers, p.t.block_bytes,
             work + PageWork::src(p.t.max_seqs, p.t.n_pages), work + PageWork::dst(p.t.max_seqs, p.t.n_pages),
             work[PageWork::kMoves], 1, p.t.status);
  fork_rows(p, first, top, &s_last);
  if (s_last) work[PageWork::kTicket] = 0;
}

// The same in one launch for at most kCopyThreads requests: every CTA checks and numbers the requests
// itself (they are few, and a second launch costs more than a CTA's 2 us), so nothing that the
// checks read may change before the last CTA is done with them.
__global__ void __launch_bounds__(kCopyThreads, 5) pages_fork_small_kernel(ForkParams p) {
  __shared__ int s_scan[33], s_first[kCopyThreads], s_child[kCopyThreads], s_src[kCopyThreads], s_dst[kCopyThreads];
  __shared__ int s_last, s_bad;
  const int i = threadIdx.x;
  const int have = min(*p.t.n_free, p.t.n_pages);
  ForkShape f{0, 0, false, false};
  bool bad = i < p.n && !fork_shape(p, i, f);
  s_child[i] = i < p.n ? p.children[i] : -1 - i;
  if (i == 0) s_bad = 0;
  __syncthreads();
  for (int k = 0; k < i && i < p.n; ++k) bad = bad || s_child[k] == s_child[i];
  if (bad) s_bad = 1;
  int total, moves;
  const int off = block_exclusive(bad ? 0 : f.fresh, s_scan, total);
  const int at = block_exclusive(!bad && f.tail ? 1 : 0, s_scan, moves);
  s_first[i] = off;
  if (!bad && f.tail && off < have) {
    s_src[at] = p.t.table[static_cast<size_t>(p.parents[i]) * p.t.max_pages + f.keep];
    s_dst[at] = p.t.free_pages[have - 1 - off];
  }
  __syncthreads();
  if (s_bad || total > have) {  // alike in every CTA
    if (i == 0 && blockIdx.x == 0) page_fail(p.t.status, s_bad ? kPageBadRequest : kPageExhausted);
    return;
  }
  copy_pages(p.t.pool, p.t.n_pages, p.t.pool, p.t.n_pages, p.t.n_layers, p.t.block_bytes, s_src, s_dst, moves, 1, p.t.status);
  fork_rows(p, s_first, have, &s_last, gridDim.x);
  if (s_last && i == 0) {
    *p.t.n_free = have - total;
    p.t.work[PageWork::kTicket] = 0;
  }
}

// ----------------------------------------------------------------------------- free
// One CTA a slot (an SM takes several), atomics on the counts, and the last CTA's scan of the bit mask of
// emptied pages, which fixes their order on the stack.  Bound by latency: the count, the row, the
// atomics, the ticket and the scan one after another, 4 us for one slot, 8 us for 512 slots of 138
// pages at most (1024-thread CTAs on one wave of SMs took 12).
__global__ void __launch_bounds__(kFreeThreads) pages_free_kernel(PageTables t, const int* slots, int n) {
  __shared__ int s_scan[33];
  __shared__ int s_held, s_last;
  int* const work = t.work;
  unsigned* const bits = reinterpret_cast<unsigned*>(work + PageWork::bits(t.max_seqs));
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int slot = slots[i];
    if (slot < 0 || slot >= t.max_seqs) {
      if (threadIdx.x == 0) page_fail(t.status, kPageBadRequest);
      continue;
    }
    // taking the count frees the slot once, however often it is listed
    if (threadIdx.x == 0) s_held = min(atomicExch(t.npages + slot, 0), t.max_pages);
    __syncthreads();
    int* row = t.table + static_cast<size_t>(slot) * t.max_pages;
    for (int j = threadIdx.x; j < s_held; j += kFreeThreads) {
      const int e = row[j];
      row[j] = -1;
      if (e < 0 || e >= t.n_pages) {
        page_fail(t.status, kDevBadPage);
        continue;
      }
      const int was = atomicSub(t.refs + e, 1);
      if (was == 1) {
        atomicOr(bits + (e >> 5), 1u << (e & 31));
      } else if (was <= 0) {  // not counted: put it back, the page is not ours to push
        atomicAdd(t.refs + e, 1);
        page_fail(t.status, kDevBadPage);
      }
    }
    __syncthreads();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(work + PageWork::kTicket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  // the emptied pages in ascending order on the stack: each thread a run of words
  const int words = (t.n_pages + 31) / 32;
  const int per = (words + kFreeThreads - 1) / kFreeThreads;
  const int w0 = min(words, static_cast<int>(threadIdx.x) * per), w1 = min(words, w0 + per);
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(__ldcg(bits + w));
  int total;
  const int base = min(max(*t.n_free, 0), t.n_pages);
  int at = base + block_exclusive(mine, s_scan, total);
  for (int w = w0; w < w1; ++w) {
    unsigned b = __ldcg(bits + w);
    if (b == 0) continue;
    bits[w] = 0;
    for (; b != 0; b &= b - 1) {
      if (at < t.n_pages) t.free_pages[at] = w * 32 + __ffs(b) - 1;
      ++at;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (base + total > t.n_pages) page_fail(t.status, kDevBadPage);  // the stack did not match refs
    *t.n_free = min(base + total, t.n_pages);
    work[PageWork::kTicket] = 0;
  }
}

// ----------------------------------------------------------------------------- compact
// Block-table entries of moved pages renamed (src is ascending), and the new free stack.
__device__ __forceinline__ void compact_tables(const PageTables& t, const int* src, const int* dst, int moves, int n_live) {
  const long long tid = static_cast<long long>(blockIdx.x) * kCopyThreads + threadIdx.x;
  const long long step = static_cast<long long>(gridDim.x) * kCopyThreads;
  const long long entries = static_cast<long long>(t.max_seqs) * t.max_pages;
  for (long long k = tid; k < entries; k += step) {
    const int e = t.table[k];
    if (e < n_live) continue;
    int lo = 0, hi = moves;  // the rank of e among the sources
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (src[mid] < e) lo = mid + 1;
      else hi = mid;
    }
    if (lo < moves && src[lo] == e) t.table[k] = dst[lo];
    else page_fail(t.status, kDevBadPage);  // an entry whose page has no references
  }
  for (long long k = tid; k < t.n_pages - n_live; k += step) t.free_pages[k] = static_cast<int>(t.n_pages - 1 - k);
}

// Listing takes 8 us for 8192 pages (two scans of the last CTA), moving goes at the copy's rate: 2000
// moves of 4 x 64 KiB, 1.07 GB, 177 us in all against 164.
// Live pages as a bit mask; the last CTA lists the moves and the new name of every moved page.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(PageTables t) {
  __shared__ int s_scan[33];
  __shared__ int s_last;
  griddep_launch_dependents();
  int* const work = t.work;
  unsigned* const bits = reinterpret_cast<unsigned*>(work + PageWork::bits(t.max_seqs));
  const int words = (t.n_pages + 31) / 32;
  const int p = blockIdx.x * kPlanThreads + threadIdx.x;
  const unsigned live = __ballot_sync(0xffffffffu, p < t.n_pages && t.refs[p] > 0);
  if ((threadIdx.x & 31) == 0 && (p >> 5) < words) bits[p >> 5] = live;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(work + PageWork::kTicket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const int per = (words + kPlanThreads - 1) / kPlanThreads;
  const int w0 = min(words, static_cast<int>(threadIdx.x) * per), w1 = min(words, w0 + per);
  int mine = 0, n_live;
  for (int w = w0; w < w1; ++w) mine += __popc(__ldcg(bits + w));
  block_exclusive(mine, s_scan, n_live);
  // bits of word w that are live at or above n_live / dead below it
  auto above = [&](int w) -> unsigned {
    const int lo = n_live - w * 32;  // ids below n_live in this word
    const unsigned keep = lo <= 0 ? 0xffffffffu : (lo >= 32 ? 0u : 0xffffffffu << lo);
    return __ldcg(bits + w) & keep;
  };
  auto holes = [&](int w) -> unsigned {
    const int lo = n_live - w * 32;
    const unsigned below = lo <= 0 ? 0u : (lo >= 32 ? 0xffffffffu : ~(0xffffffffu << lo));
    return ~__ldcg(bits + w) & below;
  };
  int n_src = 0, n_dst = 0, moves, same;
  for (int w = w0; w < w1; ++w) {
    n_src += __popc(above(w));
    n_dst += __popc(holes(w));
  }
  int a = block_exclusive(n_src, s_scan, moves);
  int b = block_exclusive(n_dst, s_scan, same);
  int* src = work + PageWork::src(t.max_seqs, t.n_pages);
  int* dst = work + PageWork::dst(t.max_seqs, t.n_pages);
  for (int w = w0; w < w1; ++w) {
    for (unsigned m = above(w); m != 0; m &= m - 1) src[a++] = w * 32 + __ffs(m) - 1;
    for (unsigned m = holes(w); m != 0; m &= m - 1) dst[b++] = w * 32 + __ffs(m) - 1;
  }
  __syncthreads();
  for (int w = w0; w < w1; ++w) bits[w] = 0;
  if (threadIdx.x == 0) {
    work[PageWork::kMoves] = moves;
    work[PageWork::kLive] = n_live;
    work[PageWork::kTicket] = 0;
    *t.n_free = t.n_pages - n_live;
  }
}

// The same as the two kernels above and below in one launch, for pools of at most kSmallPool pages:
// every CTA lists the moves itself, and the counts, which they all read, change when the last is done.
constexpr int kSmallPool = 2048;
__global__ void __launch_bounds__(kCopyThreads, 4) pages_compact_small_kernel(PageTables t, int turns) {
  __shared__ int s_scan[33], s_src[kSmallPool / 2 + 1], s_dst[kSmallPool / 2 + 1];
  __shared__ unsigned s_bits[kSmallPool / 32];
  __shared__ int s_last;
  constexpr int PER = kSmallPool / kCopyThreads;
  const int words = (t.n_pages + 31) / 32;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int q = k * kCopyThreads + threadIdx.x;
    const unsigned live = __ballot_sync(0xffffffffu, q < t.n_pages && t.refs[q] > 0);
    if ((threadIdx.x & 31) == 0) s_bits[q >> 5] = live;
  }
  __syncthreads();
  const int w = threadIdx.x;
  const unsigned mine = w < words ? s_bits[w] : 0u;
  int n_live, moves, same;
  block_exclusive(__popc(mine), s_scan, n_live);
  const int lo = n_live - w * 32;  // ids below n_live in this word
  const unsigned below = lo <= 0 ? 0u : (lo >= 32 ? 0xffffffffu : ~(0xffffffffu << lo));
  unsigned above = mine & ~below, holes = w < words ? ~mine & below : 0u;
  int a = block_exclusive(__popc(above), s_scan, moves);
  int b = block_exclusive(__popc(holes), s_scan, same);
  for (; above != 0; above &= above - 1) s_src[a++] = w * 32 + __ffs(above) - 1;
  for (; holes != 0; holes &= holes - 1) s_dst[b++] = w * 32 + __ffs(holes) - 1;
  __syncthreads();
  compact_tables(t, s_src, s_dst, moves, n_live);
  copy_pages(t.pool, t.n_pages, t.pool, t.n_pages, t.n_layers, t.block_bytes, s_src, s_dst, moves, turns, t.status);
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    s_last = atomicAdd(t.work + PageWork::kTicket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  for (int k = threadIdx.x; k < moves; k += kCopyThreads) {
    t.refs[s_dst[k]] = t.refs[s_src[k]];
    t.refs[s_src[k]] = 0;
  }
  if (threadIdx.x == 0) {
    *t.n_free = t.n_pages - n_live;
    t.work[PageWork::kTicket] = 0;
  }
}

// The moves (sources are at or above n_live, destinations below it, so they never overlap), the
// renamed counts and table entries, and the free stack.
__global__ void __launch_bounds__(kCopyThreads, 4) pages_compact_kernel(PageTables t, int turns) {
  griddep_wait();
  const int* work = t.work;
  const int moves = work[PageWork::kMoves], n_live = work[PageWork::kLive];
  const int* src = work + PageWork::src(t.max_seqs, t.n_pages);
  const int* dst = work + PageWork::dst(t.max_seqs, t.n_pages);
  compact_tables(t, src, dst, moves, n_live);
  for (int k = blockIdx.x * kCopyThreads + threadIdx.x; k < moves; k += gridDim.x * kCopyThreads) {
    t.refs[dst[k]] = t.refs[src[k]];
    t.refs[src[k]] = 0;
  }
  copy_pages(t.pool, t.n_pages, t.pool, t.n_pages, t.n_layers, t.block_bytes, src, dst, moves, turns, t.status);
}

}  // namespace llm
