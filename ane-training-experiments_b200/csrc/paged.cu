// paged.cu -- C entries of the caller-owned paged caches: argument checks, plans and launches of
// the page requests (pages.cuh) and of the attention over shared prefixes (attn_prefix.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <functional>
#include <initializer_list>
#include <new>
#include <vector>

#include "../../include/llm_cuda.h"
#include "attn_prefix.cuh"
#include "paged.h"
#include "pages.cuh"

using namespace llm;

// Sets the thread's last error (defined in llm_cuda.cu) and returns `code`.
int llm_detail_fail(int code, const char* msg);

namespace {

int fail_fmt(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return llm_detail_fail(code, buf);
}

#define CU(call)                                                                                       \
  do {                                                                                                 \
    cudaError_t e_ = (call);                                                                           \
    if (e_ != cudaSuccess) return fail_fmt(LLM_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_)); \
  } while (0)
#define RC(call)                   \
  do {                             \
    int rc_ = (call);              \
    if (rc_ != LLM_OK) return rc_; \
  } while (0)

// Makes `device` current for the scope of a call.
class DeviceScope {
 public:
  int enter(int device) {
    CU(cudaGetDevice(&prev_));
    if (prev_ == device) return LLM_OK;
    const cudaError_t e = cudaSetDevice(device);
    if (e != cudaSuccess) return fail_fmt(LLM_ERR_CUDA, "cudaSetDevice(%d) failed: %s", device, cudaGetErrorString(e));
    changed_ = true;
    return LLM_OK;
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(prev_);
  }

 private:
  int prev_ = 0;
  bool changed_ = false;
};

// Launch that may start while the stream's preceding kernel drains (the kernel waits for it).
template <typename... KArgs, typename... Args>
cudaError_t launch_dependent(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_geometry(const llm_page_cache* c) {
  if (!c) return fail_fmt(LLM_ERR_INVALID, "nil cache");
  if (c->dtype != LLM_DTYPE_F16 && c->dtype != LLM_DTYPE_BF16)
    return fail_fmt(LLM_ERR_INVALID, "cache dtype %d (LLM_DTYPE_F16 or LLM_DTYPE_BF16)", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail_fmt(LLM_ERR_UNSUPPORTED, "head_dim=%d (supported: 64, 128)", c->head_dim);
  if (c->n_layers <= 0 || c->n_pages <= 0 || c->n_kv_heads <= 0 || c->max_seqs <= 0 || c->max_pages <= 0)
    return fail_fmt(LLM_ERR_INVALID, "cache sizes must be positive");
  if (c->n_kv_heads > 1024 || c->n_pages > (1 << 26) || c->max_seqs > (1 << 24) || c->max_pages > (1 << 20))
    return fail_fmt(LLM_ERR_INVALID, "cache sizes out of range");
  if (!c->pool || !aligned(c->pool, 128)) return fail_fmt(LLM_ERR_INVALID, "the pool must be device memory aligned to 128 bytes");
  return LLM_OK;
}

// Device arrays of n int32 arguments: there, and aligned for the kernels' loads.
int check_lists(std::initializer_list<const int32_t*> lists, const char* what) {
  for (const int32_t* p : lists)
    if (!p || !aligned(p, 4)) return fail_fmt(LLM_ERR_INVALID, "nil or misaligned %s", what);
  return LLM_OK;
}

int check_tables(const llm_page_cache* c) {
  RC(check_geometry(c));
  return check_lists({c->n_free, c->status, c->npages, c->refs, c->free_pages, c->table, c->work}, "cache table");
}

PageTables tables(const llm_page_cache* c) {
  PageTables t{};
  t.pool = static_cast<uint8_t*>(c->pool);
  t.n_free = c->n_free;
  t.status = c->status;
  t.npages = c->npages;
  t.refs = c->refs;
  t.free_pages = c->free_pages;
  t.table = c->table;
  t.work = c->work;
  t.n_layers = c->n_layers;
  t.n_pages = c->n_pages;
  t.max_seqs = c->max_seqs;
  t.max_pages = c->max_pages;
  t.block_bytes = c->n_kv_heads * 2 * 16 * c->head_dim * 2;
  return t;
}

// CTAs of a launch that copies up to `moves` pages of every layer (copy_pages); 0: too many to launch.
unsigned copy_grid(const PageTables& t, long long moves, int turns = 1) {
  const long long run = static_cast<long long>(kCopyBatch) * turns;
  const long long ctas = (moves * t.n_layers * (t.block_bytes / kCopyChunk) + run - 1) / run;
  return ctas > 0x7fffffffll ? 0u : static_cast<unsigned>(std::max(1ll, ctas));
}

}  // namespace

extern "C" size_t llm_pages_work_words(int n_pages, int max_seqs) {
  if (n_pages <= 0 || max_seqs <= 0 || n_pages > (1 << 26) || max_seqs > (1 << 24)) return 0;
  return PageWork::words(max_seqs, n_pages);
}

extern "C" int llm_pages_status(int device, const llm_page_cache* c, void* stream) {
  RC(check_tables(c));
  DeviceScope dev;
  RC(dev.enter(device));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int h = 0;
  CU(cudaMemcpyAsync(&h, c->status, sizeof h, cudaMemcpyDeviceToHost, s));
  CU(cudaStreamSynchronize(s));
  if (h == 0) return LLM_OK;
  CU(cudaMemsetAsync(c->status, 0, sizeof h, s));
  CU(cudaStreamSynchronize(s));
  switch (h) {
    case kPageExhausted: return fail_fmt(LLM_ERR_OOM, "KV page pool exhausted");
    case kPageBadRequest: return fail_fmt(LLM_ERR_INVALID, "page request names a slot, page or length out of range, or a slot twice");
  }
  return fail_fmt(LLM_ERR_DEVICE, "kernel reported device error %d (%s)", h, llm_detail_device_error(h));
}

const char* llm_detail_device_error(int code) {
  switch (code) {
    case kDevWaitTimeout: return "bounded wait expired";
    case kDevBadPage: return "bad page index";
    case kPageExhausted: return "KV page pool exhausted";
    case kPageBadRequest: return "slot, page or length out of range";
  }
  return "unknown";
}

extern "C" int llm_pages_copy(int device, const llm_page_cache* from, const llm_page_cache* to, const int32_t* src,
                              const int32_t* dst, int n, void* stream) {
  RC(check_geometry(from));
  RC(check_geometry(to));
  RC(check_lists({from->status}, "cache table"));
  if (from->dtype != to->dtype || from->n_layers != to->n_layers || from->n_kv_heads != to->n_kv_heads ||
      from->head_dim != to->head_dim)
    return fail_fmt(LLM_ERR_INVALID, "the caches have different layers, heads, head_dim or dtype");
  if (n < 0) return fail_fmt(LLM_ERR_INVALID, "negative count");
  if (n == 0) return LLM_OK;
  RC(check_lists({src, dst}, "page list"));
  DeviceScope dev;
  RC(dev.enter(device));
  const PageTables a = tables(from), b = tables(to);
  const unsigned grid = copy_grid(a, n);
  if (!grid) return fail_fmt(LLM_ERR_INVALID, "%d pages in one request", n);
  pages_copy_kernel<<<grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, b, src, dst, n);
  CU(cudaGetLastError());
  return LLM_OK;
}

extern "C" int llm_pages_fork(int device, const llm_page_cache* c, const int32_t* parents, const int32_t* children,
                              const int32_t* lens, const int32_t* rooms, int n, void* stream) {
  RC(check_tables(c));
  if (n < 0 || n > c->max_seqs) return fail_fmt(LLM_ERR_INVALID, "%d requests for %d slots", n, c->max_seqs);
  if (n == 0) return LLM_OK;
  RC(check_lists({parents, children, lens, rooms}, "request array"));
  DeviceScope dev;
  RC(dev.enter(device));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ForkParams p{tables(c), parents, children, lens, rooms, n};
  const unsigned grid = copy_grid(p.t, n);
  if (!grid) return fail_fmt(LLM_ERR_INVALID, "%d requests in one call", n);
  // one launch where few requests copy little (one sequence into four: 6 us on the device against 8,
  // and 3 us less on the host)
  if (n <= kCopyThreads && grid <= 148 * 4) {
    pages_fork_small_kernel<<<grid, kCopyThreads, 0, s>>>(p);
    CU(cudaGetLastError());
    return LLM_OK;
  }
  pages_fork_plan_kernel<<<1, kPlanThreads, 0, s>>>(p);
  CU(cudaGetLastError());
  CU(launch_dependent(pages_fork_kernel, dim3(grid), dim3(kCopyThreads), 0, s, p));
  return LLM_OK;
}

extern "C" int llm_pages_free(int device, const llm_page_cache* c, const int32_t* slots, int n, void* stream) {
  RC(check_tables(c));
  if (n < 0) return fail_fmt(LLM_ERR_INVALID, "negative count");
  if (n == 0) return LLM_OK;
  RC(check_lists({slots}, "slot list"));
  DeviceScope dev;
  RC(dev.enter(device));
  pages_free_kernel<<<std::min(n, 148 * 4), kFreeThreads, 0, static_cast<cudaStream_t>(stream)>>>(tables(c), slots, n);
  CU(cudaGetLastError());
  return LLM_OK;
}

extern "C" int llm_pages_compact(int device, const llm_page_cache* c, void* stream) {
  RC(check_tables(c));
  DeviceScope dev;
  RC(dev.enter(device));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const PageTables t = tables(c);
  const unsigned all = copy_grid(t, t.n_pages / 2 + 1);
  if (!all) return fail_fmt(LLM_ERR_INVALID, "%d pages in one request", t.n_pages);
  const int few = static_cast<int>((all + 148 * 4 - 1) / (148 * 4));
  // one launch of at most four CTAs an SM (96 pages: as long on the device as two, 3 us less on the host)
  if (t.n_pages <= kSmallPool && few <= 8) {
    pages_compact_small_kernel<<<copy_grid(t, t.n_pages / 2 + 1, few), kCopyThreads, 0, s>>>(t, few);
    CU(cudaGetLastError());
    return LLM_OK;
  }
  // the host knows only a bound of the moves (half of the pool): longer CTAs where the bound makes
  // many, as most of them may find nothing to do
  const int turns = all > 148 * 16 ? 4 : 1;
  const unsigned grid = copy_grid(t, t.n_pages / 2 + 1, turns);
  pages_compact_plan_kernel<<<(t.n_pages + kPlanThreads - 1) / kPlanThreads, kPlanThreads, 0, s>>>(t);
  CU(cudaGetLastError());
  CU(launch_dependent(pages_compact_kernel, dim3(grid), dim3(kCopyThreads), 0, s, t, turns));
  return LLM_OK;
}

// ============================================================================ shared prefixes
struct llm_prefix_plan {
  int device = 0, dtype = 0, n_heads = 0, n_kv_heads = 0, head_dim = 0;
  int n_seqs = 0, n_rows = 0, max_ctx = 0, top_slot = -1;
  void* block = nullptr;  // one device allocation: items, row_info, slots, states, sums
  size_t bytes = 0;       // of it
  const PrefixItem* items[2] = {};  // [tile, columns]
  int n_items[2] = {};
  int variant = 0;  // of the tile kernel: kWide, kNarrow, kSingle
  const PrefixJoin* joins = nullptr;
  int n_joins = 0, parts = 0;
  int* tickets = nullptr;  // [n_kv_heads], where the columns' last CTA joins
  const int4* row_info = nullptr;
  float* ws_o = nullptr;
  float2* ws_ml = nullptr;
};

namespace {

enum { kTile = 0, kCols = 1 };
enum { kWide, kNarrow, kSingle };  // two streams with pairs, two without, one
constexpr int kOpenEnd = 1 << 30;
// Cost of starting and ending a CTA, in 64-position steps of its main loop.
constexpr int kItemOverhead = 4;
// (row, head) pairs that a warp of a column CTA joins itself before a launch of its own is faster.
constexpr int kInlineJoins = 4;

struct PlanGroup {
  int seq0, n_seqs, prefix;
  bool shared;
  long long rho;  // score rows per kv head
};

long long tiles_of(long long rho, int rows) { return (rho + rows - 1) / rows; }
int kind_of(long long rho) { return rho > kColRows ? kTile : kCols; }
int kernel_slots(int kind, int head_dim) { return 148 * (kind == kTile ? 1 : head_dim == 64 ? 5 : 3); }

// Positions per item of the shared prefixes: a multiple of 64 that finishes first when every CTA
// slot takes ceil(items / slots) items of that length.
int part_length(const std::vector<PlanGroup>& groups, int kind, int n_kv_heads, int slots, int tile_rows) {
  long long work = 0, longest = 0;
  for (const PlanGroup& g : groups) {
    if (!g.shared || kind_of(g.rho) != kind) continue;
    work += tiles_of(g.rho, tile_rows) * n_kv_heads * ((g.prefix + 63) / 64);
    longest = std::max<long long>(longest, (g.prefix + 63) / 64);
  }
  if (work == 0) return 64;
  const long long shortest = (longest + kMaxParts / 2 - 1) / (kMaxParts / 2);
  long long best = longest, best_cost = -1;
  for (int waves = 1; waves <= 4; ++waves) {
    for (long long c = std::max(shortest, work / (static_cast<long long>(slots) * waves)), end = c + 8; c <= end; ++c) {
      if (c < 1) continue;
      long long items = 0;
      for (const PlanGroup& g : groups)
        if (g.shared && kind_of(g.rho) == kind) items += tiles_of(g.rho, tile_rows) * n_kv_heads * (((g.prefix + 63) / 64 + c - 1) / c);
      const long long cost = ((items + slots - 1) / slots) * (std::min(c, longest) + kItemOverhead);
      if (best_cost < 0 || cost < best_cost) best = c, best_cost = cost;
    }
  }
  return static_cast<int>(std::min(best, longest) * 64);
}

// The items of a batch and the rows with several states (the caller fills in their outer rows).
// Returns the number of states in all; *most is a row's most.
long long plan_items(const int32_t* rows, const int32_t* group_sizes, const int32_t* prefixes, int n_groups, int max_ctx,
                     int group, int n_kv_heads, int head_dim, int tile_rows, std::vector<PrefixItem> (&items)[2],
                     std::vector<PrefixJoin>& joins, int* most) {
  std::vector<PlanGroup> groups;
  std::vector<int> row_start(1, 0);
  long long own_ctas = 0;
  int seq = 0;
  for (int g = 0; g < n_groups; ++g) {
    PlanGroup pg{seq, group_sizes[g], prefixes[g], false, 0};
    int active = 0;
    long long alone = 0;
    for (int i = 0; i < group_sizes[g]; ++i, ++seq) {
      const long long rho = static_cast<long long>(rows[seq]) * group;
      row_start.push_back(row_start.back() + rows[seq]);
      active += rho > 0;
      pg.rho += rho;
      alone += (rho + 127) / 128;
      own_ctas += tiles_of(rho, tile_rows) * n_kv_heads;
    }
    // Sharing pays when stacking the rows leaves fewer 128-row steps over the prefix.  One group of 2 to
    // 10 sequences of 40 to 200 score rows, time shared over not shared (geometric mean, both head
    // sizes): steps of at most 0.7 of the sequences' own 0.88 after 4096 positions (0.62..1.19) and
    // 1.00 after 512; more steps than that 0.99 after either (0.72..1.59), so those stay apart.
    pg.shared = active >= 2 && prefixes[g] > 0 && (pg.rho + 127) / 128 * 10 <= alone * 7;
    groups.push_back(pg);
  }
  // Pieces of the own ranges, when one item a sequence leaves most of the machine idle.  One sequence of
  // 16000 own positions, eight kv heads of 128: 190 us in one piece, 20.5 in pieces; 16 sequences 220
  // and 164.  From 148 CTAs on they stay whole, which costs long ranges: 24 sequences of 16000 take
  // 260 us and would 228 in pieces for 444 CTAs, 16 of them with twelve heads of 64 242 and 146.
  const int pieces = own_ctas >= 148 ? 1 : static_cast<int>(std::min<long long>(16, 296 / std::max(1ll, own_ctas)));
  const int len[2] = {part_length(groups, kTile, n_kv_heads, kernel_slots(kTile, head_dim), tile_rows),
                      part_length(groups, kCols, n_kv_heads, kernel_slots(kCols, head_dim), tile_rows)};
  *most = 0;
  // A group's states lie together: [parts][n_kv_heads][the group's score rows], from `states` on.
  long long states = 0;
  for (const PlanGroup& g : groups) {
    auto add = [&](int row0, long long rho, int pos0, int pos1, int part) {
      const long long at = part < 0 ? -1 : states + part * n_kv_heads * g.rho + (row0 - row_start[g.seq0]) * static_cast<long long>(group);
      for (long long r = tiles_of(rho, tile_rows) - 1; r >= 0; --r)  // later rows see further: longest first
        items[kind_of(rho)].push_back({row0, static_cast<int>(r * tile_rows),
                                       static_cast<int>(std::min<long long>(tile_rows, rho - r * tile_rows)), pos0, pos1,
                                       static_cast<int>(g.rho), at < 0 ? -1 : at + r * tile_rows});
    };
    int shared_parts = 0, group_parts = 0;
    if (g.shared)
      for (int pos = 0, c = len[kind_of(g.rho)]; pos < g.prefix; pos += c, ++shared_parts)
        add(row_start[g.seq0], g.rho, pos, std::min(g.prefix, pos + c), shared_parts);
    const int start = g.shared ? g.prefix : 0;
    const int bound = max_ctx - start;  // most own positions
    const int n = std::max(1, std::min(pieces, bound / 512));
    const int piece = n > 1 ? ((bound + n - 1) / n + 63) / 64 * 64 : kOpenEnd;
    for (int s = g.seq0; s < g.seq0 + g.n_seqs; ++s) {
      const long long rho = static_cast<long long>(rows[s]) * group;
      if (rho == 0) continue;
      int parts = shared_parts;
      if (n == 1) {
        add(row_start[s], rho, start, kOpenEnd, shared_parts > 0 ? parts++ : -1);
      } else {
        for (int pos = start; pos < max_ctx; pos += piece) add(row_start[s], rho, pos, pos + piece, parts++);
      }
      for (int r = 0; parts > 0 && r < rows[s]; ++r)
        joins.push_back({row_start[s] + r, parts, static_cast<int>(g.rho), 0,
                         states + (row_start[s] + r - row_start[g.seq0]) * static_cast<long long>(group)});
      group_parts = std::max(group_parts, parts);
    }
    *most = std::max(*most, group_parts);
    states += group_parts * n_kv_heads * g.rho;
  }
  for (auto& v : items)
    std::stable_sort(v.begin(), v.end(), [max_ctx](const PrefixItem& a, const PrefixItem& b) {
      auto cost = [max_ctx](const PrefixItem& i) { return (std::min(i.pos1, max_ctx) - i.pos0) * (i.n_rho > 128 ? 2ll : 1ll); };
      return cost(a) > cost(b);
    });
  return states;
}

// Time, in clocks, of a batch's tile items in one variant of the kernel: items in list order, each on
// the CTA slot that is free first.  A CTA's clocks a 64-position step and its start and end are
// measured (24 prompts of 51..203 rows after 2048 positions; two CTAs of the single variant share an
// SM's tensor core, so each takes longer): 113 us wide, 100 us single; five groups of 79 rows and
// eight heads on 14960 positions: 67 us wide, 76 us single.  Over 210 batches without a shared prefix (8
// to 64 sequences, 200 to 400 score rows, 256 to 4096 positions) its choice takes 0.91 of the wide
// variant's time, and 1.02 (head_dim 128) or 1.06 (64, whose steps are shorter than these) of the
// single one's.
double tile_clocks(const std::vector<PrefixItem>& items, int n_kv_heads, int max_ctx, int variant) {
  const int slots = variant == kSingle ? 296 : 148;
  std::vector<double> free_at(slots, 0.0);  // a heap, earliest first
  double sum = 0, longest = 0;
  const size_t ctas = items.size() * n_kv_heads;
  for (const PrefixItem& it : items) {
    const double steps = (std::min(it.pos1, max_ctx) - it.pos0 + 63) / 64;
    const double clocks = variant == kSingle ? 9000 + 2280 * steps : it.n_rho > 128 ? 13000 + 1950 * steps : 9000 + 1270 * steps;
    sum += clocks * n_kv_heads;
    longest = std::max(longest, clocks);
    for (int k = 0; ctas <= 4096 && k < n_kv_heads; ++k) {
      std::pop_heap(free_at.begin(), free_at.end(), std::greater<double>());
      free_at.back() += clocks;
      std::push_heap(free_at.begin(), free_at.end(), std::greater<double>());
    }
  }
  return ctas <= 4096 ? *std::max_element(free_at.begin(), free_at.end()) : sum / slots + longest / 2;
}

// TRACE: the kernels that record their timeline (p.trace).  They are instantiations of their own, since
// the test of a null pointer costs a small call 0.1 us of 7 on the device.
template <typename T, int HD, bool TRACE>
cudaError_t prefix_launch(const llm_prefix_plan* plan, PrefixParams p, TraceRec* const* trace, cudaStream_t s, bool prepare) {
  if (prepare) {
    // the whole carve-out for shared memory, so that CTAs of both kernels fit an SM together
    auto set = [](auto kernel, int smem) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                                         cudaSharedmemCarveoutMaxShared);
    };
    cudaError_t e = set(prefix_tile_kernel<T, HD, 2, false, TRACE>, PrefixTileCfg<T, HD, 2, false>::SMEM);
    if (e == cudaSuccess) e = set(prefix_tile_kernel<T, HD, 2, true, TRACE>, PrefixTileCfg<T, HD, 2, true>::SMEM);
    if (e == cudaSuccess) e = set(prefix_tile_kernel<T, HD, 1, false, TRACE>, PrefixTileCfg<T, HD, 1, false>::SMEM);
    if (e == cudaSuccess) e = set(prefix_cols_kernel<T, HD, TRACE>, kColsSmem<T, HD>);
    return e;
  }
  bool first = true;  // the first launch waits for the stream's earlier work as a whole
  cudaError_t e = cudaSuccess;
  if (plan->n_items[kTile] > 0) {
    const int grid = plan->n_items[kTile] * plan->n_kv_heads;
    p.items = plan->items[kTile];
    if constexpr (TRACE) p.trace = *trace++;
    auto launch = [&](auto kernel, int threads, int smem) { kernel<<<grid, threads, smem, s>>>(p); };
    using Wide = PrefixTileCfg<T, HD, 2, true>;
    using Narrow = PrefixTileCfg<T, HD, 2, false>;
    using Single = PrefixTileCfg<T, HD, 1, false>;
    if (plan->variant == kWide) launch(prefix_tile_kernel<T, HD, 2, true, TRACE>, Wide::THREADS, Wide::SMEM);
    else if (plan->variant == kNarrow) launch(prefix_tile_kernel<T, HD, 2, false, TRACE>, Narrow::THREADS, Narrow::SMEM);
    else launch(prefix_tile_kernel<T, HD, 1, false, TRACE>, Single::THREADS, Single::SMEM);
    e = cudaGetLastError();
    first = false;
  }
  if (e == cudaSuccess && plan->n_items[kCols] > 0) {
    constexpr int smem = kColsSmem<T, HD>;
    const dim3 grid(plan->n_items[kCols] * plan->n_kv_heads), block(kAttnWarps * 32);
    p.items = plan->items[kCols];
    if constexpr (TRACE) p.trace = *trace++;
    if (first) {
      prefix_cols_kernel<T, HD, TRACE><<<grid, block, smem, s>>>(p);
      e = cudaGetLastError();
    } else {
      e = launch_dependent(prefix_cols_kernel<T, HD, TRACE>, grid, block, smem, s, p);
    }
  }
  if (e == cudaSuccess && plan->n_joins > 0 && !plan->tickets) {
    if constexpr (TRACE) p.trace = *trace;
    const long long units = static_cast<long long>(plan->n_joins) * plan->n_heads;
    const dim3 grid(static_cast<unsigned>((units + kJoinWarps - 1) / kJoinWarps)), block(kJoinWarps * 32);
    e = plan->parts > 8 ? launch_dependent(prefix_join_kernel<T, HD, 20, TRACE>, grid, block, 0, s, p)
                        : launch_dependent(prefix_join_kernel<T, HD, 8, TRACE>, grid, block, 0, s, p);
  }
  return e;
}

template <bool TRACE>
cudaError_t prefix_any(const llm_prefix_plan* plan, const PrefixParams& p, TraceRec* const* trace, cudaStream_t s, bool prepare) {
  const bool bf = plan->dtype == LLM_DTYPE_BF16;
  if (plan->head_dim == 64)
    return bf ? prefix_launch<__nv_bfloat16, 64, TRACE>(plan, p, trace, s, prepare)
              : prefix_launch<__half, 64, TRACE>(plan, p, trace, s, prepare);
  return bf ? prefix_launch<__nv_bfloat16, 128, TRACE>(plan, p, trace, s, prepare)
            : prefix_launch<__half, 128, TRACE>(plan, p, trace, s, prepare);
}

// What a plan fixes of its launches.
PrefixParams plan_params(const llm_prefix_plan* plan) {
  PrefixParams p{};
  p.row_info = plan->row_info;
  p.joins = plan->joins;
  p.n_joins = plan->n_joins;
  p.tickets = plan->tickets;
  p.ws_o = plan->ws_o;
  p.ws_ml = plan->ws_ml;
  p.n_rows = plan->n_rows;
  p.n_heads = plan->n_heads;
  p.n_kv_heads = plan->n_kv_heads;
  p.max_ctx = plan->max_ctx;
  return p;
}

// Whether two of the vectors of `len` elements at r * row + h * head, r < rows and h < heads, overlap.
bool vectors_overlap(long long rows, long long heads, long long row, long long head, long long len) {
  if ((heads == 1 || head >= len) && (rows == 1 || row >= (heads - 1) * head + len)) return false;  // row by row
  if ((rows == 1 || row >= len) && (heads == 1 || head >= (rows - 1) * row + len)) return false;    // head by head
  if (rows > 1 && row < len) return true;
  for (long long h = 1; h < heads; ++h) {  // the rows whose distance is nearest to that of h heads
    const long long x = h * head, r = row > 0 ? std::min(x / row, rows - 1) : 0;
    if (x - r * row < len || (r + 1 < rows && (r + 1) * row - x < len)) return true;
  }
  return false;
}

float scale_log2(double scale) { return static_cast<float>(scale * 1.4426950408889634); }

}  // namespace

cudaError_t llm_detail_prefix_run(const llm_prefix_plan* plan, const llm_prefix_rows& r, cudaStream_t s) {
  PrefixParams p = plan_params(plan);
  p.q = r.q;
  p.out = r.out;
  p.out_f32 = r.out_f32;
  p.q_row = p.o_row = static_cast<long long>(plan->n_heads) * plan->head_dim;
  p.q_head = p.o_head = plan->head_dim;
  p.pool = static_cast<const uint8_t*>(r.layer_pool);
  p.table = r.table;
  p.ctx = r.positions;
  p.ctx_add = 1;
  p.status = r.status;
  p.n_pages = r.n_pages;
  p.max_pages = r.max_pages;
  p.scale_log2 = scale_log2(1.0 / std::sqrt(static_cast<double>(plan->head_dim)));
  if (!r.trace[0]) return prefix_any<false>(plan, p, nullptr, s, false);
  const cudaError_t e = prefix_any<true>(plan, p, nullptr, s, true);
  return e == cudaSuccess ? prefix_any<true>(plan, p, r.trace, s, false) : e;
}

size_t llm_detail_prefix_bytes(const llm_prefix_plan* plan) { return plan->bytes; }

int llm_detail_prefix_launches(const llm_prefix_plan* plan, const char* (*names)[3]) {
  int n = 0;
  auto add = [&](const char* name) {
    if (names) (*names)[n] = name;
    ++n;
  };
  if (plan->n_items[kTile] > 0) add("attention(tiles)");
  if (plan->n_items[kCols] > 0) add("attention(cols)");
  if (plan->n_joins > 0 && !plan->tickets) add("attention(join)");
  return n;
}

extern "C" int llm_prefix_plan_destroy(llm_prefix_plan* plan) {
  if (!plan) return fail_fmt(LLM_ERR_INVALID, "nil plan");
  DeviceScope dev;
  const int rc = dev.enter(plan->device);
  if (rc == LLM_OK && plan->block) cudaFree(plan->block);
  delete plan;
  return rc;
}

extern "C" int llm_prefix_plan_create(int device, int dtype, int n_heads, int n_kv_heads, int head_dim,
                                      const int32_t* slots, const int32_t* rows, int n_seqs,
                                      const int32_t* group_sizes, const int32_t* prefixes, int n_groups, int max_ctx,
                                      llm_prefix_plan** out) {
  return llm_detail_prefix_create(device, dtype, n_heads, n_kv_heads, head_dim, slots, rows, n_seqs, nullptr, group_sizes,
                                  prefixes, n_groups, max_ctx, out);
}

int llm_detail_prefix_create(int device, int dtype, int n_heads, int n_kv_heads, int head_dim, const int* slots,
                             const int* rows, int n_seqs, const int* order, const int* group_sizes, const int* prefixes,
                             int n_groups, int max_ctx, llm_prefix_plan** out) {
  if (!out) return fail_fmt(LLM_ERR_INVALID, "nil output handle");
  *out = nullptr;
  if (dtype != LLM_DTYPE_F16 && dtype != LLM_DTYPE_BF16)
    return fail_fmt(LLM_ERR_INVALID, "dtype %d (LLM_DTYPE_F16 or LLM_DTYPE_BF16)", dtype);
  if (head_dim != 64 && head_dim != 128) return fail_fmt(LLM_ERR_UNSUPPORTED, "head_dim=%d (supported: 64, 128)", head_dim);
  if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads != 0 || n_heads > 1024)
    return fail_fmt(LLM_ERR_INVALID, "n_heads=%d must be a multiple of n_kv_heads=%d", n_heads, n_kv_heads);
  if (n_seqs <= 0 || n_groups <= 0 || max_ctx <= 0 || max_ctx > (1 << 28))
    return fail_fmt(LLM_ERR_INVALID, "sequences, groups and max_ctx must be positive");
  if (!slots || !rows || !group_sizes || !prefixes) return fail_fmt(LLM_ERR_INVALID, "nil plan array");
  long long seqs = 0, total = 0;
  for (int g = 0; g < n_groups; ++g) {
    if (group_sizes[g] <= 0) return fail_fmt(LLM_ERR_INVALID, "group %d has %d sequences", g, group_sizes[g]);
    if (prefixes[g] < 0 || prefixes[g] % 16 != 0 || prefixes[g] > max_ctx)
      return fail_fmt(LLM_ERR_INVALID, "prefix %d of group %d is not a multiple of 16 within max_ctx=%d", prefixes[g], g, max_ctx);
    seqs += group_sizes[g];
  }
  if (seqs != n_seqs) return fail_fmt(LLM_ERR_INVALID, "groups of %lld sequences in all, not %d", seqs, n_seqs);
  int top = -1;
  for (int s = 0; s < n_seqs; ++s) {
    if (slots[s] < 0) return fail_fmt(LLM_ERR_INVALID, "sequence %d out of range", slots[s]);
    if (rows[s] < 0) return fail_fmt(LLM_ERR_INVALID, "sequence %d has %d rows", s, rows[s]);
    top = std::max(top, slots[s]);
    total += rows[s];
  }
  if (total > (1 << 20)) return fail_fmt(LLM_ERR_INVALID, "%lld query rows", total);
  llm_prefix_plan* p = nullptr;
  try {
    const int group = n_heads / n_kv_heads;
    std::vector<PrefixItem> items[2];
    std::vector<PrefixJoin> joins;
    // rows in plan order: sequence by sequence as listed
    std::vector<int> listed(n_seqs), start(1, 0);
    for (int s = 0; s < n_seqs; ++s) start.push_back(start.back() + rows[s]);
    std::vector<int4> info;
    info.reserve(total);
    for (int i = 0; i < n_seqs; ++i) {
      const int s = order ? order[i] : i;
      listed[i] = rows[s];
      for (int r = 0; r < rows[s]; ++r) info.push_back(make_int4(s, rows[s] - r, slots[s], start[s] + r));
    }
    int parts = 0;
    // Rows in pairs of 128-row tiles read each K/V tile once for both; single tiles spread better and
    // start and end beside one another.  Without pairs, one stream a CTA once the CTAs are more than
    // one and a half to an SM.  Two streams over one stream, without a shared prefix (144 batches of 8 to
    // 64 sequences, 60 and 120 score rows): 1.08 of its time up to 148 CTAs, 1.22 up to 222, 1.17 to 1.28
    // above; on long shared prefixes two streams are the faster: 64 rows on 32768 positions 41.2 us
    // against 43.5, eight families of 32 101 against 102.
    long long n_states = 0;
    int variant = kNarrow;
    for (int v : {kWide, kSingle}) {
      std::vector<PrefixItem> it[2];
      std::vector<PrefixJoin> jo;
      int most = 0;
      const long long st = plan_items(listed.data(), group_sizes, prefixes, n_groups, max_ctx, group, n_kv_heads, head_dim,
                                      v == kWide ? 256 : 128, it, jo, &most);
      const bool pairs = std::any_of(it[kTile].begin(), it[kTile].end(), [](const PrefixItem& i) { return i.n_rho > 128; });
      if (v == kSingle && variant == kWide &&
          tile_clocks(items[kTile], n_kv_heads, max_ctx, kWide) <= tile_clocks(it[kTile], n_kv_heads, max_ctx, kSingle))
        break;
      if (v == kSingle && variant != kWide) break;
      for (int k = 0; k < 2; ++k) items[k] = std::move(it[k]);
      joins = std::move(jo);
      parts = most;
      n_states = st;
      variant = v == kSingle ? kSingle : pairs ? kWide : items[kTile].size() * n_kv_heads > 222 ? kSingle : kNarrow;
    }
    for (PrefixJoin& j : joins) j.outer = info[j.row].w;
    DeviceScope dev;
    RC(dev.enter(device));
    p = new llm_prefix_plan;
    p->device = device;
    p->dtype = dtype;
    p->n_heads = n_heads;
    p->n_kv_heads = n_kv_heads;
    p->head_dim = head_dim;
    p->n_seqs = n_seqs;
    p->n_rows = static_cast<int>(total);
    p->max_ctx = max_ctx;
    p->top_slot = top;
    // the device block: host-built arrays first, then the workspace
    std::vector<uint8_t> host;
    auto place = [&host](const void* src, size_t bytes) -> size_t {
      const size_t at = (host.size() + 255) / 256 * 256;
      host.resize(at + bytes);
      if (bytes) memcpy(host.data() + at, src, bytes);
      return at;
    };
    size_t at_items[2];
    for (int k = 0; k < 2; ++k) {
      p->n_items[k] = static_cast<int>(items[k].size());
      at_items[k] = place(items[k].data(), items[k].size() * sizeof(PrefixItem));
    }
    p->variant = variant;
    p->n_joins = static_cast<int>(joins.size());
    p->parts = parts;
    const size_t at_joins = place(joins.data(), joins.size() * sizeof(PrefixJoin));
    const size_t at_info = place(info.data(), info.size() * sizeof(int4));
    // Few rows of column items only: the last CTA of a kv head joins them, at most kInlineJoins
    // (row, head) pairs a warp.  Four samples: 13.4 us a call, which the host bounds, against 17.8
    // with a join launch; on the device alone 7.4 us against 5.8 (a fence and a ticket).
    const std::vector<int> zeros(n_kv_heads, 0);
    const bool join_inline = items[kTile].empty() && joins.size() * group <= static_cast<size_t>(kInlineJoins * kAttnWarps);
    const size_t at_tickets = place(zeros.data(), join_inline ? zeros.size() * 4 : 0);
    const size_t states = static_cast<size_t>(n_states);
    const size_t at_ml = (host.size() + 255) / 256 * 256, at_o = (at_ml + states * 8 + 255) / 256 * 256;
    const size_t bytes = at_o + states * head_dim * 4;
    cudaError_t e = cudaMalloc(&p->block, bytes);
    if (e != cudaSuccess) {
      p->block = nullptr;
      cudaGetLastError();
      llm_prefix_plan_destroy(p);
      return fail_fmt(LLM_ERR_OOM, "cudaMalloc(%zu) failed: %s", bytes, cudaGetErrorString(e));
    }
    // A copy from pageable memory may return with its last bytes still on the way, and the first call
    // may come on a stream that is not ordered with the null stream: wait for them here.
    p->bytes = bytes;
    e = cudaMemcpy(p->block, host.data(), host.size(), cudaMemcpyHostToDevice);
    if (e == cudaSuccess) e = cudaStreamSynchronize(cudaStreamLegacy);
    if (e == cudaSuccess) e = prefix_any<false>(p, PrefixParams{}, nullptr, nullptr, true);
    if (e != cudaSuccess) {
      llm_prefix_plan_destroy(p);
      return fail_fmt(LLM_ERR_CUDA, "plan set-up failed: %s", cudaGetErrorString(e));
    }
    uint8_t* base = static_cast<uint8_t*>(p->block);
    for (int k = 0; k < 2; ++k) p->items[k] = reinterpret_cast<const PrefixItem*>(base + at_items[k]);
    p->joins = reinterpret_cast<const PrefixJoin*>(base + at_joins);
    if (join_inline && p->n_joins > 0) p->tickets = reinterpret_cast<int*>(base + at_tickets);
    p->row_info = reinterpret_cast<const int4*>(base + at_info);
    p->ws_ml = reinterpret_cast<float2*>(base + at_ml);
    p->ws_o = reinterpret_cast<float*>(base + at_o);
    *out = p;
    return LLM_OK;
  } catch (const std::bad_alloc&) {
    if (p) llm_prefix_plan_destroy(p);
    return fail_fmt(LLM_ERR_OOM, "host memory exhausted");
  }
}

extern "C" int llm_prefix_attend(llm_prefix_plan* plan, const llm_page_cache* c, int layer, const int32_t* ctx,
                                 const void* q, int64_t q_row, int64_t q_head, float scale, void* out, int64_t o_row,
                                 int64_t o_head, float* lse, void* stream) {
  if (!plan) return fail_fmt(LLM_ERR_INVALID, "nil plan");
  RC(check_geometry(c));
  RC(check_lists({c->table, c->status}, "cache table"));
  if (c->dtype != plan->dtype || c->n_kv_heads != plan->n_kv_heads || c->head_dim != plan->head_dim)
    return fail_fmt(LLM_ERR_INVALID, "the cache's dtype, heads or head_dim are not the plan's");
  if (plan->top_slot >= c->max_seqs) return fail_fmt(LLM_ERR_INVALID, "sequence %d out of range", plan->top_slot);
  if (layer < 0 || layer >= c->n_layers) return fail_fmt(LLM_ERR_INVALID, "layer %d out of range", layer);
  if (plan->n_rows == 0) return LLM_OK;
  if (!ctx || !q || !out) return fail_fmt(LLM_ERR_INVALID, "nil buffer");
  if (!aligned(ctx, 4) || !aligned(q, 16) || !aligned(out, 16) || !aligned(lse, 4))
    return fail_fmt(LLM_ERR_INVALID, "misaligned buffer (q and out need 16-byte, ctx and lse 4-byte alignment)");
  if (plan->n_rows == 1) q_row = o_row = 0;  // no address is formed with these strides
  if (plan->n_heads == 1) q_head = o_head = 0;
  for (int64_t s : {q_row, q_head, o_row, o_head})
    if (s % 8 != 0 || s < 0 || s > (int64_t{1} << 40))
      return fail_fmt(LLM_ERR_INVALID, "stride %lld (a multiple of 8 elements is needed)", static_cast<long long>(s));
  if (vectors_overlap(plan->n_rows, plan->n_heads, o_row, o_head, plan->head_dim))
    return fail_fmt(LLM_ERR_INVALID, "rows or heads of out overlap (strides %lld and %lld)", static_cast<long long>(o_row),
                    static_cast<long long>(o_head));
  if (!std::isfinite(scale)) return fail_fmt(LLM_ERR_INVALID, "scale is not finite");
  DeviceScope dev;
  RC(dev.enter(plan->device));
  PrefixParams p = plan_params(plan);
  p.q = q;
  p.out = out;
  p.lse = lse;
  p.q_row = q_row;
  p.q_head = q_head;
  p.o_row = o_row;
  p.o_head = o_head;
  p.pool = static_cast<const uint8_t*>(c->pool) +
           static_cast<size_t>(layer) * c->n_pages * c->n_kv_heads * (2 * 16 * 2) * c->head_dim;
  p.table = c->table;
  p.ctx = ctx;
  p.status = c->status;
  p.n_pages = c->n_pages;
  p.max_pages = c->max_pages;
  p.scale_log2 = scale_log2(scale > 0.f ? static_cast<double>(scale) : 1.0 / std::sqrt(static_cast<double>(plan->head_dim)));
  CU(prefix_any<false>(plan, p, nullptr, static_cast<cudaStream_t>(stream), false));
  return LLM_OK;
}
