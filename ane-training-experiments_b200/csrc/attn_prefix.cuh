// attn_prefix.cuh -- attention of a batch whose sequences share long prefixes in a paged cache.
//
// Row r of sequence s stands at position t_r = ctx_s - rows_s + r and sees positions 0..t_r:
//   o = sum_t 2^(c q.k_t - m) v_t / l,  l = sum_t 2^(c q.k_t - m),  c = scale * log2(e)
// with any m; m, l and the sum form a state that joins with another set of positions' state as
//   M = max(m, m'), l = 2^(m-M) l + 2^(m'-M) l', o = 2^(m-M) o + 2^(m'-M) o'.
// A row that sees nothing (ctx 0, or a row before position 0) gives o = 0 and lse = -inf.
#pragma once
#include "common.cuh"
#include "pages.cuh"

namespace llm {

struct PrefixParams {
  const void* q;
  void* out;
  float* lse;                 // [rows][n_heads] natural log, or nullptr
  long long q_row, q_head;    // strides in elements
  long long o_row, o_head;
  const uint8_t* pool;        // the layer's pages
  const int* table;
  const int* ctx;             // [n_seqs]
  const int* slots;           // [n_seqs]
  const int* row_start;       // [n_seqs + 1]
  const int* row_seq;         // [n_rows]
  int* status;
  int n_seqs, n_rows, n_heads, n_kv_heads, n_pages, max_pages, max_ctx;
  float scale_log2;
};

// Positions sequence s has, at most what its table row and the plan cover.
__device__ __forceinline__ int seq_ctx(const PrefixParams& p, int s) {
  const int c = p.ctx[s], most = min(p.max_ctx, p.max_pages * 16);
  if (c > most) page_fail(p.status, kPageBadRequest);
  return max(0, min(c, most));
}

// One warp per (row, head): a position at a time, lanes over the head's dimensions.
template <typename T, int HD>
__global__ void __launch_bounds__(128) prefix_rows_kernel(PrefixParams p) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (unit >= static_cast<long long>(p.n_rows) * p.n_heads) return;
  const int row = static_cast<int>(unit / p.n_heads), head = static_cast<int>(unit % p.n_heads);
  const int kvh = head / (p.n_heads / p.n_kv_heads);
  const int s = p.row_seq[row];
  const int ctx = seq_ctx(p, s);
  const int last = ctx - (p.row_start[s + 1] - row);
  const int* bt = p.table + static_cast<size_t>(p.slots[s]) * p.max_pages;
  const T* q = static_cast<const T*>(p.q) + row * p.q_row + head * p.q_head;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = ActTraits<T>::to_f(q[lane * E + e]) * p.scale_log2;
    o[e] = 0.f;
  }
  const T* block = nullptr;
  for (int t = 0; t <= last; ++t) {
    if ((t & 15) == 0) {
      int page = bt[t >> 4];
      if (page < 0 || page >= p.n_pages) {
        page_fail(p.status, kDevBadPage);
        page = 0;
      }
      block = reinterpret_cast<const T*>(p.pool) + (static_cast<size_t>(page) * p.n_kv_heads + kvh) * (2 * 16 * HD);
    }
    const int at = kv_off(t & 15, lane * E / 8) / 2 + (lane * E) % 8;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x += qv[e] * ActTraits<T>::to_f(block[at + e]);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
    const float mn = fmaxf(m, x), mu = mn == -INFINITY ? 0.f : mn;
    const float a = exp2_det_lo(m - mu), w = exp2_det_lo(x - mu);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * ActTraits<T>::to_f(block[16 * HD + at + e]);
    m = mn;
  }
  T* out = static_cast<T*>(p.out) + row * p.o_row + head * p.o_head;
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = ActTraits<T>::from_f(l > 0.f ? o[e] / l : 0.f);
  if (p.lse && lane == 0) p.lse[static_cast<size_t>(row) * p.n_heads + head] = l > 0.f ? (m + log2f(l)) * 0.69314718056f : -INFINITY;
}

}  // namespace llm
