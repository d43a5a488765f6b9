// attn_prefix.cuh -- attention of a batch whose sequences share long prefixes in a paged cache.
//
// Row r of sequence s stands at position t_r = ctx_s - rows_s + r and sees positions 0..t_r:
//   o = sum_t 2^(c q.k_t - m) v_t / l,  l = sum_t 2^(c q.k_t - m),  c = scale * log2(e)
// with any m; m, l and the sum form a state that joins with another set of positions' state as
//   M = max(m, m'), l = 2^(m-M) l + 2^(m'-M) l', o = 2^(m-M) o + 2^(m'-M) o'.
// A row that sees nothing (ctx 0, a row before position 0, or every score -inf) has l = 0 and gives
// o = 0 and lse = -inf.  A NaN score, or one of +inf (whose weight is inf - inf), makes l NaN: l is
// tested against 0 only, so that such a row leaves as NaN from every kernel.
//
// The plan cuts the work into items, each a run of score rows (query row, head of the kv head's
// group) against a run of positions of one block-table row, for every kv head: the shared
// positions of a group with all of the group's rows stacked, so that a shared page is read once
// per 256 score rows, each sequence's own positions, and pieces of long ranges.  An item that
// covers all positions of its rows writes the output; the others leave the state of each row in
// the workspace, and prefix_join_kernel joins a row's states.
// Two kernels take the items: prefix_tile_kernel up to 256 score rows on the tcgen05 tensor cores,
// prefix_cols_kernel up to 8 on warp-level MMAs (eight columns cost it nothing, and several of its
// CTAs fit an SM).  The launches run beside one another (programmatic dependent launch); the join
// waits for all of them.
#pragma once
#include "attention.cuh"
#include "common.cuh"
#include "pages.cuh"
#include "umma.cuh"

namespace llm {

struct PrefixItem {
  int row0;        // query row of score row 0's first head
  int rho0;        // score rows rho0 .. rho0 + n_rho - 1 counted from row0's first head
  int n_rho;
  int pos0, pos1;  // positions [pos0, pos1), cut at the last one a row of the item sees
  int span;        // states between one kv head's and the next
  long long state; // of score row 0 and kv head 0 in the workspace; -1: the item writes the output
};

// A query row with several states: of head h of kv head k's group, `parts` of them, from
// state + k * span + h on, span * n_kv_heads apart.
struct PrefixJoin {
  int row, parts, span, outer;  // outer: the row of out and lse
  long long state;
};

struct PrefixParams {
  const PrefixItem* items;
  const void* q;
  void* out;                  // T, or f32 when out_f32
  int out_f32;
  float* lse;                 // [rows][n_heads] natural log, or nullptr
  long long q_row, q_head;    // strides in elements
  long long o_row, o_head;
  const uint8_t* pool;        // the layer's pages
  const int* table;
  const int* ctx;             // [n_seqs] positions, less ctx_add
  int ctx_add;
  const int4* row_info;       // [n_rows] sequence, its rows from this one on, its slot, the row of q, out and lse
  const PrefixJoin* joins;    // [n_joins]
  int n_joins;
  int* tickets;               // [n_kv_heads], zero between calls: the columns' last CTA of a kv head joins; or nullptr
  float* ws_o;                // [states][HD] unnormalised sums
  float2* ws_ml;              // [states] (m in log2 units, l)
  int* status;
  int n_rows, n_heads, n_kv_heads, n_pages, max_pages, max_ctx;
  float scale_log2;
  TraceRec* trace;            // llm_trace_step; read by the TRACE instantiations only
};

// Positions sequence s has, at most what its table row and the plan cover.
__device__ __forceinline__ int seq_ctx(const PrefixParams& p, int s) {
  const int c = p.ctx[s] + p.ctx_add, most = min(p.max_ctx, p.max_pages * 16);
  if (c > most) page_fail(p.status, kPageBadRequest);
  return max(0, min(c, most));
}
// Last position that a query row sees (negative: none).
__device__ __forceinline__ int row_last(const PrefixParams& p, const int4& info) { return seq_ctx(p, info.x) - info.y; }
__device__ __forceinline__ int page_entry(const PrefixParams& p, const int* bt, int lp) {
  int e = bt[lp];
  if (e < 0 || e >= p.n_pages) {
    page_fail(p.status, kDevBadPage);
    e = 0;
  }
  return e;
}
__device__ __forceinline__ float natural_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// One warp joins the states of (row, head) and writes the output.  Lane k weighs states k and k + 32
// (kMaxParts is 64); then a lane adds its HD / 32 dimensions of BATCH states at a time: 8, or 20 where
// rows have more (18 states of 64 rows: 2.5 us after the last item against 4; but 128 registers at
// head_dim 128 against 63, which costs 4 us where 4096 rows and heads have four states each).
constexpr int kMaxParts = 64;

template <typename T, int HD, int BATCH>
__device__ __forceinline__ void join_states(const PrefixParams& p, const PrefixJoin& j, int head) {
  constexpr int V = HD / 32;
  const int lane = threadIdx.x & 31;
  const int group = p.n_heads / p.n_kv_heads;
  const int parts = j.parts;
  const size_t step = static_cast<size_t>(p.n_kv_heads) * j.span;
  const size_t at = j.state + static_cast<size_t>(head / group) * j.span + head % group;
  float2 a = make_float2(-INFINITY, 0.f), b = a;
  if (lane < parts) a = __ldcg(p.ws_ml + at + lane * step);
  if (lane + 32 < parts) b = __ldcg(p.ws_ml + at + (lane + 32) * step);
  const float M = warp_max(fmaxf(a.x, b.x));
  const float mu = M == -INFINITY ? 0.f : M;
  const float wa = exp2_det_lo(a.x - mu), wb = exp2_det_lo(b.x - mu);
  float L = a.y * wa + b.y * wb, O[V];
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
#pragma unroll
  for (int e = 0; e < V; ++e) O[e] = 0.f;
  const float* src = p.ws_o + at * HD + lane * V;
  for (int k0 = 0; k0 < parts; k0 += BATCH) {
    float v[BATCH][V], w[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int k = k0 + i;
      w[i] = __shfl_sync(0xffffffffu, k < 32 ? wa : wb, k & 31);
      if (k >= parts) w[i] = 0.f;
      if (w[i] > 0.f) {  // a state without visible positions holds no sums
        if constexpr (V == 4) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(src + k * step * HD));
          v[i][0] = x.x, v[i][1] = x.y, v[i][2] = x.z, v[i][3] = x.w;
        } else {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(src + k * step * HD));
          v[i][0] = x.x, v[i][1] = x.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[i][e] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) O[e] += v[i][e] * w[i];
  }
  const long long to = j.outer * p.o_row + head * p.o_head + lane * V;
  const float inv = L == 0.f ? 0.f : __fdiv_rn(1.0f, L);
#pragma unroll
  for (int e = 0; e < V; e += 2) {
    if (p.out_f32) *reinterpret_cast<float2*>(static_cast<float*>(p.out) + to + e) = make_float2(O[e] * inv, O[e + 1] * inv);
    else *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + to + e) = ActTraits<T>::pack2(O[e] * inv, O[e + 1] * inv);
  }
  if (p.lse && lane == 0) p.lse[static_cast<size_t>(j.outer) * p.n_heads + head] = natural_lse(M, L);
}

// ============================================================================ up to 8 score rows
// The arithmetic of attn_kernel (attention.cuh): S^T[16 positions x 8 columns] = K . Q^T, online
// softmax per column, O^T += V^T . P^T with P as two terms; warp w takes pages w, w + 4, ... of
// the item's range, and the four warps' states are joined once at the end.  Bound by HBM where the
// own ranges are long: 537 MB of 256 sequences in 88 us (6.1 TB/s, 0.93 of a plain copy).  Two pages of
// 8 KB a warp in flight and three CTAs an SM cover the latency (attn_kernel's measurements).
template <typename T, int HD>
constexpr int kColsSmem = kAttnWarps * AttnCfg<T, HD>::WARP_BYTES;

template <typename T, int HD, bool TRACE>
__global__ void __launch_bounds__(kAttnWarps * 32, HD == 64 ? 5 : 4) prefix_cols_kernel(PrefixParams p) {
  using Cfg = AttnCfg<T, HD>;
  constexpr int STAGES = Cfg::STAGES;
  constexpr int PB = Cfg::PAGE_BYTES;
  constexpr int KS = HD / 16;
  constexpr int ROWB = HD * (int)sizeof(T);
  static_assert(Cfg::FOLD_BYTES <= kColsSmem<T, HD>, "the fold area fits in the ring");

  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kAttnWarps][STAGES];
  __shared__ float s_m[8], s_l[8];
  __shared__ int s_last;

  if constexpr (TRACE) trace_start(p.trace);
  griddep_launch_dependents();
  const PrefixItem it = p.items[blockIdx.x / p.n_kv_heads];
  const int kvh = blockIdx.x % p.n_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int group = p.n_heads / p.n_kv_heads;

  // last visible position of this lane's two score columns; none for columns past the item
  const int c0 = 2 * t, c1 = 2 * t + 1;
  const int4 i0 = p.row_info[it.row0 + (it.rho0 + (c0 < it.n_rho ? c0 : 0)) / group];
  const int4 i1 = p.row_info[it.row0 + (it.rho0 + (c1 < it.n_rho ? c1 : 0)) / group];
  const int4 ig = p.row_info[it.row0 + (it.rho0 + (g < it.n_rho ? g : 0)) / group];
  // Q^T fragments: column g of the B operand is score row rho0 + g
  uint32_t qb[KS][2];
  {
    const bool ok = g < it.n_rho;
    const T* qrow = static_cast<const T*>(p.q) + ig.w * p.q_row + (kvh * group + (it.rho0 + (ok ? g : 0)) % group) * p.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qb[ks][0] = ok ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 2 * t) : 0u;
      qb[ks][1] = ok ? *reinterpret_cast<const uint32_t*>(qrow + ks * 16 + 8 + 2 * t) : 0u;
    }
  }
  const int lim0 = c0 < it.n_rho ? row_last(p, i0) : -1;
  const int lim1 = c1 < it.n_rho ? row_last(p, i1) : -1;
  int slot = lim1 > lim0 ? i1.z : i0.z;
  const int last = __reduce_max_sync(0xffffffffu, max(lim0, lim1));
  // the sequence that sees furthest names the pages (an idle one's row may be empty)
  slot = __shfl_sync(0xffffffffu, slot, __ffs(__ballot_sync(0xffffffffu, max(lim0, lim1) == last)) - 1);
  const int end = min(it.pos1, last + 1);  // positions [it.pos0, end) are read
  const int p_begin = it.pos0 >> 4, p_end = end > it.pos0 ? (end + 15) >> 4 : p_begin;

  uint8_t* wbuf = smem + warp * Cfg::WARP_BYTES;
  float* const fold_area = reinterpret_cast<float*>(smem);  // over the page ring, once it is idle
  float* const slot0 = fold_area;
  float* const slot1 = fold_area + Cfg::SLOT_FLOATS;
  const uint32_t wbase = smem_u32(wbuf);
  const uint32_t bar0 = smem_u32(&bars[warp][0]);
  const int* bt = p.table + static_cast<size_t>(slot) * p.max_pages;
  auto page_src = [&](int lp) -> const uint8_t* {
    return p.pool + (static_cast<size_t>(page_entry(p, bt, lp)) * p.n_kv_heads + kvh) * PB;
  };

  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
    fence_mbar_init();
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      const int lp = p_begin + warp + kAttnWarps * s;
      if (lp < p_end) {
        mbar_arrive_expect_tx(bar0 + 8 * s, PB);
        bulk_g2s(wbase + s * PB, page_src(lp), PB, bar0 + 8 * s);
      }
    }
  }
  __syncwarp();
  WarpState<KS> st;
  st.clear();
  int seen = 0;       // pages this warp has consumed (ring position)
  int fail_at = -1;   // ring position of an expired wait
  for (int lp = p_begin + warp; lp < p_end; lp += kAttnWarps, ++seen) {
    const int s = seen % STAGES;
    if (!mbar_wait_bounded(bar0 + 8 * s, (seen / STAGES) & 1)) {
      if (lane == 0) page_fail(p.status, kDevWaitTimeout);
      fail_at = seen;
      break;
    }
    const uint32_t kb = wbase + s * PB;
    const uint32_t vb = kb + 16 * ROWB;
    const int tok_base = lp * 16;
    if (tok_base + 16 > end) {
      // zero V rows past the range so 0-weight x stale data can never produce NaN
      uint8_t* vblk = wbuf + s * PB + 16 * ROWB;
      for (int i = lane; i < 16 * HD / 8; i += 32) {
        const int rr = i / (HD / 8), c = i % (HD / 8);
        if (tok_base + rr >= end) *reinterpret_cast<uint4*>(vblk + kv_off(rr, c)) = make_uint4(0, 0, 0, 0);
      }
      __syncwarp();
    }
    float sacc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint32_t a[4];
      const int row = (lane & 7) + 8 * ((lane >> 3) & 1);
      ldmatrix_x4(a, kb + kv_off(row, 2 * ks + (lane >> 4)));
      mma_16816(sacc, a, qb[ks][0], qb[ks][1], T());
    }
    const int tk0 = tok_base + g, tk1 = tk0 + 8;
    const int e0 = min(lim0, end - 1), e1 = min(lim1, end - 1);
    const float s0 = tk0 <= e0 ? sacc[0] * p.scale_log2 : -INFINITY;
    const float s1 = tk0 <= e1 ? sacc[1] * p.scale_log2 : -INFINITY;
    const float s2 = tk1 <= e0 ? sacc[2] * p.scale_log2 : -INFINITY;
    const float s3 = tk1 <= e1 ? sacc[3] * p.scale_log2 : -INFINITY;
    float pm0 = fmaxf(s0, s2), pm1 = fmaxf(s1, s3);
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
      pm0 = fmaxf(pm0, __shfl_xor_sync(0xffffffffu, pm0, off));
      pm1 = fmaxf(pm1, __shfl_xor_sync(0xffffffffu, pm1, off));
    }
    const float mn0 = fmaxf(st.m0, pm0), mn1 = fmaxf(st.m1, pm1);
    const float2 mu = make_float2(mn0 == -INFINITY ? 0.f : mn0, mn1 == -INFINITY ? 0.f : mn1);
    const float2 al = exp2_det_lo2(sub2_rn(make_float2(st.m0, st.m1), mu));
    const float2 p01 = exp2_det_lo2<true>(sub2_rn(make_float2(s0, s1), mu));
    const float2 p23 = exp2_det_lo2<true>(sub2_rn(make_float2(s2, s3), mu));
    st.l0 = st.l0 * al.x + (p01.x + p23.x);
    st.l1 = st.l1 * al.y + (p01.y + p23.y);
    st.m0 = mn0;
    st.m1 = mn1;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      st.o[i][0] *= al.x;
      st.o[i][1] *= al.y;
      st.o[i][2] *= al.x;
      st.o[i][3] *= al.y;
    }
    // P^T fragments of column g, positions (2t, 2t+1) and (2t+8, 2t+9), as hi + lo terms of the
    // cache's type: one term would add its 2^-9 (bf16) to every weight; the pages take longer to
    // arrive than the second term's MMAs
    const uint32_t ph01 = ActTraits<T>::pack2(p01.x, p01.y), ph23 = ActTraits<T>::pack2(p23.x, p23.y);
    const float2 h01 = ActTraits<T>::unpack2(ph01), h23 = ActTraits<T>::unpack2(ph23);
    const uint32_t pl01 = ActTraits<T>::pack2(p01.x - h01.x, p01.y - h01.y);
    const uint32_t pl23 = ActTraits<T>::pack2(p23.x - h23.x, p23.y - h23.y);
    const int srcA = 8 * t + (g >> 1), srcB = srcA + 4;
    const int sh = (g & 1) ? 16 : 0;
    auto gather = [&](uint32_t v01, uint32_t v23, uint32_t& b0, uint32_t& b1) {
      const uint32_t xa01 = __shfl_sync(0xffffffffu, v01, srcA), xa23 = __shfl_sync(0xffffffffu, v23, srcA);
      const uint32_t xb01 = __shfl_sync(0xffffffffu, v01, srcB), xb23 = __shfl_sync(0xffffffffu, v23, srcB);
      b0 = ((xa01 >> sh) & 0xffffu) | (((xb01 >> sh) & 0xffffu) << 16);
      b1 = ((xa23 >> sh) & 0xffffu) | (((xb23 >> sh) & 0xffffu) << 16);
    };
    uint32_t bh0, bh1, bl0, bl1;
    gather(ph01, ph23, bh0, bh1);
    gather(pl01, pl23, bl0, bl1);
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      uint32_t a[4];
      const int row = (lane & 7) + 8 * (lane >> 4);
      ldmatrix_x4_trans(a, vb + kv_off(row, 2 * mt + ((lane >> 3) & 1)));
      mma_16816(st.o[mt], a, bh0, bh1, T());
      mma_16816(st.o[mt], a, bl0, bl1, T());
    }
    __syncwarp();
    if (lane == 0) {
      const int nlp = lp + kAttnWarps * STAGES;
      if (nlp < p_end) {
        fence_proxy_async_smem();
        mbar_arrive_expect_tx(bar0 + 8 * s, PB);
        bulk_g2s(kb, page_src(nlp), PB, bar0 + 8 * s);
      }
    }
  }
  if (fail_at >= 0) {
    st.clear();  // an expired wait contributes nothing (the status is set)
    for (int j = fail_at + 1; j < fail_at + STAGES; ++j) {  // copies still in flight (bounded)
      if (p_begin + warp + kAttnWarps * j >= p_end) break;
      mbar_wait_bounded(bar0 + 8 * (j % STAGES), (j / STAGES) & 1);
    }
  }
#pragma unroll
  for (int off = 4; off < 32; off <<= 1) {
    st.l0 += __shfl_xor_sync(0xffffffffu, st.l0, off);
    st.l1 += __shfl_xor_sync(0xffffffffu, st.l1, off);
  }
  // (w0 + w1) + (w2 + w3), then the columns as rows [8][HD] in the fold area
  __syncthreads();
  if (warp == 1) store_slot(slot0, st, lane);
  if (warp == 3) store_slot(slot1, st, lane);
  __syncthreads();
  if (warp == 0) fold_from_slot(st, slot0, lane);
  if (warp == 2) {
    fold_from_slot(st, slot1, lane);
    store_slot(slot1, st, lane);  // each lane rewrites only the values it read
  }
  __syncthreads();
  if (warp == 0) fold_from_slot(st, slot1, lane);
  __syncthreads();
  float* const stage = fold_area;
  if (warp == 0) {
#pragma unroll
    for (int mt = 0; mt < KS; ++mt) {
      const int d = mt * 16 + g;
      stage[c0 * HD + d] = st.o[mt][0];
      stage[c1 * HD + d] = st.o[mt][1];
      stage[c0 * HD + d + 8] = st.o[mt][2];
      stage[c1 * HD + d + 8] = st.o[mt][3];
    }
    if (g == 0) {
      s_m[c0] = st.m0;
      s_m[c1] = st.m1;
      s_l[c0] = st.l0;
      s_l[c1] = st.l1;
    }
  }
  __syncthreads();
  if (it.state >= 0) {
    const size_t at = it.state + static_cast<size_t>(kvh) * it.span;
    for (int i = threadIdx.x; i < it.n_rho * HD / 4; i += kAttnWarps * 32)
      __stcg(reinterpret_cast<float4*>(p.ws_o + at * HD) + i, reinterpret_cast<const float4*>(stage)[i]);
    if (threadIdx.x < it.n_rho) __stcg(p.ws_ml + at + threadIdx.x, make_float2(s_m[threadIdx.x], s_l[threadIdx.x]));
  } else {
    for (int i = threadIdx.x; i < it.n_rho * (HD / 2); i += kAttnWarps * 32) {
      const int c = i / (HD / 2), d = 2 * (i % (HD / 2));
      const int row = p.row_info[it.row0 + (it.rho0 + c) / group].w, head = kvh * group + (it.rho0 + c) % group;
      const float l = s_l[c], inv = l == 0.f ? 0.f : __fdiv_rn(1.0f, l);
      const float x = stage[c * HD + d] * inv, y = stage[c * HD + d + 1] * inv;
      const long long at = row * p.o_row + head * p.o_head + d;
      if (p.out_f32) *reinterpret_cast<float2*>(static_cast<float*>(p.out) + at) = make_float2(x, y);
      else *reinterpret_cast<uint32_t*>(static_cast<T*>(p.out) + at) = ActTraits<T>::pack2(x, y);
      if (p.lse && d == 0) p.lse[static_cast<size_t>(row) * p.n_heads + head] = natural_lse(s_m[c], l);
    }
  }
  if (p.tickets) {  // small batches: no join launch; which CTA comes last does not change a sum's order
    const int units = p.n_joins * group;
    PrefixJoin j = p.joins[min(warp, units - 1) / group];  // the warp's first pair, fetched before it is known to be needed
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      const int n = gridDim.x / p.n_kv_heads;
      s_last = atomicAdd(p.tickets + kvh, 1) == n - 1;
      if (s_last) p.tickets[kvh] = 0;
    }
    __syncthreads();
    if (s_last) {
      __threadfence();
      for (int u = warp; u < units; u += kAttnWarps) {
        if (u != warp) j = p.joins[u / group];
        join_states<T, HD, 8>(p, j, kvh * group + u % group);
      }
    }
    if constexpr (TRACE) trace_end(p.trace);
    return;
  }
  // the launch ends after the one before it, so that whoever waits for it has waited for both; one
  // CTA sees to that, the others make room
  if constexpr (TRACE) trace_end(p.trace);
  if (blockIdx.x == gridDim.x - 1) griddep_wait();
}

// ============================================================================ up to 256 score rows
// One CTA per SM with two streams, each of 128 TMEM lanes, 256 TMEM columns (two S / P buffers of
// 64 and O) and four softmax warps with one score row per thread.  64 positions at a time a stream
// runs S = Q . K^T, softmax, P back over the S columns as hi + lo terms, O += P . V with P from
// TMEM; the reference max of a row moves only when a tile exceeds it by 2^8 (the pipeline of
// attn_prefill_tc_kernel, whose header explains it).  The two terms of P leave 2^-17 of a weight in bf16
// (2^-22 in fp16), about 2^-18 of a sum: one bf16 output in about 1700 rounds to the neighbour of
// what a sum in f32 rounds to.
//   more than 128 rows  the streams are two row tiles that share every K/V tile.  At the memory's rate
//                       an SM gets 24 bytes a clock, 1300 clocks for the 32 KB of a 64-position tile
//                       of head_dim 128; a row tile takes the tensor core 900 clocks for it (S 384,
//                       bound by re-reading Q from shared memory, P hi and lo 512): 1950 measured
//                       for two.
//   up to 128 rows      the streams take the even and the odd K/V tiles of the same rows, and are
//                       joined at the end.
// Warps 0 and 11 = bulk-copy producers, warps 1 and 2 = the streams' MMA issuers (warp 1 allocates TMEM), warps
// 3..6 stream 0, warps 7..10 stream 1.  Each stream issues PV(u), then S(u + 2) once PV(u) has read the
// P that it overwrites; S(u + 1) is done by then, and the other stream's MMAs fill the tensor core.
// Batches with pairs (WIDE) use the SM's shared memory whole.  Batches without use four stages (six
// at head_dim 64) and at most 128 registers a thread, which leaves room for a CTA of
// prefix_cols_kernel beside it: the sequences' own pages stream while the shared ones are worked on.
// Streams that take alternate tiles use an even number of stages, so that a stage serves one stream
// only: a stream that does not see the fill of a stage's previous tile (the other stream's) could
// ask for the next one while that fill is still under way, and a parity wait two phases behind
// returns at once.
// Batches of many short ranges take one stream a CTA (STREAMS = 1, 128 rows) and two CTAs an SM: what
// they wait for is a CTA's start and end, about 7 us, which then overlap.
// Measured, head_dim 128: 64 rows on 32768 positions (134 MB of K/V) 30 us beside the column CTAs, 24
// bytes a clock an SM between start and end; 24 prompts of 51 to 203 rows after 2048 positions (61.6
// GFLOP, two heads a kv head) 101 us with one stream a CTA, 113 with two.
template <typename T, int HD, int STREAMS, bool WIDE>
struct PrefixTileCfg {
  static constexpr int HALVES = HD / 64;              // 64-element halves of a K / V row
  static constexpr int SUB = 16 * 128;                // one page's half sub-block (bytes)
  static constexpr int REGION = 4 * SUB;              // 64 positions of one half (bytes)
  static constexpr int TILE_BYTES = HALVES * REGION;  // K (or V) of one 64-position tile
  static constexpr int STAGES = STREAMS == 1 ? (HD == 64 ? 5 : 2) : HD == 64 ? (WIDE ? 10 : 6) : (WIDE ? 5 : 4);  // of K and of V
  static constexpr int Q_BYTES = HALVES * 128 * 128;  // 128 rows x HD, K-major halves
  static constexpr int K_RING = (WIDE ? 2 : 1) * Q_BYTES;
  static constexpr int V_RING = K_RING + STAGES * TILE_BYTES;
  static constexpr uint32_t TMEM_COLS = 256 * STREAMS;
  static constexpr int THREADS = STREAMS == 1 ? 256 : 384;
  static constexpr float RESCALE_LOG2 = 8.0f;
  static constexpr int ROW_BYTES = HD * 4;            // of a row's sums, staged over Q and the rings
  static constexpr int META = 128 * STREAMS * (ROW_BYTES + 20);
  static constexpr int USED = V_RING + STAGES * TILE_BYTES;
  static constexpr int BARS = (USED > META ? USED : META);  // the barriers lie behind the rings
  static constexpr int SMEM = BARS + 512;
};
constexpr int kColRows = 8;  // score rows of a column item

__device__ __forceinline__ float ex2_approx(float x) {  // 2 ulp; 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// Bounded wait that polls without suspending the thread.
__device__ __forceinline__ bool mbar_poll(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kMaxWaitPolls; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
// One lane of a converged warp, chosen so that the compiler keeps warp-uniform operands in uniform
// registers (a branch on lane == 0 moved every descriptor across per MMA: 75 clocks each).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// 32 lanes x 16 columns of 32-bit from registers (tmem_st32's half)
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void streams_bar() { asm volatile("bar.sync 1, 256;\n" ::: "memory"); }

template <typename T, int HD, int STREAMS, bool WIDE, bool TRACE>
__global__ void __launch_bounds__(STREAMS == 1 ? 256 : 512, STREAMS == 1 ? 2 : 1)  // both: at most 128 registers
    prefix_tile_kernel(PrefixParams p) {
  using Cfg = PrefixTileCfg<T, HD, STREAMS, WIDE>;
  constexpr int V_WARP = STREAMS == 1 ? 7 : 11;  // fetches V
  constexpr int ST = Cfg::STAGES;
  constexpr int HALVES = Cfg::HALVES;
  constexpr int SUB = Cfg::SUB;
  constexpr int REGION = Cfg::REGION;
  constexpr int ROWB = HD * (int)sizeof(T);

  // no static shared memory: the dynamic block starts on a 1024-byte boundary, as its alignment asks
  extern __shared__ __align__(1024) uint8_t gbase[];
  struct Sync {
    uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], s_full[2][2], p_ready[2][2], pv_done[2], q_ready, drain;
    int2 s_last[8];
    uint32_t s_tmem;
  };
  static_assert(sizeof(Sync) <= 512, "room behind the rings");
  Sync& sync = *reinterpret_cast<Sync*>(gbase + Cfg::BARS);
  auto &k_full = sync.k_full, &k_empty = sync.k_empty, &v_full = sync.v_full, &v_empty = sync.v_empty;
  auto &s_full = sync.s_full, &p_ready = sync.p_ready;
  auto& pv_done = sync.pv_done;
  uint64_t &q_ready = sync.q_ready, &drain = sync.drain;
  auto& s_last = sync.s_last;
  uint32_t& s_tmem = sync.s_tmem;

  if constexpr (TRACE) trace_start(p.trace);
  const uint32_t q_s = smem_u32(gbase);
  const uint32_t k_ring = q_s + Cfg::K_RING;
  const uint32_t v_ring = q_s + Cfg::V_RING;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PrefixItem it = p.items[blockIdx.x / p.n_kv_heads];
  const int kvh = blockIdx.x % p.n_kv_heads;
  const int group = p.n_heads / p.n_kv_heads;
  const bool pair = WIDE && it.n_rho > 128;    // two row tiles
  const bool apart = pair || STREAMS == 1;     // a stream has every K/V tile; otherwise the even or the odd ones
  // warps 3..10: stream, TMEM lane, score row and the last position it sees
  const int sg = STREAMS == 2 && warp >= 7 ? 1 : 0;
  const int tl = (warp & 3) * 32 + lane;
  const int local = pair ? sg * 128 + tl : tl;
  const bool softmax_warp = warp >= 3 && warp < 3 + 4 * STREAMS;
  const bool row_ok = softmax_warp && local < it.n_rho;
  const int rho = it.rho0 + (row_ok ? local : 0);
  const int head = kvh * group + rho % group;
  const int4 info = p.row_info[it.row0 + rho / group];
  const int row = info.w;
  const int lim_row = row_ok ? row_last(p, info) : -1;
  if (softmax_warp) {
    const int m = __reduce_max_sync(0xffffffffu, lim_row);
    const int from = __ffs(__ballot_sync(0xffffffffu, lim_row == m)) - 1;
    if (lane == from) s_last[warp - 3] = make_int2(m, info.z);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(smem_u32(&k_full[s]), 1);
      mbar_init(smem_u32(&k_empty[s]), pair ? 2 : 1);
      mbar_init(smem_u32(&v_full[s]), 1);
      mbar_init(smem_u32(&v_empty[s]), pair ? 2 : 1);
    }
    for (int g = 0; g < 2; ++g) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(smem_u32(&s_full[g][b]), 1);
        mbar_init(smem_u32(&p_ready[g][b]), 128);
      }
      mbar_init(smem_u32(&pv_done[g]), 1);
    }
    mbar_init(smem_u32(&q_ready), 128 * STREAMS);
    mbar_init(smem_u32(&drain), STREAMS);
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem), Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // dependents launch only after every CTA of this grid holds its TMEM columns
  griddep_launch_dependents();

  // the sequence that sees furthest names the pages (an idle one's row may be empty)
  int2 far = s_last[0];
#pragma unroll
  for (int w = 1; w < 4 * STREAMS; ++w)
    if (s_last[w].x > far.x) far = s_last[w];
  const int last = far.x;
  const int end = min(it.pos1, last + 1);  // positions [it.pos0, end) are read
  const int nkv = end > it.pos0 ? (end - it.pos0 + 63) >> 6 : 0;
  const int page0 = it.pos0 >> 4;
  const int n_pages_it = nkv > 0 ? ((end + 15) >> 4) - page0 : 0;
  // steps of each stream; step u of stream g works on K/V tile (apart ? u : 2 u + g)
  const int n0 = apart ? nkv : (nkv + 1) >> 1, n1 = apart ? nkv : nkv >> 1;
  const int ring = apart ? ST : ST & ~1;  // stages in use
  bool failed = false;

  if (warp == 0 || warp == V_WARP) {
    // ------------------------------------------------------------ bulk-copy producers
    // Warp 0 fetches K, warp 11 V (one warp issues a copy each 50 to 80 clocks).  A warp reads the
    // block table 32 pages (8 tiles) per coalesced load, one batch ahead of use, and a lane issues
    // each copy: a page's half sub-block of K, both halves of V at once.
    const bool is_v = warp == V_WARP;
    const uint32_t stages = is_v ? v_ring : k_ring;
    const uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    const int per_page = is_v ? 1 : HALVES, size = is_v ? HALVES * SUB : SUB;
    const int j = lane / per_page, hh = lane % per_page;
    const uint32_t place = is_v ? j * HALVES * SUB : hh * REGION + j * SUB;
    const uint8_t* const src = p.pool + static_cast<size_t>(kvh) * (2 * 16 * ROWB) + (is_v ? 16 * ROWB : hh * SUB);
    const int* bt = p.table + static_cast<size_t>(far.y) * p.max_pages + page0;
    auto entries = [&](int first_page) -> int {
      const int pg = first_page + lane;
      return pg < n_pages_it ? page_entry(p, bt, pg) : 0;
    };
    int ent = entries(0), ent_next = entries(32);
    int st = 0, turn = 0;  // stage, and its uses before this one
    for (int t = 0; t < nkv; ++t) {
      if (t > 0 && (t & 7) == 0) {
        ent = ent_next;
        ent_next = entries(4 * t + 32);
      }
      const int np = min(4, n_pages_it - 4 * t);
      const size_t phys = __shfl_sync(0xffffffffu, ent, ((t & 7) << 2) + (j & 3));
      if (turn > 0 && !__all_sync(0xffffffffu, mbar_poll(smem_u32(&empty[st]), (turn + 1) & 1))) {
        failed = true;
        break;
      }
      const uint32_t bar = smem_u32(&full[st]);
      if (lane == 0) mbar_arrive_expect_tx(bar, np * HALVES * SUB);
      __syncwarp();
      if (j < np) bulk_g2s(stages + st * Cfg::TILE_BYTES + place, src + phys * p.n_kv_heads * (2 * 16 * ROWB), size, bar);
      if (++st == ring) st = 0, ++turn;
    }
    // copies still in flight must land before the CTA's shared memory goes away
    if (lane == 0)
      for (int i = 0; i < ring; ++i) {
        const int uses = turn + (i < st ? 1 : 0);
        if (uses > 0) mbar_poll(smem_u32(&full[i]), (uses - 1) & 1);
      }
  } else if (warp <= STREAMS) {
    // ------------------------------------------------------------ MMA issuer of stream warp - 1
    const int g = warp - 1;
    const int steps = __shfl_sync(0xffffffffu, g ? n1 : n0, 0);
    const uint32_t tbase = __shfl_sync(0xffffffffu, tmem, 0) + g * 256;
    constexpr uint32_t idesc_s = umma_idesc<T>(128, 64);
    constexpr uint32_t idesc_pv = umma_idesc<T>(128, HD) | (1u << 16);  // B (V) MN-major
    const uint64_t qd = sw128_desc(q_s + (pair ? g * Cfg::Q_BYTES : 0));
    const uint64_t kd0 = sw128_desc(k_ring), vd0 = sw128_desc_mn(v_ring, SUB, 1024);
    // stage and parity of the next K and of the next V tile of this stream
    int ks = apart ? 0 : g, kpar = 0, vs = ks, vpar = 0;
    auto advance = [&](int& st, int& par) {
      st += apart ? 1 : 2;
      if (st >= ring) st -= ring, par ^= 1;
    };
    // S of step u into the stream's buffer u & 1, whose P the stream's PV(u - 2) has read
    auto issue_s = [&](int u) -> bool {
      const int s = ks;
      bool ok = u < 2 || mbar_poll(smem_u32(&pv_done[g]), u & 1);
      ok = ok && mbar_poll(smem_u32(&k_full[s]), kpar);
      advance(ks, kpar);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      const uint64_t kd = kd0 + static_cast<uint64_t>(s * (Cfg::TILE_BYTES >> 4));
      const uint32_t d = tbase + (u & 1) * 64;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const int hh = k >> 2, kk = k & 3;
          umma<false>(d, qd + ((hh * 128 * 128 + 32 * kk) >> 4), kd + ((hh * REGION + 32 * kk) >> 4), idesc_s, k > 0 ? 1u : 0u);
        }
        tc_commit(smem_u32(&s_full[g][u & 1]));
        tc_commit(smem_u32(&k_empty[s]));
      }
      __syncwarp();
      return true;
    };
    auto issue_pv = [&](int u) -> bool {
      const int s = vs;
      bool ok = mbar_poll(smem_u32(&v_full[s]), vpar);
      advance(vs, vpar);
      ok = ok && mbar_poll(smem_u32(&p_ready[g][u & 1]), (u >> 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      const uint64_t vd = vd0 + static_cast<uint64_t>(s * (Cfg::TILE_BYTES >> 4));
      const uint32_t pa = tbase + (u & 1) * 64;  // P_hi at +0, P_lo at +32 (16-bit pairs)
      if (elect_one()) {
#pragma unroll
        for (int term = 0; term < 2; ++term) {
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)  // 16 positions per MMA
            umma_ts(tbase + 128, pa + term * 32 + kk * 8, vd + ((kk * HALVES * SUB) >> 4), idesc_pv, (u > 0 || term > 0 || kk > 0) ? 1u : 0u);
        }
        tc_commit(smem_u32(&pv_done[g]));
        tc_commit(smem_u32(&v_empty[s]));
      }
      __syncwarp();
      return true;
    };
    bool ok = __all_sync(0xffffffffu, mbar_poll(smem_u32(&q_ready), 0));
    if (ok && steps > 0) ok = issue_s(0);
    if (ok && steps > 1) ok = issue_s(1);
    for (int u = 0; ok && u < steps; ++u) {
      ok = issue_pv(u);
      if (ok && u + 2 < steps) ok = issue_s(u + 2);
    }
    if (!ok) failed = true;
    // every MMA of this stream has completed before O is read and TMEM is freed
    if (elect_one()) tc_commit(smem_u32(&drain));
    __syncwarp();
    mbar_poll(smem_u32(&drain), 0);
  } else if (softmax_warp) {
    // ------------------------------------------------------------ softmax / epilogue warps
    const int lim = min(lim_row, end - 1);     // last visible position of this row in the range
    const bool busy = __any_sync(0xffffffffu, row_ok);  // some row of this warp is the item's
    const uint32_t trow = tmem + sg * 256 + (static_cast<uint32_t>((warp & 3) * 32) << 16);

    // The warp's 32 Q rows -> shared memory, K-major 128B-swizzled halves; consecutive lanes on the
    // chunks of a row (one row per thread took 5 us).  Of a single tile each stream brings half.
    {
      constexpr int CH = HD / 8, N = CH;  // 16-byte chunks of a row; loads per lane for 32 rows
      const long long off = row * p.q_row + head * p.q_head;
      const unsigned rows_ok = __ballot_sync(0xffffffffu, row_ok);
      const int i0 = apart || sg == 0 ? 0 : N / 2, i1 = apart || sg == 1 ? N : N / 2;
      uint4 v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int rr = (i * 32 + lane) / CH, c = lane % CH;
        const long long o = __shfl_sync(0xffffffffu, off, rr);
        v[i] = make_uint4(0, 0, 0, 0);
        if (i >= i0 && i < i1 && (rows_ok >> rr & 1)) v[i] = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + o)[c];
      }
      uint8_t* dst = gbase + (pair ? sg * Cfg::Q_BYTES : 0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int rr = (warp & 3) * 32 + (i * 32 + lane) / CH, c = lane % CH;
        if (i >= i0 && i < i1)
          *reinterpret_cast<uint4*>(dst + (c >> 3) * 128 * 128 + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) = v[i];
      }
      fence_proxy_async_smem();
    }
    mbar_arrive(smem_u32(&q_ready));

    const float sl2 = p.scale_log2;
    float m_ref = -INFINITY, l_run = 0.f;
    bool ok = true;
    const int steps = sg ? n1 : n0;
    for (int u = 0; u < steps; ++u) {
      const int t = apart ? u : 2 * u + sg;
      // wait results are made warp-uniform: the TMEM accesses below are warp-collective
      if (!__all_sync(0xffffffffu, mbar_poll(smem_u32(&s_full[sg][u & 1]), (u >> 1) & 1))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int kbase = it.pos0 + t * 64;
      // V rows past the range were not loaded (or belong to nobody): zero them so a zero weight
      // times stale data cannot make NaN (only the last tile is ragged; its V copies land first).
      // Both streams of a pair do it, each before its own PV.
      const int valid = end - kbase;
      if (valid < 64) {
        if (!__all_sync(0xffffffffu, mbar_poll(smem_u32(&v_full[t % ring]), (t / ring) & 1))) {
          ok = false;
          break;
        }
        uint8_t* vreg = gbase + Cfg::V_RING + (t % ring) * Cfg::TILE_BYTES;
        for (int idx = tl; idx < (64 - valid) * HALVES * 8; idx += 128) {
          const int rr = valid + idx / (HALVES * 8), rem = idx % (HALVES * 8);
          *reinterpret_cast<uint4*>(vreg + ((rr >> 4) * HALVES + (rem >> 3)) * SUB + (rr & 15) * 128 + ((rem & 7) << 4)) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      if (!busy) {  // the lanes' P is never read back: whatever S left there is as good
        tc_fence_before();
        mbar_arrive(smem_u32(&p_ready[sg][u & 1]));
        continue;
      }
      const uint32_t scol = trow + (u & 1) * 64;
      float sv[64];
      {
        uint32_t ra[32], rb[32];
        tmem_ld32(scol, ra);
        tmem_ld32(scol + 32, rb);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          sv[j] = __uint_as_float(ra[j]);
          sv[32 + j] = __uint_as_float(rb[j]);
        }
      }
      if (__any_sync(0xffffffffu, kbase + 63 > lim)) {
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (kbase + j > lim) sv[j] = -INFINITY;
      }
      float m8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) m8[j] = sv[j];
#pragma unroll
      for (int j = 8; j < 64; ++j) m8[j & 7] = fmaxf(m8[j & 7], sv[j]);
      const float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                             fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7]))) * sl2;  // scale > 0
      // move the reference max only past the gap; the first visible tile always sets it
      const bool move = mx > m_ref + Cfg::RESCALE_LOG2;
      const float m_new = move ? mx : m_ref;
      const float mu = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = move ? ex2_approx(m_ref - mu) : 1.0f;
      float2 r4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) r4[k] = make_float2(0.f, 0.f);
      const float2 sl22 = make_float2(sl2, sl2), nmu = make_float2(-mu, -mu);
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 32 positions at a time: P as hi + lo over the S columns read
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 x = fma2_rn(make_float2(sv[32 * h + 2 * e], sv[32 * h + 2 * e + 1]), sl22, nmu);
          const float2 pe = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          r4[e & 3] = add2_rn(r4[e & 3], pe);
          hi[e] = ActTraits<T>::pack2(pe.x, pe.y);
          const float2 rest = sub2_rn(pe, ActTraits<T>::unpack2(hi[e]));
          lo[e] = ActTraits<T>::pack2(rest.x, rest.y);
        }
        tmem_st16(scol + 16 * h, hi);
        tmem_st16(scol + 32 + 16 * h, lo);
      }
      l_run = l_run * alpha + (((r4[0].x + r4[0].y) + (r4[1].x + r4[1].y)) + ((r4[2].x + r4[2].y) + (r4[3].x + r4[3].y)));
      m_ref = m_new;

      // O holds PV of steps < u: rescale rows whose reference moved, after PV(u - 1) completed
      if (u > 0 && __any_sync(0xffffffffu, move)) {
        if (!__all_sync(0xffffffffu, mbar_poll(smem_u32(&pv_done[sg]), (u - 1) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t v[32];
          tmem_ld32(trow + 128 + c * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
          tmem_st32(trow + 128 + c * 32, v);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(smem_u32(&p_ready[sg][u & 1]));
    }
    if (ok) {
      ok = __all_sync(0xffffffffu, mbar_poll(smem_u32(&drain), 0));
      tc_fence_after();
    }
    if (!ok) {
      failed = true;
      l_run = 0.f;  // contributes nothing
    }
    if (l_run == 0.f) m_ref = -INFINITY;  // O of a row that saw nothing is not read

    // Every MMA has completed, so Q and the rings are free: the rows' sums are staged there (16-byte
    // chunk c of a row at c ^ row, free of bank conflicts both ways) and leave a row at a time with
    // consecutive lanes on its columns.
    constexpr int CH = HD / 4;  // 16-byte chunks of a row's sums
    float4* const stage = reinterpret_cast<float4*>(gbase);
    float2* const s_ml = reinterpret_cast<float2*>(gbase + 128 * STREAMS * Cfg::ROW_BYTES);  // [128 STREAMS]
    long long* const s_off = reinterpret_cast<long long*>(s_ml + 128 * STREAMS);  // [128 STREAMS] of the output row
    float* const s_w = reinterpret_cast<float*>(s_off + 128 * STREAMS);            // [128 STREAMS]
    const int mine = sg * 128 + tl;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t v[32];
      tmem_ld32(trow + 128 + c * 32, v);
      tmem_wait_ld();
#pragma unroll
      for (int j = 0; j < 8; ++j)
        stage[mine * CH + ((c * 8 + j) ^ (lane & (CH - 1)))] =
            make_float4(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1]), __uint_as_float(v[4 * j + 2]),
                        __uint_as_float(v[4 * j + 3]));
    }
    s_ml[mine] = make_float2(m_ref, l_run);
    s_off[mine] = row * p.o_row + head * p.o_head;
    const size_t at = it.state + static_cast<size_t>(kvh) * it.span;  // of the item's score row 0
    if (!apart) streams_bar();
    float m = m_ref, l = l_run, w = l_run == 0.f ? 0.f : 1.f;  // the row's state, and this stream's weight in it
    if (!apart) {
      const float2 other = s_ml[(1 - sg) * 128 + tl];
      m = fmaxf(m_ref, other.x);
      const float mu = m == -INFINITY ? 0.f : m;
      w = ex2_approx(m_ref - mu);  // 0 where this stream saw nothing
      l = l_run * w + other.y * ex2_approx(other.x - mu);
    }
    if (row_ok && (apart || sg == 0)) {
      if (it.state >= 0) __stcg(p.ws_ml + at + local, make_float2(m, l));
      else if (p.lse) p.lse[static_cast<size_t>(row) * p.n_heads + head] = natural_lse(m, l);
    }
    s_w[mine] = it.state < 0 && l != 0.f ? __fdiv_rn(w, l) : w;
    if (apart) __syncwarp();
    else streams_bar();
    // rows of this warp: its own 32; or 16 of the tile, from both streams
    const int rows_w = apart ? 32 : 16, row_w = apart ? sg * 128 + (warp & 3) * 32 : (sg * 4 + (warp & 3)) * 16;
    const int n_w = min(rows_w, it.n_rho - row_w);
    constexpr int PER = 32 / CH;  // rows a warp stores at once
    const int c = lane % CH;
    for (int r0 = 0; r0 < n_w; r0 += 8 * PER) {
      float4 o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int k = r0 + i * PER + lane / CH, rr = row_w + (k < n_w ? k : 0);
        const float wa = s_w[rr];
        const float4 x = stage[rr * CH + (c ^ (rr & (CH - 1)))];  // not finite where the row saw nothing
        o[i] = wa != 0.f ? make_float4(x.x * wa, x.y * wa, x.z * wa, x.w * wa) : make_float4(0.f, 0.f, 0.f, 0.f);
        if (!apart) {
          const float wb = s_w[128 + rr];
          const float4 y = stage[(128 + rr) * CH + (c ^ (rr & (CH - 1)))];
          if (wb != 0.f) o[i] = make_float4(o[i].x + y.x * wb, o[i].y + y.y * wb, o[i].z + y.z * wb, o[i].w + y.w * wb);
        }
      }
      if (it.state >= 0) {
        float4* dst = reinterpret_cast<float4*>(p.ws_o + (at + row_w + r0 + lane / CH) * HD) + c;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (r0 + i * PER + lane / CH < n_w) __stcg(dst + i * PER * CH, o[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int k = r0 + i * PER + lane / CH;
          if (k >= n_w) continue;
          const long long to = s_off[row_w + k] + c * 4;
          if (p.out_f32) *reinterpret_cast<float4*>(static_cast<float*>(p.out) + to) = o[i];
          else
            *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + to) =
                make_uint2(ActTraits<T>::pack2(o[i].x, o[i].y), ActTraits<T>::pack2(o[i].z, o[i].w));
        }
      }
    }
  }
  if (failed) page_fail(p.status, kDevWaitTimeout);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
  if constexpr (TRACE) trace_end(p.trace);
}

// ============================================================================ states of a row -> output
constexpr int kJoinWarps = 4;

template <typename T, int HD, int BATCH, bool TRACE>
__global__ void __launch_bounds__(kJoinWarps * 32) prefix_join_kernel(PrefixParams p) {
  const int unit = blockIdx.x * kJoinWarps + (threadIdx.x >> 5);
  const bool on = unit < p.n_joins * p.n_heads;
  const PrefixJoin j = p.joins[on ? unit / p.n_heads : 0];
  griddep_wait();
  if constexpr (TRACE) trace_start(p.trace);
  if (on) join_states<T, HD, BATCH>(p, j, unit % p.n_heads);
  if constexpr (TRACE) trace_end(p.trace);
}

}  // namespace llm
