// paged.h -- what the context (llm_cuda.cu) uses of the paged caches' translation unit (paged.cu).
#pragma once
#include <cuda_runtime.h>

#include "../../include/llm_cuda.h"

namespace llm {
struct TraceRec;
}

// llm_prefix_plan_create for sequences listed in `order` (group by group; nullptr: as they are):
// rows, slots, ctx and the rows of q and out stay in the caller's order.
int llm_detail_prefix_create(int device, int dtype, int n_heads, int n_kv_heads, int head_dim, const int* slots,
                             const int* rows, int n_seqs, const int* order, const int* group_sizes, const int* prefixes,
                             int n_groups, int max_ctx, llm_prefix_plan** out);
// One layer of a context's decode rows: q and out [rows][n_heads][head_dim] (out f32 or the cache's
// dtype), sequence s seeing positions[s] + 1 positions.
struct llm_prefix_rows {
  const void* q;
  void* out;
  int out_f32;
  const int* positions;
  const void* layer_pool;  // the layer's pages
  const int* table;
  int n_pages, max_pages;
  int* status;
  llm::TraceRec* trace[3];  // timeline records of the launches, in their order; nullptr: none
};
cudaError_t llm_detail_prefix_run(const llm_prefix_plan* plan, const llm_prefix_rows& r, cudaStream_t s);
// Kernels of one llm_detail_prefix_run, in their order; names: nullptr, or where to put theirs.
int llm_detail_prefix_launches(const llm_prefix_plan* plan, const char* (*names)[3] = nullptr);
size_t llm_detail_prefix_bytes(const llm_prefix_plan* plan);  // device memory that it holds
// What a status word that kernels set says (DeviceError, PageError).
const char* llm_detail_device_error(int code);
