// Attention of single tokens over prefixes that requests share, their own pages and an
// exact tail: each prefix's pages are read once for all of its requests.
#include "pg_page_attention.h"

using namespace pg;

extern "C" int32_t pg_prefix_plan(const int32_t* host_prefix_requests, const int32_t* host_prefix_indptr,
                                  int32_t segments, const int32_t* host_indptr, const int32_t* host_tail_indptr,
                                  int32_t batch_size, int32_t num_qo_heads, int32_t num_kv_heads, int32_t kind,
                                  int32_t num_cus, void* workspace, int64_t workspace_bytes,
                                  pg_segment_plan_t* plan, void* stream) {
  clear_error();
  return plan_into({host_prefix_requests, host_prefix_indptr, segments, host_indptr, host_tail_indptr, batch_size,
                    num_qo_heads, num_kv_heads, kind, 0, num_cus}, workspace, workspace_bytes, plan,
                   as_stream(stream));
}

extern "C" int32_t pg_prefix_run(const pg_segment_plan_t* plan, const void* query, int64_t query_batch_stride,
                                 const void* key, const void* value, const void* key_scale,
                                 const void* value_scale, const int32_t* prefix_indices,
                                 const int32_t* prefix_last_len, const int32_t* indices,
                                 const int32_t* last_page_len, const void* tail_k, const void* tail_v,
                                 const int32_t* tail_indices, const int32_t* tail_last_len,
                                 const void* value_center, void* out, float* lse, float sm_scale,
                                 void* workspace, void* stream) {
  clear_error();
  if (!plan) return fail(PG_ERROR_INVALID_ARGUMENT, "null run argument");
  PageAttentionArgs a{};
  a.query = static_cast<const uint16_t*>(query);
  a.query_batch_stride = query_batch_stride;
  a.key = key;
  a.value = value;
  a.key_scale = static_cast<const uint16_t*>(key_scale);
  a.value_scale = static_cast<const uint16_t*>(value_scale);
  a.prefix_indices = prefix_indices;
  a.prefix_last = prefix_last_len;
  a.indices = indices;
  a.last_page_len = last_page_len;
  a.tail_k = static_cast<const uint16_t*>(tail_k);
  a.tail_v = static_cast<const uint16_t*>(tail_v);
  a.tail_indices = tail_indices;
  a.tail_last = tail_last_len;
  a.value_center = static_cast<const uint16_t*>(value_center);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  if (int32_t rc = check_attention(*plan, a, sm_scale, workspace)) return rc;
  if (plan->selected_pages) return fail(PG_ERROR_INVALID_ARGUMENT, "the plan is not one of pg_prefix_plan");
  place_work(*plan, workspace, sm_scale, a);
  const dim3 grid(static_cast<unsigned>(plan->num_items) * plan->num_kv_heads);
  const dim3 threads(kAttentionThreads);
  hipStream_t s = as_stream(stream);
  const bool wide = plan->has_prefix || a.group > kNarrowRows;
  if (plan->kind == PG_KV_INT8 && wide)
    hipLaunchKernelGGL((page_attention_kernel<true, false, true>), grid, threads, 0, s, a);
  else if (plan->kind == PG_KV_INT8)
    hipLaunchKernelGGL((page_attention_kernel<true, false, false>), grid, threads, 0, s, a);
  else if (wide)
    hipLaunchKernelGGL((page_attention_kernel<false, false, true>), grid, threads, 0, s, a);
  else
    hipLaunchKernelGGL((page_attention_kernel<false, false, false>), grid, threads, 0, s, a);
  if (int32_t rc = check_launch("prefix_attention")) return rc;
  return launch_combine(*plan, a, workspace, s);
}
