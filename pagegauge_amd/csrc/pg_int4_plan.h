// Work items of the attention over the cache held in 4 bits, and their
// planner: host C++, free of HIP.
#pragma once

#include <stdint.h>

#include <vector>

#include "pg_host.h"

namespace pg {

constexpr int kInt4Waves = 4;           // waves of a workgroup, sharing one item's pages
constexpr int kInt4GroupPages = 4;      // consecutive pages a wave takes at a time
constexpr int kInt4MaxItemPages = kInt4Waves * 64;   // a wave holds its page ids one per lane
constexpr int kInt4MaxItemsPerRequest = 4096;
constexpr int kInt4TailWeight = 4;      // an FP16 page's bytes in 4-bit pages

// One workgroup's share of a request, for one KV head: history pages [page_begin, page_end) of the page table and exact
// pages [tail_begin, tail_end) of the tail's, either perhaps empty.
struct Int4Item {
  int32_t request;
  int32_t page_begin, page_end, last_page;   // absolute; last_page: the request's final one
  int32_t tail_begin, tail_end, last_tail;
  int32_t items_in_request;
};
static_assert(sizeof(Int4Item) == 32, "work item layout");

// Validates the batch and cuts it into ``items`` (a request's are contiguous,
// ``item_ptr`` [B + 1]); a request without tokens gets one empty item.
int32_t build_int4_plan(const int32_t* host_indptr, const int32_t* host_tail_indptr,
                        int32_t batch_size, int32_t num_qo_heads, int32_t num_kv_heads,
                        int32_t num_cus, std::vector<Int4Item>& items,
                        std::vector<int32_t>& item_ptr, pg_int4_plan_t& p);

}  // namespace pg
