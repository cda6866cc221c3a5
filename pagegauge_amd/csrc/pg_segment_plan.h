// Work items of the attention over shared prefixes and over selected pages, and
// their planner: host C++, free of HIP.
#pragma once

#include <stdint.h>

#include <vector>

#include "pg_host.h"

namespace pg {

constexpr int kSegmentWaves = 4;          // waves of a workgroup
constexpr int kSegmentGroupPages = 4;     // consecutive pages a wave takes at a time
constexpr int kSegmentMaxPages = kSegmentWaves * 64;   // a wave holds its page ids one per lane
constexpr int kSegmentRows = 16;          // query rows of an item without shared tiles
constexpr int kNarrowRows = 8;            // or, with both parts of a probability in one product
constexpr int kSharedRows = 32;           // of a wave over shared tiles: items of 2 or 4 waves' rows
constexpr int kSharedMaxPages = 512;      // of an item over shared tiles, held in LDS
constexpr int kSegmentMaxSlots = 1 << 16; // partial rows of one request

// One workgroup's share, for one KV head: ``rows`` query rows over pages [page_begin,
// page_end) of a page table and exact pages [tail_begin, tail_end), either perhaps empty.
// Row i is row R = row_first + i of the segment's: query head R % group (of the KV head's)
// of request ``request`` + R / group.  Over shared tiles of 2 waves' rows each row has two
// partial rows, in slots one after the other.
struct SegmentItem {
  int32_t request, row_first, rows;
  int32_t segment;                        // of the prefix tables, or -1: the request's own table
  int32_t page_begin, page_end, last_page;    // in the table, or in a request's selection
  int32_t tail_begin, tail_end, last_tail;
  int32_t slot_at;                        // the requests' first slots: slot_base[slot_at + R / group]; -1: the output
  int32_t split;                          // added to these
  int32_t table_begin, table_pages;       // of the request, where pages are selected
  int32_t block_rows;                     // kNarrowRows, kSegmentRows, or 2 or 4 times kSharedRows: shared tiles
  int32_t reserved;
};
static_assert(sizeof(SegmentItem) == 64, "work item layout");

// A batch on the host.  ``selected`` > 0: of each request's pages only so many are read.
struct SegmentBatch {
  const int32_t* prefix_requests;         // [segments][2]
  const int32_t* prefix_indptr;           // [segments + 1]
  int32_t segments;
  const int32_t* indptr;                  // [batch_size + 1]
  const int32_t* tail_indptr;             // or null
  int32_t batch_size, num_qo_heads, num_kv_heads, kind, selected, num_cus;
};

struct SegmentWork {
  std::vector<SegmentItem> items;         // the longest first
  std::vector<int32_t> slot_ptr;          // [batch_size + 1]: partial rows of each request
  std::vector<int32_t> slot_base;         // of items' requests
};

int32_t build_segment_plan(const SegmentBatch& batch, SegmentWork& work, pg_segment_plan_t& p);

}  // namespace pg
