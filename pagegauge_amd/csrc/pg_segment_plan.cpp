// Planner of the attention over shared prefixes and over selected pages (host only).
#include "pg_segment_plan.h"

#include <algorithm>
#include <cstring>
#include <string>

namespace pg {
namespace {

int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Pages that a workgroup is worth, where there are more workgroups than fit at once.
constexpr int64_t kSmallestShare = 64;

// Pages that are read together, by ``blocks`` workgroups of query rows.
struct Unit {
  int32_t segment, request;               // segment -1: the request's own pages
  int64_t rows, pages, tail, tail_weight;
  // Two blocks of 16 rows that read the pages each are still the faster, mostly (8 requests of 4
  // heads on 16384 tokens, with the join: INT8 19.7 and 21.7 us, FP16 20.4 and 23.7; on 60000
  // 41.8 and 39.0, 47.3 and 51.0); of three the tiles are (12 requests on 16384: 25.5 and 24.9;
  // on 60000 55.3 and 41.7).
  bool shared() const { return rows > 2 * kSegmentRows; }
  // rows of one workgroup, and the partial rows that it makes of each
  int64_t block_rows() const {
    if (!shared()) return rows > kNarrowRows ? kSegmentRows : kNarrowRows;
    return rows > 2 * kSharedRows ? 4 * kSharedRows : 2 * kSharedRows;
  }
  int64_t parts() const { return block_rows() == 2 * kSharedRows ? 2 : 1; }
  int64_t blocks() const { return ceil_div(rows, block_rows()); }
  // rows of each block, evenly, in whole waves over shared tiles
  int64_t step() const {
    return !shared() ? block_rows() : ceil_div(ceil_div(rows, blocks()), kSharedRows) * kSharedRows;
  }
  int64_t weight() const { return pages + tail_weight * tail; }
  int64_t cuts(int64_t cap) const { return std::max<int64_t>(1, ceil_div(weight(), cap)); }
};

int32_t check_indptr(const int32_t* indptr, int32_t count) {
  if (!indptr) return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  for (int32_t i = 0; i < count; ++i)
    if (indptr[i] < 0 || indptr[i + 1] < indptr[i])
      return fail(PG_ERROR_INVALID_ARGUMENT, "indptr must be nonnegative and non-decreasing");
  return PG_OK;
}

}  // namespace

int32_t build_segment_plan(const SegmentBatch& b, SegmentWork& work, pg_segment_plan_t& p) {
  if (b.batch_size <= 0) return fail(PG_ERROR_INVALID_ARGUMENT, "batch size must be positive");
  if (b.num_kv_heads <= 0 || b.num_qo_heads <= 0 || b.num_qo_heads % b.num_kv_heads)
    return fail(PG_ERROR_INVALID_ARGUMENT, "query heads must be a positive multiple of KV heads");
  const int32_t group = b.num_qo_heads / b.num_kv_heads;
  if (group > 16) return fail(PG_ERROR_UNSUPPORTED, "at most 16 query heads per KV head");
  if (b.num_kv_heads > 1024) return fail(PG_ERROR_UNSUPPORTED, "at most 1024 KV heads");
  if (b.kind != PG_KV_INT8 && b.kind != PG_KV_FP16)
    return fail(PG_ERROR_INVALID_ARGUMENT, "pages must be INT8 or FP16");
  if (b.segments < 0 || (b.segments && !b.prefix_requests))
    return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  if (b.segments)
    if (int32_t rc = check_indptr(b.prefix_indptr, b.segments)) return rc;
  if (int32_t rc = check_indptr(b.indptr, b.batch_size)) return rc;
  if (b.tail_indptr)
    if (int32_t rc = check_indptr(b.tail_indptr, b.batch_size)) return rc;

  // ---- what is read together
  const int64_t tail_weight = b.kind == PG_KV_INT8 ? 2 : 1;      // of an FP16 page, by bytes
  std::vector<Unit> units;
  std::vector<bool> covered(b.batch_size, false);
  int64_t prefix_pages = 0, history = 0, tails = 0, max_pages = 0, all_pages = 0;
  for (int32_t s = 0; s < b.segments; ++s) {
    const int32_t begin = b.prefix_requests[2 * s], end = b.prefix_requests[2 * s + 1];
    if (begin < 0 || end < begin || end > b.batch_size)
      return fail(PG_ERROR_INVALID_ARGUMENT, "a prefix's requests must be a range of the batch");
    const int64_t pages = b.prefix_indptr[s + 1] - b.prefix_indptr[s];
    if (begin == end || pages == 0) continue;
    units.push_back({s, begin, static_cast<int64_t>(end - begin) * group, pages, 0, tail_weight});
    std::fill(covered.begin() + begin, covered.begin() + end, true);
    prefix_pages += pages;
  }
  for (int32_t r = 0; r < b.batch_size; ++r) {
    const int64_t all = b.indptr[r + 1] - b.indptr[r];
    const int64_t pages = b.selected > 0 ? std::min<int64_t>(all, b.selected) : all;
    const int64_t tail = b.tail_indptr ? b.tail_indptr[r + 1] - b.tail_indptr[r] : 0;
    max_pages = std::max(max_pages, all);
    all_pages += all;
    history += pages;
    tails += tail;
    if (pages || tail || !covered[r]) units.push_back({-1, r, group, pages, tail, tail_weight});
  }

  // ---- the largest share: the smallest with which everything runs at once, two
  // workgroups per CU (61 requests of 7 prefixes: 33.5 us; with shares of shared tiles
  // and of own pages apart, as below, 39.4).  Where requests and prefixes are more than
  // that, shared tiles get one workgroup per CU, which is what the matrix cores need, and
  // own pages, in half of even shares, are read beside them: the longest go first and the
  // short ones fill in behind them (256 requests on 1024 pages: shared tiles in 4 parts
  // 175 us, in 2 parts 250, in 6 parts 196, in 8 parts 215); with little of their own to
  // read shared tiles get both (the same with one exact page each: 108 us, 118 with one).
  const int64_t cus = b.num_cus > 0 ? b.num_cus : 256;
  const int64_t at_once = std::max<int64_t>(2, 2 * cus / b.num_kv_heads);
  auto items_of = [&](bool shared, int64_t cap) {
    int64_t n = 0;
    for (const Unit& u : units) n += u.shared() == shared ? u.cuts(cap) * u.blocks() : 0;
    return n;
  };
  // the smallest share in [one group of pages per wave, high] that ``fits``, or 0
  auto smallest = [](int64_t high, auto&& fits) -> int64_t {
    if (!fits(high)) return 0;
    int64_t low = kSegmentWaves * kSegmentGroupPages;
    while (low < high) {
      const int64_t middle = low + (high - low) / 2;
      if (fits(middle)) high = middle; else low = middle + 1;
    }
    return high;
  };
  int64_t shared_cap = smallest(kSharedMaxPages, [&](int64_t cap) {
    return items_of(true, cap) + items_of(false, std::min<int64_t>(cap, kSegmentMaxPages)) <= at_once;
  });
  int64_t own_cap = std::min<int64_t>(shared_cap, kSegmentMaxPages);
  if (!shared_cap) {
    int64_t weights[2] = {0, 0};
    for (const Unit& u : units) weights[u.shared()] += u.weight() * u.blocks();
    auto half_share = [&](bool shared) { return std::max(weights[shared] / at_once, kSmallestShare); };
    const int64_t shared_target = weights[0] > weights[1] / 2 ? at_once / 2 : at_once;
    shared_cap = smallest(kSharedMaxPages, [&](int64_t cap) { return items_of(true, cap) <= shared_target; });
    if (!shared_cap) shared_cap = std::min<int64_t>(kSharedMaxPages, half_share(true));
    own_cap = std::min<int64_t>(kSegmentMaxPages, half_share(false));
  }
  const int64_t shared_items = items_of(true, shared_cap);
  auto cuts_of = [&](const Unit& u) { return u.cuts(u.shared() ? shared_cap : own_cap); };
  const int64_t count = shared_items + items_of(false, own_cap);
  for (const Unit& u : units)
    if (cuts_of(u) * u.parts() > kSegmentMaxSlots) return fail(PG_ERROR_UNSUPPORTED, "too many pages in one request");
  if (count > static_cast<int64_t>(UINT32_MAX) / (kSegmentWaves * 64) / b.num_kv_heads)
    return fail(PG_ERROR_UNSUPPORTED, "too many work items");

  // ---- partial rows: a request's are those of its prefixes, then its own
  std::vector<int64_t> slots(b.batch_size, 0);
  work = SegmentWork{};
  work.items.reserve(count);
  for (const Unit& u : units) {
    const int64_t cuts = cuts_of(u);
    const bool direct = u.segment < 0 && cuts == 1 && !covered[u.request];
    const int32_t slot_at = direct ? -1 : static_cast<int32_t>(work.slot_base.size());
    const int32_t requests = static_cast<int32_t>(u.rows / group);
    if (!direct) {
      if (work.slot_base.size() + requests > INT32_MAX) return fail(PG_ERROR_UNSUPPORTED, "too many work items");
      for (int32_t r = u.request; r < u.request + requests; ++r) {
        work.slot_base.push_back(static_cast<int32_t>(slots[r]));      // from the request's first one, so far
        slots[r] += cuts * u.parts();
        if (slots[r] > kSegmentMaxSlots) return fail(PG_ERROR_UNSUPPORTED, "too many pages in one request");
      }
    }
    const bool own = u.segment < 0;
    const int32_t begin = !own ? b.prefix_indptr[u.segment] : b.selected > 0 ? 0 : b.indptr[u.request];
    const int32_t tail_begin = own && b.tail_indptr ? b.tail_indptr[u.request] : 0;
    int64_t page = 0, exact = 0;
    for (int64_t i = 0; i < cuts; ++i) {
      // cut i ends at weight w = (i + 1) W / cuts: its page, or the tail page that w falls into
      const int64_t w = (i + 1) * u.weight() / cuts;
      int64_t page_end = std::min(u.pages, w);
      int64_t exact_end = w <= u.pages ? 0 : (w - u.pages) / tail_weight;
      if (i + 1 == cuts) { page_end = u.pages; exact_end = u.tail; }
      for (int64_t row = 0; row < u.rows; row += u.step()) {
        SegmentItem it{};
        it.request = u.request;
        it.row_first = static_cast<int32_t>(row);
        it.rows = static_cast<int32_t>(std::min<int64_t>(u.step(), u.rows - row));
        it.segment = u.segment;
        it.page_begin = static_cast<int32_t>(begin + page);
        it.page_end = static_cast<int32_t>(begin + page_end);
        it.last_page = static_cast<int32_t>(begin + u.pages - 1);
        it.tail_begin = static_cast<int32_t>(tail_begin + exact);
        it.tail_end = static_cast<int32_t>(tail_begin + exact_end);
        it.last_tail = static_cast<int32_t>(tail_begin + u.tail - 1);
        it.slot_at = slot_at;
        it.block_rows = static_cast<int32_t>(u.block_rows());
        it.split = static_cast<int32_t>(i * u.parts());
        if (own) {
          it.table_begin = b.indptr[u.request];
          it.table_pages = b.indptr[u.request + 1] - b.indptr[u.request];
        }
        work.items.push_back(it);
      }
      page = page_end;
      exact = exact_end;
    }
  }
  // The longest first, which also puts the shared tiles of a full batch one to a CU and own
  // pages beside them: a CU of an XCD gets every 32nd workgroup (taken in turns, two shared ones
  // met on a CU and the batch above took 254 us instead of 200 on the same card).
  auto weight_of = [&](const SegmentItem& it) {
    return it.page_end - it.page_begin + tail_weight * (it.tail_end - it.tail_begin);
  };
  std::stable_sort(work.items.begin(), work.items.end(),
                   [&](const SegmentItem& x, const SegmentItem& y) { return weight_of(x) > weight_of(y); });

  work.slot_ptr.assign(b.batch_size + 1, 0);
  int64_t rows = 0, most = 0;
  for (int32_t r = 0; r < b.batch_size; ++r) {
    work.slot_ptr[r] = static_cast<int32_t>(rows);
    rows += slots[r];
    most = std::max(most, slots[r]);
    if (rows > INT32_MAX) return fail(PG_ERROR_UNSUPPORTED, "too many work items");
  }
  work.slot_ptr[b.batch_size] = static_cast<int32_t>(rows);
  // slots of an item's requests count from the batch's first one
  size_t at = 0;
  for (const Unit& u : units) {
    if (u.segment < 0 && !covered[u.request] && cuts_of(u) == 1) continue;
    for (int32_t r = u.request; r < u.request + u.rows / group; ++r) work.slot_base[at++] += work.slot_ptr[r];
  }

  p = pg_segment_plan_t{};
  p.batch_size = b.batch_size;
  p.num_qo_heads = b.num_qo_heads;
  p.num_kv_heads = b.num_kv_heads;
  p.kind = b.kind;
  p.num_items = static_cast<int32_t>(work.items.size());
  p.max_slots = static_cast<int32_t>(most);
  p.has_prefix = prefix_pages > 0;
  p.has_history = history > 0;
  p.has_tail = tails > 0;
  p.slot_base_count = static_cast<int32_t>(work.slot_base.size());
  p.selected_pages = b.selected;
  p.max_pages = static_cast<int32_t>(max_pages);
  int64_t offset = 0;
  auto place = [&](int64_t bytes) {
    const int64_t here = offset;
    offset = align_up(offset + bytes, 256);
    return here;
  };
  p.items_offset = place(static_cast<int64_t>(work.items.size() * sizeof(SegmentItem)));
  p.slot_ptr_offset = place((static_cast<int64_t>(b.batch_size) + 1) * 4);
  p.slot_base_offset = place(static_cast<int64_t>(work.slot_base.size()) * 4);
  p.indptr_offset = place(b.selected > 0 ? (static_cast<int64_t>(b.batch_size) + 1) * 4 : 0);
  p.scores_offset = place(b.selected > 0 ? 4 * all_pages * b.num_kv_heads : 0);
  p.partial_offset = place(rows * b.num_qo_heads * (kHeadDim + 2) * 4);
  p.partial_rows = rows;
  p.workspace_bytes = offset;
  return PG_OK;
}

}  // namespace pg

using namespace pg;

extern "C" int32_t pg_segment_plan_host(const int32_t* host_prefix_requests, const int32_t* host_prefix_indptr,
                                        int32_t segments, const int32_t* host_indptr,
                                        const int32_t* host_tail_indptr, int32_t batch_size,
                                        int32_t num_qo_heads, int32_t num_kv_heads, int32_t kind,
                                        int32_t selected_pages, int32_t num_cus, pg_segment_plan_t* plan,
                                        int32_t* items_out, int64_t items_capacity, int32_t* slot_ptr_out,
                                        int32_t* slot_base_out, int64_t slot_base_capacity) {
  clear_error();
  if (!plan) return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  return guarded([&]() -> int32_t {
    SegmentWork work;
    pg_segment_plan_t p{};
    if (int32_t rc = build_segment_plan({host_prefix_requests, host_prefix_indptr, segments, host_indptr,
                                         host_tail_indptr, batch_size, num_qo_heads, num_kv_heads, kind,
                                         selected_pages, num_cus}, work, p))
      return rc;
    if (items_out) {
      if (items_capacity < static_cast<int64_t>(work.items.size()))
        return fail(PG_ERROR_INVALID_ARGUMENT, "work-item buffer too small: need " +
                                                   std::to_string(work.items.size()) + " items");
      std::memcpy(items_out, work.items.data(), work.items.size() * sizeof(SegmentItem));
    }
    if (slot_ptr_out) std::memcpy(slot_ptr_out, work.slot_ptr.data(), work.slot_ptr.size() * sizeof(int32_t));
    if (slot_base_out) {
      if (slot_base_capacity < static_cast<int64_t>(work.slot_base.size()))
        return fail(PG_ERROR_INVALID_ARGUMENT, "slot buffer too small: need " +
                                                   std::to_string(work.slot_base.size()) + " entries");
      std::memcpy(slot_base_out, work.slot_base.data(), work.slot_base.size() * sizeof(int32_t));
    }
    *plan = p;
    return PG_OK;
  });
}
