// Planner of the attention over the cache held in 4 bits (host only).
#include "pg_int4_plan.h"

#include <algorithm>
#include <cstring>
#include <string>

namespace pg {
namespace {

int64_t align_up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A request's pages, weighted by their bytes in 4-bit pages, as one sequence:
// the history, then the exact tail.
struct Request {
  int64_t pages, tail;
  int64_t weight() const { return pages + kInt4TailWeight * tail; }
  // Cuts of at most ``cap``; no item may get more pages than its waves can hold.
  int64_t cuts(int64_t cap) const {
    if (pages > kInt4MaxItemPages) cap = std::min<int64_t>(cap, kInt4MaxItemPages);
    return std::max<int64_t>(1, ceil_div(weight(), cap));
  }
};

}  // namespace

int32_t build_int4_plan(const int32_t* host_indptr, const int32_t* host_tail_indptr,
                        int32_t batch_size, int32_t num_qo_heads, int32_t num_kv_heads,
                        int32_t num_cus, std::vector<Int4Item>& items,
                        std::vector<int32_t>& item_ptr, pg_int4_plan_t& p) {
  if (!host_indptr) return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  if (batch_size <= 0) return fail(PG_ERROR_INVALID_ARGUMENT, "batch size must be positive");
  if (num_kv_heads <= 0 || num_qo_heads <= 0 || num_qo_heads % num_kv_heads)
    return fail(PG_ERROR_INVALID_ARGUMENT, "query heads must be a positive multiple of KV heads");
  if (num_qo_heads / num_kv_heads > 16)
    return fail(PG_ERROR_UNSUPPORTED, "at most 16 query heads per KV head");
  if (num_kv_heads > 1024) return fail(PG_ERROR_UNSUPPORTED, "at most 1024 KV heads");
  std::vector<Request> requests(batch_size);
  int64_t total = 0, history = 0, exact_pages = 0;
  for (int32_t b = 0; b < batch_size; ++b) {
    Request& r = requests[b];
    r.pages = static_cast<int64_t>(host_indptr[b + 1]) - host_indptr[b];
    r.tail = host_tail_indptr ? static_cast<int64_t>(host_tail_indptr[b + 1]) - host_tail_indptr[b] : 0;
    if (host_indptr[b] < 0 || r.pages < 0 || r.tail < 0 || (host_tail_indptr && host_tail_indptr[b] < 0))
      return fail(PG_ERROR_INVALID_ARGUMENT, "indptr must be nonnegative and non-decreasing");
    total += r.weight();
    history += r.pages;
    exact_pages += r.tail;
  }
  // ``balanced``: the smallest largest share (``cap``, in weighted pages) with which the
  // batch takes no more workgroups than ``target``, but at least one group of pages
  // per wave.  Only requests of long histories have an item's limit of their own, so
  // long exact tails would be left whole where these take the target up alone (100000
  // history pages beside 4000 exact ones: 1393 us, now 393) or as many requests do (299 of
  // 41 pages beside one of 3000 exact ones: 881 us, now 133): no share exceeds two full
  // items' and twice an even one, unless a request would have too many items.
  const int64_t cus = num_cus > 0 ? num_cus : 256;
  auto items_of = [&](int64_t cap) {
    int64_t n = 0;
    for (const Request& r : requests) n += r.cuts(cap);
    return n;
  };
  const int64_t full = std::max<int64_t>(2 * kInt4MaxItemPages, ceil_div(total, kInt4MaxItemsPerRequest));
  auto balanced = [&](int64_t target) {
    int64_t low = kInt4Waves * kInt4GroupPages, high = std::max(low, total);
    if (items_of(high) > target) return std::min(high, full);
    while (low < high) {
      const int64_t cap = low + (high - low) / 2;
      if (items_of(cap) <= target) high = cap; else low = cap + 1;
    }
    return std::min(high, std::max(full, 2 * ceil_div(total, target)));
  };
  // One workgroup per CU is the better plan (49K tokens: 32 items 16.6 us, 64 items
  // 18.1; 64K 18.9 and 20.8) unless its waves cannot hold their pages (128K tokens: 33
  // items, an uneven round, 46.8 us, 64 items 33.6; 16 requests of 8K 38.3 and 34.4)
  // or requests do not divide over so few (17 requests of 3.3K: 32 items, of a whole
  // request the largest, 27.6, 64 items 24.0): then it is two.
  const int64_t one = std::max<int64_t>(1, cus / num_kv_heads);
  const int64_t two = std::max<int64_t>(1, 2 * cus / num_kv_heads);
  int64_t cap = balanced(std::max<int64_t>(batch_size, one));
  const int64_t cap2 = balanced(std::max<int64_t>(batch_size, two));
  if (cap > kInt4MaxItemPages || 10 * cap > 24 * cap2) {
    // More than two per CU are brought to whole rounds (6 requests of 13K to 70K: 66
    // items 73.4 us, 128 items 60.5; 84 of 468 to 4391 tokens 77.2 and 71; 90 of 500
    // to 8000: 141 items 105, 192 items 99), unless there are more than two rounds
    // and no request is cut yet (130 of 512 to 4000: 93.6, 192 items 101.3).
    cap = cap2;
    const int64_t n = items_of(cap), rounds = ceil_div(n, two);
    if (rounds == 2 || (rounds > 2 && rounds <= 4 && n > batch_size)) cap = balanced(rounds * two);
  }
  items.clear();
  item_ptr.assign(batch_size + 1, 0);
  int64_t most = 0;
  for (int32_t b = 0; b < batch_size; ++b) {
    const Request& r = requests[b];
    const int64_t cuts = r.cuts(cap);
    if (cuts > kInt4MaxItemsPerRequest)
      return fail(PG_ERROR_UNSUPPORTED, "too many pages in one request");
    item_ptr[b] = static_cast<int32_t>(items.size());
    const int32_t begin = host_indptr[b], tail = host_tail_indptr ? host_tail_indptr[b] : 0;
    // cut i ends at weight w = (i + 1) W / cuts: its history page, or the
    // tail page that w falls into
    int64_t page = 0, exact = 0;
    for (int64_t i = 0; i < cuts; ++i) {
      const int64_t w = (i + 1) * r.weight() / cuts;
      int64_t page_end = std::min(r.pages, w);
      int64_t exact_end = w <= r.pages ? 0 : (w - r.pages) / kInt4TailWeight;
      if (i + 1 == cuts) { page_end = r.pages; exact_end = r.tail; }
      items.push_back({b, static_cast<int32_t>(begin + page), static_cast<int32_t>(begin + page_end),
                       static_cast<int32_t>(begin + r.pages - 1), static_cast<int32_t>(tail + exact),
                       static_cast<int32_t>(tail + exact_end), static_cast<int32_t>(tail + r.tail - 1),
                       static_cast<int32_t>(cuts)});
      page = page_end;
      exact = exact_end;
    }
    most = std::max(most, cuts);
  }
  if (items.size() > UINT32_MAX / (kInt4Waves * 64)) return fail(PG_ERROR_UNSUPPORTED, "too many work items");
  item_ptr[batch_size] = static_cast<int32_t>(items.size());
  p = pg_int4_plan_t{};
  p.batch_size = batch_size;
  p.num_qo_heads = num_qo_heads;
  p.num_kv_heads = num_kv_heads;
  p.has_tail = exact_pages > 0;
  p.has_history = history > 0;
  p.num_items = static_cast<int32_t>(items.size());
  p.max_items_per_request = static_cast<int32_t>(most);
  p.items_offset = 0;
  p.item_ptr_offset = align_up(static_cast<int64_t>(items.size() * sizeof(Int4Item)), 256);
  p.partial_offset = p.item_ptr_offset + align_up((batch_size + 1) * 4, 256);
  const int64_t rows = most > 1 ? static_cast<int64_t>(items.size()) * num_qo_heads : 0;
  p.workspace_bytes = p.partial_offset + rows * (kHeadDim + 2) * 4;
  return PG_OK;
}

}  // namespace pg

using namespace pg;

extern "C" int32_t pg_int4_plan_host(const int32_t* host_indptr, const int32_t* host_tail_indptr,
                                     int32_t batch_size, int32_t num_qo_heads, int32_t num_kv_heads,
                                     int32_t num_cus, pg_int4_plan_t* plan, int32_t* items_out,
                                     int64_t items_capacity, int32_t* item_ptr_out) {
  clear_error();
  if (!plan) return fail(PG_ERROR_INVALID_ARGUMENT, "null plan argument");
  return guarded([&]() -> int32_t {
    std::vector<Int4Item> items;
    std::vector<int32_t> item_ptr;
    pg_int4_plan_t p{};
    if (int32_t rc = build_int4_plan(host_indptr, host_tail_indptr, batch_size, num_qo_heads,
                                     num_kv_heads, num_cus, items, item_ptr, p))
      return rc;
    if (items_out) {
      if (items_capacity < static_cast<int64_t>(items.size()))
        return fail(PG_ERROR_INVALID_ARGUMENT, "work-item buffer too small: need " +
                                                   std::to_string(items.size()) + " items");
      std::memcpy(items_out, items.data(), items.size() * sizeof(Int4Item));
    }
    if (item_ptr_out) std::memcpy(item_ptr_out, item_ptr.data(), item_ptr.size() * sizeof(int32_t));
    *plan = p;
    return PG_OK;
  });
}
