// Host-side fuzz of the planner of shared prefixes and selected pages
// (pg_segment_plan_host), built with AddressSanitizer and UndefinedBehaviorSanitizer by
// tests/test_segment_plan_sanitized.py.  Random batches and malformed ones; of every
// accepted plan the items stay within their tables and the limits that the kernels
// assume, each request's pages and rows are read once in all (by count), and partial rows
// stay within their request's; rejected inputs leave a message.
// Usage: segment_plan_fuzz <seed> <iterations>; prints "ok <plans> <rejections>".
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "pagegauge_hip.h"
#include "pg_segment_plan.h"

namespace {

int failures = 0;

void check(bool cond, const char* what, int iteration) {
  if (!cond) {
    std::fprintf(stderr, "iteration %d: %s\n", iteration, what);
    if (++failures > 20) std::exit(1);
  }
}

}  // namespace

int main(int argc, char** argv) {
  if (argc < 3) return 2;
  std::mt19937 rng(static_cast<unsigned>(std::atoi(argv[1])));
  const int iterations = std::atoi(argv[2]);
  auto pick = [&](int low, int high) { return std::uniform_int_distribution<int>(low, high)(rng); };
  int plans = 0, rejected = 0;
  for (int n = 0; n < iterations; ++n) {
    const int batch = pick(1, 24), hkv = pick(1, 9), group = pick(1, 16), segments = pick(0, 4);
    const int selected = segments == 0 && pick(0, 2) == 0 ? pick(1, 400) : 0;
    auto length = [&]() { return pick(0, 3) ? pick(0, 40) : pick(0, 3) ? pick(0, 3000) : pick(0, 200000); };
    auto table = [&](int count) {
      std::vector<int32_t> indptr(count + 1, pick(0, 5));
      for (int i = 0; i < count; ++i) indptr[i + 1] = indptr[i] + length();
      return indptr;
    };
    std::vector<int32_t> own = table(batch), tail = table(batch), prefix = table(segments), requests;
    for (int s = 0; s < segments; ++s) {
      const int a = pick(0, batch), b = pick(0, batch);
      requests.push_back(a < b ? a : b);
      requests.push_back(a < b ? b : a);
    }
    int kind = pick(0, 1), heads = hkv * group, cus = pick(0, 2) ? 256 : pick(-1, 400);
    if (pick(0, 9) == 0) {                 // something wrong
      switch (pick(0, 6)) {
        case 0: own[pick(0, batch)] = -1; break;
        case 1: own[pick(0, batch)] = 2147483647; break;
        case 2: if (segments) requests[pick(0, 2 * segments - 1)] = pick(-3, batch + 3); break;
        case 3: heads += 1; break;
        case 4: kind = pick(2, 5); break;
        case 5: if (segments) prefix[pick(0, segments)] = pick(-2, 2147483647); break;
        default: tail[pick(0, batch)] = pick(-2, 1000000); break;
      }
    }
    const bool with_tail = pick(0, 3) != 0;
    pg_segment_plan_t plan{};
    auto call = [&](int32_t* items, int64_t room, int32_t* slot_ptr, int32_t* slot_base, int64_t base_room) {
      return pg_segment_plan_host(requests.data(), prefix.data(), segments, own.data(),
                                  with_tail ? tail.data() : nullptr, batch, heads, hkv, kind, selected, cus, &plan,
                                  items, room, slot_ptr, slot_base, base_room);
    };
    if (call(nullptr, 0, nullptr, nullptr, 0) != PG_OK) {
      ++rejected;
      check(pg_last_error()[0] != 0, "a rejection without a message", n);
      continue;
    }
    ++plans;
    std::vector<pg::SegmentItem> items(plan.num_items);
    std::vector<int32_t> slot_ptr(batch + 1), slot_base(plan.slot_base_count);
    check(call(reinterpret_cast<int32_t*>(items.data()), plan.num_items, slot_ptr.data(), slot_base.data(),
               plan.slot_base_count) == PG_OK, "the second call", n);
    const int g = heads / hkv;
    std::vector<int64_t> read(batch, 0), exact(batch, 0), slots(batch, 0);
    for (const pg::SegmentItem& it : items) {
      const bool shared = it.block_rows > pg::kSegmentRows;
      const int parts = it.block_rows == 2 * pg::kSharedRows ? 2 : 1;
      check(it.rows > 0 && it.rows <= it.block_rows && it.row_first >= 0, "rows", n);
      check(it.page_end >= it.page_begin && it.page_end - it.page_begin <= (shared ? pg::kSharedMaxPages : pg::kSegmentMaxPages),
            "pages of an item", n);
      check(it.tail_end >= it.tail_begin && it.tail_end - it.tail_begin <= pg::kSegmentMaxPages, "exact pages of an item", n);
      const int last = it.request + (it.row_first + it.rows - 1) / g;
      check(it.request >= 0 && last < batch, "requests of an item", n);
      if (it.segment >= 0)
        check(it.segment < segments && it.page_begin >= prefix[it.segment] && it.page_end <= prefix[it.segment + 1] &&
              it.page_end > it.page_begin && last < requests[2 * it.segment + 1], "a prefix's table", n);
      else if (selected)
        check(it.page_begin >= 0 && it.page_end <= selected && it.page_end <= own[it.request + 1] - own[it.request],
              "a selection's table", n);
      else
        check(it.page_begin >= own[it.request] && it.page_end <= own[it.request + 1], "a request's table", n);
      for (int row = it.row_first; row < it.row_first + it.rows; ++row) {
        const int request = it.request + row / g;
        read[request] += it.page_end - it.page_begin;
        exact[request] += it.tail_end - it.tail_begin;
        slots[request] += it.slot_at >= 0 ? parts : 0;
        if (it.slot_at < 0) continue;
        check(it.slot_at + row / g < plan.slot_base_count, "slot_base", n);
        const int64_t slot = static_cast<int64_t>(slot_base[it.slot_at + row / g]) + it.split;
        check(slot >= slot_ptr[request] && slot + parts <= slot_ptr[request + 1], "a partial row", n);
      }
    }
    for (int b = 0; b < batch; ++b) {
      int64_t pages = own[b + 1] - own[b];
      if (selected && pages > selected) pages = selected;
      for (int s = 0; s < segments; ++s)
        if (requests[2 * s] <= b && b < requests[2 * s + 1]) pages += prefix[s + 1] - prefix[s];
      check(read[b] == pages * g, "pages of a request", n);
      check(exact[b] == (with_tail ? static_cast<int64_t>(tail[b + 1] - tail[b]) * g : 0), "exact pages of a request", n);
      check(slots[b] == static_cast<int64_t>(slot_ptr[b + 1] - slot_ptr[b]) * g, "partial rows of a request", n);
      check(slot_ptr[b + 1] - slot_ptr[b] <= plan.max_slots, "most partial rows", n);
    }
    check(plan.partial_rows == slot_ptr[batch], "partial rows", n);
    check(plan.items_offset + static_cast<int64_t>(items.size()) * 64 <= plan.slot_ptr_offset &&
          plan.slot_ptr_offset + 4 * (batch + 1) <= plan.slot_base_offset &&
          plan.slot_base_offset + 4 * static_cast<int64_t>(slot_base.size()) <= plan.indptr_offset &&
          plan.indptr_offset <= plan.scores_offset && plan.scores_offset <= plan.partial_offset &&
          plan.partial_offset + plan.partial_rows * heads * 520 <= plan.workspace_bytes, "the workspace", n);
    if (selected)
      check(plan.partial_offset - plan.scores_offset >= 4ll * (own[batch] - own[0]) * hkv, "room for scores", n);
  }
  if (failures) return 1;
  std::printf("ok %d %d\n", plans, rejected);
  return 0;
}
