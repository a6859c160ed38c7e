// Which rows of the experts' products are cleared: those of no segment, each
// once or more, and none of a segment, whatever the segments' order; and which
// rows a segment has.  Built and run by tests/test_experts_shapes.py (no GPU needed).  Prints "ok".
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "cusort_experts.cuh"

using namespace cusort_b200;

struct OneLane {
  int lane = 0, count = 1;
  int highest(int v) const { return v; }
  int lowest(int v) const { return v; }
};

static int bad = 0;

// A plan of segments that do not overlap: shuffled experts, gaps between them, rows behind; empty experts anywhere.
static void check(int experts, int most, int gap, int all, bool shuffled, unsigned seed) {
  std::mt19937 rng(seed);
  std::vector<int> order(experts), first(experts), count(experts);
  for (int e = 0; e < experts; ++e) order[e] = e;
  if (shuffled) std::shuffle(order.begin(), order.end(), rng);
  int at = gap ? rng() % (gap + 1) : 0;
  for (int e : order) {
    count[e] = rng() % 3 ? rng() % (most + 1) : 0;
    first[e] = at;
    at += count[e] + (gap ? rng() % (gap + 1) : 0);
  }
  for (int e : order)
    if (count[e] == 0 && shuffled) first[e] = rng() % (at + 1);
  const int capacity = at;
  std::vector<int> cleared(capacity, 0);
  const Segments s{first.data(), count.data(), nullptr};
  for (int me = 0; me < all; ++me)
    other_rows(s, experts, capacity, me, all, OneLane(), [&](int begin, int end) {
      if (begin < 0 || begin > end || end > capacity) {
        ++bad;
        std::printf("rows %d to %d of %d\n", begin, end, capacity);
        return;
      }
      for (int r = begin; r < end; ++r) ++cleared[r];
    });
  std::vector<int> there(capacity, 0);
  for (int e = 0; e < experts; ++e)
    for (int r = first[e]; r < first[e] + count[e]; ++r) ++there[r];
  for (int r = 0; r < capacity; ++r)
    if ((cleared[r] > 0) != (there[r] == 0)) {
      if (++bad < 20)
        std::printf("%d experts, seed %u: row %d is %s\n", experts, seed, r, there[r] ? "cleared" : "left");
    }
}

// As many rows as there may be, of which the first ones belong to an expert: the parts begin and end where they should.
static void check_most(int capacity, int taken, int all) {
  int first = 0, count = taken;
  const Segments s{&first, &count, nullptr};
  int64_t next = taken;
  for (int me = 0; me < all; ++me)
    other_rows(s, 1, capacity, me, all, OneLane(), [&](int begin, int end) {
      if (begin == end) return;  // before a segment that begins at row 0
      if (begin != next || end < begin || end > capacity) {
        ++bad;
        std::printf("part %d of %d: rows %d to %d of %d, %lld come next\n", me, all, begin, end, capacity,
                    (long long)next);
      }
      next = end;
    });
  if (next != capacity) ++bad, std::printf("%lld of %d rows\n", (long long)next, capacity);
}

// The rows r with offset <= r < offset + count, of those there are.
static void check_segment(int offset, int count, int capacity) {
  const SegmentArgs a{&count, &offset, 1, capacity};
  const int2 got = segment(a, 0);
  const int64_t begin = std::max<int64_t>(offset, 0), end = std::min<int64_t>((int64_t)offset + count, capacity);
  const int64_t rows = std::max<int64_t>(end - begin, 0);
  if (got.y != rows || (rows > 0 && got.x != begin) || got.x < 0 || got.x > capacity) {
    ++bad;
    std::printf("offset %d, count %d of %d rows: %d from %d on\n", offset, count, capacity, got.y, got.x);
  }
}

int main() {
  for (int capacity : {1, 40, INT32_MAX - 1025})
    for (int offset : {0, 1, 39, 40, 41, -1, -5, -100, INT32_MAX, INT32_MIN, -INT32_MAX})
      for (int count : {0, 1, 5, 6, 40, 41, 140, 1 << 30, INT32_MAX, -1, INT32_MIN})
        check_segment(offset, count, capacity);
  for (int capacity : {INT32_MAX - 1024, INT32_MAX - 1500, INT32_MAX - 5000})
    for (int taken : {0, 1, 700})
      for (int all : {1, 148, 2368, 4736}) check_most(capacity, taken, all);
  for (unsigned seed = 0; seed < 40; ++seed)
    for (int experts : {1, 2, 7, 64, 300})
      for (int gap : {0, 5})
        for (int all : {1, 6, 148, 1184}) check(experts, 9, gap, all, seed % 4 != 0, seed);
  if (bad == 0) std::printf("ok\n");
  return bad != 0;
}
