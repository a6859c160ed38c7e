// What the forms of the 16-bit experts' products read of tensor memory and of
// shared memory, against what they have there.  Built and run by
// tests/test_experts_shapes.py (no GPU needed).  Prints a line for each read
// that goes too far, then "ok" if there was none.
#include <cstdint>
#include <cstdio>

#include "cusort_experts.cuh"

using namespace cusort_b200;

static int bad = 0;

#define EXPECT(name, condition, ...)      \
  do {                                    \
    if (!(condition)) {                   \
      ++bad;                              \
      std::printf("%s: ", name);          \
      std::printf(__VA_ARGS__);           \
      std::printf("\n");                  \
    }                                     \
  } while (0)

template <typename Shape>
static void check(const char* name) {
  const int columns = Shape::kColumns, own = Shape::kSumColumns;
  EXPECT(name, columns >= 32 && columns <= 512 && (columns & (columns - 1)) == 0,
         "%d columns of tensor memory cannot be allocated", columns);
  // the instruction's width, in whole steps, and what the storing warps read, 32 columns at a time
  for (int rows = 1; rows <= Shape::kRows; ++rows) {
    const int width = (rows + Shape::kRowStep - 1) / Shape::kRowStep * Shape::kRowStep;
    EXPECT(name, width <= own, "sums of %d rows fill %d columns of %d", rows, width, own);
    for (int sum = 0; sum < 2; ++sum)
      for (int c = 0; c < rows; c += kSumLoad) {
        const int begin = sum * own + c, end = begin + kSumLoad;
        EXPECT(name, end <= columns, "columns %d to %d are read of sum %d, %d are allocated", begin, end - 1, sum,
               columns);
        EXPECT(name, end <= (sum + 1) * own, "columns %d to %d are read of sum %d, the other's among them", begin,
               end - 1, sum);
      }
  }
  // 128 lanes of weights: of 64 columns the rest is what lies behind, up to the end of what the stages and the
  // storing warps have
  const uint32_t last = (Shape::kStages - 1) * Shape::kStage + (Shape::kSub - 1) * Shape::kStep;
  const uint32_t end = last + kTileM * kBlockK * 2, there = Shape::kStages * Shape::kStage + Shape::kStaging;
  EXPECT(name, end <= there, "weights are read up to byte %u of %u", end, there);
}

int main() {
  check<ProductFewestNarrow>("fewest rows, 64 columns");
  check<ProductFewest>("fewest rows");
  check<ProductFew>("few rows");
  check<ProductMany>("many rows");
  if (bad == 0) std::printf("ok\n");
  return bad != 0;
}
