// Which keys rows of packed attention look through one by one: all that stand in front of them or at their place, none behind the text's last one.
#include "../../csrc/ops/packed_keys.hpp"
#include "_test.h"

using namespace mccl::ops::packed;

TEST_CASE(rows_of_a_tile_stay_within_the_keys_of_their_text) {
  for (int m : {1, 2, 28, 100, 127, 128, 129, 255, 256, 257, 412}) {
    // a tile's 128 rows from any of the text's positions on: the last ones may stand up to 127 positions behind its keys
    for (int pos = -130; pos < m + kRows; ++pos) {
      for (int b = 0; b * kRows < m; ++b) {
        const BlockKeys keys = block_keys(b, pos, m);
        CHECK(keys.first == b * kRows);
        for (int j = b * kRows; j < (b + 1) * kRows; ++j) CHECK((j < keys.end) == (j < m && j <= pos));
        CHECK(keys.end <= m && keys.end <= (b + 1) * kRows);
      }
    }
  }
}

int main() { return run_all_tests(); }
