// Host check of the length that the division of work counts for a sequence (csrc/paged_model.hpp), up to the
// largest capacities, counts and lengths that a call may have.
#include "paged_model.hpp"

#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#define CHECK(x)                                                        \
  do {                                                                  \
    if (!(x)) {                                                         \
      std::printf("line %d: %s\n", __LINE__, #x);                       \
      std::exit(1);                                                     \
    }                                                                   \
  } while (0)

int main() {
  const int top = (int)pa::kPagedMaxPos;
  const int sizes[] = {0, 1, 2, 63, 64, 1000, top / 2, top / 2 + 1, top - 1, top};
  for (int capacity : sizes)
    for (int count : sizes)
      for (int length : sizes) {
        if (capacity == 0) continue;
        const pa::SeqRows s = pa::seq_rows(0, count, length, top);
        const pa::SeqRows w = pa::held_rows(s, capacity);
        CHECK(w.first == s.first && w.count == s.count);
        CHECK(w.length == std::min<int64_t>(length, (int64_t)capacity + count));
        for (int i : {0, count / 2, count - 1}) {   // the same keys, and the same places within the capacity
          if (i < 0 || i >= count) continue;
          CHECK(pa::keys_seen(w, i, capacity, true) == pa::keys_seen(s, i, capacity, true));
          CHECK(pa::keys_seen(w, i, capacity, false) == pa::keys_seen(s, i, capacity, false));
          const int a = pa::new_token_pos(s, i), b = pa::new_token_pos(w, i);
          CHECK(a == b || (a >= capacity && b >= capacity));
        }
        const pa::TileShape t = pa::make_tiles(1, 16);
        CHECK(pa::tiles_cost(w, t, false, pa::tiles_of(w, t)) >= 0 && pa::tiles_cost(w, t, true, pa::tiles_of(w, t)) >= 0);
      }
  std::printf("ok\n");
  return 0;
}
