// The window of a mask that a step of keys sees (csrc/paged_model.hpp), bit by bit, on the host.
#include <cstdio>
#include <random>
#include <vector>

#include "paged_model.hpp"

int main() {
  std::mt19937 rng(1);
  for (int words : {1, 2, 3, 5, 32}) {
    std::vector<uint32_t> m(words);
    for (uint32_t& x : m) x = rng();
    for (int j0 = -200; j0 < 32 * words + 200; ++j0) {
      const uint32_t got = pa::mask_window(j0, words, [&](int i) {
        if (i < 0 || i >= words) std::printf("word %d of %d is read\n", i, words), std::exit(1);
        return m[i];
      });
      for (int b = 0; b < 32; ++b) {
        const int j = j0 + b;
        const uint32_t want = j < 0 ? 1 : j < 32 * words ? m[j / 32] >> j % 32 & 1 : 0;
        if ((got >> b & 1) != want) return std::printf("words %d, j0 %d, bit %d\n", words, j0, b), 1;
      }
    }
    for (int j0 : {-(1 << 30), (1 << 30)})   // far before and behind
      if (pa::mask_window(j0, words, [&](int) { return 0u; }) != (j0 < 0 ? ~0u : 0u)) return std::printf("far %d\n", j0), 1;
  }
  std::puts("ok");
}
