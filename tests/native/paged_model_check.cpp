// Host checks of the paged cache's index arithmetic (csrc/paged_model.hpp): page numbers against plain
// division, and a sequence's rows and visible keys under offsets and lengths of any value.
#include "paged_model.hpp"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <initializer_list>

#define CHECK(x)                                                        \
  do {                                                                  \
    if (!(x)) {                                                         \
      std::printf("line %d: %s\n", __LINE__, #x);                       \
      std::exit(1);                                                     \
    }                                                                   \
  } while (0)

static uint32_t rnd() {
  static uint64_t s = 88172645463325252ull;
  s ^= s << 13, s ^= s >> 7, s ^= s << 17;
  return (uint32_t)(s >> 16);
}

int main() {
  const uint32_t top = 1u << 30;
  auto check_div = [&](uint32_t d) {
    const pa::PageDiv p = pa::make_page_div(d);
    auto one = [&](uint64_t n) { CHECK(n >= 2ull * top || pa::page_of((uint32_t)n, p) == n / d); };
    for (uint64_t n = 0; n < 200; ++n) one(n);
    for (uint64_t q = 1; q * d < 2ull * top && q < 300; ++q) one(q * d - 1), one(q * d), one(q * d + 1);
    for (int i = 0; i < 200; ++i) one(rnd() % (2ull * top));
    one(2ull * top - 1), one(2ull * top - 2), one((2ull * top - 1) / d * d), one((2ull * top - 1) / d * d - 1);
  };
  for (uint32_t d = 1; d < 5000; ++d) check_div(d);
  for (int i = 0; i < 5000; ++i) check_div(rnd() % top + 1);
  for (uint32_t d : {top, top - 1, top / 2, top / 2 + 1, 65535u, 65536u, 65537u}) check_div(d);

  const int odd[] = {INT32_MIN, INT32_MIN + 1, -1000, -1, 0, 1, 2, 7, 63, 64, 1000, (1 << 30) - 1, 1 << 30, INT32_MAX};
  for (int tokens : {1, 2, 64, 1000, 1 << 30})
    for (int b : odd)
      for (int e : odd)
        for (int len : odd) {
          const pa::SeqRows s = pa::seq_rows(b, e, len, tokens);
          CHECK(s.first >= 0 && s.count >= 0 && (int64_t)s.first + s.count <= tokens && s.length >= 0);
          for (int cap : {1, 64, 1 << 30})
            for (int i : {0, s.count / 2, s.count - 1}) {
              if (i < 0) continue;
              const int64_t pos = (int64_t)s.length - s.count + i;
              CHECK(pa::new_token_pos(s, i) == pos);
              const int64_t c = pos + 1 < 0 ? 0 : pos + 1 > cap ? cap : pos + 1;
              CHECK(pa::keys_seen(s, i, cap, true) == c);
              CHECK(pa::keys_seen(s, i, cap, false) == (s.length < cap ? s.length : cap));
            }
        }
  std::printf("ok\n");
  return 0;
}
