// The paged cache's index arithmetic on the host: prints "ok" or the first fault.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include "kernels/paged_common.h"

using namespace grxk;

static void fail(const char* what, long long a, long long b) {
  std::printf("%s: %lld %lld\n", what, a, b);
  std::exit(1);
}

int main() {
  // Division by every page size up to 4096 and around the powers of two.
  std::vector<int> sizes;
  for (int d = 1; d <= 4096; ++d) sizes.push_back(d);
  for (int b = 12; b < 31; ++b)
    for (int e = -2; e <= 2; ++e) sizes.push_back((1 << b) + e);
  sizes.push_back(0x7fffffff - 255);
  for (int d : sizes) {
    const PageDiv v = page_div(d);
    auto check = [&](long long n) {
      if (n >= 0 && n <= 0x7fffffff && div_page(v, (int)n) != n / d) fail("division", n, d);
    };
    const long long last = 0x7fffffff / d;
    for (long long q : {0ll, 1ll, 2ll, 3ll, 1000ll, last / 2, last - 1, last})
      for (int e = -2; e <= 2; ++e) check(q * d + e);
    check(0x7fffffff);
    unsigned x = 12345u + (unsigned)d;
    for (int i = 0; i < 200; ++i) {
      x = x * 1664525u + 1013904223u;
      check(x >> 1);
    }
  }
  // Slots of two sequences of room 20 on 9 pages of 5, some of which do not exist.
  const int table[2 * 6] = {8, 0, -1, 3, 77, 77, 9, 2147483647, -2147483647 - 1, 5, 77, 77};
  const int lengths[2] = {0, 0};
  const PagedView v = {table, 6, lengths, 9, 5, 20, page_div(5)};
  const int want[2][4] = {{8, 0, -1, 3}, {-1, -1, -1, 5}};
  for (int b = 0; b < 2; ++b)
    for (int slot = 0; slot < 40; ++slot) {
      int page = -2, row = -2;
      const bool there = find_slot(v, b, slot, &page, &row);
      const bool should = slot < 20 && want[b][slot / 5] >= 0;
      if (there != should) fail("slot", b, slot);
      if (there && (page != want[b][slot / 5] || row != slot % 5)) fail("place", b, slot);
    }
  for (int n : {-2147483647 - 1, -1, 0, 1, 19, 20, 21, 2147483647})
    if (clamp_length(n, 20) != (n < 0 ? 0 : n > 20 ? 20 : n)) fail("length", n, 20);
  // Order of the weights' keys.
  const float up[] = {-__builtin_inff(), -3e38f, -1.0f, -1e-45f, 0.0f, 1e-45f, 1.0f, 1.0000001f, 3e38f,
                      __builtin_inff(), __builtin_nanf("")};
  auto key = [](float f) {
    uint32_t u;
    std::memcpy(&u, &f, 4);
    return order_key(u);
  };
  for (int i = 0; i + 1 < (int)(sizeof up / sizeof up[0]); ++i)
    if (key(up[i]) >= key(up[i + 1])) fail("order", i, i + 1);
  if (key(0.0f) != key(-0.0f)) fail("zeros", 0, 0);
  if (key(-__builtin_nanf("")) != key(__builtin_nanf(""))) fail("nan", 0, 0);
  std::printf("ok\n");
  return 0;
}
