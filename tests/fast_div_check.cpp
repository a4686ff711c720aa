// CPU check of the page division (fe2o3_amd/csrc/kv_cache.hpp, FastDiv)
// against the division itself: every divisor up to 4096, then powers of two
// and their neighbours and pseudo-random divisors up to 2^31 - 1, each at the
// multiples of the divisor and one either side of them, spread over the whole
// range of n, and at the range's ends.
#include <stdio.h>

#include "../fe2o3_amd/csrc/kv_cache.hpp"

static unsigned long long bad = 0, tried = 0;

static void check(uint32_t d) {
  const kv_cache::FastDiv f = kv_cache::FastDiv::of(d);
  const uint32_t last = 0x7fffffffu;
  auto one = [&](uint64_t n) {
    if (n > last) return;
    ++tried;
    if (f.div((uint32_t)n) != (uint32_t)n / d) ++bad;
  };
  const uint64_t most = last / d;
  const uint64_t step = most / 500u + 1u;
  for (uint64_t q = 0; q <= most; q += step)
    for (int64_t e = -1; e <= 1; ++e) one(q * d + e);
  for (int64_t e = -1; e <= 1; ++e) one(most * d + e);
  for (uint64_t n = last - 64u; n <= last; ++n) one(n);
}

int main() {
  for (uint32_t d = 1; d <= 4096u; ++d) check(d);
  for (int b = 12; b < 31; ++b)
    for (int e = -2; e <= 2; ++e) check((1u << b) + e);
  check(0x7fffffffu);
  check(0x7ffffffeu);
  uint64_t x = 88172645463325252ull;
  for (int i = 0; i < 20000; ++i) {
    x ^= x << 13;
    x ^= x >> 7;
    x ^= x << 17;
    const uint32_t d = (uint32_t)(x & 0x7fffffffu) >> (i % 20);
    check(d == 0 ? 1 : d);
  }
  printf("tried %llu bad %llu\n", tried, bad);
  return bad == 0 ? 0 : 1;
}
