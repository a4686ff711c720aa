// CPU check of the e4m3 cache write's quotients (fe2o3_amd/csrc/kv_cache.hpp,
// RowScale): for every bf16 magnitude as a row's largest and bf16 values of both
// signs up to it, the code of the quotient is that of the division.  Every value
// within 2^22 of the largest (smaller ones are below a quarter of the least code's
// half), below that both zeros and every 61st.  Rows that RowScale leaves to the
// division are counted.
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "../fe2o3_amd/csrc/fp8_codec.hpp"
#include "../fe2o3_amd/csrc/kv_cache.hpp"

static float of_bf16(uint32_t b) {
  const uint32_t bits = b << 16;
  float f;
  memcpy(&f, &bits, 4);
  return f;
}
static uint8_t code(float f) {
  uint32_t bits;
  memcpy(&bits, &f, 4);
  return fe2o3::e4m3_from_bits(bits);
}

int main() {
  unsigned long long bad = 0, tried = 0, rows = 0;
#pragma omp parallel for reduction(+ : bad, tried, rows) schedule(dynamic, 64)
  for (int a = 0; a < 0x7f80; ++a) {
    const kv_cache::RowScale s(of_bf16(a));
    if (s.scale != fmaxf(of_bf16(a), 1.17549435e-38f) / 448.0f) ++bad;
    if (!s.usual) continue;
    ++rows;
    const int from = a > 22 * 128 ? a - 22 * 128 : 0;
    for (int m = 0; m <= a; m += m < from ? (m + 61 < from ? 61 : from - m) : 1)
      for (uint32_t sign = 0; sign <= 0x8000u; sign += 0x8000u) {
        const float x = of_bf16(m | sign);
        ++tried;
        if (code(s.quotient(x)) != code(x / s.scale)) ++bad;
      }
  }
  printf("rows %llu tried %llu bad %llu\n", rows, tried, bad);
  return bad == 0 ? 0 : 1;
}
