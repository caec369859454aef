// kv8_floor_sum of csrc/sdv_kv8_sums.h against the sum itself, term by term.  Prints "<sums> sums, <differences> differences".
#include <cstdio>
#define __device__
#define __forceinline__ inline
#include "sdv_kv8_sums.h"

static uint64_t sums, differences, state = 1;
static uint32_t draw(uint32_t n) {  // below n
  state = state * 6364136223846793005ull + 1442695040888963407ull;
  return (uint32_t)((state >> 33) % n);
}

template <int TR>
static void check(uint32_t most, uint32_t keys, uint32_t G, uint32_t b) {
  uint64_t want = 0;
  for (uint32_t i = 0; i < most; ++i) {
    want += ((uint64_t)TR * i + b) / ((uint64_t)keys * G);
    if (want >> 31) return;
    if (i < 300 || i + 1 == most) {
      ++sums;
      differences += sdv::kv8_floor_sum<TR>(i + 1, keys, G, b) != want;
    }
  }
}

template <int TR>
static void checks() {
  for (uint32_t G = 1; G <= 40; ++G)
    for (uint32_t unit = 0; unit < 6; ++unit)
      for (int turn = 0; turn < 12; ++turn) {
        const uint32_t keys = 64u << unit, ctx = turn < 4 ? turn : draw(turn < 8 ? 5000 : (1u << 30) / G);
        check<TR>(1 + draw(turn < 8 ? 300 : 20000), keys, G, ctx * G + TR + keys * G - 1);  // as the plan asks for it
        check<TR>(1 + draw(300), keys, G, draw(1u << 30));
      }
}

int main() {
  checks<16>();
  checks<32>();
  checks<256>();
  printf("%llu sums, %llu differences\n", (unsigned long long)sums, (unsigned long long)differences);
  return differences != 0;
}
