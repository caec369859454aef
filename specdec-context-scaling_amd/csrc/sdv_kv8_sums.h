// The sum of the units of a sequence's tiles, of which the i-th has ceil((ctx G + TR (i + 1)) / (keys G)) with TR
// rows a tile, G rows a token and `keys` keys a unit, TR and `keys` powers of two: a sum of floors.
#pragma once

#include <cstdint>

namespace sdv {

// Sum over i < n of floor((TR i + b) / (keys G)); n > 0, and the sum is below 2^31.
//
// With TR <= keys a term is floor((i + c) / q) for c = floor(b / TR) and q = keys G / TR.  Take out the whole part of
// c / q, n times.  Of the terms left, which are 0 .. t, all but the last stand q times (the 0s less often, but
// they add nothing): q t (t - 1) / 2, and t for each i past q t, with x = c mod q + n and t = floor(x / q).
//
// With R = TR / keys > 1 a term is floor((R i + c) / G) for c = floor(b / keys).  Take out the whole part of c / G.
// The terms rise in K = floor((R (n - 1) + c) / G) steps, and the k-th leaves the first ceil((k G - c) / R) terms below
// it: the sum is n K - sum over k of floor(z_k / R) with z_k = k G + R - 1 - c.  R floor(z / R) is z - z mod R, whose
// second part repeats after R steps.
template <int TR>
__device__ __forceinline__ uint32_t kv8_floor_sum(uint32_t n, uint32_t keys, uint32_t G, uint32_t b) {
  if (TR <= 64 || TR <= keys) {
    const uint32_t q = keys / TR * G, c = b / TR, whole = c / q;
    const uint32_t x = c - whole * q + n, t = x / q;
    return n * whole + q * (t * (t - 1) / 2) + t * (x - t * q);
  }
  const uint32_t R = TR / keys;
  uint32_t c = b / keys;
  const uint32_t whole = c / G;
  c -= whole * G;
  const uint32_t K = (R * (n - 1) + c) / G;
  const uint32_t z0 = R - 1 - c;  // modulo 2^32
  uint64_t left = 0;              // sum of z_k mod R over 1 <= k <= K
  for (uint32_t k = 1; k <= R; ++k) left += (uint64_t)((z0 + k * G) & (R - 1)) * (K / R + (k <= K % R));
  const uint64_t below = ((int64_t)(int32_t)z0 * K + (uint64_t)K * (K + 1) / 2 * G - left) / R;
  return n * whole + (uint32_t)((uint64_t)n * K - below);
}

}  // namespace sdv
