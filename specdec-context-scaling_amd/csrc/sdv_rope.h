// Rotary positions on the device: the angles of eight frequencies and the rotation of 16 dimensions.
//
// A pair (x, y) at position p becomes scale * (x cos t - y sin t, x sin t + y cos t), t = p * inv_freq[i].  The
// first `rotary` dimensions of a head are pairs, (i, i + rotary / 2) or, interleaved, (2i, 2i + 1); the rest pass.
//
// A unit is 16 dimensions whose pairs lie within it: two pieces of eight, rotary / 2 apart or side by side, of
// frequencies 8u .. 8u + 7.  Units from rotary / 16 on pass.
//
// The angle is taken in turns and in 64 bits, p * inv_freq / 2 pi less its nearest whole number, so that a far
// position loses nothing (2^20 radians would leave an fp32 angle 2^-4 off); what is left goes to fp32 (2^-24 of
// it) and through sincospi.
#pragma once

#include "sdv_internal.h"

namespace sdv {

struct RopeArgs {
  const double* inv_freq;  // radians per position, rotary / 2
  int units;               // rotary / 16
  float scale;
  float sign;              // -1: the inverse rotation (the transpose)
};

// Cosine and sine of frequency i at `pos`, with the scale and the sign.
__device__ __forceinline__ void rope_angle(const RopeArgs& r, int i, int pos, float& c, float& s) {
  const double p = (double)pos * 0.15915494309189535, f = r.inv_freq[i];  // 1 / (2 pi)
  sincospif(2.0f * (float)__builtin_fma(p, f, -rint(p * f)), &s, &c);
  c *= r.scale;
  s *= r.scale * r.sign;
}

// First dimension of a unit's two pieces.
template <bool IL>
__device__ __forceinline__ int rope_piece(const RopeArgs& r, int u, int which) {
  if (IL || u >= r.units) return 16 * u + 8 * which;
  return 8 * (u + which * r.units);
}

// A unit's 16 values, rotated, in fp32.
template <bool IL>
__device__ __forceinline__ void rope_rotate(uint4 w0, uint4 w1, const float* c, const float* s, float (&y)[16]) {
  const auto at = [&](int k) {
    const uint32_t w = k < 8 ? (&w0.x)[k >> 1] : (&w1.x)[(k & 7) >> 1];
    return (k & 1) ? bf16_hi(w) : bf16_lo(w);
  };
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int a = IL ? 2 * i : i, b = IL ? 2 * i + 1 : i + 8;
    const float x0 = at(a), x1 = at(b);
    y[a] = __builtin_fmaf(x0, c[i], -(x1 * s[i]));  // written out, so that every kernel rounds alike
    y[b] = __builtin_fmaf(x0, s[i], x1 * c[i]);
  }
}

__device__ __forceinline__ uint4 rope_pack8(const float* y) {
  return make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
}

// What the entry points refuse.
inline int rope_check(const void* inv_freq, int32_t rotary_dim, int32_t interleaved, int32_t head_dim) {
  if (!inv_freq) return SDV_ERR_NULL;
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % 16 || interleaved < 0 || interleaved > 1) return SDV_ERR_SHAPE;
  return reinterpret_cast<uintptr_t>(inv_freq) % 8 ? SDV_ERR_ALIGN : SDV_OK;
}

}  // namespace sdv
