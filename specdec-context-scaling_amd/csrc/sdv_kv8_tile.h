// What the kernels that move rows into and out of the kv8 cache share (sdv_kv8_cache.hip, sdv_rope.hip): which
// page block a wavefront has, the quantization of a row, and the writing of a block's V.
#pragma once

#include "sdv_kv8.h"

namespace sdv {

struct Kv8CacheArgs {
  Kv8Rows r;
  const int32_t* pos;  // seq_lens (append: the rows end there) or starts (gather: they begin there)
  int32_t length;      // every sequence's length where an append's pos is nullptr
  void* k;             // packed BF16 rows
  void* v;
  int64_t k_stride, v_stride;  // elements between tokens
  uint8_t* k_pages;
  uint8_t* v_pages;
  float* scales;
  int kv_heads;
};

// The wavefront's page block: its sequence, logical block, and which tokens t0 <= t < t1 of the block
// are the call's, the first of them packed row `row` - t0.  ENDS: `pos` holds where the rows end.  SKIP: rows before
// position 0 are left out (else their blocks count on downwards, -1 and so on).
struct Kv8Tile {
  int b, block, t0, t1, row;
};

template <bool ENDS, bool SKIP = true>
__device__ __forceinline__ bool kv8_tile(const Kv8CacheArgs& a, int tile, Kv8Tile& out) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int base = 0; base < a.r.batch; base += kWave) {
    const int b = base + lane;
    int first = 0, n = 0, p0 = 0, count = 0;
    if (b < a.r.batch) {
      kv8_rows(a.r, b, first, n);
      if constexpr (ENDS) {
        p0 = max(a.pos ? a.pos[b] : a.length, 0) - n;
        const int skip = SKIP ? max(-p0, 0) : 0;  // rows before position 0 (a length below the row count) have no slot
        first += skip;
        n -= skip;
        p0 += skip;
      } else {
        p0 = min(max(a.pos[b], INT32_MIN / 2), INT32_MAX - a.r.total);  // no sum below overflows
      }
      if (n > 0) count = ((p0 + n - 1) >> 4) - (p0 >> 4) + 1;
    }
    const int end = (int)kv8_lane_scan((uint32_t)count);
    const uint64_t past = __ballot(tile < end);
    if (past != 0) {
      const int src = __builtin_ctzll(past);
      const int s_first = __builtin_amdgcn_readlane(first, src), s_n = __builtin_amdgcn_readlane(n, src),
                s_p0 = __builtin_amdgcn_readlane(p0, src);
      const int j = tile - (__builtin_amdgcn_readlane(end, src) - __builtin_amdgcn_readlane(count, src));
      out.b = base + src;
      out.block = (s_p0 >> 4) + j;
      out.t0 = max(s_p0 - out.block * kBlock, 0);
      out.t1 = min(s_p0 + s_n - out.block * kBlock, kBlock);
      out.row = s_first + out.block * kBlock - s_p0;  // row of the block's token 0
      return true;
    }
    tile -= __builtin_amdgcn_readlane(end, kWave - 1);
  }
  return false;
}

// ---------------------------------------------------------------------------- write
// Scale of a row from its max-abs bits; r = RN(1/s); fast: quotient_rn's codes equal the IEEE
// quotient's (tests/native/quotient_check.c walks Q = 448, tests/native/quotient_check_int8.c Q = 127).
template <int FMT>
__device__ __forceinline__ void kv8_scale(uint32_t ab, float& s, float& r, bool& fast, bool& finite) {
  const float amax = __uint_as_float(ab);
  float sc = amax / (FMT == kFp8 ? 448.0f : 127.0f);
  if (sc == 0.0f) sc = 1.0f;
  finite = ab < 0x7F800000u;
  fast = ab == 0 || (ab >= kFastMinAmaxBits && finite);
  s = finite ? sc : __builtin_nanf("");
  r = 1.0f / sc;
}

template <int FMT>
__device__ __forceinline__ uint32_t kv8_encode(float q) {
  if constexpr (FMT == kFp8) return e4m3fn_encode(q);
  return (uint32_t)(int)__builtin_rintf(q) & 0xFFu;
}

// Four quotients as codes, the first in the low byte.
template <int FMT>
__device__ __forceinline__ uint32_t kv8_pack4(float a, float b, float c, float d) {
  if constexpr (FMT == kFp8) {
    const uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, (int)w, true);
  } else {
    // adding 1.5 * 2^23 rounds to the nearest integer, ties to even, and leaves it in the low bits
    constexpr float kRound = 12582912.0f;
    const uint32_t ab = __builtin_amdgcn_perm(__float_as_uint(b + kRound), __float_as_uint(a + kRound), 0x0C0C0400u);
    const uint32_t cd = __builtin_amdgcn_perm(__float_as_uint(d + kRound), __float_as_uint(c + kRound), 0x0C0C0400u);
    return ab | cd << 16;
  }
}

__device__ __forceinline__ float bf16_at(uint4 v, int k) {
  const uint32_t w = (&v.x)[k >> 1];
  return (k & 1) ? bf16_hi(w) : bf16_lo(w);
}

// Max of bit patterns over each run of U (4 or 8) lanes, in all of them.
template <int U>
__device__ __forceinline__ uint32_t unit_max_bits(uint32_t v) {
  if constexpr (U == 8) return row_max_bits<8>(v);
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));  // quad [1,0,3,2]
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));  // quad [2,3,0,1]
}

// Tokens t.t0 .. t.t1 - 1 of a block's V, quantized and written: lane (r, p) of the wavefront has tokens r*J ..
// r*J+J-1, dimensions 8p .. 8p+7, in vw (whatever it has of tokens that are not the call's is not written).  lds_v: D
// pieces of 16 bytes, the wavefront's own.
template <int D, int FMT>
__device__ __forceinline__ void kv8_write_v(const Kv8Tile& t, const uint4 (&vw)[kBlock * D / 8 / kWave], uint8_t* vp, float* sp, uint4* lds_v) {
  constexpr int LPR = D / 8, RPW = kWave / LPR, J = kBlock / RPW;
  const int lane = threadIdx.x & (kWave - 1), r = lane / LPR, p = lane % LPR;
  float s[J], rcp[J];
  bool fast[J], finite[J];
#pragma unroll
  for (int j = 0; j < J; ++j)
    kv8_scale<FMT>(row_max_bits<LPR>(abs_max_bits8(vw[j])), s[j], rcp[j], fast[j], finite[j]);
  uint32_t packed[8];  // dimension 8p + k: token r*J + j's code in byte j
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < J; ++j) q[j] = fast[j] ? quotient_rn(bf16_at(vw[j], k), s[j], rcp[j]) : 0.0f;
    packed[k] = kv8_pack4<FMT>(q[0], q[1], q[2], q[3]);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    if (fast[j] || !finite[j]) continue;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      packed[k] = (packed[k] & ~(0xFFu << (8 * j))) | kv8_encode<FMT>(bf16_at(vw[j], k) / s[j]) << (8 * j);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int tok = r * J + j;
    if (p == 0 && tok >= t.t0 && tok < t.t1) sp[kBlock + tok] = s[j];
  }
  if (t.t1 - t.t0 < kBlock) {  // a sequence's first or last block: bytes
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int tok = r * J + j;
      if (tok < t.t0 || tok >= t.t1) continue;
#pragma unroll
      for (int k = 0; k < 8; ++k) vp[(8 * p + k) * kBlock + tok] = (uint8_t)(packed[k] >> (8 * j));
    }
    return;
  }
  uint8_t* mine = reinterpret_cast<uint8_t*>(lds_v);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint8_t* dst = mine + (8 * p + k) * kBlock + r * J;
    if (J == 4)
      *reinterpret_cast<uint32_t*>(dst) = packed[k];
    else
      *reinterpret_cast<uint16_t*>(dst) = (uint16_t)packed[k];
  }
  __syncthreads();
#pragma unroll
  for (int d = lane; d < D; d += kWave) reinterpret_cast<uint4*>(vp)[d] = lds_v[d];
}

// ---------------------------------------------------------------------------- host
// Checks and grid that the entry points share.  Every sequence's rows touch at most
// min(n, (n + 30) / 16) blocks, a wavefront each; a launch has fewer than 2^32 threads along x.
inline int64_t kv8_cache_tiles(int32_t total, int32_t batch) {
  const int64_t tiles = (int64_t)total / kBlock + 2 * (int64_t)batch;
  return tiles < total ? tiles : total;
}

inline int kv8_cache_check(const void* k, const void* v, int64_t k_stride, int64_t v_stride, int32_t total,
                           const void* k_pages, const void* v_pages, const float* scales, int32_t num_blocks,
                           int32_t format, const int32_t* table, int32_t max_blocks, const int32_t* cu,
                           const int32_t* pos, int32_t batch, int32_t kv_heads, int32_t head_dim) {
  if (!k || !v || !k_pages || !v_pages || !scales || !table || !cu) return SDV_ERR_NULL;
  if (total < 0 || num_blocks <= 0 || max_blocks <= 0 || batch <= 0 || kv_heads <= 0 || kv_heads > 65535) return SDV_ERR_SHAPE;
  if (max_blocks > INT32_MAX / kBlock || total > INT32_MAX / 2 || batch > INT32_MAX / 4) return SDV_ERR_SHAPE;
  if (kv8_cache_tiles(total, batch) >= (1LL << 32) / kWave) return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  if (format != SDV_KV8_FP8 && format != SDV_KV8_INT8) return SDV_ERR_UNSUPPORTED;
  const int64_t row = (int64_t)kv_heads * head_dim;
  if (k_stride < row || v_stride < row) return SDV_ERR_SHAPE;
  if (!aligned(k, 16) || !aligned(v, 16) || k_stride % 8 || v_stride % 8 || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
      !aligned(scales, 16) || !aligned(table, 4) || !aligned(cu, 4) || !aligned(pos, 4))
    return SDV_ERR_ALIGN;
  return SDV_OK;
}

inline Kv8CacheArgs kv8_cache_args(void* k, void* v, int64_t k_stride, int64_t v_stride, int32_t total, void* k_pages,
                                   void* v_pages, float* scales, int32_t num_blocks, const int32_t* table,
                                   int32_t max_blocks, const int32_t* cu, const int32_t* pos, int32_t length, int32_t batch,
                                   int32_t kv_heads) {
  return {{cu, table, max_blocks, num_blocks, batch, total}, pos, length, k, v, k_stride, v_stride,
          static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages), scales, kv_heads};
}

inline dim3 kv8_cache_grid(int32_t total, int32_t batch, int32_t kv_heads) {
  return dim3((unsigned)kv8_cache_tiles(total, batch), (unsigned)kv_heads);
}

}  // namespace sdv
