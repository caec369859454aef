// The 8-bit KV cache (kv8): page layout, code conversions and the arguments its kernels share.
//
// Per block of 16 tokens and KV head, one byte a value (E4M3FN or two's-complement int8):
//   K [4][D/16][4][16]  token 4p + r, dimension 16c + j at [p][c][r][j]
//   V [D][16]           dimension-major
//   scales [2][16]      fp32, K's 16 tokens, then V's
// The attention kernels take the codes as BF16 MFMA operands (every code is exact in BF16).  K's
// order makes the 16 key rows of one 16x16x32 MFMA -- four tokens 4p..4p+3 from each of four blocks
// -- 256-byte runs in memory, and leaves lane group g of the product with all of block g's tokens,
// which is what the V operand of the next product needs: no lane exchange between the two.
//
// Codes are always finite: a row that holds an infinity or a NaN has codes 0 and scale NaN.  It
// reads back as NaN, gives NaN to every query that sees it, and nothing to one that does not.
#pragma once

#include "sdv_internal.h"

namespace sdv {

constexpr int kFp8 = SDV_KV8_FP8, kInt8 = SDV_KV8_INT8;

// Where the rows of each sequence lie: rows cu[b] .. cu[b+1]-1 of the packed tensors.  Entries are
// clamped to the tensor, so that no value reads or writes past it.
struct Kv8Rows {
  const int32_t* cu;
  const int32_t* table;
  int32_t max_blocks;
  int32_t num_blocks;
  int32_t batch;
  int32_t total;
};

__device__ __forceinline__ void kv8_rows(const Kv8Rows& r, int b, int& first, int& n) {
  first = min(max(r.cu[b], 0), r.total);
  n = min(max(r.cu[b + 1], 0), r.total) - first;
  if (n < 0) n = 0;
}

// Physical block of logical block j of sequence b, or -1.
__device__ __forceinline__ int kv8_block(const Kv8Rows& r, int b, int j) {
  if (j < 0 || j >= r.max_blocks) return -1;
  const int id = r.table[(int64_t)b * r.max_blocks + j];
  return id >= 0 && id < r.num_blocks ? id : -1;
}

// Eight codes (two dwords) as BF16, exactly.
template <int FMT>
__device__ __forceinline__ bf16x8 kv8_bf16x8(uint32_t lo, uint32_t hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  uint4 w;
  if constexpr (FMT == kFp8) {
    w.x = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    w.y = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    w.z = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    w.w = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    // an integer up to 127 has at most seven bits: BF16 is the upper half of its fp32
    const auto pair = [](uint32_t a, uint32_t b) {
      return __builtin_amdgcn_perm(__float_as_uint((float)(int8_t)b), __float_as_uint((float)(int8_t)a), 0x07060302u);
    };
    w.x = pair(lo, lo >> 8);
    w.y = pair(lo >> 16, lo >> 24);
    w.z = pair(hi, hi >> 8);
    w.w = pair(hi >> 16, hi >> 24);
  }
  return __builtin_bit_cast(bf16x8, w);
}

// Code in byte `sel` of a dword as fp32 (sel is a constant after unrolling).
template <int FMT>
__device__ __forceinline__ float kv8_decode(uint32_t w, int sel) {
  if constexpr (FMT == kFp8) return e4m3fn_decode(w, sel);
  return (float)(int8_t)(w >> (8 * sel));
}

// Inclusive sum over a wavefront's lanes (DPP row shifts, then row broadcasts).
__device__ __forceinline__ uint32_t kv8_lane_scan(uint32_t x) {
  int v = (int)x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return (uint32_t)v;
}

}  // namespace sdv
