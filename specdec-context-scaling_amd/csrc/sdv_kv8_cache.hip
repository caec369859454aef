// The 8-bit KV cache's write and read-back (layout and codes: sdv_kv8.h).
//
// Write: per (token, KV head) and for K and V alike, m = max|x|, s = m / Q with Q = 448 (E4M3FN) or
// 127 (int8), an IEEE fp32 division, 1 for a row of zeros; code = RNE(x / s).  A row whose maximum is
// not finite has scale NaN and codes 0.  Read-back: bf16(code * s), one fp32 product.
//
// Both kernels give one wavefront one page block of one sequence and KV head, whichever of the call's
// rows fall in it (the rows of a sequence are consecutive positions, so a block's rows lie together
// in the packed tensors).  Whole blocks then move in 16-byte pieces wherever a sequence starts in the
// packed tensor; only a sequence's first and last block are written in bytes.  A wavefront finds its
// block by a scan over the sequences' block counts.
//
// Bound by memory where there is enough to move: reading 112,000 positions of 16 sequences back (174 MB
// read and written, 2 x 128) takes 30 to 34 us, 5.1 to 5.8 TB/s, a large copy's rate.  Small calls are three
// loads one after another (lengths, block id, rows) between the ends of a launch: 32 tokens 4.8 us, a
// chunk of 2048 5.3, of which a kernel that does nothing but a small fill is 1.8 (GPU time in a graph;
// eager calls 4.7 and 5.1).  A workgroup is one wavefront, so that a chunk of 2048 rows is 256 of them.
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
// are the call's, the first of them packed row `row` - t0.  ENDS: `pos` holds where the rows end.
struct Kv8Tile {
  int b, block, t0, t1, row;
};

template <bool ENDS>
__device__ __forceinline__ bool kv8_tile(const Kv8CacheArgs& a, int tile, Kv8Tile& out) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int base = 0; base < a.r.batch; base += kWave) {
    const int b = base + lane;
    int first = 0, n = 0, p0 = 0, count = 0;
    if (b < a.r.batch) {
      kv8_rows(a.r, b, first, n);
      if constexpr (ENDS) {
        p0 = max(a.pos ? a.pos[b] : a.length, 0) - n;
        const int skip = max(-p0, 0);  // rows before position 0 (a length below the row count) have no slot
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

template <int D, int FMT>
__global__ __launch_bounds__(64) void kv8_append_kernel(Kv8CacheArgs a) {
  constexpr int LPR = D / 8;        // lanes per token row: 16 bytes of BF16 each
  constexpr int RPW = kWave / LPR;  // token rows per wave-wide load (4 or 8)
  constexpr int J = kBlock / RPW;   // loads (4 or 2)
  __shared__ uint4 lds_v[D];        // V codes of the block, [D][16]

  Kv8Tile t;
  if (!kv8_tile<true>(a, (int)blockIdx.x, t)) return;  // wave-uniform
  const int id = kv8_block(a.r, t.b, t.block);
  if (id < 0) return;
  const int lane = threadIdx.x, r = lane / LPR, p = lane % LPR, kvh = blockIdx.y;
  const uint16_t* kin = static_cast<const uint16_t*>(a.k) + kvh * D + 8 * p;
  const uint16_t* vin = static_cast<const uint16_t*>(a.v) + kvh * D + 8 * p;
  const int64_t page = (int64_t)id * a.kv_heads + kvh;
  uint8_t* kp = a.k_pages + page * (kBlock * D);
  uint8_t* vp = a.v_pages + page * (kBlock * D);
  float* sp = a.scales + page * (2 * kBlock);

  // V: lane (r, p) holds tokens r*J .. r*J+J-1, so that it packs their codes per dimension; K: token
  // j*RPW + r in load j, so that the lanes of one store hold consecutive bytes of the page.  Tokens
  // that are not the call's re-read a row that is.
  uint4 kw[J], vw[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int kt = min(max(j * RPW + r, t.t0), t.t1 - 1), vt = min(max(r * J + j, t.t0), t.t1 - 1);
    kw[j] = load_stream16(kin + (int64_t)(t.row + kt) * a.k_stride);
    vw[j] = load_stream16(vin + (int64_t)(t.row + vt) * a.v_stride);
  }

  // K
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int tok = j * RPW + r;
    float s, rcp;
    bool fast, finite;
    kv8_scale<FMT>(row_max_bits<LPR>(abs_max_bits8(kw[j])), s, rcp, fast, finite);
    float q[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) q[k] = fast ? quotient_rn(bf16_at(kw[j], k), s, rcp) : 0.0f;
    uint2 c = make_uint2(kv8_pack4<FMT>(q[0], q[1], q[2], q[3]), kv8_pack4<FMT>(q[4], q[5], q[6], q[7]));
    if (!fast && finite) {  // max-abs in (0, 2^-60): the IEEE division, value by value (rare)
      c = make_uint2(0, 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) (&c.x)[k >> 2] |= kv8_encode<FMT>(bf16_at(kw[j], k) / s) << (8 * (k & 3));
    }
    if (tok >= t.t0 && tok < t.t1) {
      *reinterpret_cast<uint2*>(kp + (tok >> 2) * (4 * D) + (p >> 1) * 64 + (tok & 3) * 16 + (p & 1) * 8) = c;
      if (p == 0) sp[tok] = s;
    }
  }

  // V
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

// ---------------------------------------------------------------------------- read-back
// The rows are written past the caches' reused lines: what is read back is mostly more than they hold
// (112,000 positions 35.6 -> 32.2 us, 8192 4.8 -> 4.3; with K's codes read that way too 33.9 and 4.4).
__device__ __forceinline__ void kv8_store_stream(uint16_t* p, uint4 v) {
  __builtin_nontemporal_store(u32x4_t{v.x, v.y, v.z, v.w}, reinterpret_cast<u32x4_t*>(p));
}

template <int D, int FMT>
__global__ __launch_bounds__(64) void kv8_gather_kernel(Kv8CacheArgs a) {
  constexpr int LPR = D / 8, RPW = kWave / LPR, J = kBlock / RPW;
  // V codes, [D][16], with 16 bytes between runs of eight dimensions: the lanes of a read lie 144
  // bytes apart and meet 64 different banks
  __shared__ uint4 lds_v[D + D / 8];

  Kv8Tile t;
  if (!kv8_tile<false>(a, (int)blockIdx.x, t)) return;
  const int id = kv8_block(a.r, t.b, t.block);
  const int lane = threadIdx.x, r = lane / LPR, p = lane % LPR, kvh = blockIdx.y;
  uint16_t* kout = static_cast<uint16_t*>(a.k) + kvh * D + 8 * p;
  uint16_t* vout = static_cast<uint16_t*>(a.v) + kvh * D + 8 * p;
  if (id < 0) {  // no such block: zeros
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int tok = j * RPW + r;
      if (tok < t.t0 || tok >= t.t1) continue;
      *reinterpret_cast<uint4*>(kout + (int64_t)(t.row + tok) * a.k_stride) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(vout + (int64_t)(t.row + tok) * a.v_stride) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const int64_t page = (int64_t)id * a.kv_heads + kvh;
  const uint8_t* kp = a.k_pages + page * (kBlock * D);
  const uint8_t* vp = a.v_pages + page * (kBlock * D);
  const float* sp = a.scales + page * (2 * kBlock);
  uint2 kw[J];
  float ks[J], vs[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int tok = j * RPW + r;
    kw[j] = *reinterpret_cast<const uint2*>(kp + (tok >> 2) * (4 * D) + (p >> 1) * 64 + (tok & 3) * 16 + (p & 1) * 8);
    ks[j] = sp[tok];
    vs[j] = sp[kBlock + r * J + j];
  }
#pragma unroll
  for (int d = lane; d < D; d += kWave) lds_v[d + d / 8] = load_stream16(vp + d * kBlock);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int tok = j * RPW + r;
    uint4 o;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
      const uint32_t w = (&kw[j].x)[k >> 2];
      (&o.x)[k >> 1] = pack_bf16x2(kv8_decode<FMT>(w, k & 3) * ks[j], kv8_decode<FMT>(w, (k & 3) + 1) * ks[j]);
    }
    if (tok >= t.t0 && tok < t.t1) kv8_store_stream(kout + (int64_t)(t.row + tok) * a.k_stride, o);
  }
  uint32_t packed[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(lds_v) + (8 * p + k + p) * kBlock + r * J;
    packed[k] = J == 4 ? *reinterpret_cast<const uint32_t*>(src) : *reinterpret_cast<const uint16_t*>(src);
  }
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int tok = r * J + j;
    uint4 o;
#pragma unroll
    for (int k = 0; k < 8; k += 2)
      (&o.x)[k >> 1] = pack_bf16x2(kv8_decode<FMT>(packed[k], j) * vs[j], kv8_decode<FMT>(packed[k + 1], j) * vs[j]);
    if (tok >= t.t0 && tok < t.t1) kv8_store_stream(vout + (int64_t)(t.row + tok) * a.v_stride, o);
  }
}

}  // namespace sdv

using namespace sdv;

// Checks and grid that both entry points share.  Every sequence's rows touch at most
// min(n, (n + 30) / 16) blocks.
static int kv8_cache_check(const void* k, const void* v, int64_t k_stride, int64_t v_stride, int32_t total,
                           const void* k_pages, const void* v_pages, const float* scales, int32_t num_blocks,
                           int32_t format, const int32_t* table, int32_t max_blocks, const int32_t* cu,
                           const int32_t* pos, int32_t batch, int32_t kv_heads, int32_t head_dim) {
  if (!k || !v || !k_pages || !v_pages || !scales || !table || !cu) return SDV_ERR_NULL;
  if (total < 0 || num_blocks <= 0 || max_blocks <= 0 || batch <= 0 || kv_heads <= 0 || kv_heads > 65535) return SDV_ERR_SHAPE;
  if (max_blocks > INT32_MAX / kBlock || total > INT32_MAX / 2 || batch > INT32_MAX / 4) return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  if (format != SDV_KV8_FP8 && format != SDV_KV8_INT8) return SDV_ERR_UNSUPPORTED;
  const int64_t row = (int64_t)kv_heads * head_dim;
  if (k_stride < row || v_stride < row) return SDV_ERR_SHAPE;
  if (!aligned(k, 16) || !aligned(v, 16) || k_stride % 8 || v_stride % 8 || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
      !aligned(scales, 16) || !aligned(table, 4) || !aligned(cu, 4) || !aligned(pos, 4))
    return SDV_ERR_ALIGN;
  return SDV_OK;
}

static Kv8CacheArgs kv8_cache_args(void* k, void* v, int64_t k_stride, int64_t v_stride, int32_t total, void* k_pages,
                                   void* v_pages, float* scales, int32_t num_blocks, const int32_t* table,
                                   int32_t max_blocks, const int32_t* cu, const int32_t* pos, int32_t length, int32_t batch,
                                   int32_t kv_heads) {
  return {{cu, table, max_blocks, num_blocks, batch, total}, pos, length, k, v, k_stride, v_stride,
          static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages), scales, kv_heads};
}

static dim3 kv8_cache_grid(int32_t total, int32_t batch, int32_t kv_heads) {
  const int64_t tiles = (int64_t)total / kBlock + 2 * (int64_t)batch;
  return dim3((unsigned)(tiles < total ? tiles : total), (unsigned)kv_heads);
}

extern "C" int sdv_kv8_append(const void* k_new, const void* v_new, int64_t k_stride, int64_t v_stride, int32_t total_rows,
                              void* k_pages, void* v_pages, float* scales, int32_t num_blocks, int32_t format,
                              const int32_t* block_table, int32_t max_blocks_per_seq, const int32_t* cu_rows,
                              const int32_t* seq_lens, int32_t max_seq_len, int32_t batch, int32_t kv_heads,
                              int32_t head_dim, void* stream) {
  if (!seq_lens && max_seq_len <= 0) return SDV_ERR_SHAPE;
  const int st = kv8_cache_check(k_new, v_new, k_stride, v_stride, total_rows, k_pages, v_pages, scales, num_blocks, format,
                                 block_table, max_blocks_per_seq, cu_rows, seq_lens, batch, kv_heads, head_dim);
  if (st != SDV_OK || total_rows == 0) return st;
  const Kv8CacheArgs a = kv8_cache_args(const_cast<void*>(k_new), const_cast<void*>(v_new), k_stride, v_stride, total_rows, k_pages,
                                        v_pages, scales, num_blocks, block_table, max_blocks_per_seq, cu_rows, seq_lens,
                                        max_seq_len, batch, kv_heads);
  const dim3 grid = kv8_cache_grid(total_rows, batch, kv_heads), block(kWave);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128 && format == SDV_KV8_FP8)
    hipLaunchKernelGGL((kv8_append_kernel<128, kFp8>), grid, block, 0, s, a);
  else if (head_dim == 128)
    hipLaunchKernelGGL((kv8_append_kernel<128, kInt8>), grid, block, 0, s, a);
  else if (format == SDV_KV8_FP8)
    hipLaunchKernelGGL((kv8_append_kernel<64, kFp8>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((kv8_append_kernel<64, kInt8>), grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}

extern "C" int sdv_kv8_gather(const void* k_pages, const void* v_pages, const float* scales, int32_t num_blocks, int32_t format,
                              const int32_t* block_table, int32_t max_blocks_per_seq, const int32_t* cu_rows,
                              const int32_t* starts, int32_t batch, int32_t total_rows, int32_t kv_heads, int32_t head_dim,
                              void* k_out, void* v_out, int64_t k_stride, int64_t v_stride, void* stream) {
  if (!starts) return SDV_ERR_NULL;
  const int st = kv8_cache_check(k_out, v_out, k_stride, v_stride, total_rows, k_pages, v_pages, scales, num_blocks, format,
                                 block_table, max_blocks_per_seq, cu_rows, starts, batch, kv_heads, head_dim);
  if (st != SDV_OK || total_rows == 0) return st;
  const Kv8CacheArgs a = kv8_cache_args(k_out, v_out, k_stride, v_stride, total_rows, const_cast<void*>(k_pages),
                                        const_cast<void*>(v_pages), const_cast<float*>(scales), num_blocks, block_table,
                                        max_blocks_per_seq, cu_rows, starts, 0, batch, kv_heads);
  const dim3 grid = kv8_cache_grid(total_rows, batch, kv_heads), block(kWave);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128 && format == SDV_KV8_FP8)
    hipLaunchKernelGGL((kv8_gather_kernel<128, kFp8>), grid, block, 0, s, a);
  else if (head_dim == 128)
    hipLaunchKernelGGL((kv8_gather_kernel<128, kInt8>), grid, block, 0, s, a);
  else if (format == SDV_KV8_FP8)
    hipLaunchKernelGGL((kv8_gather_kernel<64, kFp8>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((kv8_gather_kernel<64, kInt8>), grid, block, 0, s, a);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}
