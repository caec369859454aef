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
#include "sdv_kv8_tile.h"

namespace sdv {

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

  kv8_write_v<D, FMT>(t, vw, vp, sp, lds_v);
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
