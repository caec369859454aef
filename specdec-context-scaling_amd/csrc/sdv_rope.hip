// Rotary positions of packed rows, and of a step's rows on their way into the kv8 cache (formula: sdv_rope.h).
#include "sdv_kv8_tile.h"
#include "sdv_rope.h"

namespace sdv {

// ---------------------------------------------------------------------------- rows of q and k
struct RopeRows {
  RopeArgs rope;
  const int32_t* positions;
  int rows;
  const uint16_t* in[2];  // q, k
  uint16_t* out[2];
  int64_t in_stride[2], out_stride[2];  // elements between rows
  int heads[2];
};

constexpr int kRopeThreads = 256, kRopeGroup = 8;  // threads and heads of a workgroup

// A workgroup has kRopeGroup heads of as many rows as it has threads for.  A thread loads one unit and, meanwhile, works out one
// of the rows' angles for all heads of the workgroup.  32 rows of 14 heads of 128: 2.5 us in a graph (2.9 with each lane's eight
// angles its own), of which an empty launch takes 2.1; 8191 rows of 16 heads of 64 7.4 us (8.1), 4.5 TB/s.  Those move what
// a copy moves in 4.5 us: the rest is the start and some 190 vector instructions a thread, whose loads, sines and stores follow
// one another in every thread at the same time.
template <int D, bool IL>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeRows a) {
  constexpr int U = D / 16, A = D / 2, RB = kRopeThreads / A;  // units and angles of a row; rows
  __shared__ __align__(16) float cs[2][RB][A];
  const int tid = threadIdx.x, r = tid / A, u = tid % U, heads = a.heads[0] + a.heads[1];
  const int64_t row = (int64_t)blockIdx.x * RB + r;
  const int h = blockIdx.y * kRopeGroup + tid % A / U, k = h >= a.heads[0];
  const bool has = row < a.rows && h < heads, turn = u < a.rope.units;
  const int d0 = rope_piece<IL>(a.rope, u, 0), d1 = rope_piece<IL>(a.rope, u, 1);
  const int at = (h - (k ? a.heads[0] : 0)) * D;
  uint4 w[2];
  if (has) {
    w[0] = *reinterpret_cast<const uint4*>(a.in[k] + row * a.in_stride[k] + at + d0);
    w[1] = *reinterpret_cast<const uint4*>(a.in[k] + row * a.in_stride[k] + at + d1);
  }
  if (row < a.rows && tid % A < 8 * a.rope.units) rope_angle(a.rope, tid % A, a.positions[row], cs[0][r][tid % A], cs[1][r][tid % A]);
  __syncthreads();
  if (!has) return;
  if (turn) {
    float y[16];
    rope_rotate<IL>(w[0], w[1], &cs[0][r][8 * u], &cs[1][r][8 * u], y);
    w[0] = rope_pack8(y);
    w[1] = rope_pack8(y + 8);
  }
  uint16_t* dst = a.out[k] + row * a.out_stride[k] + at;
  *reinterpret_cast<uint4*>(dst + d0) = w[0];
  *reinterpret_cast<uint4*>(dst + d1) = w[1];
}

// ---------------------------------------------------------------------------- a step's rows
struct Kv8RopeArgs {
  Kv8CacheArgs c;
  RopeArgs rope;
  const int32_t* positions;  // per packed row, or nullptr: the row's position in its sequence
  const uint16_t* q;
  uint16_t* q_out;
  int64_t q_stride, out_stride;
  int q_heads;
};

constexpr int kRopeHeads = 4;  // query heads of a wavefront; 2048 tokens with 1, 2, 4, 6, 8: 8.0, 7.5, 7.2, 7.5, 7.3 us in a graph

// A lane's eight angles of token `tok`, one of first .. first + n of a page block.  Of up to kRopeFew tokens the lanes work out
// the angles in turns and share them: a lane's own eight, one after another, kept a step of one token a sequence waiting (32
// of them 4.2 us in a graph, 3.7 like this), where a full block has work for every lane either way (2048 tokens 7.3 us, 9.1 with
// their angles shared).
constexpr int kRopeFew = 2;

template <int D>
__device__ __forceinline__ void rope_token(const Kv8RopeArgs& a, const Kv8Tile& t, int first, int n, int tok, int u, bool turn,
                                           float (&cs)[2][kRopeFew][D / 2], float (&c)[8], float (&s)[8]) {
  constexpr int A = D / 2;
  const auto pos = [&](int tok) { return a.positions ? a.positions[t.row + tok] : t.block * kBlock + tok; };
  if (n <= kRopeFew) {  // wave-uniform
    for (int e = threadIdx.x; e < n * A; e += kWave)
      if (e % A < 8 * a.rope.units) rope_angle(a.rope, e % A, pos(first + e / A), cs[0][e / A][e % A], cs[1][e / A][e % A]);
    __syncthreads();  // of one wavefront
    const int i = min(max(tok - first, 0), n - 1);
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = cs[0][i][8 * u + k], s[k] = cs[1][i][8 * u + k];
  } else if (turn) {
#pragma unroll
    for (int k = 0; k < 8; ++k) rope_angle(a.rope, 8 * u + k, pos(min(max(tok, first), first + n - 1)), c[k], s[k]);
  }
}

// Workgroups (x, y) of one wavefront: x a page block of a sequence, whichever of the call's rows fall in it; y a KV head, whose K
// is rotated, quantized and written, or one whose V is written (as by kv8_append_kernel), or kRopeHeads query heads of as
// many of its tokens as a load has rows.  So many wavefronts share the angles of no more than four heads, but each is little
// more than its loads one after another (lengths, rows, pages), which are what a call takes: with K, V and all tokens of the
// heads in one wavefront each a step of 2048 tokens took 8.9 us in a graph, 7.0 like this (7.3 with rope_token).  28,719 rows of 51
// sequences, which are more than the caches hold: 45 us, 4.9 TB/s (with 6 heads a wavefront 46, with 12 49).
template <int D, int FMT, bool IL>
__global__ __launch_bounds__(64) void kv8_rope_append_kernel(Kv8RopeArgs a) {
  constexpr int U = D / 16;      // lanes per row: a unit each
  constexpr int R = kWave / U;   // rows of a wave-wide load (8 or 16)
  constexpr int P = kBlock / R;  // loads of a block
  __shared__ union {
    uint4 v[D];
    float cs[2][kRopeFew][D / 2];
  } lds;
  const int lane = threadIdx.x, u = lane % U, rr = lane / U, y = blockIdx.y;
  const int d0 = rope_piece<IL>(a.rope, u, 0), d1 = rope_piece<IL>(a.rope, u, 1);
  const bool turn = u < a.rope.units;
  Kv8Tile t;

  if (y >= 2 * a.c.kv_heads) {  // query heads
    if (!kv8_tile<true, false>(a.c, (int)blockIdx.x, t)) return;
    const int part = (y - 2 * a.c.kv_heads) % P, h0 = (y - 2 * a.c.kv_heads) / P * kRopeHeads;
    const int first = max(t.t0, part * R), n = min(t.t1, (part + 1) * R) - first;
    if (n <= 0) return;
    // of R rows, 2^lg are tokens and the others more heads of theirs
    int lg = 0;
    while ((1 << lg) < n) ++lg;
    const int step = R >> lg, hs = rr >> lg, tok = first + (rr & ((1 << lg) - 1));
    const int64_t row = t.row + min(tok, t.t1 - 1);
    const uint16_t* src = a.q + row * a.q_stride;
    const auto has = [&](int i) { return i * step + hs < kRopeHeads && h0 + i * step + hs < a.q_heads && tok < first + n; };
    uint4 w[kRopeHeads][2];
#pragma unroll
    for (int i = 0; i < kRopeHeads; ++i) {
      if (!has(i)) continue;
      w[i][0] = *reinterpret_cast<const uint4*>(src + (h0 + i * step + hs) * D + d0);
      w[i][1] = *reinterpret_cast<const uint4*>(src + (h0 + i * step + hs) * D + d1);
    }
    float c[8], s[8];
    rope_token<D>(a, t, first, n, tok, u, turn, lds.cs, c, s);
#pragma unroll
    for (int i = 0; i < kRopeHeads; ++i) {
      if (!has(i)) continue;
      if (turn) {
        float z[16];
        rope_rotate<IL>(w[i][0], w[i][1], c, s, z);
        w[i][0] = rope_pack8(z);
        w[i][1] = rope_pack8(z + 8);
      }
      uint16_t* dst = a.q_out + row * a.out_stride + (h0 + i * step + hs) * D;
      *reinterpret_cast<uint4*>(dst + d0) = w[i][0];
      *reinterpret_cast<uint4*>(dst + d1) = w[i][1];
    }
    return;
  }

  // Tokens that are not the call's re-read a row that is; rows are loaded before it is known whether they have a block.
  if (!kv8_tile<true>(a.c, (int)blockIdx.x, t)) return;  // wave-uniform
  const int kvh = y % a.c.kv_heads;
  if (y >= a.c.kv_heads) {  // V, as kv8_write_v has it
    constexpr int LPR = D / 8, JV = kBlock * LPR / kWave;
    const uint16_t* vin = static_cast<const uint16_t*>(a.c.v) + kvh * D + 8 * (lane % LPR);
    uint4 vw[JV];
#pragma unroll
    for (int j = 0; j < JV; ++j) {
      const int tok = min(max(lane / LPR * JV + j, t.t0), t.t1 - 1);
      vw[j] = *reinterpret_cast<const uint4*>(vin + (int64_t)(t.row + tok) * a.c.v_stride);
    }
    const int id = kv8_block(a.c.r, t.b, t.block);
    if (id < 0) return;
    const int64_t page = (int64_t)id * a.c.kv_heads + kvh;
    kv8_write_v<D, FMT>(t, vw, a.c.v_pages + page * (kBlock * D), a.c.scales + page * (2 * kBlock), lds.v);
    return;
  }

  // K: lane (rr, u) holds unit u of token j*R + rr
  uint4 kw[P][2];
  const uint16_t* kin = static_cast<const uint16_t*>(a.c.k) + kvh * D;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int tok = min(max(j * R + rr, t.t0), t.t1 - 1);
    const uint16_t* src = kin + (int64_t)(t.row + tok) * a.c.k_stride;
    kw[j][0] = *reinterpret_cast<const uint4*>(src + d0);
    kw[j][1] = *reinterpret_cast<const uint4*>(src + d1);
  }
  const int id = kv8_block(a.c.r, t.b, t.block);
  if (id < 0) return;
  const int64_t page = (int64_t)id * a.c.kv_heads + kvh;
  uint8_t* kp = a.c.k_pages + page * (kBlock * D);
  float* sp = a.c.scales + page * (2 * kBlock);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    if (t.t1 <= j * R || t.t0 >= (j + 1) * R) continue;  // none of the call's tokens
    const int tok = j * R + rr;
    float z[16], c[8], s[8];
    rope_token<D>(a, t, t.t0, t.t1 - t.t0, tok, u, turn, lds.cs, c, s);
    if (turn) {
      rope_rotate<IL>(kw[j][0], kw[j][1], c, s, z);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) z[k] = bf16_at(kw[j][k >> 3], k & 7);
    }
    uint32_t ab = 0;
#pragma unroll
    for (int k = 0; k < 16; ++k) ab = max(ab, __float_as_uint(z[k]) & 0x7FFFFFFFu);
    ab = unit_max_bits<U>(ab);
    constexpr float kQ = FMT == kFp8 ? 448.0f : 127.0f;
    float scale = __uint_as_float(ab) / kQ;
    if (scale == 0.0f) scale = 1.0f;
    const bool finite = ab < 0x7F800000u;
    // the largest quotient passes Q where the scale is below fp32's normal numbers
#pragma unroll
    for (int k = 0; k < 16; ++k) z[k] = finite ? fminf(fmaxf(z[k] / scale, -kQ), kQ) : 0.0f;
    if (tok >= t.t0 && tok < t.t1) {
      uint8_t* dst = kp + (tok >> 2) * (4 * D) + (tok & 3) * 16;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int d = k == 0 ? d0 : d1;
        *reinterpret_cast<uint2*>(dst + (d >> 4) * 64 + (d & 8)) =
            make_uint2(kv8_pack4<FMT>(z[8 * k], z[8 * k + 1], z[8 * k + 2], z[8 * k + 3]),
                       kv8_pack4<FMT>(z[8 * k + 4], z[8 * k + 5], z[8 * k + 6], z[8 * k + 7]));
      }
      if (u == 0) sp[tok] = finite ? scale : __builtin_nanf("");
    }
  }
}

}  // namespace sdv

using namespace sdv;

// A launch has fewer than 2^32 threads along x: of more rows (2^25 of 128 dimensions, 2^26 of 64) one for each so many.
template <int D, bool IL>
static void rope_launch(const RopeRows& a, hipStream_t st) {
  constexpr int rows = kRopeThreads / (D / 2), most = (1 << 23) * rows;
  const unsigned groups = (unsigned)((a.heads[0] + a.heads[1] + kRopeGroup - 1) / kRopeGroup);
  for (int first = 0; first < a.rows; first += most) {
    RopeRows x = a;
    x.rows = a.rows - first < most ? a.rows - first : most;
    x.positions += first;
    for (int k = 0; k < 2; ++k) {
      if (x.heads[k] == 0) continue;
      x.in[k] += first * x.in_stride[k];
      x.out[k] += first * x.out_stride[k];
    }
    hipLaunchKernelGGL((rope_kernel<D, IL>), dim3((unsigned)((x.rows + rows - 1) / rows), groups), dim3(kRopeThreads), 0, st, x);
  }
}

extern "C" int sdv_rope(const void* q, int64_t q_stride, int32_t q_heads, const void* k, int64_t k_stride, int32_t k_heads,
                        const int32_t* positions, const double* inv_freq, int32_t rotary_dim, int32_t interleaved, float scale,
                        int32_t inverse, int32_t rows, int32_t head_dim, void* q_out, int64_t q_out_stride, void* k_out,
                        int64_t k_out_stride, void* stream) {
  if (!q || !q_out || !positions || (k_heads > 0 && (!k || !k_out))) return SDV_ERR_NULL;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  const int st = rope_check(inv_freq, rotary_dim, interleaved, head_dim);
  if (st != SDV_OK) return st;
  if (rows < 0 || q_heads <= 0 || k_heads < 0 || q_heads > 32767 || k_heads > 32767 || rows > INT32_MAX / 2 || inverse < 0 || inverse > 1)
    return SDV_ERR_SHAPE;
  const int64_t qr = (int64_t)q_heads * head_dim, kr = (int64_t)k_heads * head_dim;
  if (q_stride < qr || q_out_stride < qr || (k_heads > 0 && (k_stride < kr || k_out_stride < kr))) return SDV_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(q_out, 16) || q_stride % 8 || q_out_stride % 8 || !aligned(positions, 4)) return SDV_ERR_ALIGN;
  if (k_heads > 0 && (!aligned(k, 16) || !aligned(k_out, 16) || k_stride % 8 || k_out_stride % 8)) return SDV_ERR_ALIGN;
  if (rows == 0) return SDV_OK;
  const RopeRows a = {{inv_freq, rotary_dim / 16, scale, inverse ? -1.0f : 1.0f}, positions, rows,
                      {static_cast<const uint16_t*>(q), static_cast<const uint16_t*>(k)},
                      {static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_out)}, {q_stride, k_stride}, {q_out_stride, k_out_stride},
                      {q_heads, k_heads}};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128)
    interleaved ? rope_launch<128, true>(a, s) : rope_launch<128, false>(a, s);
  else
    interleaved ? rope_launch<64, true>(a, s) : rope_launch<64, false>(a, s);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}

template <int D, int FMT>
static void kv8_rope_launch(const Kv8RopeArgs& a, bool interleaved, dim3 grid, hipStream_t st) {
  if (interleaved)
    hipLaunchKernelGGL((kv8_rope_append_kernel<D, FMT, true>), grid, dim3(kWave), 0, st, a);
  else
    hipLaunchKernelGGL((kv8_rope_append_kernel<D, FMT, false>), grid, dim3(kWave), 0, st, a);
}

extern "C" int sdv_kv8_rope_append(const void* q, int64_t q_stride, void* q_out, int64_t q_out_stride, int32_t q_heads,
                                   const void* k_new, const void* v_new, int64_t k_stride, int64_t v_stride, int32_t total_rows,
                                   void* k_pages, void* v_pages, float* scales, int32_t num_blocks, int32_t format,
                                   const int32_t* block_table, int32_t max_blocks_per_seq, const int32_t* cu_rows,
                                   const int32_t* seq_lens, int32_t max_seq_len, int32_t batch, int32_t kv_heads, int32_t head_dim,
                                   const int32_t* positions, const double* inv_freq, int32_t rotary_dim, int32_t interleaved,
                                   float scale, void* stream) {
  if (!q || !q_out) return SDV_ERR_NULL;
  if (!seq_lens && max_seq_len <= 0) return SDV_ERR_SHAPE;
  int st = kv8_cache_check(k_new, v_new, k_stride, v_stride, total_rows, k_pages, v_pages, scales, num_blocks, format, block_table,
                           max_blocks_per_seq, cu_rows, seq_lens, batch, kv_heads, head_dim);
  if (st != SDV_OK) return st;
  st = rope_check(inv_freq, rotary_dim, interleaved, head_dim);
  if (st != SDV_OK) return st;
  if (q_heads <= 0 || q_heads > 65535 || kv_heads > 16383) return SDV_ERR_SHAPE;
  const int64_t row = (int64_t)q_heads * head_dim;
  if (q_stride < row || q_out_stride < row) return SDV_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(q_out, 16) || q_stride % 8 || q_out_stride % 8 || !aligned(positions, 4)) return SDV_ERR_ALIGN;
  if (total_rows == 0) return SDV_OK;
  const Kv8RopeArgs a = {kv8_cache_args(const_cast<void*>(k_new), const_cast<void*>(v_new), k_stride, v_stride, total_rows, k_pages,
                                        v_pages, scales, num_blocks, block_table, max_blocks_per_seq, cu_rows, seq_lens, max_seq_len,
                                        batch, kv_heads),
                         {inv_freq, rotary_dim / 16, scale, 1.0f}, positions, static_cast<const uint16_t*>(q),
                         static_cast<uint16_t*>(q_out), q_stride, q_out_stride, q_heads};
  dim3 grid = kv8_cache_grid(total_rows, batch, kv_heads);
  grid.y = (unsigned)(2 * kv_heads + (q_heads + kRopeHeads - 1) / kRopeHeads * (head_dim / 64));  // a part per load of a block
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (head_dim == 128)
    format == SDV_KV8_FP8 ? kv8_rope_launch<128, kFp8>(a, interleaved, grid, s) : kv8_rope_launch<128, kInt8>(a, interleaved, grid, s);
  else
    format == SDV_KV8_FP8 ? kv8_rope_launch<64, kFp8>(a, interleaved, grid, s) : kv8_rope_launch<64, kInt8>(a, interleaved, grid, s);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}
