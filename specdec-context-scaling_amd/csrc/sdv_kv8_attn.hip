// Attention of ragged query rows over the 8-bit KV cache (layout: sdv_kv8.h; shares: sdv_kv8_plan.h).
//
//   x_j = scale * s^K_j * (q . c^K_j),   out = sum_j e^(x_j - M) s^V_j c^V_j / sum_j e^(x_j - M)
//
// over the keys j that the row sees, in one pass over them with a running maximum and sum.  The
// codes c are exact in BF16, so q.c is exact products summed in fp32 on the matrix cores, and the
// scales multiply the fp32 scores and probabilities.  The one rounding before the output's is
// e^(..) s^V to BF16, the operand of its product (half a step, 2^-9 of each term; the terms' errors
// are independent).
#include "sdv_kv8_plan.h"

namespace sdv {

// The value of lane `P` of each group of four lanes.
template <int P>
__device__ __forceinline__ float quad_lane(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), P * 0x55, 0xF, 0xF, true));
}

__device__ __forceinline__ float4 quad_lane4(float4 v, int p) {  // p is a constant after unrolling
  switch (p) {
    case 0: return make_float4(quad_lane<0>(v.x), quad_lane<0>(v.y), quad_lane<0>(v.z), quad_lane<0>(v.w));
    case 1: return make_float4(quad_lane<1>(v.x), quad_lane<1>(v.y), quad_lane<1>(v.z), quad_lane<1>(v.w));
    case 2: return make_float4(quad_lane<2>(v.x), quad_lane<2>(v.y), quad_lane<2>(v.z), quad_lane<2>(v.w));
    default: return make_float4(quad_lane<3>(v.x), quad_lane<3>(v.y), quad_lane<3>(v.z), quad_lane<3>(v.w));
  }
}

// Bits of a dword's bytes 4w..4w+3 that belong to the first n tokens of a block.
__device__ __forceinline__ uint32_t kv8_keep(int n, int w) {
  const int k = n - 4 * w;
  return k >= 4 ? ~0u : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
}

// A running maximum is moved only by a score more than 2^8 times its exponential: until then the
// probabilities are at most 2^8, and BF16 and fp32 hold them as exactly as they hold those below 1.
constexpr float kKv8Slack = 8.0f;

// ---------------------------------------------------------------------------- few rows
// Tiles of 16 or 32 rows: single tokens and verify blocks.  Each of a workgroup's four wavefronts
// streams every fourth step of the tile with all of its rows; their sums meet in LDS at its end.
//
// A step is four page blocks.  S^T = K Q^T on v_mfma_f32_16x16x32_bf16: MFMA p takes tokens 4p..4p+3 of
// the four blocks as its 16 key rows, so that lane (n, g) of its result holds row n and tokens 4p + r
// of block g, and after all four MFMAs every token of block g: with the 16 tokens as its k-slots that
// is the B operand of O^T = V^T P^T as it stands (A: lane (d, g) the 16 codes of dimension d in block g,
// one 16-byte load).
template <int D, int FMT, int RT>
__global__ __launch_bounds__(kKv8Threads, D == 128 && RT == 2 ? 1 : 2) void kv8_rows_kernel(Kv8AttnArgs a) {
  constexpr int TR = 16 * RT, KI = D / 64, KS = D / 32, DT = D / 16;
  constexpr int kWaves = kKv8Threads / kWave, kRow = D + 4;
  __shared__ __align__(16) float lds_o[kWaves][TR][kRow];
  __shared__ float lds_m[kWaves][TR], lds_l[kWaves][TR];
  __shared__ Kv8PlanLds lds_plan;

  Kv8Cut cut = {};
  Kv8Place<TR> at;
  if (!at.begin(a, lds_plan, (int)blockIdx.x, (int)gridDim.x)) {
    if (threadIdx.x == 0) a.cuts[blockIdx.x] = cut;
    return;
  }
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n = lane & 15, g = lane >> 4;
  const int64_t page_bytes = (int64_t)kBlock * D;
  bool first_part = true;

  for (;;) {
    const Kv8Seq seq = at.seq;
    const int b = at.b, kvh = at.kvh;
    const int s0 = (int)(at.u - at.tile0), s1 = (int)min(at.steps, at.end - at.tile0);
    const int row0 = at.i * TR, rows = min(seq.n * a.G - row0, TR);

    // query operand: lane (n, g), k-step 2i + h: dimensions (4i + g)*16 + 8h .. +7
    bf16x8 qop[RT][KS];
    int lim[RT];          // last key that the row sees; with a tree, the context's last
    uint64_t bits[RT];    // new tokens that it sees (tree)
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = row0 + 16 * rt + n, tok = r / a.G, head = r - tok * a.G;
      const bool live = 16 * rt + n < rows;
      const uint16_t* src = a.q + (int64_t)(seq.first + (live ? tok : 0)) * a.q_stride + (int64_t)(kvh * a.G + (live ? head : 0)) * D;
#pragma unroll
      for (int kk = 0; kk < KS; ++kk)
        qop[rt][kk] = *reinterpret_cast<const bf16x8*>(src + (4 * (kk >> 1) + g) * 16 + 8 * (kk & 1));
      lim[rt] = seq.tree ? seq.ctx - 1 : seq.ctx + (live ? tok : 0);
      bits[rt] = seq.tree && live ? a.tree[seq.first + tok] : 0;
    }
    // keys up to here are seen by every row of the tile
    const int all = seq.tree ? seq.ctx - 1 : seq.ctx + row0 / a.G;

    f32x4 o[RT][DT];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -INFINITY;
      l[rt] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int32_t* table = a.r.table + (int64_t)b * a.r.max_blocks;
    // block id of this lane's K and V block in a step; -1: none
    const auto block_id = [&](int step, int k) {
      const int j = step * 4 + k;
      const int id = table[min(j, a.r.max_blocks - 1)];
      return j < a.r.max_blocks && id >= 0 && id < a.r.num_blocks ? id : -1;
    };
    uint4 kw[4][KI], vw[DT];
    float4 sk, sv, sk_next, sv_next;
    const auto load_k = [&](int id) {
      const uint8_t* src = a.k_pages + ((int64_t)max(id, 0) * a.kv_heads + kvh) * page_bytes + g * 64 + (n & 3) * 16;
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int i = 0; i < KI; ++i) kw[p][i] = load_stream16(src + p * (4 * D) + i * 256);
    };
    const auto load_s = [&](int id) {
      const float* src = a.scales + ((int64_t)max(id, 0) * a.kv_heads + kvh) * (2 * kBlock) + 4 * (n & 3);
      sk_next = *reinterpret_cast<const float4*>(src);
      sv_next = *reinterpret_cast<const float4*>(src + kBlock);
    };
    const auto load_v = [&](int id) {
      const uint8_t* src = a.v_pages + ((int64_t)max(id, 0) * a.kv_heads + kvh) * page_bytes + n * kBlock;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vw[dt] = load_stream16(src + dt * (16 * kBlock));
    };

    int step = s0 + wave;
    int idk = -1, idv = -1, idk_next = -1, idv_next = -1;
    if (step < s1) {
      idk = block_id(step, n >> 2);
      idv = block_id(step, g);
      idk_next = block_id(step + kWaves, n >> 2);
      idv_next = block_id(step + kWaves, g);
      load_k(idk);
      load_s(idv);
      load_v(idv);
    }
    for (; step < s1; step += kWaves) {
      sk = sk_next;
      sv = sv_next;
      f32x4 s[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int p = 0; p < 4; ++p) s[rt][p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
          const uint4 w = kw[p][kk >> 1];
          const bf16x8 kop = (kk & 1) ? kv8_bf16x8<FMT>(w.z, w.w) : kv8_bf16x8<FMT>(w.x, w.y);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop, qop[rt][kk], s[rt][p], 0, 0, 0);
        }
      // the next step's K goes into the registers that are free now; the one after's block ids first,
      // so that waiting for them later does not wait for the data in between
      const int idv_now = idv;
      const bool more = step + kWaves < s1;
      if (more) {
        idk = idk_next;
        idv = idv_next;
        idk_next = block_id(step + 2 * kWaves, n >> 2);
        idv_next = block_id(step + 2 * kWaves, g);
        load_k(idk);
        load_s(idv);
      }

      const bool masked = step * kKv8Step + kKv8Step - 1 > all || __any(idv_now < 0);
      const int key0 = step * kKv8Step + g * kBlock;  // this lane's first token
      const auto seen = [&](int rt, int t) {
        const int key = key0 + t;
        if (key <= lim[rt]) return idv_now >= 0;
        const int j = key - seq.ctx;
        return idv_now >= 0 && key < seq.T && j < 64 && ((bits[rt] >> j) & 1);
      };
      bf16x8 pop[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float y[16];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float4 k4 = quad_lane4(sk, p);
#pragma unroll
          for (int r = 0; r < 4; ++r) y[4 * p + r] = s[rt][p][r] * ((&k4.x)[r] * a.c);
        }
        if (masked) {
#pragma unroll
          for (int t = 0; t < 16; ++t) y[t] = seen(rt, t) ? y[t] : -INFINITY;
        }
        float mx = y[0];
#pragma unroll
        for (int t = 1; t < 16; ++t) mx = fmaxf(mx, y[t]);
        if (__any(mx > m[rt] + kKv8Slack)) {
          float2 pr = lane_pair<16>(mx);
          mx = fmaxf(pr.x, pr.y);
          pr = lane_pair<32>(mx);
          mx = fmaxf(fmaxf(pr.x, pr.y), m[rt]);
          const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mx);
          l[rt] *= f;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
          m[rt] = mx;
        }
        const float ms = m[rt] == -INFINITY ? 0.0f : m[rt];
        uint32_t w[8];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const float4 v4 = quad_lane4(sv, p);
          float e[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = __builtin_amdgcn_exp2f(y[4 * p + r] - ms);
            l[rt] += x;
            e[r] = x * (&v4.x)[r];
            // the scale of a token that the row does not see may be anything
            if (masked) e[r] = seen(rt, 4 * p + r) ? e[r] : 0.0f;
          }
          w[2 * p] = pack_bf16x2(e[0], e[1]);
          w[2 * p + 1] = pack_bf16x2(e[2], e[3]);
        }
        pop[rt][0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
        pop[rt][1] = __builtin_bit_cast(bf16x8, make_uint4(w[4], w[5], w[6], w[7]));
      }
      if (masked) {  // codes behind the sequence's end, or of no block, may decode to NaN
        const int valid = idv_now < 0 ? 0 : seq.T - key0;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          vw[dt].x &= kv8_keep(valid, 0);
          vw[dt].y &= kv8_keep(valid, 1);
          vw[dt].z &= kv8_keep(valid, 2);
          vw[dt].w &= kv8_keep(valid, 3);
        }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 v0 = kv8_bf16x8<FMT>(vw[dt].x, vw[dt].y), v1 = kv8_bf16x8<FMT>(vw[dt].z, vw[dt].w);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pop[rt][0], o[rt][dt], 0, 0, 0);
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pop[rt][1], o[rt][dt], 0, 0, 0);
        }
      }
      if (more) load_v(idv);
    }

    // the wavefronts' sums: lane (n, g) holds row n, dimensions 16 dt + 4g + i
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float2 pr = lane_pair<16>(l[rt]);
      pr = lane_pair<32>(pr.x + pr.y);
      if (g == 0) {
        lds_m[wave][16 * rt + n] = m[rt];
        lds_l[wave][16 * rt + n] = pr.x + pr.y;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(&lds_o[wave][16 * rt + n][16 * dt + 4 * g]) = o[rt][dt];
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == (int)at.steps;
    const int slot = 2 * at.w + (first_part ? 0 : 1);
    float* part = a.part + (int64_t)slot * (TR * (D + 2));
    for (int e = tid; e < rows * (D / 4); e += kKv8Threads) {
      const int r = e / (D / 4), d = 4 * (e % (D / 4));
      float mm = lds_m[0][r];
#pragma unroll
      for (int k = 1; k < kWaves; ++k) mm = fmaxf(mm, lds_m[k][r]);
      float ll = 0.0f;
      f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < kWaves; ++k) {
        const float f = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(lds_m[k][r] - mm);
        ll += lds_l[k][r] * f;
        acc += *reinterpret_cast<const f32x4*>(&lds_o[k][r][d]) * f;
      }
      if (whole) {
        const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;  // a row that sees nothing: 0
        const int t = (row0 + r) / a.G, head = row0 + r - t * a.G;
        uint2 w = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
        *reinterpret_cast<uint2*>(a.out + (int64_t)(seq.first + t) * a.out_stride + (int64_t)(kvh * a.G + head) * D + d) = w;
      } else {
        *reinterpret_cast<f32x4*>(part + r * D + d) = acc;
        if (d == 0) {
          part[TR * D + r] = mm;
          part[TR * D + TR + r] = ll;
        }
      }
    }
    if (!whole && s0 == 0) {
      cut.parts = at.owner(at.tile0 + at.steps - 1) - at.w + 1;
      cut.slot = slot;
      cut.first = seq.first;
      cut.n = seq.n;
      cut.kvh = kvh;
      cut.i = at.i;
    }
    first_part = false;
    at.u = at.tile0 + (uint32_t)s1;
    if (at.u >= at.end || !at.next(a)) break;
    __syncthreads();
  }
  if (tid == 0) a.cuts[blockIdx.x] = cut;
}

// ---------------------------------------------------------------------------- shared tiles
// The parts of the tile that workgroup x's range cuts, summed in their order: a thread per four
// dimensions of a row.
template <int D, int TR>
__global__ __launch_bounds__(256) void kv8_merge_kernel(Kv8AttnArgs a) {
  const Kv8Cut cut = a.cuts[blockIdx.x];
  const int e = (int)(blockIdx.y * 256 + threadIdx.x), r = e / (D / 4), d = 4 * (e % (D / 4));
  const int row = cut.i * TR + r;
  if (cut.parts == 0 || row >= cut.n * a.G) return;
  constexpr int kPart = TR * (D + 2);
  const float* first = a.part + (int64_t)cut.slot * kPart;
  const float* rest = a.part + (int64_t)(cut.slot & ~1) * kPart;  // part k >= 1: + 2k slots
  const auto part = [&](int k) { return k == 0 ? first : rest + (int64_t)2 * k * kPart; };
  float mm = -INFINITY;
  for (int k = 0; k < cut.parts; ++k) mm = fmaxf(mm, part(k)[TR * D + r]);
  float ll = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int k = 0; k < cut.parts; ++k) {
    const float* p = part(k);
    const float f = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(p[TR * D + r] - mm);
    ll += p[TR * D + TR + r] * f;
    acc += *reinterpret_cast<const f32x4*>(p + r * D + d) * f;
  }
  const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
  const int t = row / a.G, head = row - t * a.G;
  uint2 w = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  *reinterpret_cast<uint2*>(a.out + (int64_t)(cut.first + t) * a.out_stride + (int64_t)(cut.kvh * a.G + head) * D + d) = w;
}

}  // namespace sdv

using namespace sdv;

// Rows per tile: 16 where a sequence's rows fit one tile of 16, else 32.
static int kv8_tile_rows(int32_t G, int32_t max_q_len) { return (int64_t)G * max_q_len <= 16 ? 16 : 32; }

constexpr int kKv8Grid = 512;  // two workgroups per CU

// Most units of a call, or -1 where they or the row and key counts pass what the plan's 32-bit sums hold.
static int64_t kv8_units(int32_t batch, int32_t total, int32_t G, int32_t kv_heads, int32_t max_len, int tile) {
  if (((int64_t)max_len + total) * G > (1 << 30)) return -1;
  const int64_t tiles = (int64_t)total * G / tile + batch;
  const int64_t units = tiles * (((int64_t)max_len + total) / kKv8Step + 1) * kv_heads;
  return units > INT32_MAX ? -1 : units;
}

static size_t kv8_workspace(int tile, int32_t head_dim) {
  return kKv8Grid * sizeof(Kv8Cut) + (size_t)kKv8Grid * 2 * tile * (head_dim + 2) * sizeof(float);
}

static int kv8_attn_sizes(int32_t batch, int32_t total, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                          int32_t max_len) {
  if (batch <= 0 || total < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || max_q_len <= 0 || max_len <= 0)
    return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  if (batch > INT32_MAX / 4 || total > INT32_MAX / 2) return SDV_ERR_SHAPE;
  const int32_t G = q_heads / kv_heads;
  return kv8_units(batch, total, G, kv_heads, max_len, kv8_tile_rows(G, max_q_len)) < 0 ? SDV_ERR_SHAPE : SDV_OK;
}

extern "C" size_t sdv_kv8_attention_workspace_size(int32_t batch, int32_t total_rows, int32_t q_heads, int32_t kv_heads,
                                                   int32_t head_dim, int32_t max_q_len, int32_t max_seq_len) {
  if (kv8_attn_sizes(batch, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len) != SDV_OK) return 0;
  return kv8_workspace(kv8_tile_rows(q_heads / kv_heads, max_q_len), head_dim);
}

template <int D, int FMT, int RT>
static void kv8_launch(const Kv8AttnArgs& a, int grid, hipStream_t st) {
  hipLaunchKernelGGL((kv8_rows_kernel<D, FMT, RT>), dim3((unsigned)grid), dim3(kKv8Threads), 0, st, a);
  hipLaunchKernelGGL((kv8_merge_kernel<D, 16 * RT>), dim3((unsigned)grid, 16 * RT * D / 1024), dim3(256), 0, st, a);
}

extern "C" int sdv_kv8_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, const float* scales,
                                 int32_t num_blocks, int32_t format, const int32_t* block_table, int32_t max_blocks_per_seq,
                                 const int32_t* cu_rows, const int32_t* seq_lens, const uint64_t* tree_mask, int32_t batch,
                                 int32_t total_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                                 int32_t max_seq_len, float scale, void* workspace, size_t workspace_bytes, void* out,
                                 int64_t out_stride, void* stream) {
  if (!q || !k_pages || !v_pages || !scales || !block_table || !cu_rows || !out) return SDV_ERR_NULL;
  const int sizes = kv8_attn_sizes(batch, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len);
  if (sizes != SDV_OK) return sizes;
  if (num_blocks <= 0 || max_blocks_per_seq <= 0 || max_blocks_per_seq > INT32_MAX / kBlock) return SDV_ERR_SHAPE;
  if (format != SDV_KV8_FP8 && format != SDV_KV8_INT8) return SDV_ERR_UNSUPPORTED;
  if (tree_mask && max_q_len > 64) return SDV_ERR_UNSUPPORTED;
  const int64_t row = (int64_t)q_heads * head_dim;
  if (q_stride < row || out_stride < row) return SDV_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride % 8 || out_stride % 8 || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
      !aligned(scales, 16) || !aligned(block_table, 4) || !aligned(cu_rows, 4) || !aligned(seq_lens, 4) || !aligned(tree_mask, 8))
    return SDV_ERR_ALIGN;
  const int G = q_heads / kv_heads, tile = kv8_tile_rows(G, max_q_len);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < kv8_workspace(tile, head_dim)) return SDV_ERR_WORKSPACE;
  if (total_rows == 0) return SDV_OK;

  Kv8AttnArgs a;
  a.r = {cu_rows, block_table, max_blocks_per_seq, num_blocks, batch, total_rows};
  a.lens = seq_lens;
  a.tree = tree_mask;
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.k_pages = static_cast<const uint8_t*>(k_pages);
  a.v_pages = static_cast<const uint8_t*>(v_pages);
  a.scales = scales;
  a.G = G;
  a.kv_heads = kv_heads;
  a.max_len = max_seq_len;
  a.c = (float)((double)scale * 1.4426950408889634);
  a.min_units = kKv8Threads / kWave;
  a.cuts = static_cast<Kv8Cut*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kKv8Grid * sizeof(Kv8Cut));
  const int64_t most = kv8_units(batch, total_rows, G, kv_heads, max_seq_len, tile) / a.min_units;
  const int grid = (int)(most < 1 ? 1 : most < kKv8Grid ? most : kKv8Grid);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool fp8 = format == SDV_KV8_FP8;
  if (head_dim == 128 && tile == 16)
    fp8 ? kv8_launch<128, kFp8, 1>(a, grid, st) : kv8_launch<128, kInt8, 1>(a, grid, st);
  else if (head_dim == 128)
    fp8 ? kv8_launch<128, kFp8, 2>(a, grid, st) : kv8_launch<128, kInt8, 2>(a, grid, st);
  else if (tile == 16)
    fp8 ? kv8_launch<64, kFp8, 1>(a, grid, st) : kv8_launch<64, kInt8, 1>(a, grid, st);
  else
    fp8 ? kv8_launch<64, kFp8, 2>(a, grid, st) : kv8_launch<64, kInt8, 2>(a, grid, st);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}
