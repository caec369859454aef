// Few rows over the 8-bit KV cache: a tile of 16 or 32 query rows over a range of its keys, by one workgroup.
// Included by sdv_kv8_attn.hip and sdv_kv8_shared.hip.
#pragma once

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

// Sums of up to 2^30 terms of 2^8 |V| pass fp32's range where V's scales are above 2^81.  From the first
// scale of 2^64 on a wavefront takes its maxima to be 2^48 times as large: its sums are that much smaller
// then, and the least probability that counts is 2^-78 (2^-126 otherwise).  Looking for one costs a call
// over 2048 keys 0.1 us of 7.8.
constexpr float kKv8LargeScale = 18446744073709551616.0f, kKv8Raise = 48.0f;

constexpr int kKv8Threads = 256;  // of the kernel for few rows
constexpr int kKv8Grid = 512;     // its workgroups: two per CU

// A sequence's blocks, and the visibility of its new tokens (by packed row) where that is a tree's, else nullptr.
struct Kv8View {
  const int32_t* table;
  int max_blocks;
  int num_blocks;
  const uint64_t* bits;
  __device__ __forceinline__ bool named(int j) const { return j < max_blocks && table[j] >= 0 && table[j] < num_blocks; }
};

// The maximum that stands for a row none of whose scores of keys lo .. hi - 1 is above -inf: -inf where
// it sees none of the keys, the lowest finite number where it does (scores of an infinite q, or NaN).  Both
// sums are 0 or NaN; over all keys the first is an output of 0 and the second 0 / 0.  Looked for block by
// block, since it hardly ever comes to this: keys up to the row's own position, or the context and its
// mask's tokens, in blocks that the table names.  (As a check of each output's sum in kv8_write and the
// merges the code that this takes made a call over 2048 keys 0.2 us longer, 7.7 to 7.9.)
template <class Named>
__device__ __forceinline__ float kv8_lowest(const uint64_t* tree, int max_blocks, const Kv8Seq& s, int tok, int lo, int hi, const Named& named) {
  const int last = min(s.tree ? s.ctx - 1 : s.ctx + tok, hi - 1);
  bool any = false;
  for (int j = lo / kBlock; !any && j < max_blocks && j * kBlock <= last; ++j) any = named(j);
  if (s.tree) {
    const uint64_t bits = tree[s.first + tok];
    for (int j = max(lo - s.ctx, 0); !any && j < min(min(hi - s.ctx, s.n), 64); ++j) any = ((bits >> j) & 1) != 0 && named((s.ctx + j) >> 4);
  }
  return any ? -3.4028235e38f : -INFINITY;
}

// ---------------------------------------------------------------------------- few rows
// Tiles of 16 or 32 rows: single tokens and verify blocks.  Each of a workgroup's four wavefronts
// streams every fourth step of the tile with all of its rows; their sums meet in LDS at its end.
//
// A wavefront's step is four page blocks, or two where it has two row tiles (with four their registers
// do not leave two wavefronts a SIMD: 32 sequences of 2048 to 32768 keys, five rows each, 95 us, so 77).  S^T = K Q^T on
// v_mfma_f32_16x16x32_bf16: of four blocks, MFMA p takes tokens 4p..4p+3 of each as its 16 key rows, so
// that lane (n, g) of its result holds row n and tokens 4p + r of block g, and after all four MFMAs every
// token of block g: with the 16 tokens as its k-slots that is the B operand of O^T = V^T P^T as it stands
// (A: lane (d, g) the 16 codes of dimension d in block g, one 16-byte load).  Of two blocks, lane group
// g has tokens 8 (g % 2) + 4p + r of block g / 2.  The matrix cores have time to spare here, so P goes
// in as two BF16 operands, the rounded value and what the rounding left (16 bits in all), over BF16's
// whole range of scales.
//
// Long batches are bound by memory: single tokens of 32 sequences of 2048 to 32768 keys (293 MB of pages,
// 2 KV heads of 128) take 55 to 57 us, 5.2 TB/s, a large copy's rate; the matrix cores are busy a tenth of
// it.  Short calls are bound by latencies, each a microsecond or more: lengths, page ids, the pages,
// the merge's count, and the parts.  One token over 2048 keys takes 7.5 us, over 32768 18.5.
template <int D, int RT>
struct Kv8RowsLds {
  __align__(16) float o[kKv8Threads / kWave][16 * RT][D + 4];  // the wavefronts' sums
  float m[kKv8Threads / kWave][16 * RT], l[kKv8Threads / kWave][16 * RT];
  __align__(16) uint16_t q[RT == 1 ? 8 : 16 * RT * D];
};

// Steps s0 .. s1 - 1 of the tile that begins with row row0 of the sequence and has `rows` of them; each wavefront's sums
// to lds.
// AGAIN: the pages are read by other tiles as well, and by way of the caches.
template <int D, int FMT, int RT, bool AGAIN = false>
__device__ __forceinline__ void kv8_rows_tile(const Kv8AttnArgs& a, const Kv8View& w, const Kv8Seq& seq, int kvh, int row0, int rows,
                                              int s0, int s1, Kv8RowsLds<D, RT>& lds) {
  constexpr int KI = D / 64, KS = D / 32, DT = D / 16, kWaves = kKv8Threads / kWave;
  constexpr int PG = RT == 1 ? 4 : 2;  // page blocks of a wavefront's step, and MFMAs of its q.k^T
  constexpr int NT = 4 * PG;           // a lane's tokens of them
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n = lane & 15, g = lane >> 4;
  const int64_t page_bytes = (int64_t)kBlock * D;
  // the lane's place in a step: block and token of the key row that it loads, of the tokens that it holds
  const int kblk = PG == 4 ? n >> 2 : n >> 3, vblk = PG == 4 ? g : g >> 1;
  const int kpart = PG == 4 ? 0 : 2 * (n >> 2 & 1), vtok = PG == 4 ? 0 : 8 * (g & 1);

  // block id of this lane's K and V block in a step; -1: none
  const auto block_id = [&](int step, int k) {
    const int j = step * PG + k;
    const int id = w.table[min(j, w.max_blocks - 1)];
    return j < w.max_blocks && id >= 0 && id < w.num_blocks ? id : -1;
  };
  int step = s0 * (4 / PG) + wave;
  const int last = s1 * (4 / PG);
  int idk = block_id(step, kblk), idv = block_id(step, vblk);
  int idk_next = block_id(step + kWaves, kblk), idv_next = block_id(step + kWaves, vblk);

  // query operand: lane (n, g), k-step 2i + h: dimensions (4i + g)*16 + 8h .. +7.  One row tile of it
  // stays in registers; of two tiles it would not leave two wavefronts a SIMD, and lies in LDS.
  bf16x8 qreg[RT == 1 ? KS : 1];
  int lim[RT];          // last key that the row sees; with a tree, the context's last
  uint64_t bits[RT];    // new tokens that it sees (tree)
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + n, tok = r / a.G, head = r - tok * a.G;
    const bool live = 16 * rt + n < rows;
    const uint16_t* src = a.q + (int64_t)(seq.first + (live ? tok : 0)) * a.q_stride + (int64_t)(kvh * a.G + (live ? head : 0)) * D;
    if constexpr (RT == 1) {
#pragma unroll
      for (int kk = 0; kk < KS; ++kk) qreg[kk] = *reinterpret_cast<const bf16x8*>(src + (4 * (kk >> 1) + g) * 16 + 8 * (kk & 1));
    } else {
      for (int kk = wave; kk < KS; kk += kWaves)
        *reinterpret_cast<uint4*>(&lds.q[(rt * KS + kk) * 512 + lane * 8]) =
            *reinterpret_cast<const uint4*>(src + (4 * (kk >> 1) + g) * 16 + 8 * (kk & 1));
    }
    lim[rt] = seq.tree ? seq.ctx - 1 : seq.ctx + (live ? tok : 0);
    bits[rt] = w.bits && live ? w.bits[seq.first + tok] : 0;
  }
  // keys up to here are seen by every row of the tile
  const int all = seq.tree ? seq.ctx - 1 : seq.ctx + row0 / a.G;

  f32x4 o[RT][DT];
  float m[RT], l[RT], raise = 0.0f;  // raise: wave-uniform
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }

  const auto load16 = [](const uint8_t* p) { return AGAIN ? *reinterpret_cast<const uint4*>(p) : load_stream16(p); };
  uint4 kw[PG][KI];
  uint32_t vw[DT][PG];
  float4 sk, sv, sk_next, sv_next;
  const auto load_k = [&](int id) {
    const uint8_t* src = a.k_pages + ((int64_t)max(id, 0) * a.kv_heads + kvh) * page_bytes + kpart * (4 * D) + g * 64 + (n & 3) * 16;
#pragma unroll
    for (int p = 0; p < PG; ++p)
#pragma unroll
      for (int i = 0; i < KI; ++i) kw[p][i] = load16(src + p * (4 * D) + i * 256);
  };
  const auto load_s = [&](int id) {
    const float* src = a.scales + ((int64_t)max(id, 0) * a.kv_heads + kvh) * (2 * kBlock) + vtok + 4 * (n & (PG - 1));
    sk_next = *reinterpret_cast<const float4*>(src);
    sv_next = *reinterpret_cast<const float4*>(src + kBlock);
  };
  const auto load_v = [&](int id) {
    const uint8_t* src = a.v_pages + ((int64_t)max(id, 0) * a.kv_heads + kvh) * page_bytes + n * kBlock + vtok;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if constexpr (PG == 4) {
        const uint4 x = load16(src + dt * (16 * kBlock));
        vw[dt][0] = x.x;
        vw[dt][1] = x.y;
        vw[dt][2] = x.z;
        vw[dt][3] = x.w;
      } else {
        const uint64_t* at = reinterpret_cast<const uint64_t*>(src + dt * (16 * kBlock));
        const uint64_t w = AGAIN ? *at : __builtin_nontemporal_load(at);
        vw[dt][0] = (uint32_t)w;
        vw[dt][1] = (uint32_t)(w >> 32);
      }
    }
  };
  if (step < last) {
    load_k(idk);
    load_s(idv);
    load_v(idv);
  }
  if constexpr (RT > 1) __syncthreads();  // lds.q
  for (; step < last; step += kWaves) {
    sk = sk_next;
    sv = sv_next;
    f32x4 s[RT][PG];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int p = 0; p < PG; ++p) s[rt][p] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (RT > 1) asm volatile("" ::: "memory");  // the operand is read again each step
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      bf16x8 qop[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        if constexpr (RT == 1)
          qop[rt] = qreg[kk];
        else
          qop[rt] = *reinterpret_cast<const bf16x8*>(&lds.q[(rt * KS + kk) * 512 + lane * 8]);
      }
#pragma unroll
      for (int p = 0; p < PG; ++p) {
        const uint4 w = kw[p][kk >> 1];
        const bf16x8 kop = (kk & 1) ? kv8_bf16x8<FMT>(w.z, w.w) : kv8_bf16x8<FMT>(w.x, w.y);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kop, qop[rt], s[rt][p], 0, 0, 0);
      }
    }
    // The next step's K goes into the registers that are free now; the one after's block ids first, so
    // that waiting for them later does not wait for the data in between.
    const int idv_now = idv;
    const bool more = step + kWaves < last;
    if (more) {
      idk = idk_next;
      idv = idv_next;
      idk_next = block_id(step + 2 * kWaves, kblk);
      idv_next = block_id(step + 2 * kWaves, vblk);
      load_k(idk);
      load_s(idv);
    }

    const bool masked = (step + 1) * (PG * kBlock) - 1 > all || __any(idv_now < 0);
    const int key0 = step * (PG * kBlock) + vblk * kBlock + vtok;  // this lane's first token
    // which of this lane's tokens each of its rows sees
    uint32_t vis[RT];
    if (masked) {
      const auto first = [](int k) { return (1u << min(max(k, 0), NT)) - 1u; };
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        vis[rt] = first(lim[rt] + 1 - key0);
        const int sh = key0 - seq.ctx;  // the token behind bit 0 of the mask, from this lane's first
        if (seq.tree && sh > -NT && sh < 64) vis[rt] |= (uint32_t)(sh >= 0 ? bits[rt] >> sh : bits[rt] << -sh) & first(seq.T - key0);
        if (idv_now < 0) vis[rt] = 0;
      }
    }
    const auto seen = [&](int rt, int t) { return ((vis[rt] >> t) & 1) != 0; };
    if (masked) {  // codes behind the sequence's end, or of no block, may decode to NaN
      const int valid = idv_now < 0 ? 0 : seq.T - key0;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int p = 0; p < PG; ++p) vw[dt][p] &= kv8_keep(valid, p);
      }
    }
    const float raised = raise;
    if (__any(fmaxf(fmaxf(sv.x, sv.y), fmaxf(sv.z, sv.w)) >= kKv8LargeScale)) raise = kKv8Raise;
    constexpr int NH = PG / 2;  // p.V products per dimension tile, 32 tokens each
    bf16x8 hi[RT][NH], lo[RT][NH];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float y[NT];
#pragma unroll
      for (int p = 0; p < PG; ++p) {
        const float4 k4 = quad_lane4(sk, p);
#pragma unroll
        for (int r = 0; r < 4; ++r) y[4 * p + r] = s[rt][p][r] * ((&k4.x)[r] * a.c);
      }
      if (masked) {
#pragma unroll
        for (int t = 0; t < NT; ++t) y[t] = seen(rt, t) ? y[t] : -INFINITY;
      }
      float mx = y[0];
#pragma unroll
      for (int t = 1; t < NT; ++t) mx = fmaxf(mx, y[t]);
      if (__any(mx > m[rt] + kKv8Slack) || raise != raised) {
        float2 pr = lane_pair<16>(mx);
        mx = fmaxf(pr.x, pr.y);
        pr = lane_pair<32>(mx);
        mx = fmaxf(fmaxf(pr.x, pr.y), m[rt]);
        const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[rt] - mx + (raised - raise));
        l[rt] *= f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
        m[rt] = mx;
      }
      const float ms = m[rt] == -INFINITY ? 0.0f : m[rt] + raise;
      uint32_t wh[2 * PG], wl[2 * PG];
#pragma unroll
      for (int p = 0; p < PG; ++p) {
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
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w = pack_bf16x2(e[2 * h], e[2 * h + 1]);
          wh[2 * p + h] = w;
          wl[2 * p + h] = pack_bf16x2(e[2 * h] - bf16_lo(w), e[2 * h + 1] - bf16_hi(w));
        }
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        hi[rt][h] = __builtin_bit_cast(bf16x8, make_uint4(wh[4 * h], wh[4 * h + 1], wh[4 * h + 2], wh[4 * h + 3]));
        lo[rt][h] = __builtin_bit_cast(bf16x8, make_uint4(wl[4 * h], wl[4 * h + 1], wl[4 * h + 2], wl[4 * h + 3]));
      }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const bf16x8 v = kv8_bf16x8<FMT>(vw[dt][2 * h], vw[dt][2 * h + 1]);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, hi[rt][h], o[rt][dt], 0, 0, 0);
          o[rt][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, lo[rt][h], o[rt][dt], 0, 0, 0);
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
      lds.m[wave][16 * rt + n] = m[rt] + raise;
      lds.l[wave][16 * rt + n] = pr.x + pr.y;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(&lds.o[wave][16 * rt + n][16 * dt + 4 * g]) = o[rt][dt];
  }
}

// Four dimensions of row r of the tile: the wavefronts' sums as one, with their maximum and their sum of exponentials.
template <int D, int RT>
__device__ __forceinline__ f32x4 kv8_rows_sum(const Kv8RowsLds<D, RT>& lds, int r, int d, float& mm, float& ll) {
  constexpr int kWaves = kKv8Threads / kWave;
  mm = lds.m[0][r];
#pragma unroll
  for (int k = 1; k < kWaves; ++k) mm = fmaxf(mm, lds.m[k][r]);
  ll = 0.0f;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    const float f = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(lds.m[k][r] - mm);
    ll += lds.l[k][r] * f;
    acc += *reinterpret_cast<const f32x4*>(&lds.o[k][r][d]) * f;
  }
  return acc;
}

}  // namespace sdv
