// 128 query rows over a range of a prefix's keys, all of which every row sees, by one workgroup.
// Included by sdv_kv8_shared.hip.
//
// A wavefront has 32 rows; the four share stages of 64 keys, whose codes are converted once on their way to LDS, two
// buffers of them.  Products are v_mfma_f32_32x32x16: S^T = K Q^T in BF16 (codes and q as they are), O^T = V^T P^T in
// FP16.  Lane (g, n) of a product holds row n and tokens 8j + 4g + i of a unit of 32 keys (two blocks): with those as
// its k-slots that is the B operand of the next product as it stands, and V is laid out for it.  V is fp16(code) *
// fp16(scale * 2^(b - E)), E the exponent of the largest V scale of the item's keys and b such that the largest code
// stays under 2^15; p is held as 2^7 p: 11 bits each, and how far that is off is worked out in sdv_kv8_chunk.h.  An item
// whose V scales lie more than kWideBand binades apart is not computed this way.
//
// Two units are at work at once, the products of a third behind them: K Q^T of the one ahead, the scores of this one,
// V^T P^T of the one behind, a matrix instruction at a time among the others' work (none of them waits for another).  So
// a stage's buffer has K of units 2s + 1 and 2s + 2, scales of the scores of 2s and 2s + 1, V of 2s - 1 and 2s, and V's
// scales of the stage after it.
//
// Units take exp2(s - m) against the maximum so far; one that would bring a lane's sum to 2^8 p is done again with a new
// maximum, from products that are still in registers.  Blocks that the table does not name are taken as zeros, with scores
// of NaN, which end up there as well and become -inf.  A token whose V scale is NaN has its V taken as 0 and its scores as
// NaN.
#pragma once

#include "sdv_kv8_rows.h"

namespace sdv {

typedef float f32x16 __attribute__((ext_vector_type(16)));

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kWideRows = 32 * (kKv8Threads / kWave);
constexpr int kWideBand = 18;           // an FP16 scale is a normal number from 2^(E - 19) on
constexpr float kWideBits = 7.0f, kWideBound = 32768.0f;  // 2^7 p, and a lane's sum of 16 of them

template <int D>
struct Kv8WideLds {
  uint4 k[2][2][D / 16][kWave];  // [buffer][unit][16 dimensions][lane (g, n): key n, dimensions 8g ..]
  uint4 v[2][4][D / 32][kWave];  // [buffer][block][32 dimensions][lane (g, d): tokens 4g .. 4g+3, 8+4g .. of dimension d]
  float ks[2][kKv8Step];         // K's scales times the softmax's
  _Float16 vs[2][4][kBlock];     // V's, of the next stage's blocks
  int gone[2][4];                // whether the table does not name a block
  float spare[kKv8Threads];
  uint32_t most[kKv8Threads / kWave], least[kKv8Threads / kWave];
};

__device__ __forceinline__ uint32_t wide_f16x2(float lo, float hi) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}

// Four codes as FP16, exactly, times their tokens' scales (FP16 pairs).
template <int FMT>
__device__ __forceinline__ uint2 wide_v4(uint32_t w, uint32_t s01, uint32_t s23) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  f16x2 lo, hi;
  if constexpr (FMT == kFp8) {
    lo = (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
    hi = (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
  } else {
    // with the sign bit turned a code is c + 128; under the bits 0x6400 that is 1024 + c + 128 in FP16
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
  }
  return make_uint2(__builtin_bit_cast(uint32_t, lo * __builtin_bit_cast(f16x2, s01)), __builtin_bit_cast(uint32_t, hi * __builtin_bit_cast(f16x2, s23)));
}

// Rows row0 .. row0 + rows - 1 of those that begin with packed row `first`; steps s0 .. s1 - 1 of T keys (whole blocks), s0 < s1.
// acc, m and l: the lane's sums, maximum (that of its row) and half of its sum of exponentials, the sums in units of
// 2^(E - b), all of them times 2^7.  False: nothing done, the V scales lie too far apart.
template <int D, int FMT>
__device__ __forceinline__ bool kv8_wide_tile(const Kv8AttnArgs& a, const Kv8View& w, int first, int T, int kvh, int row0, int rows, int s0,
                                              int s1, int& E, Kv8WideLds<D>& lds, f32x16 (&acc)[D / 32], float& m, float& l) {
  constexpr int KS = D / 16, DT = D / 32;
  constexpr int NP = D / 64;                // 16-byte pieces of a stage's K, and of its V, per thread
  constexpr int TB = kKv8Threads * NP / 4;  // threads of a block
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int g = lane >> 5, n = lane & 31;
  const int64_t page_bytes = (int64_t)kBlock * D;

  // a thread's pieces: of blocks blk, blk + 4 / NP ...: K of a token's 16 dimensions, V of a dimension's 16 tokens, and a scale
  const int blk = __builtin_amdgcn_readfirstlane(tid / TB), in = tid % TB;
  const int ktok = in & 15, kc = in >> 4;
  const int ksrc = (ktok >> 2) * (4 * D) + kc * 64 + (ktok & 3) * 16, vsrc = in * kBlock;
  const int lo = 4 * s0, hi = min(min(T / kBlock, w.max_blocks), 4 * s1);
  // What a stage's buffer takes: K and V's scales from block 4s + 2 on, the scores' scales from 4s, V from 4s - 2.  The
  // table is read two stages ahead, in front of the pages, so that waiting for it does not wait for those.
  int idk[NP], ids[NP], idv[NP];  // of the stage that is fetched, wave-uniform
  int raw_k[NP], raw_s[NP];       // of the one after it, as the table has them
  uint4 kw[NP], vw[NP];           // on their way
  float sk[NP], sv[NP];
  int of_k[NP], of_v[NP], of_s[NP];  // their ids
  // All bits where the table names the block, without a branch (see stash_s).
  const auto named = [](int id) { return (uint32_t)~(id >> 31); };
  const auto mask = [](uint4 x, uint32_t keep) { return make_uint4(x.x & keep, x.y & keep, x.z & keep, x.w & keep); };
  const auto look = [&](int s) {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int x = 4 * s + blk + j * (4 / NP);
      raw_k[j] = w.table[min(max(x + 2, 0), w.max_blocks - 1)];
      raw_s[j] = w.table[min(max(x, 0), w.max_blocks - 1)];
    }
  };
  const auto valid = [&](int x, int id) { return x >= lo && x < hi && id >= 0 && id < w.num_blocks ? id : -1; };
  const auto ids_of = [&](int s) {  // from what look(s) has found; V's blocks are K's of the stage before
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const int x = 4 * s + blk + j * (4 / NP);
      idv[j] = idk[j];
      idk[j] = valid(x + 2, __builtin_amdgcn_readfirstlane(raw_k[j]));
      ids[j] = valid(x, __builtin_amdgcn_readfirstlane(raw_s[j]));
    }
  };
  const auto page = [&](int id) { return (int64_t)max(id, 0) * a.kv_heads + kvh; };
  const auto fetch_k = [&]() {
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      of_k[j] = idk[j];
      kw[j] = *reinterpret_cast<const uint4*>(a.k_pages + page(idk[j]) * page_bytes + ksrc);
      // lanes 0 .. 15 of a block: a scale of the scores and the same token's of V; 16 .. 31: one of V of the next stage
      const float* own = a.scales + page(in < 16 ? ids[j] : idk[j]) * (2 * kBlock);
      sk[j] = own[in & 15];
      sv[j] = own[kBlock + (in & 15)];
    }
  };
  const auto fetch = [&]() {
    fetch_k();
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      of_v[j] = idv[j];
      of_s[j] = ids[j];
      vw[j] = *reinterpret_cast<const uint4*>(a.v_pages + page(idv[j]) * page_bytes + vsrc);
    }
  };
  const auto stash_k = [&](int buf, int j, uint4 x, int id) {
    const int b = blk + j * (4 / NP);
    x = mask(x, named(id));
    uint4* kd = &lds.k[buf][b >> 1][kc][(b & 1) * 16 + ktok];
    kd[0] = __builtin_bit_cast(uint4, kv8_bf16x8<FMT>(x.x, x.y));
    kd[32] = __builtin_bit_cast(uint4, kv8_bf16x8<FMT>(x.z, x.w));
  };
  const auto stash_v = [&](int buf, int j) {  // with the scales in the other buffer
    const int b = blk + j * (4 / NP);
    const uint4 x = mask(vw[j], named(of_v[j]));
    const uint4* sp = reinterpret_cast<const uint4*>(lds.vs[buf ^ 1][b]);
    const uint4 s0_ = sp[0], s1_ = sp[1];
    const uint2 a0 = wide_v4<FMT>(x.x, s0_.x, s0_.y), a1 = wide_v4<FMT>(x.y, s0_.z, s0_.w);
    const uint2 a2 = wide_v4<FMT>(x.z, s1_.x, s1_.y), a3 = wide_v4<FMT>(x.w, s1_.z, s1_.w);
    uint4* vd = &lds.v[buf][b][in >> 5][in & 31];
    vd[0] = make_uint4(a0.x, a0.y, a2.x, a2.y);
    vd[32] = make_uint4(a1.x, a1.y, a3.x, a3.y);
  };
  // Without a branch, which would part the steps that this stands among: the lanes that have none write elsewhere.
  const auto stash_vs = [&](int buf, int j, float x, int id, float to_e) {
    const int b = blk + j * (4 / NP);
    x = __uint_as_float((__float_as_uint(x) >= 0x7F800000u ? 0u : __float_as_uint(x)) & named(id));
    *(in >= 16 && in < 32 ? &lds.vs[buf][b][in & 15] : reinterpret_cast<_Float16*>(&lds.spare[tid])) = (_Float16)(x * to_e);
  };
  const auto stash_s = [&](int buf, int j, float to_e) {
    const int b = blk + j * (4 / NP);
    // NaN where there is no block, or V is NaN: all bits
    const float x = __uint_as_float((sv[j] == sv[j] ? __float_as_uint(sk[j] * a.c) : ~0u) | ~named(of_s[j]));
    *(in < 16 ? &lds.ks[buf][b * 16 + (in & 15)] : &lds.spare[tid]) = x;
    *(in == 0 ? &lds.gone[buf][b] : reinterpret_cast<int*>(&lds.spare[tid])) = of_s[j] < 0;
    stash_vs(buf, j, sv[j], of_k[j], to_e);
  };

  // The first loads, of the table, of q and then of the pages, all at once.  Unit 2 s0's K lies in the other buffer, as the
  // stage before would have it, and so do V's first scales.
#pragma unroll
  for (int j = 0; j < NP; ++j) idk[j] = -1;
  look(s0 - 1);
  int raw_k0[NP], raw_s0[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    raw_k0[j] = raw_k[j];
    raw_s0[j] = raw_s[j];
  }
  look(s0);
  // V's scales of all of the item's blocks, four at a time (more of them in a loop)
  constexpr int kScan = 2;
  int raw_v[kScan];
#pragma unroll
  for (int i = 0; i < kScan; ++i) raw_v[i] = w.table[min(lo + (tid + i * kKv8Threads) / 4, w.max_blocks - 1)];
  const int r = wave * 32 + n;  // this lane's row (past the last, the tile's first: never stored)
  const int rr = row0 + (r < rows ? r : 0), tok = rr / a.G, head = rr - tok * a.G;
  const uint16_t* src = a.q + (int64_t)(first + tok) * a.q_stride + (int64_t)(kvh * a.G + head) * D + 8 * g;
  bf16x8 q[KS];
#pragma unroll
  for (int kk = 0; kk < KS; ++kk) q[kk] = *reinterpret_cast<const bf16x8*>(src + kk * 16);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = (f32x16)0.0f;
  m = -INFINITY;
  l = 0.0f;
  uint4 kw_first[NP];
  float sv_first[NP];
  int of_first[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int x = 4 * (s0 - 1) + blk + j * (4 / NP);
    of_first[j] = valid(x + 2, __builtin_amdgcn_readfirstlane(raw_k0[j]));
    const int64_t page0 = page(of_first[j]);
    kw_first[j] = *reinterpret_cast<const uint4*>(a.k_pages + page0 * page_bytes + ksrc);
    sv_first[j] = a.scales[page0 * (2 * kBlock) + kBlock + (in & 15)];
    idk[j] = of_first[j];
  }
  ids_of(s0);
  look(s0 + 1);
  fetch();
  float4 scan[kScan];
#pragma unroll
  for (int i = 0; i < kScan; ++i) {
    const int id = valid(lo + (tid + i * kKv8Threads) / 4, raw_v[i]);
    scan[i] = *reinterpret_cast<const float4*>(a.scales + page(id) * (2 * kBlock) + kBlock + 4 * (tid & 3));
    if (id < 0) scan[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  uint32_t most = 0, least = 0;  // of the bits; the least as what is missing to an infinity's
  const auto scale_in = [&](float4 v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = __float_as_uint((&v.x)[i]);  // scales are not negative
      const bool counts = x < 0x7F800000u && x != 0;
      most = max(most, counts ? x : 0u);
      least = max(least, counts ? 0x7F800000u - x : 0u);
    }
  };
#pragma unroll
  for (int i = 0; i < kScan; ++i) scale_in(scan[i]);
  for (int e = tid + kScan * kKv8Threads; e < 4 * (hi - lo); e += kKv8Threads) {
    const int id = valid(lo + e / 4, w.table[lo + e / 4]);
    if (id >= 0) scale_in(*reinterpret_cast<const float4*>(a.scales + page(id) * (2 * kBlock) + kBlock + 4 * (e & 3)));
  }
  most = wave_max_nonneg_bits(most);
  least = wave_max_nonneg_bits(least);
  if (lane == 0) {
    lds.most[wave] = most;
    lds.least[wave] = least;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kKv8Threads / kWave; ++k) {
    most = max(most, lds.most[k]);
    least = max(least, lds.least[k]);
  }
  E = max((int)(__builtin_amdgcn_readfirstlane(most) >> 23) - 127, -120);
  const int floor = 127 + E - kWideBand;
  if (floor > 0 && 0x7F800000u - __builtin_amdgcn_readfirstlane(least) < (uint32_t)floor << 23) return false;
  const float to_e = __uint_as_float((uint32_t)(127 + (FMT == kFp8 ? 5 : 7) - E) << 23);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    stash_k(1, j, kw_first[j], of_first[j]);
    stash_vs(1, j, sv_first[j], of_first[j], to_e);
    stash_k(0, j, kw[j], of_k[j]);
  }
  __syncthreads();
  f32x16 sc = (f32x16)0.0f;  // products of the unit whose scores come next
#pragma unroll
  for (int kk = 0; kk < KS; ++kk)
    sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, lds.k[1][1][kk][lane]), q[kk], sc, 0, 0, 0);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    stash_v(0, j);
    stash_s(0, j, to_e);
  }
  ids_of(s0 + 1);
  look(s0 + 2);
  fetch();
  __syncthreads();

  uint32_t pw[8];  // p of the unit whose p.V comes next: two operands
#pragma unroll
  for (int i = 0; i < 8; ++i) pw[i] = 0;
  const auto operand = [&](int h) { return __builtin_bit_cast(f16x8, make_uint4(pw[4 * h], pw[4 * h + 1], pw[4 * h + 2], pw[4 * h + 3])); };

  // Of two workgroups of a CU the older one's wavefronts go first, and it is done a quarter earlier; then the other has the CU to
  // itself, which it does not fill.  By turns of four stages they end together: 75.3 -> 73.0 us, with the merge, for 32 x 5
  // rows over 32768 tokens, 79.5 -> 76.8 for 64 x 5 over 16384 (in a graph of 20 calls).
  const int older = blockIdx.x < gridDim.x / 2 ? 1 : 0;
  for (int s = s0; s < s1; ++s) {
    if (((s - s0) >> 2 & 1) == older)
      __builtin_amdgcn_s_setprio(1);
    else
      __builtin_amdgcn_s_setprio(0);
    const int buf = (s - s0) & 1;
    const int4 about = *reinterpret_cast<const int4*>(lds.gone[buf]);
#pragma unroll
    for (int un = 0; un < 2; ++un) {
      constexpr int NG = KS, EPG = 16 / NG, kAhead = 2;
      static_assert(KS == 2 * DT, "a step has one matrix instruction of q.k^T and one of p.V");
      const auto kop = [&](int i) { return __builtin_bit_cast(bf16x8, lds.k[buf][un][i][lane]); };
      const auto vop = [&](int i) { return __builtin_bit_cast(f16x8, lds.v[buf][2 * un + i / DT][i % DT][lane]); };
      const auto k4 = [&](int j) { return *reinterpret_cast<const float4*>(&lds.ks[buf][32 * un + 8 * j + 4 * g]); };
      bf16x8 ok[kAhead];
      f16x8 ov[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        ok[i] = kop(i);
        ov[i] = vop(i);
      }
      float4 kq = k4(0), kq_next = k4(1);
      f32x16 sn = (f32x16)0.0f;
      uint32_t pn[8];
      float y[16], p[16], s4[4];
      const float nm = kWideBits - m;
      const auto expo = [&](int e) {
        y[e] = __builtin_fmaf(sc[e], (&kq.x)[e & 3], nm);
        if ((e & 3) == 3 && e < 15) {
          kq = kq_next;
          if (e < 11) kq_next = k4(e / 4 + 2);
        }
      };
      const auto take = [&](int e) {
        s4[e & 3] = e < 4 ? p[e] : s4[e & 3] + p[e];
        if (e & 1) pn[e / 2] = wide_f16x2(p[e - 1], p[e]);
      };
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ok[i % kAhead], q[i], sn, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < EPG; ++k) {
          const int e = i * EPG + k;
          expo(e);
          if (e >= EPG) p[e - EPG] = __builtin_amdgcn_exp2f(y[e - EPG]);
        }
        acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ov[i % kAhead], operand(i / DT), acc[i % DT], 0, 0, 0);
        if (i + kAhead < NG) {
          ok[i % kAhead] = kop(i + kAhead);
          ov[i % kAhead] = vop(i + kAhead);
        }
#pragma unroll
        for (int k = 0; k < EPG; ++k) {
          const int e = i * EPG + k;
          if (e >= 2 * EPG) take(e - 2 * EPG);
        }
        if (un == 0 && i < NP) stash_k(buf ^ 1, i, kw[i], of_k[i]);
        if (un == 0 && i >= NP && i < 2 * NP) {
          stash_v(buf ^ 1, i - NP);
          stash_s(buf ^ 1, i - NP, to_e);
        }
        if (un == 0 && i == 2 * NP) {
          ids_of(s + 2);
          look(s + 3);
          fetch();
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int e = 16 - 2 * EPG; e < 16; ++e) {
        if (e >= 16 - EPG) p[e] = __builtin_amdgcn_exp2f(y[e]);
        take(e);
      }
      float sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
      if (__any(!(sum < kWideBound))) {
        const bool g0 = __builtin_amdgcn_readfirstlane(un == 0 ? about.x : about.z) != 0, g1 = __builtin_amdgcn_readfirstlane(un == 0 ? about.y : about.w) != 0;
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 x = k4(j);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[4 * j + i] = (j < 2 ? g0 : g1) ? -INFINITY : sc[4 * j + i] * (&x.x)[i];
            mx = fmaxf(mx, y[4 * j + i]);
          }
        }
        const float2 pr = lane_pair<32>(mx);
        mx = fmaxf(fmaxf(pr.x, pr.y), m);
        const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
        l *= f;
        m = mx;
        const float up = mx == -INFINITY ? 0.0f : kWideBits - mx;
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(y[e] + up), p1 = __builtin_amdgcn_exp2f(y[e + 1] + up);
          sum += p0 + p1;
          pn[e / 2] = wide_f16x2(p0, p1);
        }
      }
      l += sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) pw[i] = pn[i];
      sc = sn;
    }
    __syncthreads();
  }
  __builtin_amdgcn_s_setprio(0);
  // the last unit's p.V
#pragma unroll
  for (int i = 0; i < 2 * DT; ++i)
    acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, lds.v[(s1 - s0) & 1][i / DT][i % DT][lane]), operand(i / DT), acc[i % DT], 0, 0, 0);
  return true;
}

}  // namespace sdv
