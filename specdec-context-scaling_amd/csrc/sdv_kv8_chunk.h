// Many rows over the 8-bit KV cache: prompt chunks, trees, and batches that hold one.
// Included by sdv_kv8_attn.hip.
//
// A workgroup of eight wavefronts takes a tile of 256 rows, 32 per wavefront, and streams stages of 64
// keys, two units of 32.  Products are v_mfma_f32_32x32x16: S^T = K Q^T in BF16 (codes and q as they
// are), O^T = V^T P^T in FP16, which holds P and V to 11 bits.  Lane (g, n) of a product holds row n
// and tokens 8j + 4g + i of the unit's two blocks: with those as its k-slots that is the B operand of
// the next product as it stands.
//
// Each stage's codes are converted once per workgroup on their way to LDS: K to BF16, V to
// fp16(code) * fp16(scale * 2^(b - E)), E the exponent of the largest V scale of the tile's keys so
// far (the sums are rescaled where it grows) and b such that the largest code stays under 2^15.  K's scale
// times the softmax's multiplies the scores.  p is held as 2^7 p.  The scales of a window of 64 stages are
// worked out before its loop and lie in LDS.
//
// How far that is off: each of V's two roundings is 2^-12 of a value, or 2^-25 where the product is below
// FP16's normal numbers, which is 2^(E - 30) or less.  The scale must be a normal number itself, or its
// rounding would be multiplied by the code.  So a window with scales below 2^(E - 18), as small V beside a row
// of zeros (scale 1) has them, is gone over twice, the second time for those alone, in units 2^18 times
// as small, and with no part in the sum of exponentials.  (Sums may lie 2^36 below the largest E so far; scales
// smaller still are off by up to 2^(E - 39).)  p is off by 2^-12 of it, or by 2^-32 where it is below 2^-21.
// Noticing such windows takes 1.3 us of a chunk's 45 to 115; a second loop that keeps V's codes as they are and
// puts its scale into two operands of p took the registers of the first (2048 rows over 8192 keys 720 us
// instead of 113).
//
// A token whose V scale is NaN has its V taken as 0 and its scores as NaN: that makes NaN of the rows
// that see it, and of no others.
//
// Bound by the matrix cores and what keeps them waiting: 2048 rows of 12 heads over 8192 keys (90 GFLOP,
// head_dim 128) take 113 to 116 us, 0.79 PFLOP/s, where a large product of the library reaches 1.27 at the
// clocks that such work runs at (1.7 to 1.8 GHz).  A stage takes 3400 cycles for 2080 of MFMA on each SIMD
// (without the scores 2600, without them and the conversions 2200); starts take 7 to 9 us (the plan 1.4,
// then page ids, scales and codes, one after another) and the parts' launch 8 to 12 (45 MB of them).
// 256 rows: a stage's conversion and its reads from LDS serve all of them; with 128 (four wavefronts)
// both would double.  Wave priorities move nothing.
//
// Softmax in one pass: units that all rows see take exp2(s - m) against the maximum so far; one that
// would bring a lane's sum over it to 2^8 (a score 8 above m in base 2, or more than one near that) is
// done again with a new maximum, from products that are still in registers.  Units that need a mask,
// and a segment's first, take the maximum first.
#pragma once

#include <type_traits>

namespace sdv {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kChunkWaves = 8;
constexpr int kChunkRows = 32 * kChunkWaves;
constexpr int kChunkThreads = kWave * kChunkWaves;
constexpr int kChunkGrid = 256;      // workgroups, one per CU
constexpr int kChunkStages = 64;     // of a window, whose page ids and scales are held in LDS
constexpr int kChunkTokens = kKv8Step * kChunkStages;
constexpr int kChunkBand = 18;       // binades of V's scales that one pass over a window serves
constexpr float kChunkBits = 7.0f;   // p is held as 2^7 p
constexpr float kChunkBound = 32768.0f;  // of a lane's 16 of them in a unit: each stays under FP16's largest

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
}

// Four codes as FP16, exactly.
template <int FMT>
__device__ __forceinline__ uint2 chunk_f16x4(uint32_t w) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (FMT == kFp8) {
    return make_uint2(__builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                      __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)));
  } else {
    // with the sign bit turned a code is c + 128; under the bits 0x6400 that is 1024 + c + 128 in FP16
    const uint32_t u = w ^ 0x80808080u;
    const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    const f16x2 lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
    const f16x2 hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
  }
}

// Four V codes times their tokens' scales (FP16 pairs), as FP16.
template <int FMT>
__device__ __forceinline__ uint2 chunk_v4(uint32_t w, uint32_t s01, uint32_t s23) {
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  const uint2 c = chunk_f16x4<FMT>(w);
  const f16x2 lo = __builtin_bit_cast(f16x2, c.x) * __builtin_bit_cast(f16x2, s01);
  const f16x2 hi = __builtin_bit_cast(f16x2, c.y) * __builtin_bit_cast(f16x2, s23);
  return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// A tile that begins in a workgroup's range and is cut by its end.  Its first part lies in `slot`
// (2w or 2w + 1), the later ones in the first slots of the ranges that follow: 2(w + 1), 2(w + 2), ...
struct Kv8Cut {
  int parts;     // 0: none
  int slot;
  int first, n;  // the sequence's packed rows
  int kvh, i;    // KV head and tile
  int pad[2];
};

// A part: [wavefront][32-dimension tile][4][lane] pieces of 16 bytes, then [wavefront][lane] (maximum, sum).
// The pieces are divided by the part's sum of exponentials: before that those of a large V pass fp32's range.
template <int D>
constexpr int chunk_part() {
  return kChunkRows * D + kChunkThreads * 2;
}

template <int D, int FMT>
__global__ __launch_bounds__(kChunkThreads) __attribute__((amdgpu_waves_per_eu(2))) void kv8_chunk_kernel(Kv8AttnArgs a) {
  constexpr int W = kChunkWaves, NB = 3;
  constexpr int KS = D / 16;              // MFMA steps of a unit's q.k^T
  constexpr int DT = D / 32;              // 32-dimension tiles of the output
  constexpr int kUnit = 32 * D * 2;       // bytes of a unit's K, and of its V
  constexpr int kBlk = kUnit / 2;
  constexpr int kVAt = 2 * kUnit;         // a stage: K of two units, then V of two
  __shared__ __align__(16) uint8_t ring[NB][4 * kUnit];
  __shared__ __align__(16) float lds_ks[kChunkTokens + 32];  // the window's scales of the scores (one unit is read past it)
  __shared__ __align__(16) _Float16 lds_vs[kChunkTokens];    // and of V
  __shared__ int lpb[kChunkTokens / kBlock];                 // its page ids; -1: no block
  __shared__ uint32_t s_max[W], s_bad[W], s_low[W];
  __shared__ Kv8PlanLds<kChunkThreads> lds_plan;

  Kv8Cut cut = {};
  Kv8Place<kChunkRows, kChunkThreads> at;
  if (!at.begin(a, lds_plan, (int)blockIdx.x, (int)gridDim.x)) {
    if (threadIdx.x == 0) a.cuts[blockIdx.x] = cut;
    return;
  }
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 5, n = lane & 31;
  const int64_t page_bytes = (int64_t)kBlock * D;
  // this wavefront's share of a stage: half of block `wave / 2`'s K, and of its V
  const int blk = wave >> 1, half = wave & 1;
  // lane's piece of K and V in a page, and where it goes
  const int t16 = lane & 15;
  const int kc = (lane >> 4) + 4 * half;  // K chunk: 16 dimensions of head_dim 128, 8 of 64
  const int ksrc = (t16 >> 2) * (4 * D) + (t16 & 3) * 16 + (D == 128 ? kc * 64 : (kc >> 1) * 64 + (kc & 1) * 8);
  const int kdst = (blk >> 1) * kUnit + (blk & 1) * kBlk + (D == 128 ? 2 * kc : kc) * 256 + t16 * 16;
  const int vd = D == 128 ? 64 * half + lane : lane;  // V dimension; of 64 a half of its tokens
  const int vsrc = vd * kBlock + (D == 128 ? 0 : 8 * half);
  const int vdst = kVAt + (blk >> 1) * kUnit + (blk & 1) * kBlk + (vd >> 5) * 1024 + (vd & 31) * 16 + (D == 128 ? 0 : 8 * half);
  const int vtok = (blk & 1) * kBlock + (D == 128 ? 0 : 8 * half);  // the piece's first token in its unit
  const unsigned kofs = (unsigned)((n >> 4) * kBlk + g * 256 + (n & 15) * 16);
  bool first_part = true;

  for (;;) {
    const Kv8Seq seq = at.seq;
    const int b = at.b, kvh = at.kvh;
    const uint32_t last_unit = min(at.units_of, at.end - at.tile0);
    int slo, shi, steps;
    if (!at.part(a, slo, shi, steps)) break;  // the range ends within the tile's start
    const int row0 = at.i * kChunkRows, rows = min(seq.n * a.G - row0, kChunkRows);
    const int nbk = (seq.T + kBlock - 1) / kBlock;
    const int32_t* table = a.r.table + (int64_t)b * a.r.max_blocks;

    // Page ids of a window, of a thread's tokens (four at a time, tokens 4 (tid + 512 i)) and of the
    // pieces that go first: unit 0's K and stage 0.  Loaded before all else, since the scales and codes
    // wait for them.
    constexpr int kTok = kChunkTokens / 4 / kChunkThreads;
    int idt[kTok], id_k0, id_k1, id_v1;
    const auto load_ids = [&](int wlo) {
      const int last = 4 * min(kChunkStages, shi - wlo) - 1;  // block of the window
      const auto id_of = [&](int j) { return 4 * wlo + j < nbk ? kv8_block(a.r, b, 4 * wlo + j) : -1; };
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const int j = (tid + kChunkThreads * i) / 4;
        idt[i] = j <= last ? id_of(j) : -1;
      }
      id_k0 = id_of(blk & 1);
      id_k1 = id_of(2 + blk);  // units 1 and 2: blocks 2 .. 5, clamped like the loop's
      if (2 + blk > last) id_k1 = id_of(last - 1 + (blk & 1));
      id_v1 = id_of(blk & 1);  // units 0 (for -1) and 0
    };
    load_ids(slo);

    // this lane's row (of a wavefront without rows, or past the last, the tile's first: never stored)
    const int r = wave * 32 + n;
    const bool rv = r < rows;
    const int rr = row0 + (rv ? r : 0), tok = rr / a.G, head = kvh * a.G + rr - tok * a.G;
    const uint16_t* src = a.q + (int64_t)(seq.first + tok) * a.q_stride + (int64_t)head * D;
    bf16x8 qop[KS];
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) qop[kk] = *reinterpret_cast<const bf16x8*>(src + kk * 16 + g * 8);
    // last key that the row sees (with a tree, the context's last), and the new tokens of a tree
    const int lim = !rv ? -1 : seq.tree ? seq.ctx - 1 : seq.ctx + tok;
    const uint64_t bits = seq.tree && rv ? a.tree[seq.first + tok] : 0;
    const bool active = wave * 32 < rows;  // the wavefront has rows
    // units that all of its rows see
    const int all = seq.tree ? seq.ctx - 1 : seq.ctx + (row0 + min(wave * 32, rows - 1)) / a.G;
    const int ufull = max(all + 1, 0) >> 5;

    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = (f32x16)0.0f;
    float m = -INFINITY, l = 0.0f;
    int e_acc = -120, e_top = -120;  // exponent that the sums are relative to, the largest it has been

    bool low = false;  // second pass over a window: its small V scales
    for (int wlo = slo; wlo < shi;) {                      // windows; workgroup-uniform
      const int nit = min(kChunkStages, shi - wlo);        // stages
      // Units of the window (32 keys): x = 0 .. 2 nit - 1, the first at key 32 ux0.  The loop multiplies
      // q.k^T one unit ahead of the scores and p.V one unit behind them: buffer s holds K of units
      // 2s + 1, 2s + 2 and V of units 2s - 1, 2s.  Past the window's ends the nearest unit is loaded;
      // its products are not used, or meet p = 0.
      const int ux0 = 2 * wlo, nx = 2 * nit;
      const auto unit_at = [&](int x) { return min(max(x, 0), nx - 1); };

      // ---- a stage on its way to LDS
      uint4 kw, vw;  // codes (head_dim 64: the first half)
      uint4 sw[2];   // V's scales of the piece's tokens
      int vblk;      // tokens of the piece's block that the sequence has
      // the piece's block in the window, of K and of V
      const auto kblock = [&](int s) { return 2 * unit_at(2 * s + 1 + (blk >> 1)) + (blk & 1); };
      const auto vblock = [&](int s) { return 2 * unit_at(2 * s - 1 + (blk >> 1)) + (blk & 1); };
      const auto fetch = [&](const uint8_t* pages, uint32_t at_byte, int id) {
        const uint8_t* p = pages + ((int64_t)max(id, 0) * a.kv_heads + kvh) * page_bytes;
        if constexpr (D == 128) return *reinterpret_cast<const uint4*>(p + at_byte);
        const uint2 w = *reinterpret_cast<const uint2*>(p + at_byte);
        return make_uint4(w.x, w.y, 0, 0);
      };
      const auto fetch_k = [&](int id) { kw = fetch(a.k_pages, (uint32_t)ksrc, id); };
      const auto fetch_v = [&](int s, int id) {
        vw = fetch(a.v_pages, (uint32_t)vsrc, id);
        vblk = id < 0 ? 0 : seq.T - (2 * ux0 + vblock(s)) * kBlock;
      };
      const auto stash_k = [&](uint8_t* buf, int h) {
        if (D == 128 && h == 1)
          *reinterpret_cast<bf16x8*>(buf + kdst + 256) = kv8_bf16x8<FMT>(kw.z, kw.w);
        else if (h == 0)
          *reinterpret_cast<bf16x8*>(buf + kdst) = kv8_bf16x8<FMT>(kw.x, kw.y);
      };
      const auto read_vs = [&](int s) {
        const _Float16* src = &lds_vs[32 * unit_at(2 * s - 1 + (blk >> 1)) + vtok];
        sw[0] = *reinterpret_cast<const uint4*>(src);
        if constexpr (D == 128) sw[1] = *reinterpret_cast<const uint4*>(src + 8);
      };
      // tokens 0..3 and 8..11 of the piece's block (h = 0), or 4..7 and 12..15
      const auto stash_v = [&](uint8_t* buf, int h) {
        // codes of no token of the sequence may decode to NaN (scalar masks: no branch among the steps)
        const int k = D == 128 ? vblk : vblk - 8 * half;
        (&vw.x)[h] &= kv8_keep(k, h);
        if constexpr (D == 128) (&vw.x)[h + 2] &= kv8_keep(k, h + 2);
        const uint2 a0 = h == 0 ? chunk_v4<FMT>(vw.x, sw[0].x, sw[0].y) : chunk_v4<FMT>(vw.y, sw[0].z, sw[0].w);
        if constexpr (D == 128) {
          const uint2 a2 = h == 0 ? chunk_v4<FMT>(vw.z, sw[1].x, sw[1].y) : chunk_v4<FMT>(vw.w, sw[1].z, sw[1].w);
          *reinterpret_cast<uint4*>(buf + vdst + 512 * h) = make_uint4(a0.x, a0.y, a2.x, a2.y);
        } else {
          *reinterpret_cast<uint2*>(buf + vdst + 512 * h) = a0;
        }
      };

      // the first loads
      const int block0 = 4 * wlo;
      fetch_k(__builtin_amdgcn_readfirstlane(id_k0));
      const uint4 kw_first = kw;
      fetch_k(__builtin_amdgcn_readfirstlane(id_k1));
      fetch_v(0, __builtin_amdgcn_readfirstlane(id_v1));

      // scales of the window
      const int quad = (tid & 3) * 4;
      float4 kst[kTok], vst[kTok];
      uint32_t mine = 0;
      bool wrong = false;
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const int j = (tid + kChunkThreads * i) / 4;  // block of the window
        wrong = wrong || (j < 4 * nit && block0 + j < nbk && idt[i] < 0);
      }
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const float* sp = a.scales + ((int64_t)max(idt[i], 0) * a.kv_heads + kvh) * (2 * kBlock) + quad;
        kst[i] = *reinterpret_cast<const float4*>(sp);
        vst[i] = *reinterpret_cast<const float4*>(sp + kBlock);
      }
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const int t0 = (block0 + (tid + kChunkThreads * i) / 4) * kBlock + quad;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float &k = (&kst[i].x)[c], &v = (&vst[i].x)[c];
          k = v == v ? k * a.c : v;
          const uint32_t ab = __float_as_uint(v);  // scales are not negative
          if (idt[i] < 0 || t0 + c >= seq.T || ab >= 0x7F800000u) v = 0.0f;
          mine = max(mine, __float_as_uint(v));
        }
      }
      mine = wave_max_nonneg_bits(mine);
      __syncthreads();  // the last window's are no longer read
      if (lane == 0) s_max[wave] = mine;
      if (lane == 0) s_bad[wave] = 0;
      if (wrong) s_bad[wave] = 1;
      __syncthreads();
      uint32_t largest = 0, any_bad = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        largest = max(largest, s_max[i]);
        any_bad |= s_bad[i];
      }
      const bool bad = __builtin_amdgcn_readfirstlane(any_bad) != 0;
      // the sums in units of the window's exponent, or of the small scales'
      const int e = low ? e_acc - kChunkBand : max(e_acc, (int)(__builtin_amdgcn_readfirstlane(largest) >> 23) - 127);
      e_top = max(e_top, e);
      const int e_split = low ? e : e < max(e_top - kChunkBand, kChunkBand - 120) ? -127 : e - kChunkBand;
      const uint32_t split = (uint32_t)(127 + e_split) << 23;
      bool below = false;
#pragma unroll
      for (int i = 0; i < kTok; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float& v = (&vst[i].x)[c];
          const bool small = __float_as_uint(v) < split;
          below = below || (small && v != 0.0f);
          if (small != low) v = 0.0f;
        }
      if (lane == 0) s_low[wave] = 0;
      if (below) s_low[wave] = 1;
      const float l_top = l, m_top = m;
      if (e != e_acc) {
        const float f = __builtin_amdgcn_ldexpf(1.0f, max(e_acc - e, -126));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
        e_acc = e;
      }
      const float to_e = __uint_as_float((uint32_t)(127 + (FMT == kFp8 ? 5 : 7) - e) << 23);
#pragma unroll
      for (int i = 0; i < kTok; ++i) {
        const int t = tid + kChunkThreads * i;
        *reinterpret_cast<float4*>(&lds_ks[4 * t]) = kst[i];
        *reinterpret_cast<uint2*>(&lds_vs[4 * t]) = make_uint2(pack_f16x2(vst[i].x * to_e, vst[i].y * to_e), pack_f16x2(vst[i].z * to_e, vst[i].w * to_e));
        if ((tid & 3) == 0) lpb[t / 4] = idt[i];
      }
      __syncthreads();

      uint8_t *cur = ring[0], *nxt = ring[1], *third = ring[2];
      const auto rotate = [&]() {
        uint8_t* const t = cur;
        cur = nxt;
        nxt = third;
        third = t;
      };

      // ---- products and scores
      constexpr int NM = KS + 2 * DT, SPM = 16 / NM, kAhead = 4;
      static_assert(KS == 2 * DT && NM * SPM == 16, "q.k^T and p.V steps alternate");
      const auto operand = [&](const uint8_t* sb, int mstep) {  // step of unit mstep / NM: k step or tile i
        const int un = mstep / NM, i = (mstep % NM) / 2;
        return (mstep & 1) ? *reinterpret_cast<const uint4*>(sb + kVAt + un * kUnit + i * 1024 + lane * 16)
                           : *reinterpret_cast<const uint4*>(sb + un * kUnit + i * 512 + kofs);
      };
      uint4 op[kAhead];
      f32x16 sc;       // products of the unit whose scores come next
      uint32_t pw[8];  // p of the unit whose p.V product comes next: two MFMA operands
      const auto pop = [&](int h) {
        return __builtin_bit_cast(f16x8, make_uint4(pw[4 * h], pw[4 * h + 1], pw[4 * h + 2], pw[4 * h + 3]));
      };
      const auto scale4 = [&](int x, int j) { return *reinterpret_cast<const float4*>(&lds_ks[32 * x + 8 * j + 4 * g]); };
      // scores of unit x from its products with a maximum of their own: sums and maximum moved as they
      // need, p to pn, their sum returned
      const auto renew = [&](int x, uint32_t (&pn)[8]) {
        float y[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float4 k4 = scale4(x, j);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[4 * j + i] = sc[4 * j + i] * (&k4.x)[i];
        }
        const int k0 = 32 * (ux0 + x) + 4 * g;  // key of element 0; element e is key k0 + 8 (e / 4) + e % 4
        const auto first = [](int k) { return k >= 32 ? ~0u : k <= 0 ? 0u : (1u << k) - 1u; };
        uint32_t vis = first(lim + 1 - k0);
        const int sh = k0 - seq.ctx;
        if (seq.tree && sh > -32 && sh < 64) vis |= (uint32_t)(sh >= 0 ? bits >> sh : bits << -sh) & first(seq.T - k0);
        // the lane's keys of the first block are bits 0..3 and 8..11, of the second 16..19 and 24..27
        if (lpb[2 * unit_at(x)] < 0) vis &= 0xFFFF0000u;
        if (lpb[2 * unit_at(x) + 1] < 0) vis &= 0x0000FFFFu;
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          y[e] = (vis >> (8 * (e >> 2) + (e & 3))) & 1 ? y[e] : -INFINITY;
          mx = fmaxf(mx, y[e]);
        }
        const float2 pr = lane_pair<32>(mx);
        mx = fmaxf(fmaxf(pr.x, pr.y), m);
        const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= f;
        l *= f;
        m = mx;
        const float nm = mx == -INFINITY ? 0.0f : kChunkBits - mx;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float p0 = __builtin_amdgcn_exp2f(y[e] + nm), p1 = __builtin_amdgcn_exp2f(y[e + 1] + nm);
          sum += p0 + p1;
          pn[e / 2] = pack_f16x2(p0, p1);
        }
        return sum;
      };
      const auto publish = [&]() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
      };
      float4 kq[4];  // the scores' scales, two groups of four ahead
      const int nfast = !active || bad ? 0 : min(nit, max(0, (ufull - ux0) >> 1));

      // One iteration is two units of NM steps.  A step issues one MFMA -- q.k^T of the next unit and
      // p.V of the one before in turn -- reads the LDS operand of the step kAhead later and works on
      // 16 / NM scores of this unit.  The three do not depend on each other, and the scheduling
      // barriers hold the order.  The first unit's steps also convert and write the next stage, whose
      // loads went out an iteration ago, to the third buffer, and send the loads of the stage after it;
      // the barrier at its end publishes the stage.
      const auto body = [&](int it, bool fast) {
        f32x16 sn = (f32x16)0.0f;
        uint32_t pn[8];
        int idk = 0, idv = 0;
#pragma unroll
        for (int un = 0; un < 2; ++un) {
          // A step works on the exponent of one score (or two), the exponential of the one before and the
          // sum and conversion of the one before that: none waits for another.
          const float nm = kChunkBits - m;
          float y[16], p[16], s4[4];
          const auto expo = [&](int e) {
            const int j = e >> 2;
            y[e] = __builtin_fmaf(sc[e], (&kq[j].x)[e & 3], nm);
            if ((e & 3) == 3) kq[j] = scale4(2 * it + un + 1, j);  // of the next unit
          };
          const auto take = [&](int e) {
            s4[e & 3] = e < 4 ? p[e] : s4[e & 3] + p[e];
            if (e & 1) pn[e / 2] = pack_f16x2(p[e - 1], p[e]);
          };
#pragma unroll
          for (int mm = 0; mm < NM; ++mm) {
            const int ms = un * NM + mm, i = mm / 2;
            if (mm & 1)
              acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, op[ms % kAhead]), pop(i / DT), acc[i % DT], 0, 0, 0);
            else
              sn = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, op[ms % kAhead]), qop[i], mm == 0 ? (f32x16)0.0f : sn, 0, 0, 0);
            op[ms % kAhead] = ms + kAhead < 2 * NM ? operand(cur, ms + kAhead) : operand(nxt, ms + kAhead - 2 * NM);
            if (fast) {
#pragma unroll
              for (int k = 0; k < SPM; ++k) {
                const int e = mm * SPM + k;
                if (e >= 2 * SPM) take(e - 2 * SPM);
                if (e >= SPM) p[e - SPM] = __builtin_amdgcn_exp2f(y[e - SPM]);
                expo(e);
              }
            }
            if (un == 0) {
              if (mm == 0) {
                read_vs(it + 1);
                idk = lpb[kblock(it + 2)];
                idv = lpb[vblock(it + 2)];
                stash_k(nxt, 0);
              }
              if (mm == (NM > 8 ? 2 : 1)) stash_k(nxt, 1);
              if (mm == (NM > 8 ? 4 : 2)) stash_v(nxt, 0);
              if (mm == (NM > 8 ? 6 : 3)) stash_v(nxt, 1);
              if (mm == (NM > 8 ? 8 : 4)) fetch_k(__builtin_amdgcn_readfirstlane(idk));
              if (mm == (NM > 8 ? 9 : 4)) fetch_v(it + 2, __builtin_amdgcn_readfirstlane(idv));
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          float sum = 0.0f;
          if (fast) {
#pragma unroll
            for (int e = 16 - 2 * SPM; e < 16; ++e) {
              if (e >= 16 - SPM) p[e] = __builtin_amdgcn_exp2f(y[e]);
              take(e);
            }
            sum = (s4[0] + s4[1]) + (s4[2] + s4[3]);
          }
          if (!fast || __any(rv && !(sum < kChunkBound))) sum = renew(2 * it + un, pn);
          if (!fast) {
#pragma unroll
            for (int j = 0; j < 4; ++j) kq[j] = scale4(2 * it + un + 1, j);
          }
          l += sum;
#pragma unroll
          for (int w = 0; w < 8; ++w) pw[w] = pn[w];
          sc = sn;
          if (un == 0) publish();
        }
        rotate();
      };

      const auto stash = [&](uint8_t* buf) {
        stash_k(buf, 0);
        stash_k(buf, 1);
        stash_v(buf, 0);
        stash_v(buf, 1);
      };
      const auto fetch_stage = [&](int s) {
        fetch_k(__builtin_amdgcn_readfirstlane(lpb[kblock(s)]));
        fetch_v(s, __builtin_amdgcn_readfirstlane(lpb[vblock(s)]));
      };
      read_vs(0);
      stash(cur);
      kw = kw_first;
      stash_k(third, 0);
      stash_k(third, 1);
      fetch_stage(1);
      publish();
      if (active) {
        sc = (f32x16)0.0f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
          sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*reinterpret_cast<const bf16x8*>(third + kUnit + kk * 512 + kofs), qop[kk], sc, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 8; ++w) pw[w] = 0;
#pragma unroll
        for (int ms = 0; ms < kAhead; ++ms) op[ms] = operand(cur, ms);
#pragma unroll
        for (int j = 0; j < 4; ++j) kq[j] = scale4(0, j);
      }
      int it = 0;
      if (active) {
        body(it++, false);
        for (; it < nfast; ++it) body(it, true);
        for (; it < nit; ++it) body(it, false);
        // the last unit's p.V
#pragma unroll
        for (int i = 0; i < 2 * DT; ++i)
          acc[i % DT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, operand(cur, 2 * i + 1)), pop(i / DT), acc[i % DT], 0, 0, 0);
      } else {  // a wavefront without rows loads its share
        for (; it < nit; ++it) {
          read_vs(it + 1);
          stash(nxt);
          fetch_stage(it + 2);
          publish();
          rotate();
        }
      }
      uint32_t any_low = 0;
#pragma unroll
      for (int i = 0; i < W; ++i) any_low |= s_low[i];
      if (low && m_top != m)
        l = l_top * __builtin_amdgcn_exp2f(m_top - m);  // counted in the first pass
      else if (low)
        l = l_top;
      low = !low && __builtin_amdgcn_readfirstlane(any_low) != 0;
      if (!low) wlo += kChunkStages;
      if (wlo < shi) load_ids(wlo);
    }

    // the sums in units of 1
    const float unit = __builtin_amdgcn_ldexpf(1.0f, e_acc - (FMT == kFp8 ? 5 : 7));
    const float2 pr = lane_pair<32>(l);
    l = pr.x + pr.y;
    if (__builtin_expect(rv && m == -INFINITY, 0)) m = kv8_lowest(a, b, seq, tok, slo * kKv8Step, shi * kKv8Step);
    const bool whole = slo == 0 && shi == steps;
    // a row that sees nothing: 0; a part without exponentials has no weight
    const float inv = m == -INFINITY || (!whole && l == 0.0f) ? 0.0f : unit / l;
    if (whole) {
      if (rv) {
        uint16_t* dst = a.out + (int64_t)(seq.first + tok) * a.out_stride + (int64_t)head * D + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint2*>(dst + dt * 32 + 8 * j) = make_uint2(pack_bf16x2(acc[dt][4 * j] * inv, acc[dt][4 * j + 1] * inv),
                                                                          pack_bf16x2(acc[dt][4 * j + 2] * inv, acc[dt][4 * j + 3] * inv));
      }
    } else {
      const int slot = 2 * at.w + (first_part ? 0 : 1);
      float* part = a.part + (int64_t)slot * chunk_part<D>();
      if (active) {
        float4* p4 = reinterpret_cast<float4*>(part) + wave * (DT * 4 * 64) + lane;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            p4[(dt * 4 + j) * 64] = make_float4(acc[dt][4 * j] * inv, acc[dt][4 * j + 1] * inv, acc[dt][4 * j + 2] * inv, acc[dt][4 * j + 3] * inv);
        reinterpret_cast<float2*>(part + kChunkRows * D)[tid] = make_float2(m, l);
      }
      if (slo == 0) {
        cut.parts = at.parts(a);
        cut.slot = slot;
        cut.first = seq.first;
        cut.n = seq.n;
        cut.kvh = kvh;
        cut.i = at.i;
      }
    }
    first_part = false;
    at.u = at.tile0 + last_unit;
    if (at.u >= at.end || !at.next(a)) break;
    __syncthreads();  // lpb and the ring
  }
  if (tid == 0) a.cuts[blockIdx.x] = cut;
}

// The parts of the x-th cut tile, in their order: 32 rows of 32 dimensions a
// workgroup, a thread four dimensions of a row (a piece of lane n or n + 32).  Four parts are in flight
// where there are no more (2048 rows over 8192 keys: most tiles have four), else 16.
template <int D>
__global__ __launch_bounds__(256) void kv8_chunk_merge_kernel(Kv8AttnArgs a, int ranges) {
  constexpr int DT = D / 32, kPart = chunk_part<D>();
  static_assert(kChunkGrid == 256, "a thread per range");
  // the x-th range that cuts a tile
  __shared__ int s_count[4], s_range;
  const int tid = threadIdx.x;
  const uint64_t cuts = __ballot(tid < ranges && a.cuts[min(tid, ranges - 1)].parts > 0);
  if ((tid & 63) == 0) s_count[tid >> 6] = __popcll(cuts);
  if (tid == 0) s_range = -1;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) before += k < (tid >> 6) ? s_count[k] : 0;
  before += __popcll(cuts & ((1ull << (tid & 63)) - 1));
  if ((cuts >> (tid & 63) & 1) && before == (int)blockIdx.x) s_range = tid;
  __syncthreads();
  if (s_range < 0) return;
  const Kv8Cut cut = a.cuts[s_range];
  const int wave = blockIdx.y / DT, dt = blockIdx.y % DT, lane = threadIdx.x & 63, j = threadIdx.x >> 6, n = lane & 31;
  const int row = cut.i * kChunkRows + wave * 32 + n;
  if (row >= cut.n * a.G) return;
  const auto part = [&](int k) { return a.part + (int64_t)(k == 0 ? cut.slot : (cut.slot & ~1) + 2 * k) * kPart; };
  float m = -INFINITY, l = 0.0f;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  const auto add = [&](auto batch, int k0) {
    constexpr int kBatch = decltype(batch)::value;
    float2 st[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {  // past the last part its own again, not counted
      const float* p = part(min(k0 + k, cut.parts - 1));
      st[k] = reinterpret_cast<const float2*>(p + kChunkRows * D)[wave * 64 + n];
      v[k] = reinterpret_cast<const float4*>(p)[wave * (DT * 4 * 64) + (dt * 4 + j) * 64 + lane];
    }
    float mx = m;
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (k0 + k < cut.parts) mx = fmaxf(mx, st[k].x);
    // the mean so far and the parts' means, weighted by their sums of exponentials
    float w[kBatch], before = mx == -INFINITY ? l : l * __builtin_amdgcn_exp2f(m - mx);
    l = before;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      w[k] = k0 + k >= cut.parts ? 0.0f : mx == -INFINITY ? st[k].y : st[k].y * __builtin_amdgcn_exp2f(st[k].x - mx);
      l += w[k];
    }
    m = mx;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    before *= inv;
    sum = make_float4(sum.x * before, sum.y * before, sum.z * before, sum.w * before);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float x = w[k] * inv;
      sum = make_float4(sum.x + v[k].x * x, sum.y + v[k].y * x, sum.z + v[k].z * x, sum.w + v[k].w * x);
    }
  };
  if (cut.parts <= 4) {
    add(std::integral_constant<int, 4>(), 0);
  } else {
    for (int k0 = 0; k0 < cut.parts; k0 += 16) add(std::integral_constant<int, 16>(), k0);
  }
  if (m != -INFINITY && l == 0.0f) sum = make_float4(NAN, NAN, NAN, NAN);  // scores of -inf alone
  const int tok = row / a.G, head = cut.kvh * a.G + row - tok * a.G;
  *reinterpret_cast<uint2*>(a.out + (int64_t)(cut.first + tok) * a.out_stride + (int64_t)head * D + 32 * dt + 8 * j + 4 * (lane >> 5)) =
      make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w));
}

}  // namespace sdv
