// Attention of ragged query rows over the 8-bit KV cache (layout: sdv_kv8.h; shares: sdv_kv8_plan.h).
//
//   x_j = scale * s^K_j * (q . c^K_j),   out = sum_j e^(x_j - M) s^V_j c^V_j / sum_j e^(x_j - M)
//
// over the keys j that the row sees, in one pass over them with a running maximum and sum.  The
// codes c are exact in BF16, so q.c is exact products summed in fp32 on the matrix cores, and K's
// scales multiply the fp32 scores.  The one rounding before the output's is that of the operands of
// the second product: e^(..) s^V to 16 bits here, e^(..) and s^V c^V to FP16 in the kernel for many
// rows.  (With e^(..) s^V as one BF16 operand, 2^-9 of each term, the outputs' error against 64 bits
// was 2.7e-3, of which BF16 outputs alone make 1.6e-3.)
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

// Counts of finished parts, per slot and range; every call leaves its slot's zero, as the loader does.
static __device__ uint32_t kv8_counts[SDV_KV8_SLOTS][kKv8Grid];

// The maximum that stands for a row none of whose scores of keys lo .. hi - 1 is above -inf: -inf where
// it sees none of the keys, the lowest finite number where it does (scores of an infinite q, or NaN).  Both
// sums are 0 or NaN; over all keys the first is an output of 0 and the second 0 / 0.  Looked for block by
// block, since it hardly ever comes to this: keys up to the row's own position, or the context and its
// mask's tokens, in blocks that the table names.  (As a check of each output's sum in kv8_write and the
// merges the code that this takes made a call over 2048 keys 0.2 us longer, 7.7 to 7.9.)
__device__ __forceinline__ float kv8_lowest(const Kv8AttnArgs& a, int b, const Kv8Seq& s, int tok, int lo, int hi) {
  const int last = min(s.tree ? s.ctx - 1 : s.ctx + tok, hi - 1);
  bool any = false;
  for (int j = lo / kBlock; !any && j < a.r.max_blocks && j * kBlock <= last; ++j) any = kv8_block(a.r, b, j) >= 0;
  if (s.tree) {
    const uint64_t bits = a.tree[s.first + tok];
    for (int j = max(lo - s.ctx, 0); !any && j < min(min(hi - s.ctx, s.n), 64); ++j)
      any = ((bits >> j) & 1) != 0 && kv8_block(a.r, b, (s.ctx + j) >> 4) >= 0;
  }
  return any ? -3.4028235e38f : -INFINITY;
}

// ---------------------------------------------------------------------------- shared tiles
// The parts of a tile that several ranges share: each workgroup leaves its sums in a slot of the
// workspace and counts itself in done[first range]; the one that finds all others counted adds the
// parts up in range order (so the result does not depend on which one it is) and clears the count.
// Nothing waits.  Parts are written and read with device scope (sc1: through to the memory that all
// XCDs see), 16 bytes at a time, and every wavefront waits for its stores before the barrier before
// the count.  Fences that write back or drop an XCD's L2 instead cost its other workgroups more (a
// batch of 32 sequences 56 -> 59 us with an acquire fence per merge).
typedef unsigned int kv8_u32x4 __attribute__((ext_vector_type(4)));
constexpr int kDeviceScope = 16;  // sc1

__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv8_parts(float* part, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(part, 0, bytes, 0x00027000);
}
__device__ __forceinline__ void kv8_put(__amdgpu_buffer_rsrc_t r, int at, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(kv8_u32x4, v), r, at, 0, kDeviceScope);
}
__device__ __forceinline__ f32x4 kv8_get(__amdgpu_buffer_rsrc_t r, int at) {
  return __builtin_bit_cast(f32x4, (kv8_u32x4)__builtin_amdgcn_raw_buffer_load_b128(r, at, 0, kDeviceScope));
}

// True in the workgroup that finishes last of `parts`.  All its threads call it; *lds_flag is theirs.
__device__ __forceinline__ bool kv8_last(uint32_t* done, int parts, int* lds_flag) {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t before = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *lds_flag = before + 1 == (uint32_t)parts;
    if (before + 1 == (uint32_t)parts) __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  asm volatile("" ::: "memory");
  return *lds_flag != 0;
}

// A tile's rows: row0 .. row0 + rows - 1 of the sequence whose packed rows begin at `first`.
struct Kv8TileRows {
  int row0, rows, first, kvh;
};

// Four dimensions of row r of a tile: the sum over the keys divided by that of the exponentials, m their maximum.
template <int D>
__device__ __forceinline__ void kv8_write(const Kv8AttnArgs& a, const Kv8TileRows& t, int r, int d, f32x4 acc, float m, float l) {
  const float inv = m == -INFINITY ? 0.0f : 1.0f / l;  // a row that sees nothing: 0
  const int tok = (t.row0 + r) / a.G, head = t.row0 + r - tok * a.G;
  *reinterpret_cast<uint2*>(a.out + (int64_t)(t.first + tok) * a.out_stride + (int64_t)(t.kvh * a.G + head) * D + d) =
      make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
}

// Adds up a tile's parts: slot 2 w0 + skip, then 2 (w0 + 1), 2 (w0 + 2), ...  A batch of them at a time:
// their maxima and sums by way of LDS, 16 pieces of 16 bytes a thread in flight beside them (a load that
// goes past the caches takes about a microsecond).
template <int D, int TR>
__device__ __forceinline__ void kv8_merge(const Kv8AttnArgs& a, __amdgpu_buffer_rsrc_t mem, int w0, int skip, int parts,
                                          Kv8TileRows t, float2* lds) {
  constexpr int kItems = TR * D / 4 / kKv8Threads;  // four-dimension pieces of the tile per thread
  constexpr int kPart = TR * (D + 4), kBatch = 16 / kItems;
  constexpr int kStats = (kBatch * TR + kKv8Threads - 1) / kKv8Threads;
  const int tid = threadIdx.x;
  const auto part_of = [&](int k) { return (2 * w0 + (k == 0 ? skip : 2 * k)) * kPart * 4; };
  float mm[kItems], ll[kItems];
  f32x4 acc[kItems];
  int piece[kItems], row[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    piece[i] = min(tid + i * kKv8Threads, t.rows * (D / 4) - 1);
    row[i] = piece[i] / (D / 4);
    mm[i] = -INFINITY;
    ll[i] = 0.0f;
    acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int k0 = 0; k0 < parts; k0 += kBatch) {
    f32x4 st[kStats], x[kBatch][kItems];
#pragma unroll
    for (int j = 0; j < kStats; ++j) {  // past the last part its own again, not counted
      const int e = tid + j * kKv8Threads;
      st[j] = kv8_get(mem, part_of(min(k0 + e / TR, parts - 1)) + (TR * D + 4 * (e % TR)) * 4);
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
#pragma unroll
      for (int i = 0; i < kItems; ++i) x[k][i] = kv8_get(mem, part_of(min(k0 + k, parts - 1)) + 16 * piece[i]);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kStats; ++j) {
      const int e = tid + j * kKv8Threads;
      if (e < kBatch * TR) lds[e] = k0 + e / TR < parts ? make_float2(st[j][0], st[j][1]) : make_float2(-INFINITY, 0.0f);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      float mx = mm[i];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) mx = fmaxf(mx, lds[k * TR + row[i]].x);
      const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mm[i] - mx);
      acc[i] *= f;
      ll[i] *= f;
      mm[i] = mx;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float2 s = lds[k * TR + row[i]];
        const float w = k0 + k >= parts ? 0.0f : mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s.x - mx);
        ll[i] += s.y * w;
        acc[i] += x[k][i] * w;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    if (tid + i * kKv8Threads < t.rows * (D / 4)) kv8_write<D>(a, t, row[i], 4 * (piece[i] % (D / 4)), acc[i], mm[i], ll[i]);
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
template <int D, int FMT, int RT>
__global__ __launch_bounds__(kKv8Threads, 2) void kv8_rows_kernel(Kv8AttnArgs a) {
  constexpr int TR = 16 * RT, KI = D / 64, KS = D / 32, DT = D / 16;
  constexpr int kWaves = kKv8Threads / kWave, kRow = D + 4, kPart = TR * (D + 4);
  constexpr int PG = RT == 1 ? 4 : 2;  // page blocks of a wavefront's step, and MFMAs of its q.k^T
  constexpr int NT = 4 * PG;           // a lane's tokens of them
  __shared__ __align__(16) float lds_o[kWaves][TR][kRow];
  __shared__ float lds_m[kWaves][TR], lds_l[kWaves][TR];
  __shared__ __align__(16) uint16_t lds_q[RT == 1 ? 8 : TR * D];
  __shared__ Kv8PlanLds<kKv8Threads> lds_plan;
  static_assert(sizeof(lds_o) + sizeof(lds_m) + sizeof(lds_l) + sizeof(lds_q) + sizeof(lds_plan) <= 80 * 1024, "two workgroups per CU");

  Kv8Place<TR, kKv8Threads> at;
  if (!at.begin(a, lds_plan, (int)blockIdx.x, (int)gridDim.x)) return;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int n = lane & 15, g = lane >> 4;
  const int64_t page_bytes = (int64_t)kBlock * D;
  // the lane's place in a step: block and token of the key row that it loads, of the tokens that it holds
  const int kblk = PG == 4 ? n >> 2 : n >> 3, vblk = PG == 4 ? g : g >> 1;
  const int kpart = PG == 4 ? 0 : 2 * (n >> 2 & 1), vtok = PG == 4 ? 0 : 8 * (g & 1);
  bool first_part = true;

  for (;;) {
    const Kv8Seq seq = at.seq;
    const int b = at.b, kvh = at.kvh;
    const uint32_t last_unit = min(at.units_of, at.end - at.tile0);
    int s0, s1, steps;
    if (!at.part(a, s0, s1, steps)) break;  // the range ends within the tile's start
    const int row0 = at.i * TR, rows = min(seq.n * a.G - row0, TR);

    const int32_t* table = a.r.table + (int64_t)b * a.r.max_blocks;
    // block id of this lane's K and V block in a step; -1: none
    const auto block_id = [&](int step, int k) {
      const int j = step * PG + k;
      const int id = table[min(j, a.r.max_blocks - 1)];
      return j < a.r.max_blocks && id >= 0 && id < a.r.num_blocks ? id : -1;
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
          *reinterpret_cast<uint4*>(&lds_q[(rt * KS + kk) * 512 + lane * 8]) =
              *reinterpret_cast<const uint4*>(src + (4 * (kk >> 1) + g) * 16 + 8 * (kk & 1));
      }
      lim[rt] = seq.tree ? seq.ctx - 1 : seq.ctx + (live ? tok : 0);
      bits[rt] = seq.tree && live ? a.tree[seq.first + tok] : 0;
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

    uint4 kw[PG][KI];
    uint32_t vw[DT][PG];
    float4 sk, sv, sk_next, sv_next;
    const auto load_k = [&](int id) {
      const uint8_t* src = a.k_pages + ((int64_t)max(id, 0) * a.kv_heads + kvh) * page_bytes + kpart * (4 * D) + g * 64 + (n & 3) * 16;
#pragma unroll
      for (int p = 0; p < PG; ++p)
#pragma unroll
        for (int i = 0; i < KI; ++i) kw[p][i] = load_stream16(src + p * (4 * D) + i * 256);
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
          const uint4 w = load_stream16(src + dt * (16 * kBlock));
          vw[dt][0] = w.x;
          vw[dt][1] = w.y;
          vw[dt][2] = w.z;
          vw[dt][3] = w.w;
        } else {
          const uint64_t w = __builtin_nontemporal_load(reinterpret_cast<const uint64_t*>(src + dt * (16 * kBlock)));
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
    if constexpr (RT > 1) __syncthreads();  // lds_q
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
            qop[rt] = *reinterpret_cast<const bf16x8*>(&lds_q[(rt * KS + kk) * 512 + lane * 8]);
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
        lds_m[wave][16 * rt + n] = m[rt] + raise;
        lds_l[wave][16 * rt + n] = pr.x + pr.y;
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(&lds_o[wave][16 * rt + n][16 * dt + 4 * g]) = o[rt][dt];
    }
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = 2 * at.w + (first_part ? 0 : 1);
    const __amdgpu_buffer_rsrc_t parts_mem = kv8_parts(a.part, 2 * at.ranges * kPart * 4);
    const int part = slot * kPart * 4;  // byte offsets: at most 1024 parts of 32 rows
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
      if (__builtin_expect(mm == -INFINITY, 0)) mm = kv8_lowest(a, b, seq, (row0 + r) / a.G, s0 * kKv8Step, s1 * kKv8Step);
      if (whole) {
        kv8_write<D>(a, {row0, rows, seq.first, kvh}, r, d, acc, mm, ll);
      } else {
        kv8_put(parts_mem, part + (r * D + d) * 4, acc);
        if (d == 0) kv8_put(parts_mem, part + (TR * D + 4 * r) * 4, f32x4{mm, ll, 0.0f, 0.0f});
      }
    }
    if (!whole) {
      const int w0 = at.first_range(a), parts = at.parts(a);
      uint32_t* done = a.done ? a.done : kv8_counts[a.slot];
      if (kv8_last(done + w0, parts, lds_plan.T)) {
        kv8_merge<D, TR>(a, parts_mem, w0, at.second_part(a), parts, {row0, rows, seq.first, kvh},
                         reinterpret_cast<float2*>(&lds_o[0][0][0]));
      }
    }
    first_part = false;
    at.u = at.tile0 + last_unit;
    if (at.u >= at.end || !at.next(a)) break;
    __syncthreads();
  }
}

}  // namespace sdv

#include "sdv_kv8_chunk.h"

using namespace sdv;

constexpr int kKv8Start = 5;  // steps that starting a tile costs, about

// Most tiles of one KV head, and most units of a call, or -1 where they or the row and key counts pass
// what the plan's 32-bit sums hold.
static int64_t kv8_tiles(int32_t batch, int32_t total, int32_t G, int tile) {
  const int64_t cut = (int64_t)total * G / tile + batch;
  return cut < (int64_t)total * G ? cut : (int64_t)total * G;
}
static int64_t kv8_units(int32_t batch, int32_t total, int32_t G, int32_t kv_heads, int32_t max_len, int tile, int unit, int start) {
  if (((int64_t)max_len + total) * G > (1 << 30)) return -1;
  const int64_t units = kv8_tiles(batch, total, G, tile) * (((int64_t)max_len + total) / (kKv8Step << unit) + 1 + start) * kv_heads;
  return units > INT32_MAX ? -1 : units;
}

// Rows per tile: 16 or 32 where a sequence's rows fit that.  With more rows 256, whose stages serve more of
// them (1800 over 32768 keys 82 us, in tiles of 32 195), or 32 where all tiles of those together have at
// most eight steps for each workgroup of the device: the many small ones start sooner and their parts need
// no second launch.  2 KV heads of 128, tiles of 32 and of 256, in us (with a fill of 1.8): 300 tokens' 1800
// rows 12 and 25, 288 rows over 2048 keys 14 and 23, 144 over 8192 (1280 steps) 20 and 25, 1200 over 2048
// (2432) 21 and 28; of four sequences of 8192 48 rows each (2560) 24 and 24, 144 each (5632) 33 and 32, 288
// each (10240) 42 and 37; 1200 over 8192 (9728) 44 and 36.  With other heads the two are even at 6400 steps
// (14/2/64, 26 and 27), 8192 (20/1/64, 30 and 30) and 4096 to 8192 (32/8/128, 27 and 25, 31 and 31); at less than
// 3000 tiles of 32 take 0.5 to 0.8 of the time, past 10000 1.2 to 1.8.
static int kv8_tile_rows(int32_t batch, int32_t total, int32_t G, int32_t kv_heads, int32_t max_q_len, int32_t max_len) {
  const int64_t rows = (int64_t)G * max_q_len, steps = ((int64_t)max_len + kKv8Step - 1) / kKv8Step;
  if (rows <= 32) return rows <= 16 ? 16 : 32;
  return kv8_tiles(batch, total, G, 32) * kv_heads <= 8 * kKv8Grid / steps ? 32 : kChunkRows;
}

static size_t kv8_workspace(int tile, int32_t head_dim) {
  if (tile == kChunkRows)
    return SDV_KV8_SYNC_BYTES + kChunkGrid * (sizeof(Kv8Cut) + 2 * sizeof(float) * (head_dim == 128 ? chunk_part<128>() : chunk_part<64>()));
  return SDV_KV8_SYNC_BYTES + (size_t)kKv8Grid * 2 * tile * (head_dim + 4) * sizeof(float);
}
static_assert(kKv8Grid * sizeof(uint32_t) == SDV_KV8_SYNC_BYTES / 2, "a count per range");

static int kv8_attn_sizes(int32_t batch, int32_t total, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                          int32_t max_len) {
  if (batch <= 0 || total < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || max_q_len <= 0 || max_len <= 0)
    return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  if (batch > INT32_MAX / 4 || total > INT32_MAX / 2) return SDV_ERR_SHAPE;
  const int32_t G = q_heads / kv_heads;
  return kv8_units(batch, total, G, kv_heads, max_len, kv8_tile_rows(batch, total, G, kv_heads, max_q_len, max_len), 0, kKv8Start) < 0 ? SDV_ERR_SHAPE : SDV_OK;
}

extern "C" size_t sdv_kv8_attention_workspace_size(int32_t batch, int32_t total_rows, int32_t q_heads, int32_t kv_heads,
                                                   int32_t head_dim, int32_t max_q_len, int32_t max_seq_len) {
  if (kv8_attn_sizes(batch, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len) != SDV_OK) return 0;
  return kv8_workspace(kv8_tile_rows(batch, total_rows, q_heads / kv_heads, kv_heads, max_q_len, max_seq_len), head_dim);
}

template <int D, int FMT, int RT>
static void kv8_launch(const Kv8AttnArgs& a, int grid, hipStream_t st) {
  hipLaunchKernelGGL((kv8_rows_kernel<D, FMT, RT>), dim3((unsigned)grid), dim3(kKv8Threads), 0, st, a);
}

template <int D, int FMT>
static void kv8_launch_chunk(Kv8AttnArgs a, int grid, int64_t tiles, hipStream_t st) {
  a.cuts = reinterpret_cast<Kv8Cut*>(a.part);
  a.part += kChunkGrid * sizeof(Kv8Cut) / sizeof(float);
  hipLaunchKernelGGL((kv8_chunk_kernel<D, FMT>), dim3((unsigned)grid), dim3(kChunkThreads), 0, st, a);
  const unsigned cuts = (unsigned)(tiles < grid ? tiles : grid);  // at most
  hipLaunchKernelGGL((kv8_chunk_merge_kernel<D>), dim3(cuts, kChunkWaves * D / 32), dim3(256), 0, st, a, grid);
}

extern "C" int sdv_kv8_attention_slot(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, const float* scales,
                                      int32_t num_blocks, int32_t format, const int32_t* block_table, int32_t max_blocks_per_seq,
                                      const int32_t* cu_rows, const int32_t* seq_lens, const uint64_t* tree_mask, int32_t batch,
                                      int32_t total_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                                      int32_t max_seq_len, float scale, void* workspace, size_t workspace_bytes, int32_t slot,
                                      void* out, int64_t out_stride, void* stream) {
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
  const int G = q_heads / kv_heads, tile = kv8_tile_rows(batch, total_rows, G, kv_heads, max_q_len, max_seq_len);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < kv8_workspace(tile, head_dim)) return SDV_ERR_WORKSPACE;
  if (slot < -1 || slot >= SDV_KV8_SLOTS) return SDV_ERR_WORKSPACE;
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
  a.done = slot < 0 ? static_cast<uint32_t*>(workspace) : nullptr;
  a.slot = slot;
  a.cuts = nullptr;
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + SDV_KV8_SYNC_BYTES);
  // Units.  Where the device holds a workgroup for every unit of every tile, each takes one: the call is
  // as long as its latencies, and a second tile would double them (GPU time, 2 KV heads, with a fill of
  // 1.8 us before each call: eight sequences
  // of 1000 to 4096 keys, five rows each, 31 us in equal ranges of single steps and 19 so; one of 2048
  // keys 12 and 9).  A unit is four steps, one per wavefront; of a tile's S steps longer ones make less
  // to add up, and the shortest calls have units of about the root of S / 8 of them (16 rows; 2S / 8, 32:
  // their parts are larger).  One row in us, at 4, 8 and 16 steps: 8192 keys 12.3 11.8 16.3, 32768 keys
  // 26 20 20, 131072 keys 51 52 35; five rows: 8192 keys 21 19 26, 32768 keys 50 35 34.  Units of eight
  // also where ones of four would not fit (eight sequences of 8192 keys, one row each, 14 us, in ranges
  // 19) and where a sequence's several tiles would then stand two a CU (576 rows over 2048 keys 16 us, with
  // four 19).  At 16 steps units and ranges are even (sixteen sequences 19.9 and 21.8, of mixed lengths 18.4
  // and 18.1).  With other heads (14/2/64, 20/1/64, 32/8/128; 27 sizes of 1 to 16 sequences, 2048 to 131072 keys) the
  // unit is the best or within 11% of it but for the longest contexts of one sequence, where a longer one would
  // take up to a fifth off (20/1/64, one row over 32768 keys 23 and 19; 32/8/128, four rows 28 and 22).
  const int64_t tiles = kv8_tiles(batch, total_rows, G, tile) * kv_heads;
  const int64_t steps = ((int64_t)max_seq_len + kKv8Step - 1) / kKv8Step;
  const int most_grid = tile == kChunkRows ? kChunkGrid : kKv8Grid;
  const auto fits = [&](int unit, int grid) { return tiles * (((steps - 1) >> unit) + 1) <= grid; };
  int unit = 2;
  if (tile != kChunkRows) {
    while ((int64_t)128 << (2 * unit) < steps * tile) ++unit;
    if (unit == 2 && !fits(2, (int64_t)G * max_q_len > 32 ? kKv8Grid / 2 : kKv8Grid)) unit = 3;
  }
  a.unit = fits(unit, most_grid) ? unit : 0;
  a.start = a.unit == 0 ? kKv8Start : 0;
  const int64_t most = kv8_units(batch, total_rows, G, kv_heads, max_seq_len, tile, a.unit, a.start);
  const int grid = (int)(most < most_grid ? most : most_grid);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool fp8 = format == SDV_KV8_FP8;
  if (tile == kChunkRows && head_dim == 128)
    fp8 ? kv8_launch_chunk<128, kFp8>(a, grid, tiles, st) : kv8_launch_chunk<128, kInt8>(a, grid, tiles, st);
  else if (tile == kChunkRows)
    fp8 ? kv8_launch_chunk<64, kFp8>(a, grid, tiles, st) : kv8_launch_chunk<64, kInt8>(a, grid, tiles, st);
  else if (head_dim == 128 && tile == 16)
    fp8 ? kv8_launch<128, kFp8, 1>(a, grid, st) : kv8_launch<128, kInt8, 1>(a, grid, st);
  else if (head_dim == 128)
    fp8 ? kv8_launch<128, kFp8, 2>(a, grid, st) : kv8_launch<128, kInt8, 2>(a, grid, st);
  else if (tile == 16)
    fp8 ? kv8_launch<64, kFp8, 1>(a, grid, st) : kv8_launch<64, kInt8, 1>(a, grid, st);
  else
    fp8 ? kv8_launch<64, kFp8, 2>(a, grid, st) : kv8_launch<64, kInt8, 2>(a, grid, st);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}

extern "C" int sdv_kv8_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, const float* scales,
                                 int32_t num_blocks, int32_t format, const int32_t* block_table, int32_t max_blocks_per_seq,
                                 const int32_t* cu_rows, const int32_t* seq_lens, const uint64_t* tree_mask, int32_t batch,
                                 int32_t total_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                                 int32_t max_seq_len, float scale, void* workspace, size_t workspace_bytes, void* out,
                                 int64_t out_stride, void* stream) {
  return sdv_kv8_attention_slot(q, q_stride, k_pages, v_pages, scales, num_blocks, format, block_table, max_blocks_per_seq, cu_rows,
                                seq_lens, tree_mask, batch, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len, scale,
                                workspace, workspace_bytes, -1, out, out_stride, stream);
}
