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
#include "sdv_kv8_rows.h"

namespace sdv {

// Counts of finished parts, per slot and range; every call leaves its slot's zero, as the loader does.
static __device__ uint32_t kv8_counts[SDV_KV8_SLOTS][kKv8Grid];

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

template <int D, int FMT, int RT>
__global__ __launch_bounds__(kKv8Threads, 2) void kv8_rows_kernel(Kv8AttnArgs a) {
  constexpr int TR = 16 * RT, kPart = TR * (D + 4);
  __shared__ Kv8RowsLds<D, RT> lds;
  __shared__ Kv8PlanLds<kKv8Threads> lds_plan;
  static_assert(sizeof(lds) + sizeof(lds_plan) <= 80 * 1024, "two workgroups per CU");

  Kv8Place<TR, kKv8Threads> at;
  if (!at.begin(a, lds_plan, (int)blockIdx.x, (int)gridDim.x)) return;
  const int tid = threadIdx.x;
  bool first_part = true;

  for (;;) {
    const Kv8Seq seq = at.seq;
    const int b = at.b, kvh = at.kvh;
    const uint32_t last_unit = min(at.units_of, at.end - at.tile0);
    int s0, s1, steps;
    if (!at.part(a, s0, s1, steps)) break;  // the range ends within the tile's start
    const int row0 = at.i * TR, rows = min(seq.n * a.G - row0, TR);

    const Kv8View view = {a.r.table + (int64_t)b * a.r.max_blocks, a.r.max_blocks, a.r.num_blocks, a.tree};
    kv8_rows_tile<D, FMT, RT>(a, view, seq, kvh, row0, rows, s0, s1, lds);
    __syncthreads();
    const bool whole = s0 == 0 && s1 == steps;
    const int slot = 2 * at.w + (first_part ? 0 : 1);
    const __amdgpu_buffer_rsrc_t parts_mem = kv8_parts(a.part, 2 * at.ranges * kPart * 4);
    const int part = slot * kPart * 4;  // byte offsets: at most 1024 parts of 32 rows
    for (int e = tid; e < rows * (D / 4); e += kKv8Threads) {
      const int r = e / (D / 4), d = 4 * (e % (D / 4));
      float mm, ll;
      const f32x4 acc = kv8_rows_sum<D, RT>(lds, r, d, mm, ll);
      if (__builtin_expect(mm == -INFINITY, 0)) mm = kv8_lowest(a.tree, view.max_blocks, seq, (row0 + r) / a.G, s0 * kKv8Step, s1 * kKv8Step, [&](int j) { return view.named(j); });
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
                         reinterpret_cast<float2*>(&lds.o[0][0][0]));
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
