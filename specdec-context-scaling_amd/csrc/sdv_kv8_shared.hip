// Attention over the 8-bit KV cache of sequences that begin with the same pages (definition: sdv_kv8_attn.hip).
//
// A group is consecutive sequences whose first P tokens (whole blocks) are the same pages.  Its rows lie together in the
// packed tensors, so a group's prefix is one more sequence: all of its rows, each of which sees all P keys.  A sequence's
// own part is the sequence it was with its first P keys left out.  Every tile of either leaves its sums with their
// maximum and their sum of exponentials; a second launch adds those up for each row:
//
//   M = max_k m_k,   out = sum_k e^(m_k - M) acc_k / sum_k e^(m_k - M) l_k
//
// Tiles of 32 rows of a prefix, and of 16 or 32 of a sequence, are cut into ranges as in kv8_rows_kernel, and computed
// by its code; a prefix's pages are read once per 32 rows of the group, from memory once.
#include "sdv_kv8_rows.h"

namespace sdv {

// What one launch leaves for the next, of a prefix or a sequence: units of its tiles, and which parts are theirs.
struct Kv8SharedTiles {
  uint32_t unit0;  // units before it, of one KV head
  uint32_t tile0;  // tiles before it, likewise
  uint32_t units;  // of each of its tiles, those of its start among them; 0: no tiles
  int first, n;    // its packed rows
  int pad[3];
};
struct Kv8SharedPlan {
  uint32_t per_head, tiles;  // units and tiles of a KV head
  uint32_t share, rest;      // every range has `share` units, the first `rest` one more
  int start;
  int pad[3];
};

struct Kv8SharedArgs {
  Kv8AttnArgs a;
  const int32_t* cu_groups;
  const int32_t* prefix;
  int groups, max_prefix;
  uint32_t parts;  // that the workspace holds: more than tables whose entries do not decrease ever need
  Kv8SharedPlan* plan;
  Kv8SharedTiles* of;  // per prefix, then per sequence
};

constexpr int kSharedModes = 4;   // units of 4, 8, 16 and 32 steps, one a workgroup where there is one for each
constexpr int kSharedStart = 5;   // else single steps, and so many that stand for a tile's start

// Prefix v, or sequence v - groups: its rows, keys and blocks.
struct Kv8SharedSeq {
  Kv8Seq seq;
  int skip;   // blocks of the table in front of its first key
  int table;  // whose table
  int steps;  // of 64 keys, of each tile
};

template <int TP, int TS>
__device__ __forceinline__ Kv8SharedSeq kv8_shared_seq(const Kv8SharedArgs& s, int v) {
  const Kv8AttnArgs& a = s.a;
  Kv8SharedSeq x;
  x.skip = 0;
  if (v < s.groups) {
    const int b0 = min(max(s.cu_groups[v], 0), a.r.batch), b1 = min(max(s.cu_groups[v + 1], b0), a.r.batch);
    x.table = min(b0, a.r.batch - 1);
    const int first = min(max(a.r.cu[b0], 0), a.r.total), end = min(max(a.r.cu[b1], 0), a.r.total);
    const int P = b0 < b1 ? min(max(s.prefix[x.table], 0), s.max_prefix) & ~(kBlock - 1) : 0;
    x.seq.first = first;
    x.seq.n = P > 0 ? max(end - first, 0) : 0;
    x.seq.T = x.seq.ctx = P;
    x.seq.tiles = (x.seq.n * a.G + TP - 1) / TP;
    x.seq.tree = true;  // of no visible new tokens
  } else {
    const int b = v - s.groups;
    int first, n;
    kv8_rows(a.r, b, first, n);
    const int P = min(max(s.prefix[b], 0), s.max_prefix) & ~(kBlock - 1);
    const int T = (a.lens ? min(max(a.lens[b], 0), a.max_len) : a.max_len) - P;
    x.table = b;
    x.skip = P / kBlock;
    x.seq = kv8_seq_of<TS>(a, first, T > 0 ? n : 0, T);
    x.seq.ctx = T - n;
  }
  x.steps = (max(x.seq.T, 0) + kKv8Step - 1) >> kKv8StepBits;
  return x;
}

__device__ __forceinline__ uint32_t kv8_shared_units(const Kv8SharedSeq& x, int unit) {
  return (uint32_t)(x.steps + (1 << unit) - 1) >> unit;
}

struct Kv8SharedLds {
  uint4 run[kKv8Threads];  // units and tiles of the wavefront's runs up to and with this one, units and tiles of this one
  uint32_t total[kKv8Threads / kWave][kSharedModes + 2];
};

// A workgroup's place among the units: as Kv8Place, over prefixes and sequences.
template <int TP, int TS>
struct Kv8SharedPlace {
  uint32_t per_head, tiles, share, rest;
  int unit, start;
  int ranges;
  uint32_t u, end;
  int kvh, v, i;
  Kv8SharedSeq x;
  uint32_t tile0, units_of;  // the tile's first unit and its units
  uint32_t ordinal;          // tiles before it, of all KV heads

  __device__ __forceinline__ bool begin(const Kv8SharedArgs& s, Kv8SharedLds& lds, int w, int grid) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int count = s.groups + s.a.r.batch, per_run = (count + kKv8Threads - 1) / kKv8Threads;
    uint32_t mine[kSharedModes + 2] = {};  // units at each size, at single steps, tiles
    for (int k = 0; k < per_run; ++k) {
      const int y = tid * per_run + k;
      if (y >= count) break;
      const Kv8SharedSeq q = kv8_shared_seq<TP, TS>(s, y);
#pragma unroll
      for (int m = 0; m < kSharedModes; ++m) mine[m] += (uint32_t)q.seq.tiles * kv8_shared_units(q, m + 2);
      mine[kSharedModes] += (uint32_t)q.seq.tiles * (uint32_t)(q.steps + kSharedStart);
      mine[kSharedModes + 1] += (uint32_t)q.seq.tiles;
    }
    uint32_t scan[kSharedModes + 2];
#pragma unroll
    for (int m = 0; m < kSharedModes + 2; ++m) {
      scan[m] = kv8_lane_scan(mine[m]);
      if (lane == kWave - 1) lds.total[wave][m] = scan[m];
    }
    __syncthreads();
    uint32_t total[kSharedModes + 2];
#pragma unroll
    for (int m = 0; m < kSharedModes + 2; ++m) {
      total[m] = 0;
#pragma unroll
      for (int k = 0; k < kKv8Threads / kWave; ++k) total[m] += lds.total[k][m];
      total[m] = __builtin_amdgcn_readfirstlane(total[m]);
    }
    tiles = total[kSharedModes + 1];
    int mode = kSharedModes;
#pragma unroll
    for (int m = kSharedModes - 1; m >= 0; --m)
      if (total[m] * (uint32_t)s.a.kv_heads <= (uint32_t)grid) mode = m;
    unit = mode == kSharedModes ? 0 : mode + 2;
    start = mode == kSharedModes ? kSharedStart : 0;
    uint32_t upto = scan[kSharedModes], of_run = mine[kSharedModes];
    per_head = total[kSharedModes];
#pragma unroll
    for (int m = 0; m < kSharedModes; ++m)
      if (m == mode) {
        upto = scan[m];
        of_run = mine[m];
        per_head = total[m];
      }
    lds.run[tid] = make_uint4(upto, scan[kSharedModes + 1], of_run, mine[kSharedModes + 1]);
    const uint32_t units = per_head * (uint32_t)s.a.kv_heads;
    ranges = (int)min((uint32_t)grid, units);
    share = ranges > 0 ? units / (uint32_t)ranges : 0;
    rest = units - share * (uint32_t)ranges;
    __syncthreads();
    if (w == 0) {  // what the second launch needs
      uint32_t u0 = 0, t0 = 0;
      for (int k = 0; k < wave; ++k) {
        u0 += lds.run[k * kWave + kWave - 1].x;
        t0 += lds.run[k * kWave + kWave - 1].y;
      }
      u0 += upto - of_run;
      t0 += scan[kSharedModes + 1] - mine[kSharedModes + 1];
      for (int k = 0; k < per_run; ++k) {
        const int y = tid * per_run + k;
        if (y >= count) break;
        const Kv8SharedSeq q = kv8_shared_seq<TP, TS>(s, y);
        const uint32_t each = q.seq.tiles > 0 ? kv8_shared_units(q, unit) + (uint32_t)start : 0;
        s.of[y] = {u0, t0, each, q.seq.first, q.seq.n, {0, 0, 0}};
        u0 += (uint32_t)q.seq.tiles * each;
        t0 += (uint32_t)q.seq.tiles;
      }
      if (tid == 0) *s.plan = {per_head, tiles, share, rest, start, {0, 0, 0}};
    }
    if (w >= ranges) return false;
    u = (uint32_t)w * share + min((uint32_t)w, rest);
    end = u + share + ((uint32_t)w < rest ? 1 : 0);
    kvh = (int)(u / per_head);
    uint32_t rem = u - (uint32_t)kvh * per_head;
    tile0 = (uint32_t)kvh * per_head;
    ordinal = (uint32_t)kvh * tiles;
    // the wavefront whose runs hold the unit, then the run: the first that ends behind it
    int wv = 0;
#pragma unroll
    for (int k = 0; k < kKv8Threads / kWave - 1; ++k) {
      const uint4 r = lds.run[k * kWave + kWave - 1];
      if (wv == k && rem >= r.x) {
        rem -= r.x;
        tile0 += r.x;
        ordinal += r.y;
        wv = k + 1;
      }
    }
    wv = __builtin_amdgcn_readfirstlane(wv);
    rem = __builtin_amdgcn_readfirstlane(rem);
    const uint4 run = lds.run[wv * kWave + lane];
    const int at = min(__popcll(__ballot(run.x <= rem)), kWave - 1);
    const uint32_t before = __builtin_amdgcn_readlane(run.x, at) - __builtin_amdgcn_readlane(run.z, at);
    rem -= before;
    tile0 += before;
    ordinal += __builtin_amdgcn_readlane(run.y, at) - __builtin_amdgcn_readlane(run.w, at);
    for (v = (wv * kWave + at) * per_run;; ++v) {
      if (v >= count) return false;  // not reached: the runs hold the unit
      x = kv8_shared_seq<TP, TS>(s, v);
      units_of = kv8_shared_units(x, unit) + (uint32_t)start;
      const uint32_t all = (uint32_t)x.seq.tiles * units_of;
      if (rem < all) break;
      rem -= all;
      tile0 += all;
      ordinal += (uint32_t)x.seq.tiles;
    }
    i = (int)(rem / units_of);
    tile0 += (uint32_t)i * units_of;
    ordinal += (uint32_t)i;
    return true;
  }

  // The tile after this one; false past the last (not reached while u < end).
  __device__ __forceinline__ bool next(const Kv8SharedArgs& s) {
    tile0 += units_of;
    ++ordinal;
    if (++i < x.seq.tiles) return true;
    i = 0;
    do {
      if (++v >= s.groups + s.a.r.batch) {
        v = 0;
        if (++kvh >= s.a.kv_heads) return false;
      }
      x = kv8_shared_seq<TP, TS>(s, v);
    } while (x.seq.tiles == 0);
    units_of = kv8_shared_units(x, unit) + (uint32_t)start;
    return true;
  }
};

// A part: [32][D] sums, then [32] (maximum, sum of exponentials).
template <int D>
constexpr int shared_part() {
  return 32 * (D + 2);
}

// RS: row tiles of 16 of a sequence's tile.
template <int D, int FMT, int RS>
__global__ __launch_bounds__(kKv8Threads, 2) void kv8_shared_kernel(Kv8SharedArgs s) {
  constexpr int RP = 2;
  __shared__ Kv8RowsLds<D, RP> lds;
  __shared__ Kv8SharedLds lds_plan;
  static_assert(sizeof(Kv8RowsLds<D, RS>) <= sizeof(lds), "a sequence's tile uses the same memory");
  const Kv8AttnArgs& a = s.a;
  Kv8SharedPlace<16 * RP, 16 * RS> at;
  const int w = (int)blockIdx.x;
  if (!at.begin(s, lds_plan, w, (int)gridDim.x)) return;
  for (;;) {
    const uint32_t last_unit = min(at.units_of, at.end - at.tile0);
    const int lo = max((int)(at.u - at.tile0) - at.start, 0), hi = (int)last_unit - at.start;
    if (lo >= hi) break;  // the range ends within the tile's start
    const bool prefix = at.v < s.groups;
    const int TR = prefix ? 16 * RP : 16 * RS;
    const Kv8Seq seq = at.x.seq;
    const int row0 = at.i * TR, rows = min(seq.n * a.G - row0, TR);
    // a tile of early rows sees fewer keys than its sequence's last
    int steps = at.x.steps;
    if (!seq.tree) steps = min(steps, max(seq.ctx + (row0 + rows - 1) / a.G + kKv8Step, 0) >> kKv8StepBits);
    const int s0 = min(lo << at.unit, steps), s1 = min(hi << at.unit, steps);
    const Kv8View view = {a.r.table + (int64_t)at.x.table * a.r.max_blocks + at.x.skip, a.r.max_blocks - at.x.skip, a.r.num_blocks,
                          prefix ? nullptr : a.tree};
    const uint32_t slot = at.ordinal + (uint32_t)w;  // each part's own: from one to the next the tile or the range is another
    if (slot >= s.parts) break;
    float* part = a.part + (int64_t)slot * shared_part<D>();
    const auto leave = [&](const auto& sums) {
      __syncthreads();
      for (int e = threadIdx.x; e < rows * (D / 4); e += kKv8Threads) {
        const int r = e / (D / 4), d = 4 * (e % (D / 4));
        float mm, ll;
        const f32x4 acc = kv8_rows_sum(sums, r, d, mm, ll);
        if (__builtin_expect(mm == -INFINITY, 0)) {
          Kv8Seq c = seq;
          c.tree = !prefix && seq.tree;
          const int until = prefix ? min(s1 * kKv8Step, seq.T) : s1 * kKv8Step;
          mm = kv8_lowest(a.tree, view.max_blocks, c, (row0 + r) / a.G, s0 * kKv8Step, until, [&](int j) { return view.named(j); });
        }
        *reinterpret_cast<f32x4*>(part + r * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(part + 32 * D + 2 * r) = make_float2(mm, ll);
      }
    };
    if (RS == RP || prefix) {
      kv8_rows_tile<D, FMT, RP>(a, view, seq, at.kvh, row0, rows, s0, s1, lds);
      leave(lds);
    } else {
      auto& few = reinterpret_cast<Kv8RowsLds<D, RS>&>(lds);
      kv8_rows_tile<D, FMT, RS>(a, view, seq, at.kvh, row0, rows, s0, s1, few);
      leave(few);
    }
    at.u = at.tile0 + last_unit;
    if (at.u >= at.end || !at.next(s)) break;
    __syncthreads();
  }
}

// The rows of a packed token and KV head: the parts of the prefix's tile and of the sequence's that hold them, added up.
constexpr int kSharedMergeThreads = 256;

template <int D, int TS>
__global__ __launch_bounds__(kSharedMergeThreads) void kv8_shared_merge_kernel(Kv8SharedArgs s) {
  const Kv8AttnArgs& a = s.a;
  __shared__ int found[2];
  const int tid = threadIdx.x, token = blockIdx.x, kvh = blockIdx.y;
  if (tid < 2) found[tid] = 0;
  __syncthreads();
  // the sequence: as many end at or before the token; the group: as many end at or before the sequence
  for (int x = tid; x < a.r.batch; x += kSharedMergeThreads) {
    const uint64_t before = __ballot(min(max(a.r.cu[x + 1], 0), a.r.total) <= token);
    if ((tid & (kWave - 1)) == 0) atomicAdd(&found[0], __popcll(before));
  }
  __syncthreads();
  const int b = found[0];
  if (b >= a.r.batch || token < min(max(a.r.cu[b], 0), a.r.total)) return;  // behind the last sequence
  for (int x = tid; x < s.groups; x += kSharedMergeThreads) {
    const uint64_t before = __ballot(s.cu_groups[x + 1] <= b);
    if ((tid & (kWave - 1)) == 0) atomicAdd(&found[1], __popcll(before));
  }
  __syncthreads();
  const int g = found[1];
  const Kv8SharedPlan plan = *s.plan;
  const bool grouped = g < s.groups && s.cu_groups[g] <= b;
  Kv8SharedTiles of[2] = {s.of[grouped ? g : 0], s.of[s.groups + b]};
  if (!grouped) of[0].units = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (token < of[k].first || token - of[k].first >= of[k].n) of[k].units = 0;
  const auto owner = [&](uint32_t x) {
    const uint32_t split = plan.rest * (plan.share + 1);
    return x < split ? x / (plan.share + 1) : plan.rest + (x - split) / plan.share;
  };
  for (int e = tid; e < a.G * (D / 4); e += kSharedMergeThreads) {
    const int head = e / (D / 4), d = 4 * (e % (D / 4));
    float m = -INFINITY, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (of[k].units == 0) continue;
      const int TR = k == 0 ? 32 : TS;
      const int row = (token - of[k].first) * a.G + head, i = row / TR, r = row - i * TR;
      const uint32_t t0 = (uint32_t)kvh * plan.per_head + of[k].unit0 + (uint32_t)i * of[k].units;
      const uint32_t first = owner(t0 + (uint32_t)plan.start), last = owner(t0 + of[k].units - 1);
      const uint32_t slot = (uint32_t)kvh * plan.tiles + of[k].tile0 + (uint32_t)i + first;
      const float* part = a.part + (int64_t)slot * shared_part<D>();
      for (uint32_t j = 0; j <= last - first && slot + j < s.parts; ++j, part += shared_part<D>()) {
        const float2 st = *reinterpret_cast<const float2*>(part + 32 * D + 2 * r);
        const f32x4 y = *reinterpret_cast<const f32x4*>(part + r * D + d);
        const float mx = fmaxf(m, st.x);
        const float f0 = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx), f1 = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.x - mx);
        l = l * f0 + st.y * f1;
        acc = acc * f0 + y * f1;
        m = mx;
      }
    }
    const float inv = m == -INFINITY ? 0.0f : 1.0f / l;  // a row that sees nothing: 0
    *reinterpret_cast<uint2*>(a.out + (int64_t)token * a.out_stride + (int64_t)(kvh * a.G + head) * D + d) =
        make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  }
}

}  // namespace sdv

using namespace sdv;

// Most tiles of one KV head.
static int64_t shared_tiles(int32_t batch, int32_t groups, int32_t total, int32_t G, int tile) {
  const int64_t rows = (int64_t)total * G, own = rows / tile + batch, prefix = rows / 32 + groups;
  return (own < rows ? own : rows) + (prefix < rows ? prefix : rows);
}

static int shared_tile(int32_t G, int32_t max_q_len) { return (int64_t)G * max_q_len <= 16 ? 16 : 32; }

// The plan's sums are 32 bits wide, and a part's number a 31-bit one.
static int shared_sizes(int32_t batch, int32_t groups, int32_t total, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                        int32_t max_len, int32_t max_prefix) {
  if (batch <= 0 || groups < 0 || groups > batch || total < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || kv_heads > 65535 ||
      max_q_len <= 0 || max_len <= 0 || max_prefix < 0)
    return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  if (batch > INT32_MAX / 4 || total > INT32_MAX / 2) return SDV_ERR_SHAPE;
  const int32_t G = q_heads / kv_heads;
  if (((int64_t)max_len + max_prefix + total) * G > (1 << 30)) return SDV_ERR_SHAPE;
  const int64_t tiles = shared_tiles(batch, groups, total, G, shared_tile(G, max_q_len)) * kv_heads;
  const int64_t longest = max_len > max_prefix ? max_len : max_prefix;
  return tiles > INT32_MAX / 8 || tiles * (longest / kKv8Step + 1 + kSharedStart) > INT32_MAX ? SDV_ERR_SHAPE : SDV_OK;
}

static size_t shared_tables(int32_t batch, int32_t groups) {
  return round_up(sizeof(Kv8SharedPlan) + ((size_t)batch + groups) * sizeof(Kv8SharedTiles), 256);
}

static int64_t shared_parts(int32_t batch, int32_t groups, int32_t total, int32_t G, int32_t kv_heads, int32_t max_q_len) {
  return shared_tiles(batch, groups, total, G, shared_tile(G, max_q_len)) * kv_heads + kKv8Grid;
}

static size_t shared_workspace(int32_t batch, int32_t groups, int32_t total, int32_t G, int32_t kv_heads, int32_t head_dim, int32_t max_q_len) {
  return shared_tables(batch, groups) +
         (size_t)shared_parts(batch, groups, total, G, kv_heads, max_q_len) * sizeof(float) * (head_dim == 128 ? shared_part<128>() : shared_part<64>());
}

extern "C" size_t sdv_kv8_shared_attention_workspace_size(int32_t batch, int32_t groups, int32_t total_rows, int32_t q_heads,
                                                          int32_t kv_heads, int32_t head_dim, int32_t max_q_len, int32_t max_seq_len,
                                                          int32_t max_prefix_len) {
  if (shared_sizes(batch, groups, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len, max_prefix_len) != SDV_OK) return 0;
  return shared_workspace(batch, groups, total_rows, q_heads / kv_heads, kv_heads, head_dim, max_q_len);
}

template <int D, int FMT>
static void shared_launch(const Kv8SharedArgs& s, int tile, hipStream_t st) {
  const dim3 grid(kKv8Grid), merge((unsigned)s.a.r.total, (unsigned)s.a.kv_heads);
  if (tile == 16) {
    hipLaunchKernelGGL((kv8_shared_kernel<D, FMT, 1>), grid, dim3(kKv8Threads), 0, st, s);
    hipLaunchKernelGGL((kv8_shared_merge_kernel<D, 16>), merge, dim3(kSharedMergeThreads), 0, st, s);
  } else {
    hipLaunchKernelGGL((kv8_shared_kernel<D, FMT, 2>), grid, dim3(kKv8Threads), 0, st, s);
    hipLaunchKernelGGL((kv8_shared_merge_kernel<D, 32>), merge, dim3(kSharedMergeThreads), 0, st, s);
  }
}

extern "C" int sdv_kv8_shared_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, const float* scales,
                                        int32_t num_blocks, int32_t format, const int32_t* block_table, int32_t max_blocks_per_seq,
                                        const int32_t* cu_rows, const int32_t* seq_lens, const uint64_t* tree_mask,
                                        const int32_t* cu_groups, const int32_t* prefix_lens, int32_t batch, int32_t groups,
                                        int32_t total_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                                        int32_t max_seq_len, int32_t max_prefix_len, float scale, void* workspace,
                                        size_t workspace_bytes, void* out, int64_t out_stride, void* stream) {
  if (!q || !k_pages || !v_pages || !scales || !block_table || !cu_rows || !cu_groups || !prefix_lens || !out) return SDV_ERR_NULL;
  const int sizes = shared_sizes(batch, groups, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len, max_prefix_len);
  if (sizes != SDV_OK) return sizes;
  if (num_blocks <= 0 || max_blocks_per_seq <= 0 || max_blocks_per_seq > INT32_MAX / kBlock) return SDV_ERR_SHAPE;
  if (max_prefix_len > (int64_t)max_blocks_per_seq * kBlock) return SDV_ERR_SHAPE;
  if (format != SDV_KV8_FP8 && format != SDV_KV8_INT8) return SDV_ERR_UNSUPPORTED;
  if (tree_mask && max_q_len > 64) return SDV_ERR_UNSUPPORTED;
  const int64_t row = (int64_t)q_heads * head_dim;
  if (q_stride < row || out_stride < row) return SDV_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride % 8 || out_stride % 8 || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
      !aligned(scales, 16) || !aligned(block_table, 4) || !aligned(cu_rows, 4) || !aligned(seq_lens, 4) || !aligned(tree_mask, 8) ||
      !aligned(cu_groups, 4) || !aligned(prefix_lens, 4))
    return SDV_ERR_ALIGN;
  const int G = q_heads / kv_heads;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < shared_workspace(batch, groups, total_rows, G, kv_heads, head_dim, max_q_len))
    return SDV_ERR_WORKSPACE;
  if (total_rows == 0) return SDV_OK;

  Kv8SharedArgs s;
  Kv8AttnArgs& a = s.a;
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
  a.unit = a.start = 0;
  a.done = nullptr;
  a.slot = -1;
  a.cuts = nullptr;
  s.cu_groups = cu_groups;
  s.prefix = prefix_lens;
  s.groups = groups;
  s.max_prefix = max_prefix_len;
  s.parts = (uint32_t)shared_parts(batch, groups, total_rows, G, kv_heads, max_q_len);
  s.plan = static_cast<Kv8SharedPlan*>(workspace);
  s.of = reinterpret_cast<Kv8SharedTiles*>(s.plan + 1);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + shared_tables(batch, groups));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int tile = shared_tile(G, max_q_len);
  if (head_dim == 128)
    format == SDV_KV8_FP8 ? shared_launch<128, kFp8>(s, tile, st) : shared_launch<128, kInt8>(s, tile, st);
  else
    format == SDV_KV8_FP8 ? shared_launch<64, kFp8>(s, tile, st) : shared_launch<64, kInt8>(s, tile, st);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}
