// Attention over the 8-bit KV cache of sequences that begin with the same pages (definition: sdv_kv8_attn.hip).
//
// A group is consecutive sequences whose first P tokens (whole blocks) are the same pages.  Its rows lie together in the
// packed tensors, so a group's prefix is one more sequence: all of its rows, each of which sees all P keys.  A sequence's
// own part is the sequence it was with its first P keys left out.  Tiles of 32 or 128 rows of a prefix, and of 16 or 32 of
// a sequence, are cut along their keys into items, one a workgroup where there is one for each, and computed by
// kv8_rows_tile, those of 128 rows by kv8_wide_tile.  Every item leaves its sums with their maximum and their sum of exponentials; a second launch adds
// those up for each row:
//
//   M = max_k m_k,   out = sum_k e^(m_k - M) acc_k / sum_k e^(m_k - M) l_k
//
// The items of one stretch of a prefix's keys, one for each of its tiles, stand one after another and go to the
// workgroups of one XCD, whose L2 then serves all of them but the first.
#include "sdv_kv8_wide.h"

namespace sdv {

struct Kv8SharedArgs {
  Kv8AttnArgs a;
  const int32_t* cu_groups;
  const int32_t* prefix;
  int groups, max_prefix;
  bool wide;          // tiles of a prefix have kWideRows rows, else 32
  uint32_t parts[2];  // that the workspace holds, of prefixes and of sequences: no fewer than tables need whose entries do not decrease
  float* part[2];
  struct Kv8SharedRow* rows;  // per packed token
};

// Where the parts of a packed token's rows lie: of the prefix (k = 0) and of the sequence.  Row r = row0[k] + head of KV
// head h: part base[k] + h * per_head[k] + c * tiles[k] + r / tile for each of the chunks c < chunks[k].
struct Kv8SharedRow {
  uint32_t base[2], per_head[2];
  int tiles[2], chunks[2], row0[2];
  int pad[6];
};

constexpr int kSharedStart = 5;   // steps that starting an item costs, about
constexpr int kSharedWide = 3;    // a step's time with kWideRows rows; with tiles of 16 rows of a sequence it is 1, of 32 2, about
constexpr int kSharedShort = 4;   // steps of those that an item has at least: its part costs as much

// Prefix v, or sequence v - groups: its rows, keys and blocks.
struct Kv8SharedSeq {
  int first, n;  // packed rows
  int T;         // keys; of a sequence those behind the prefix
  int table;     // whose table
  int skip;      // blocks of the table in front of the first key
  int tiles;
  __device__ __forceinline__ uint32_t steps() const { return (uint32_t)(max(T, 0) + kKv8Step - 1) >> kKv8StepBits; }
};

// From the tables' entries: rows first .. end - 1, a prefix of P tokens, and of a sequence its length.
__device__ __forceinline__ Kv8SharedSeq kv8_shared_prefix(const Kv8SharedArgs& s, int b0, int b1, int first, int end, int P) {
  Kv8SharedSeq x;
  x.table = min(b0, s.a.r.batch - 1);
  x.skip = 0;
  x.first = min(max(first, 0), s.a.r.total);
  x.T = b0 < b1 ? min(max(P, 0), s.max_prefix) & ~(kBlock - 1) : 0;
  x.n = x.T > 0 ? max(min(max(end, 0), s.a.r.total) - x.first, 0) : 0;
  x.tiles = s.wide ? (x.n * s.a.G + kWideRows - 1) / kWideRows : (x.n * s.a.G + 31) / 32;
  return x;
}
template <int TS>
__device__ __forceinline__ Kv8SharedSeq kv8_shared_own(const Kv8SharedArgs& s, int b, int first, int end, int P, int len) {
  Kv8SharedSeq x;
  P = min(max(P, 0), s.max_prefix) & ~(kBlock - 1);
  x.table = b;
  x.skip = P / kBlock;
  x.first = min(max(first, 0), s.a.r.total);
  x.T = (s.a.lens ? min(max(len, 0), s.a.max_len) : s.a.max_len) - P;
  x.n = x.T > 0 ? max(min(max(end, 0), s.a.r.total) - x.first, 0) : 0;  // none: nothing behind the prefix
  x.tiles = (x.n * s.a.G + TS - 1) / TS;
  return x;
}

template <int TS>
__device__ __forceinline__ Kv8SharedSeq kv8_shared_seq(const Kv8SharedArgs& s, int v) {
  const Kv8AttnArgs& a = s.a;
  if (v < s.groups) {
    const int b0 = min(max(s.cu_groups[v], 0), a.r.batch), b1 = min(max(s.cu_groups[v + 1], b0), a.r.batch);
    return kv8_shared_prefix(s, b0, b1, a.r.cu[b0], a.r.cu[b1], s.prefix[min(b0, a.r.batch - 1)]);
  }
  const int b = v - s.groups;
  return kv8_shared_own<TS>(s, b, a.r.cu[b], a.r.cu[b + 1], s.prefix[b], a.lens ? a.lens[b] : 0);
}

// The tables in LDS, where a workgroup has a thread for each prefix and sequence: all of them in one load each, where a
// prefix's rows would be a second one after its sequences.
struct Kv8SharedTables {
  int cu[kKv8Threads + 1], prefix[kKv8Threads];
};

struct Kv8SharedLds {
  uint32_t sum[kKv8Threads / kWave][2];  // steps, by the time that they take, and tiles
  uint32_t less[kKv8Threads / kWave];  // items of all prefixes and sequences, of fewer steps
  uint2 run[kKv8Threads];  // items of prefixes, and of sequences, of the wavefront's runs up to and with this one
};

// A call's items, in this order: (prefixes, then sequences) x (KV head) x (v) x (chunk of its keys) x (tile).
template <int TS>
struct Kv8SharedItems {
  int count, per_run;       // prefixes and sequences; of a thread's run
  uint32_t length[2];       // steps of an item of a prefix, and of a sequence, at most: they take as long
  uint32_t per_head[2];     // items of a KV head
  uint32_t items;

  // The item that is being computed.
  Kv8SharedSeq x;
  int kvh, tile, chunk, v;
  uint32_t chunks;

  __device__ __forceinline__ uint32_t chunks_of(int i, uint32_t steps) const { return (steps + length[i] - 1) / length[i]; }

  // seqs: a run's last prefix or sequence, its only one where the runs hold one each.
  __device__ __forceinline__ void begin(const Kv8SharedArgs& s, Kv8SharedLds& lds, Kv8SharedSeq* seqs, uint32_t grid) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const uint32_t heads = (uint32_t)s.a.kv_heads, weight = s.wide ? kSharedWide : 1, own = s.wide ? TS / 16 : 1;
    count = s.groups + s.a.r.batch;
    per_run = (count + kKv8Threads - 1) / kKv8Threads;
    uint32_t steps = 0, tiles = 0;
    const auto count_in = [&](int y, const Kv8SharedSeq& q) {
      steps += (uint32_t)q.tiles * q.steps() * (y < s.groups ? weight : own);
      tiles += (uint32_t)q.tiles;
      seqs[tid] = q;
    };
    if (per_run == 1) {
      Kv8SharedTables& tables = *reinterpret_cast<Kv8SharedTables*>(seqs + kKv8Threads);
      const int b = tid - s.groups;
      const bool has = b >= 0 && tid < count;
      int g0 = 0, g1 = 0, len = 0;
      if (tid < s.groups) {
        g0 = s.cu_groups[tid];
        g1 = s.cu_groups[tid + 1];
      }
      if (has) {
        const int first = s.a.r.cu[b], P = s.prefix[b];
        if (s.a.lens) len = s.a.lens[b];
        tables.cu[b] = first;
        tables.prefix[b] = P;
      }
      if (tid == 0) tables.cu[s.a.r.batch] = s.a.r.cu[s.a.r.batch];
      __syncthreads();
      if (tid < s.groups) {
        const int b0 = min(max(g0, 0), s.a.r.batch), b1 = min(max(g1, b0), s.a.r.batch);
        count_in(tid, kv8_shared_prefix(s, b0, b1, tables.cu[b0], tables.cu[b1], tables.prefix[min(b0, s.a.r.batch - 1)]));
      } else if (has) {
        count_in(tid, kv8_shared_own<TS>(s, b, tables.cu[b], tables.cu[b + 1], tables.prefix[b], len));
      }
    } else {
      for (int k = 0; k < per_run; ++k) {
        const int y = tid * per_run + k;
        if (y >= count) break;
        count_in(y, kv8_shared_seq<TS>(s, y));
      }
    }
    steps = kv8_lane_scan(steps);
    tiles = kv8_lane_scan(tiles);
    if (lane == kWave - 1) {
      lds.sum[wave][0] = steps;
      lds.sum[wave][1] = tiles;
    }
    __syncthreads();
    steps = tiles = 0;
#pragma unroll
    for (int k = 0; k < kKv8Threads / kWave; ++k) {
      steps += lds.sum[k][0];
      tiles += lds.sum[k][1];
    }
    steps = __builtin_amdgcn_readfirstlane(steps) * heads;
    tiles = __builtin_amdgcn_readfirstlane(tiles) * heads;
    // A tile of n steps has at most n / length + 1 chunks, so with an even share of the steps over the workgroups that the tiles
    // leave (and two for each XCD, which takes an eighth of either kind's items, rounded up) there is a workgroup for every
    // item.  Where the tiles alone are too many for that: an even share of the steps and starts.
    const bool fits = 2 * tiles <= grid - 16;
    uint32_t each = fits ? steps / (grid - 16 - tiles) + 1 : (steps + kSharedStart * tiles) / grid + 1;
    const auto share = [&](uint32_t each) {
      length[1] = ((each + own - 1) / own + 3) & ~3u;
      length[0] = s.wide ? max((each + kSharedWide - 1) / kSharedWide, (uint32_t)kSharedShort) : length[1];
    };
    const auto items_of = [&]() {
      uint2 n = make_uint2(0, 0);
      for (int k = 0; k < per_run; ++k) {
        const int y = tid * per_run + k;
        if (y >= count) break;
        const Kv8SharedSeq q = per_run == 1 ? seqs[tid] : kv8_shared_seq<TS>(s, y);
        const uint32_t c = (uint32_t)q.tiles * chunks_of(y < s.groups ? 0 : 1, q.steps());
        n.x += y < s.groups ? c : 0;
        n.y += y < s.groups ? 0 : c;
      }
      return n;
    };
    uint2 mine;
    bool taken = false;
    // That is what it takes where every tile ends in a short item.  As a rule there is a workgroup for each with items half way to
    // where none does: then they are taken, with tiles of kWideRows (32 x 5 rows over 32768 tokens 76.2 -> 72.9 us; with
    // tiles of 32, whose steps are short, the more parts take longer: 32 x 1 over 8192 20.3 -> 24.3).
    if (s.wide && fits) {
      share((each + steps / grid + 1) / 2);
      mine = items_of();
      const uint32_t n = kv8_lane_scan(min(mine.x, 1023u) | min(mine.y, 1023u) << 16);  // more do not fit anyway
      if (lane == kWave - 1) lds.less[wave] = n;
      __syncthreads();
      uint32_t p = 0, q = 0;
#pragma unroll
      for (int k = 0; k < kKv8Threads / kWave; ++k) {
        p += lds.less[k] & 0xFFFF;
        q += lds.less[k] >> 16;
      }
      taken = (__builtin_amdgcn_readfirstlane(p) * heads + 7) / 8 + (__builtin_amdgcn_readfirstlane(q) * heads + 7) / 8 <= grid / 8;
    }
    if (!taken) {
      share(each);
      mine = items_of();
    }
    lds.run[tid] = make_uint2(kv8_lane_scan(mine.x), kv8_lane_scan(mine.y));
    __syncthreads();
    per_head[0] = per_head[1] = 0;
#pragma unroll
    for (int k = 0; k < kKv8Threads / kWave; ++k) {
      per_head[0] += lds.run[k * kWave + kWave - 1].x;
      per_head[1] += lds.run[k * kWave + kWave - 1].y;
    }
    per_head[0] = __builtin_amdgcn_readfirstlane(per_head[0]);
    per_head[1] = __builtin_amdgcn_readfirstlane(per_head[1]);
    items = (per_head[0] + per_head[1]) * heads;
  }

  // Items before those of prefix or sequence y (of one KV head and its kind).
  __device__ __forceinline__ uint32_t before(const Kv8SharedArgs& s, const Kv8SharedLds& lds, int y) const {
    const int i = y < s.groups ? 0 : 1, run = y / per_run;
    uint32_t n = run % kWave ? (&lds.run[run - 1].x)[i] : 0;
    for (int k = 0; k < run / kWave; ++k) n += (&lds.run[k * kWave + kWave - 1].x)[i];
    for (int k = run * per_run; k < y; ++k) {
      if ((k < s.groups ? 0 : 1) != i) continue;
      const Kv8SharedSeq q = kv8_shared_seq<TS>(s, k);
      n += (uint32_t)q.tiles * chunks_of(i, q.steps());
    }
    return n;
  }

  // The item of this number (< items); seqs: as begin left them, or nullptr.
  __device__ __forceinline__ bool find(const Kv8SharedArgs& s, const Kv8SharedLds& lds, const Kv8SharedSeq* seqs, uint32_t item) {
    const int lane = threadIdx.x & (kWave - 1);
    const uint32_t prefixes = per_head[0] * (uint32_t)s.a.kv_heads;
    const int i = item < prefixes ? 0 : 1;
    uint32_t rem = item - (i ? prefixes : 0);
    kvh = (int)(rem / per_head[i]);
    rem -= (uint32_t)kvh * per_head[i];
    // the wavefront whose runs hold the item, then the run: the first that ends behind it
    int wv = 0;
#pragma unroll
    for (int k = 0; k < kKv8Threads / kWave - 1; ++k) {
      const uint32_t n = (&lds.run[k * kWave + kWave - 1].x)[i];
      if (wv == k && rem >= n) {
        rem -= n;
        wv = k + 1;
      }
    }
    wv = __builtin_amdgcn_readfirstlane(wv);
    rem = __builtin_amdgcn_readfirstlane(rem);
    const uint32_t upto = (&lds.run[wv * kWave + lane].x)[i];
    const int at = min(__popcll(__ballot(upto <= rem)), kWave - 1);
    if (at > 0) rem -= __builtin_amdgcn_readlane(upto, at - 1);
    v = (wv * kWave + at) * per_run;
    if (per_run == 1) {
      x = seqs ? seqs[v] : kv8_shared_seq<TS>(s, v);
    } else {
      for (;; ++v) {
        if (v >= count) return false;  // not reached: the runs hold the item
        if ((v < s.groups ? 0 : 1) != i) continue;
        x = kv8_shared_seq<TS>(s, v);
        const uint32_t n = (uint32_t)x.tiles * chunks_of(i, x.steps());
        if (rem < n) break;
        rem -= n;
      }
    }
    x.first = __builtin_amdgcn_readfirstlane(x.first);
    x.n = __builtin_amdgcn_readfirstlane(x.n);
    x.T = __builtin_amdgcn_readfirstlane(x.T);
    x.table = __builtin_amdgcn_readfirstlane(x.table);
    x.skip = __builtin_amdgcn_readfirstlane(x.skip);
    x.tiles = __builtin_amdgcn_readfirstlane(x.tiles);
    if (x.tiles <= 0) return false;  // not reached
    chunks = chunks_of(i, x.steps());
    chunk = (int)(rem / (uint32_t)x.tiles);
    tile = (int)(rem - (uint32_t)chunk * (uint32_t)x.tiles);
    return true;
  }

  // The row table's entry of a packed token.
  __device__ __forceinline__ void describe(const Kv8SharedArgs& s, const Kv8SharedLds& lds, int token) const {
    const Kv8AttnArgs& a = s.a;
    Kv8SharedRow row = {};
    // the sequence: as many end at or before the token; its group: as many end at or before it
    int b = 0, g = 0;
    for (int hi = a.r.batch; b < hi;) {
      const int mid = (b + hi) / 2;
      if (min(max(a.r.cu[mid + 1], 0), a.r.total) <= token) b = mid + 1; else hi = mid;
    }
    for (int hi = s.groups; g < hi;) {
      const int mid = (g + hi) / 2;
      if (s.cu_groups[mid + 1] <= b) g = mid + 1; else hi = mid;
    }
    const int of[2] = {g < s.groups && s.cu_groups[g] <= b ? g : -1, b < a.r.batch ? s.groups + b : -1};
    // in no sequence
    row.row0[0] = b < a.r.batch && token >= min(max(a.r.cu[b], 0), a.r.total) ? 0 : -1;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (row.row0[0] < 0 || of[k] < 0) continue;
      const Kv8SharedSeq q = kv8_shared_seq<TS>(s, of[k]);
      if (token < q.first || token - q.first >= q.n) continue;
      row.row0[k] = (token - q.first) * a.G;
      row.tiles[k] = q.tiles;
      row.chunks[k] = (int)chunks_of(k, q.steps());
      row.per_head[k] = per_head[k];
      row.base[k] = before(s, lds, of[k]);
    }
    s.rows[token] = row;
  }
};

// A part of a tile of TR rows: [TR][D] sums, then [TR] (maximum, sum of exponentials).
template <int D>
constexpr int shared_part(int TR) {
  return TR * (D + 2);
}

// RS: row tiles of 16 of a sequence's tile.
template <int D, int FMT, int RS>
__global__ __launch_bounds__(kKv8Threads, 2) void kv8_shared_kernel(Kv8SharedArgs s) {
  constexpr int RP = 2;
  __shared__ Kv8RowsLds<D, RP> lds;
  __shared__ Kv8SharedLds lds_plan;
  static_assert(sizeof(Kv8RowsLds<D, RS>) <= sizeof(lds) && sizeof(Kv8WideLds<D>) <= sizeof(lds), "every kind of tile uses the same memory");
  const Kv8AttnArgs& a = s.a;
  Kv8SharedItems<16 * RS> at;
  const uint32_t grid = gridDim.x, w = blockIdx.x;
  static_assert(sizeof(lds.o) >= kKv8Threads * sizeof(Kv8SharedSeq) + sizeof(Kv8SharedTables), "room for the plan until the first sums");
  static_assert(sizeof(lds) + sizeof(lds_plan) <= 80 * 1024, "two workgroups per CU");
  const Kv8SharedSeq* seqs = reinterpret_cast<Kv8SharedSeq*>(&lds.o);
  at.begin(s, lds_plan, reinterpret_cast<Kv8SharedSeq*>(&lds.o), grid);
  // Workgroups w, w + 8, ... share an XCD: an eighth of the prefixes' items, one after another, and of the sequences' are
  // theirs.
  const uint32_t prefixes = at.per_head[0] * (uint32_t)a.kv_heads, mine_p = (prefixes + 7) / 8, mine_s = (at.items - prefixes + 7) / 8;
  for (uint32_t j = w >> 3; j < mine_p + mine_s; j += grid >> 3) {
    const uint32_t item = j < mine_p ? (w & 7) * mine_p + j : prefixes + (w & 7) * mine_s + (j - mine_p);
    if (item >= (j < mine_p ? prefixes : at.items)) continue;
    if (!at.find(s, lds_plan, seqs, item)) break;
    __syncthreads();
    seqs = nullptr;
    const bool prefix = at.v < s.groups, wide = prefix && s.wide;
    const uint32_t slot = prefix ? item : item - prefixes;
    if (slot >= s.parts[prefix ? 0 : 1]) break;
    const int TR = wide ? kWideRows : prefix ? 16 * RP : 16 * RS;
    const Kv8SharedSeq x = at.x;
    const int row0 = at.tile * TR, rows = min(x.n * a.G - row0, TR);
    Kv8Seq seq;
    seq.first = x.first;
    seq.n = x.n;
    seq.T = x.T;
    seq.ctx = prefix ? x.T : x.T - x.n;
    seq.tiles = x.tiles;
    seq.tree = prefix || a.tree != nullptr;  // of a prefix every row sees all keys: a tree's context
    int steps = (int)x.steps();
    int each = (steps + (int)at.chunks - 1) / (int)at.chunks;
    if (!wide) each = (each + 3) & ~3;
    // a tile of early rows sees fewer keys than its sequence's last
    if (!seq.tree) steps = min(steps, max(seq.ctx + (row0 + rows - 1) / a.G + kKv8Step, 0) >> kKv8StepBits);
    const int s0 = min(at.chunk * each, steps), s1 = min(s0 + each, steps);
    const Kv8View view = {a.r.table + (int64_t)x.table * a.r.max_blocks + x.skip, a.r.max_blocks - x.skip, a.r.num_blocks,
                          prefix ? nullptr : a.tree};
    float* part = s.part[prefix ? 0 : 1] + (int64_t)slot * shared_part<D>(TR);
    const auto lowest = [&](int r) {
      Kv8Seq c = seq;
      c.tree = !prefix && seq.tree;
      const int until = prefix ? min(s1 * kKv8Step, seq.T) : s1 * kKv8Step;
      return kv8_lowest(a.tree, view.max_blocks, c, (row0 + r) / a.G, s0 * kKv8Step, until, [&](int j) { return view.named(j); });
    };
    const auto leave = [&](const auto& sums, int at_row, int count) {  // of a tile of few rows, from row at_row of the part on
      __syncthreads();
      for (int e = threadIdx.x; e < count * (D / 4); e += kKv8Threads) {
        const int r = e / (D / 4), d = 4 * (e % (D / 4));
        float mm, ll;
        const f32x4 acc = kv8_rows_sum(sums, r, d, mm, ll);
        if (__builtin_expect(mm == -INFINITY, 0)) mm = lowest(at_row + r);
        *reinterpret_cast<f32x4*>(part + (at_row + r) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(part + TR * D + 2 * (at_row + r)) = make_float2(mm, ll);
      }
    };
    Kv8WideLds<D>& lds_wide = reinterpret_cast<Kv8WideLds<D>&>(lds);
    int E = 0;
    f32x16 acc[D / 32];
    float m, l;
    if (wide && kv8_wide_tile<D, FMT>(a, view, x.first, x.T, at.kvh, row0, rows, s0, s1, E, lds_wide, acc, m, l)) {
      // in units of 1; where V is large enough for the sums of 2^30 keys to pass fp32's range, as of a maximum 2^48 times as large
      const float raise = E >= 64 ? kKv8Raise : 0.0f;
      const float unit = __builtin_amdgcn_ldexpf(1.0f, E - (FMT == kFp8 ? 5 : 7) - (int)(kWideBits + raise));
      const int lane = threadIdx.x & (kWave - 1), g = lane >> 5, r = (int)threadIdx.x / kWave * 32 + (lane & 31);
      const float2 pr = lane_pair<32>(l);
      if (r < rows) {
        m = __builtin_expect(m == -INFINITY, 0) ? lowest(r) : m + raise;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<f32x4*>(part + r * D + 32 * dt + 8 * j + 4 * g) =
                f32x4{acc[dt][4 * j] * unit, acc[dt][4 * j + 1] * unit, acc[dt][4 * j + 2] * unit, acc[dt][4 * j + 3] * unit};
        if (g == 0) *reinterpret_cast<float2*>(part + TR * D + 2 * r) = make_float2(m, __builtin_amdgcn_ldexpf(pr.x + pr.y, -(int)(kWideBits + raise)));
      }
    } else if (prefix) {
      for (int k = 0; k < rows; k += 16 * RP) {  // a tile of kWideRows as several of few rows
        const int count = min(rows - k, 16 * RP);
        __syncthreads();
        kv8_rows_tile<D, FMT, RP, true>(a, view, seq, at.kvh, row0 + k, count, s0, s1, lds);
        leave(lds, k, count);
      }
    } else {
      auto& few = reinterpret_cast<Kv8RowsLds<D, RS>&>(lds);
      kv8_rows_tile<D, FMT, RS>(a, view, seq, at.kvh, row0, rows, s0, s1, few);
      leave(few, 0, rows);
    }
    __syncthreads();
  }
  // the row table, from the last workgroups on, which have the least to do
  for (uint32_t token = (grid - 1 - w) * kKv8Threads + threadIdx.x; token < (uint32_t)a.r.total; token += grid * kKv8Threads)
    at.describe(s, lds_plan, (int)token);
}

// The rows of a packed token and KV head: their parts added up, four dimensions a thread, the parts of a row by as many
// groups of threads as have kSharedMergeBatch of them in flight each (at most eight groups).
constexpr int kSharedMergeThreads = 512, kSharedMergeBatch = 8, kSharedMergeHeads = 4;  // heads of a workgroup

template <int D, int TS>
__global__ __launch_bounds__(kSharedMergeThreads) void kv8_shared_merge_kernel(Kv8SharedArgs s) {
  constexpr int LN = D / 4, GR = kSharedMergeThreads / LN;
  __shared__ f32x4 lds_acc[GR][LN];
  __shared__ float2 lds_ml[GR];
  const Kv8AttnArgs& a = s.a;
  const int tid = threadIdx.x, token = blockIdx.x, kvh = blockIdx.y;
  const Kv8SharedRow row = s.rows[token];
  if (row.row0[0] < 0) return;  // in no sequence
  const int n0 = row.chunks[0], n = n0 + row.chunks[1], TP = s.wide ? kWideRows : 32;
  int lg = 0;
  while (lg < 3 && (kSharedMergeBatch << lg) < n) ++lg;
  const int group = tid / LN, ln = tid % LN, d = 4 * ln;
  const int first = (int)blockIdx.z * kSharedMergeHeads, end = min(first + kSharedMergeHeads, a.G);
  for (int h0 = first; h0 < end; h0 += GR >> lg) {
    const int head = h0 + (group >> lg);
    const bool live = head < end;
    const int r0 = row.row0[0] + min(head, a.G - 1), r1 = row.row0[1] + min(head, a.G - 1);
    const uint32_t base0 = row.base[0] + (uint32_t)kvh * row.per_head[0] + (uint32_t)(r0 / TP);
    const uint32_t base1 = row.base[1] + (uint32_t)kvh * row.per_head[1] + (uint32_t)(r1 / TS);
    const float* const own = s.part[1] + (r1 % TS) * D + d;
    const float* const prefix = s.part[0] + (r0 % TP) * D + d;
    float m = -INFINITY, l = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = group & ((1 << lg) - 1); live && k0 < n; k0 += kSharedMergeBatch << lg) {
      float2 st[kSharedMergeBatch];
      f32x4 y[kSharedMergeBatch];
#pragma unroll
      for (int k = 0; k < kSharedMergeBatch; ++k) {  // past the last part that again, not counted
        const int c = min(k0 + (k << lg), n - 1);
        const uint32_t x0 = min(base0 + (uint32_t)(c * row.tiles[0]), s.parts[0] - 1), x1 = min(base1 + (uint32_t)((c - n0) * row.tiles[1]), s.parts[1] - 1);
        const float* const part = c < n0 ? prefix + (int64_t)x0 * shared_part<D>(TP) : own + (int64_t)x1 * shared_part<D>(TS);
        const int stats = c < n0 ? (TP - r0 % TP) * D + 2 * (r0 % TP) - d : (TS - r1 % TS) * D + 2 * (r1 % TS) - d;
        st[k] = *reinterpret_cast<const float2*>(part + stats);
        y[k] = *reinterpret_cast<const f32x4*>(part);
      }
      float mx = m;
#pragma unroll
      for (int k = 0; k < kSharedMergeBatch; ++k) mx = fmaxf(mx, st[k].x);
      const float f = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
      l *= f;
      acc *= f;
      m = mx;
#pragma unroll
      for (int k = 0; k < kSharedMergeBatch; ++k) {
        const float w = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st[k].x - mx);
        if (k0 + (k << lg) < n) {
          l += st[k].y * w;
          acc += y[k] * w;
        }
      }
    }
    if (lg > 0) {  // the groups' sums
      __syncthreads();
      lds_acc[group][ln] = acc;
      if (ln == 0) lds_ml[group] = make_float2(m, l);
      __syncthreads();
      const int g0 = group & ~((1 << lg) - 1);
      m = -INFINITY;
      for (int k = 0; k < 1 << lg; ++k) m = fmaxf(m, lds_ml[g0 + k].x);
      l = 0.0f;
      acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int k = 0; k < 1 << lg; ++k) {
        const float w = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(lds_ml[g0 + k].x - m);
        l += lds_ml[g0 + k].y * w;
        acc += lds_acc[g0 + k][ln] * w;
      }
      if (group != g0) continue;
    }
    if (!live) continue;
    const float inv = m == -INFINITY ? 0.0f : 1.0f / l;  // a row that sees nothing: 0
    *reinterpret_cast<uint2*>(a.out + (int64_t)token * a.out_stride + (int64_t)(kvh * a.G + head) * D + d) =
        make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  }
}

}  // namespace sdv

using namespace sdv;

static int shared_tile(int32_t G, int32_t max_q_len) { return (int64_t)G * max_q_len <= 16 ? 16 : 32; }

// Rows of a prefix's tile, or 0 where a call takes longer here than in sdv_kv8_attention, which reads the prefix again for
// every sequence, from the caches: it has one launch, and tiles of 256 of a sequence's own rows.  From 204 sizes of one group
// (2 to 64 sequences, 1, 5 and 24 rows each, prefixes of 256 to 32768, heads 12/2/128 and 14/2/64), GPU time in us, sdv_kv8_attention
// first, then tiles of 32 and of 128 rows, 12/2/128:
//   up to 16 rows a sequence and KV head, by the keys not read again: the ways meet between 200 and 250 thousand (4 x 1 over 32768
//     26 24 30, 8 x 1 over 16384 21 22 27, 16 x 1 over 8192 19 19 26, 32 x 1 over 4096 17 17 23; with heads of 64 19 17 20, 15 16 19,
//     15 15 18, 14 14 17), and twice as many are worth the other launch: 8 x 1 over 32768 30 26 33, 32 x 1 over 8192 24 20 28,
//     64 x 1 over 8192 38 29 34;
//   up to 64, by the prefix: 2 x 5 over 1024 13 14 19 and over 4096 18 15 21, 16 x 5 over 1024 14 16 22 and over 4096 25 24 27;
//   more: 8 x 24 over 4096 31 34 39, 32 x 24 over 8192 81 134 88;
//   and of the two kinds of tiles, by a group's rows times its prefix: 8 x 5 over 32768 50 41 42, 32 x 5 over 8192 43 44 42, 64 x 1 over
//     32768 126 65 50, 32 x 5 over 32768 112 109 71, 64 x 5 over 32768 217 206 131; with heads of 64 from a third of that on (32 x 1 over
//     16384 27 23 23, 64 x 1 over 4096 18 17 19).
// Over all of the sizes this takes 1.2% longer than the fastest of the three for each.  It has no more than the counts and the
// longest prefix, and is that of batches of one group: sequences that share nothing count as if they did, and one with many rows
// keeps all from sharing.  kv8_attention would be faster for 62 single tokens over 8392 tokens of their own and a pair that shares
// 8192 (57 74 70, taken: 74; with 2000 of their own 22 31 29), for 56 such and 8 that share (55 71 61), for 16 pairs (27 30 38)
// and for 56 blocks of 5 rows over 4000 and 8 that share 4096 (45 58 50); with 32 that share and 32 that do not it is 49 51 46.
constexpr int64_t kSharedKeys = 1 << 18, kSharedPrefix = 1 << 12, kSharedWideKeys = 8 << 20;
static int shared_rows(int32_t batch, int32_t groups, int32_t total, int32_t G, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                       int32_t max_prefix) {
  const int64_t own = (int64_t)G * max_q_len;
  if (groups <= 0 || batch == groups || own > 64) return 0;
  if (own <= 16 ? (int64_t)(batch - groups) * max_prefix * kv_heads < kSharedKeys : max_prefix < kSharedPrefix) return 0;
  const int64_t keys = (int64_t)total * G / groups * max_prefix * kv_heads / 2;
  return keys >= (head_dim == 128 ? kSharedWideKeys : kSharedWideKeys / 3) ? kWideRows : 32;
}

// Most tiles of all KV heads' prefixes (k = 0) and sequences.
static int64_t shared_tiles(int k, bool wide, int32_t batch, int32_t groups, int32_t total, int32_t G, int32_t kv_heads, int32_t max_q_len) {
  const int64_t rows = (int64_t)total * G;
  const int64_t cut = k == 0 ? rows / (wide ? kWideRows : 32) + groups : rows / shared_tile(G, max_q_len) + batch;
  return (cut < rows ? cut : rows) * kv_heads;
}

// The plan's sums are 32 bits wide, and a part's number a 31-bit one.
static int shared_sizes(int32_t batch, int32_t groups, int32_t total, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                        int32_t max_len, int32_t max_prefix) {
  if (batch <= 0 || groups < 0 || groups > batch || total < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_heads > 65535 ||
      max_q_len <= 0 || max_len <= 0 || max_prefix < 0)
    return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  if (batch > INT32_MAX / 4 || total > INT32_MAX / 2) return SDV_ERR_SHAPE;
  const int32_t G = q_heads / kv_heads;
  if (((int64_t)max_len + max_prefix + total) * G > (1 << 30)) return SDV_ERR_SHAPE;
  const int64_t prefixes = shared_tiles(0, false, batch, groups, total, G, kv_heads, max_q_len), own = shared_tiles(1, false, batch, groups, total, G, kv_heads, max_q_len);
  if (prefixes + own > INT32_MAX / 8) return SDV_ERR_SHAPE;
  const int64_t steps = prefixes * (max_prefix / kKv8Step + 1) * kSharedWide + own * 2 * (max_len / kKv8Step + 1) + (prefixes + own) * kSharedStart;
  return steps > INT32_MAX / 4 ? SDV_ERR_SHAPE : SDV_OK;
}

static size_t shared_tables(int32_t total) { return round_up((size_t)total * sizeof(Kv8SharedRow), 256); }

// Parts of prefixes and of sequences: a chunk has an even share of all steps at least.
static int64_t shared_parts(int k, bool wide, int32_t batch, int32_t groups, int32_t total, int32_t G, int32_t kv_heads, int32_t max_q_len) {
  return shared_tiles(k, wide, batch, groups, total, G, kv_heads, max_q_len) + kKv8Grid;
}
static size_t shared_part_bytes(int k, bool wide, int32_t G, int32_t head_dim, int32_t max_q_len) {
  const int rows = k == 1 ? shared_tile(G, max_q_len) : wide ? kWideRows : 32;
  return sizeof(float) * (head_dim == 128 ? shared_part<128>(rows) : shared_part<64>(rows));
}

static size_t shared_workspace(bool wide, int32_t batch, int32_t groups, int32_t total, int32_t G, int32_t kv_heads, int32_t head_dim, int32_t max_q_len) {
  size_t bytes = shared_tables(total);
  for (int k = 0; k < 2; ++k)
    bytes += (size_t)shared_parts(k, wide, batch, groups, total, G, kv_heads, max_q_len) * shared_part_bytes(k, wide, G, head_dim, max_q_len);
  return bytes;
}

extern "C" int32_t sdv_kv8_shared_attention_tile_rows(int32_t batch, int32_t groups, int32_t total_rows, int32_t q_heads, int32_t kv_heads,
                                                      int32_t head_dim, int32_t max_q_len, int32_t max_seq_len, int32_t max_prefix_len) {
  if (shared_sizes(batch, groups, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len, max_prefix_len) != SDV_OK) return 0;
  return shared_rows(batch, groups, total_rows, q_heads / kv_heads, kv_heads, head_dim, max_q_len, max_prefix_len);
}

extern "C" size_t sdv_kv8_shared_attention_workspace_size(int32_t batch, int32_t groups, int32_t total_rows, int32_t q_heads,
                                                          int32_t kv_heads, int32_t head_dim, int32_t max_q_len, int32_t max_seq_len,
                                                          int32_t max_prefix_len, int32_t tile_rows) {
  if (shared_sizes(batch, groups, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len, max_prefix_len) != SDV_OK) return 0;
  if (tile_rows != 32 && tile_rows != kWideRows) return 0;
  return shared_workspace(tile_rows != 32, batch, groups, total_rows, q_heads / kv_heads, kv_heads, head_dim, max_q_len);
}

template <int D, int FMT, int RS>
static void shared_launch(const Kv8SharedArgs& s, hipStream_t st) {
  hipLaunchKernelGGL((kv8_shared_kernel<D, FMT, RS>), dim3(kKv8Grid), dim3(kKv8Threads), 0, st, s);
  constexpr int most = 1 << 22;  // tokens of a launch, which has fewer than 2^32 threads along x
  for (int first = 0; first < s.a.r.total; first += most) {
    Kv8SharedArgs x = s;
    x.rows += first;
    x.a.out += first * x.a.out_stride;
    const int n = s.a.r.total - first < most ? s.a.r.total - first : most;
    const dim3 merge((unsigned)n, (unsigned)s.a.kv_heads, (unsigned)((s.a.G + kSharedMergeHeads - 1) / kSharedMergeHeads));
    hipLaunchKernelGGL((kv8_shared_merge_kernel<D, 16 * RS>), merge, dim3(kSharedMergeThreads), 0, st, x);
  }
}

template <int D, int FMT>
static void shared_launch(const Kv8SharedArgs& s, int tile, hipStream_t st) {
  tile == 16 ? shared_launch<D, FMT, 1>(s, st) : shared_launch<D, FMT, 2>(s, st);
}

extern "C" int sdv_kv8_shared_attention(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, const float* scales,
                                        int32_t num_blocks, int32_t format, const int32_t* block_table, int32_t max_blocks_per_seq,
                                        const int32_t* cu_rows, const int32_t* seq_lens, const uint64_t* tree_mask,
                                        const int32_t* cu_groups, const int32_t* prefix_lens, int32_t batch, int32_t groups,
                                        int32_t total_rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t max_q_len,
                                        int32_t max_seq_len, int32_t max_prefix_len, int32_t tile_rows, float scale, void* workspace,
                                        size_t workspace_bytes, void* out, int64_t out_stride, void* stream) {
  if (!q || !k_pages || !v_pages || !scales || !block_table || !cu_rows || !cu_groups || !prefix_lens || !out) return SDV_ERR_NULL;
  const int sizes = shared_sizes(batch, groups, total_rows, q_heads, kv_heads, head_dim, max_q_len, max_seq_len, max_prefix_len);
  if (sizes != SDV_OK) return sizes;
  if (num_blocks <= 0 || max_blocks_per_seq <= 0 || max_blocks_per_seq > INT32_MAX / kBlock) return SDV_ERR_SHAPE;
  if (max_prefix_len > (int64_t)max_blocks_per_seq * kBlock) return SDV_ERR_SHAPE;
  if (format != SDV_KV8_FP8 && format != SDV_KV8_INT8) return SDV_ERR_UNSUPPORTED;
  if (tree_mask && max_q_len > 64) return SDV_ERR_UNSUPPORTED;
  if (tile_rows != 32 && tile_rows != kWideRows) return SDV_ERR_UNSUPPORTED;
  const int64_t row = (int64_t)q_heads * head_dim;
  if (q_stride < row || out_stride < row) return SDV_ERR_SHAPE;
  if (!aligned(q, 16) || !aligned(out, 16) || q_stride % 8 || out_stride % 8 || !aligned(k_pages, 16) || !aligned(v_pages, 16) ||
      !aligned(scales, 16) || !aligned(block_table, 4) || !aligned(cu_rows, 4) || !aligned(seq_lens, 4) || !aligned(tree_mask, 8) ||
      !aligned(cu_groups, 4) || !aligned(prefix_lens, 4))
    return SDV_ERR_ALIGN;
  const int G = q_heads / kv_heads;
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < shared_workspace(tile_rows != 32, batch, groups, total_rows, G, kv_heads, head_dim, max_q_len))
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
  s.wide = tile_rows != 32;
  for (int k = 0; k < 2; ++k) s.parts[k] = (uint32_t)shared_parts(k, s.wide, batch, groups, total_rows, G, kv_heads, max_q_len);
  s.rows = static_cast<Kv8SharedRow*>(workspace);
  a.part = nullptr;
  char* const parts = static_cast<char*>(workspace) + shared_tables(total_rows);
  s.part[0] = reinterpret_cast<float*>(parts);
  s.part[1] = reinterpret_cast<float*>(parts + s.parts[0] * shared_part_bytes(0, s.wide, G, head_dim, max_q_len));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int tile = shared_tile(G, max_q_len);
  if (head_dim == 128)
    format == SDV_KV8_FP8 ? shared_launch<128, kFp8>(s, tile, st) : shared_launch<128, kInt8>(s, tile, st);
  else
    format == SDV_KV8_FP8 ? shared_launch<64, kFp8>(s, tile, st) : shared_launch<64, kInt8>(s, tile, st);
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}
