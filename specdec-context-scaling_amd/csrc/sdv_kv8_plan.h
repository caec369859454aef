// How the attention of ragged rows over a kv8 cache is shared out.
//
// A sequence's query rows (token-major: row r is token r / G, head r % G of the KV head's group) are
// cut into tiles of TR rows; a tile streams the keys its last row sees in steps of 64.  The steps of
// all tiles, in the order (KV head, sequence, tile), are one sequence that is cut into equal
// contiguous ranges, one per workgroup: single tokens over long contexts, prompt chunks and
// batches of both are then equally long for every workgroup, and a workgroup crosses at most two
// tiles that it shares.  Where there are fewer steps than that takes, a tile's steps are counted in
// units of several, each one workgroup's.  Lengths are read on the device; every workgroup works out
// its own range.
//
// The units of a sequence's tiles up to the i-th sum in closed form: of u keys each, tile j has
// ceil((ctx G + TR (j + 1)) / (u G)) (the last one ceil(T / u)), a sum of floors of a linear
// function, which takes as many turns as Euclid's algorithm on (u G, TR).
#pragma once

#include "sdv_kv8.h"

namespace sdv {

constexpr int kKv8Step = 64;  // keys per step: four page blocks

struct Kv8AttnArgs {
  Kv8Rows r;
  const int32_t* lens;   // nullptr: every sequence has max_len tokens
  const uint64_t* tree;  // visibility of a sequence's new tokens among themselves, or nullptr: causal
  const uint16_t* q;
  uint16_t* out;
  int64_t q_stride, out_stride;  // elements between tokens
  const uint8_t* k_pages;
  const uint8_t* v_pages;
  const float* scales;
  int G, kv_heads, max_len;
  float c;         // softmax scale times log2 e
  int unit;        // steps per unit
  uint32_t* done;  // per range: finished parts of the shared tile that begins in it; 0 between calls
  float* part;     // two slots per range: [TR][D] sums, then [TR][4]: maximum, sum of exponentials, -, -
};

// Sum of floor((a i + b) / m) over i < n.
__device__ __forceinline__ uint32_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  uint32_t ans = 0;
  while (n > 0) {
    if (a >= m) {
      ans += (uint32_t)((uint64_t)n * (n - 1) / 2) * (a / m);
      a %= m;
    }
    if (b >= m) {
      ans += n * (b / m);
      b %= m;
    }
    const uint32_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const uint32_t t = m;
    m = a;
    a = t;
  }
  return ans;
}

struct Kv8Seq {
  int first, n, T, ctx;
  int tiles;
  bool tree;
};

template <int TR>
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnArgs& a, int b) {
  Kv8Seq s;
  kv8_rows(a.r, b, s.first, s.n);
  s.T = a.lens ? min(max(a.lens[b], 0), a.max_len) : a.max_len;
  s.ctx = s.T - s.n;
  s.tiles = (s.n * a.G + TR - 1) / TR;
  int tree = a.tree != nullptr;
  asm("" : "+v"(tree));  // else the compiler writes the kernels out twice, with and without
  s.tree = __builtin_amdgcn_readfirstlane(tree);
  return s;
}

// Units of `unit` steps of the tiles before the i-th (i < tiles), of the i-th, and of all.
template <int TR>
__device__ __forceinline__ uint32_t kv8_before(const Kv8Seq& s, int G, int i, int unit) {
  const uint32_t keys = kKv8Step * unit;
  if (s.tree) return (uint32_t)i * (((uint32_t)max(s.T, 1) + keys - 1) / keys);
  const uint32_t m = keys * G;
  return floor_sum((uint32_t)i, m, TR, (uint32_t)(max(s.ctx, 0) * G + TR) + m - 1);
}

template <int TR>
__device__ __forceinline__ uint32_t kv8_steps(const Kv8Seq& s, int G, int i, int unit) {
  const uint32_t keys = kKv8Step * unit;
  if (s.tree) return ((uint32_t)max(s.T, 1) + keys - 1) / keys;
  const int ctx = max(s.ctx, 0);
  if (i == s.tiles - 1) return ((uint32_t)(ctx + s.n) + keys - 1) / keys;
  const uint32_t m = keys * G;
  return ((uint32_t)(ctx * G + TR * (i + 1)) + m - 1) / m;
}

template <int TR>
__device__ __forceinline__ uint32_t kv8_seq_units(const Kv8Seq& s, int G, int unit) {
  return s.tiles == 0 ? 0 : kv8_before<TR>(s, G, s.tiles - 1, unit) + kv8_steps<TR>(s, G, s.tiles - 1, unit);
}

// Inclusive sum over a wavefront's lanes (DPP row shifts, then row broadcasts).
__device__ __forceinline__ uint32_t kv8_lane_scan(uint32_t x) {
  int v = (int)x;
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
  return (uint32_t)v;
}

constexpr int kKv8Threads = 256;

struct Kv8PlanLds {
  uint32_t run[kKv8Threads + 1];  // units before each run of sequences (a run per thread)
  uint32_t wave[kKv8Threads / kWave];
};

// A workgroup's place among the units.
template <int TR>
struct Kv8Place {
  uint32_t per_head;   // units of one KV head
  uint32_t units;      // of all
  uint32_t share, rest;  // every range has `share` units, the first `rest` one more
  int ranges;          // workgroups with a range
  int w;               // this one's
  uint32_t u, end;     // next unit, end of the range
  int kvh, b, i;       // the tile that holds u
  Kv8Seq seq;
  uint32_t tile0, units_of;  // its first unit and its units

  __device__ __forceinline__ uint32_t start(int x) const { return (uint32_t)x * share + min((uint32_t)x, rest); }
  __device__ __forceinline__ int owner(uint32_t x) const {
    const uint32_t split = rest * (share + 1);
    return (int)(x < split ? x / (share + 1) : rest + (x - split) / share);
  }

  // False: no range for this workgroup.  `grid` workgroups, this one `index`.
  __device__ __forceinline__ bool begin(const Kv8AttnArgs& a, Kv8PlanLds& lds, int index, int grid) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int per_run = (a.r.batch + kKv8Threads - 1) / kKv8Threads;
    if (a.r.batch == 1) {
      per_head = kv8_seq_units<TR>(kv8_seq<TR>(a, 0), a.G, a.unit);
    } else {
      uint32_t mine = 0;
      for (int k = 0; k < per_run; ++k) {
        const int x = tid * per_run + k;
        if (x < a.r.batch) mine += kv8_seq_units<TR>(kv8_seq<TR>(a, x), a.G, a.unit);
      }
      const uint32_t scan = kv8_lane_scan(mine);
      if (lane == kWave - 1) lds.wave[tid / kWave] = scan;
      __syncthreads();
      uint32_t before = 0;
      per_head = 0;
#pragma unroll
      for (int k = 0; k < kKv8Threads / kWave; ++k) {
        const uint32_t v = lds.wave[k];
        before += k < tid / kWave ? v : 0;
        per_head += v;
      }
      lds.run[tid] = before + scan - mine;
      if (tid == 0) lds.run[kKv8Threads] = per_head;
      __syncthreads();
    }
    per_head = __builtin_amdgcn_readfirstlane(per_head);
    units = per_head * (uint32_t)a.kv_heads;
    if (units == 0) return false;
    ranges = (int)min((uint32_t)grid, units);
    w = index;
    if (w >= ranges) return false;
    share = units / (uint32_t)ranges;
    rest = units - share * (uint32_t)ranges;
    u = start(w);
    end = start(w + 1);
    kvh = (int)(u / per_head);
    uint32_t rem = u - (uint32_t)kvh * per_head;
    tile0 = (uint32_t)kvh * per_head;
    b = 0;
    if (a.r.batch > 1) {
      // the last run that begins at or before rem; runs of no units share their start with the next
      int lo = 0, hi = kKv8Threads;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (lds.run[mid] <= rem)
          lo = mid;
        else
          hi = mid;
      }
      lo = __builtin_amdgcn_readfirstlane(lo);
      b = lo * per_run;
      const uint32_t base = __builtin_amdgcn_readfirstlane(lds.run[lo]);
      rem -= base;
      tile0 += base;
      for (;; ++b) {
        if (b >= a.r.batch) return false;  // not reached: the runs hold the unit
        seq = kv8_seq<TR>(a, b);
        const uint32_t n = kv8_seq_units<TR>(seq, a.G, a.unit);
        if (rem < n) break;
        rem -= n;
        tile0 += n;
      }
    } else {
      seq = kv8_seq<TR>(a, 0);
    }
    // the tile: the lanes test 64 of them at a time
    i = 0;
    for (int count = seq.tiles; count > 1;) {
      const int stride = (count + kWave - 1) / kWave;
      const bool at = lane * stride < count && kv8_before<TR>(seq, a.G, i + min(lane * stride, count - 1), a.unit) <= rem;
      const int k = __popcll(__ballot(at)) - 1;
      i += k * stride;
      count = min(stride, count - k * stride);
    }
    i = __builtin_amdgcn_readfirstlane(i);
    tile0 += __builtin_amdgcn_readfirstlane(kv8_before<TR>(seq, a.G, i, a.unit));
    units_of = kv8_steps<TR>(seq, a.G, i, a.unit);
    return true;
  }

  // The tile after this one; false past the last (not reached while u < end).
  __device__ __forceinline__ bool next(const Kv8AttnArgs& a) {
    tile0 += units_of;
    if (++i >= seq.tiles) {
      i = 0;
      do {
        if (++b >= a.r.batch) {
          b = 0;
          if (++kvh >= a.kv_heads) return false;
        }
        seq = kv8_seq<TR>(a, b);
      } while (seq.tiles == 0);
    }
    units_of = kv8_steps<TR>(seq, a.G, i, a.unit);
    return true;
  }
};

}  // namespace sdv
