// How the attention of ragged rows over a kv8 cache is shared out.
//
// A sequence's query rows (token-major: row r is token r / G, head r % G of the KV head's group) are
// cut into tiles of TR rows; a tile streams the keys its last row sees in steps of 64.  The steps of
// all tiles, in the order (KV head, sequence, tile), are one sequence that is cut into equal
// contiguous ranges, one per workgroup: single tokens over long contexts, prompt chunks and
// batches of both are then equally long for every workgroup, and a workgroup crosses at most two
// tiles that it shares.  A tile's steps are preceded by a few that stand for what starting it costs.
// Where the device has a workgroup for each, steps are counted in units of several, each one
// workgroup's.  Lengths are read on the device, so that a recorded call follows them; every workgroup
// works out its own range, in 1 to 1.5 us.
//
// The units of a sequence's tiles up to the i-th sum in closed form (sdv_kv8_sums.h): of u keys each,
// tile j has ceil((ctx G + TR (j + 1)) / (u G)), the last one ceil(T / u).
#pragma once

#include "sdv_kv8.h"
#include "sdv_kv8_sums.h"

namespace sdv {

constexpr int kKv8StepBits = 6, kKv8Step = 1 << kKv8StepBits;  // keys per step: four page blocks

struct Kv8Cut;

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
  int unit;        // steps per unit, as a power of two
  int start;       // units that stand for a tile's start
  uint32_t* done;  // per range: finished parts of the shared tile that begins in it; 0 between calls; or nullptr:
  int slot;        //   a slot of kv8_counts
  Kv8Cut* cuts;    // per workgroup, of the kernels whose parts a second launch adds up
  float* part;     // two slots per range: [TR][D] sums, then [TR][4]: maximum, sum of exponentials, -, -
};

struct Kv8Seq {
  int first, n, T, ctx;
  int tiles;
  bool tree;
};

template <int TR>
__device__ __forceinline__ Kv8Seq kv8_seq_of(const Kv8AttnArgs& a, int first, int n, int T) {
  Kv8Seq s;
  s.first = first;
  s.n = n;
  s.T = T;
  s.ctx = T - n;
  s.tiles = (n * a.G + TR - 1) / TR;
  int tree = a.tree != nullptr;
  asm("" : "+v"(tree));  // else the compiler writes the kernels out twice, with and without
  s.tree = __builtin_amdgcn_readfirstlane(tree);
  return s;
}

template <int TR>
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnArgs& a, int b) {
  int first, n;
  kv8_rows(a.r, b, first, n);
  return kv8_seq_of<TR>(a, first, n, a.lens ? min(max(a.lens[b], 0), a.max_len) : a.max_len);
}

// Units of 2^unit steps of the tiles before the i-th (i < tiles), of the i-th, and of all; `start` are
// added to each tile.
template <int TR>
__device__ __forceinline__ uint32_t kv8_steps_before(const Kv8Seq& s, int G, int i, int unit) {
  const uint32_t keys = (uint32_t)kKv8Step << unit;
  if (s.tree) return (uint32_t)i * (((uint32_t)max(s.T, 1) + keys - 1) >> (kKv8StepBits + unit));
  if (i == 0) return 0;
  return kv8_floor_sum<TR>((uint32_t)i, keys, (uint32_t)G, (uint32_t)(max(s.ctx, 0) * G + TR) + keys * G - 1);
}

template <int TR>
__device__ __forceinline__ uint32_t kv8_steps(const Kv8Seq& s, int G, int i, int unit) {
  const uint32_t keys = (uint32_t)kKv8Step << unit;
  if (s.tree) return ((uint32_t)max(s.T, 1) + keys - 1) >> (kKv8StepBits + unit);
  const int ctx = max(s.ctx, 0);
  if (i == s.tiles - 1) return ((uint32_t)(ctx + s.n) + keys - 1) >> (kKv8StepBits + unit);
  const uint32_t m = keys * G;
  return ((uint32_t)(ctx * G + TR * (i + 1)) + m - 1) / m;
}

template <int TR>
__device__ __forceinline__ uint32_t kv8_before(const Kv8Seq& s, const Kv8AttnArgs& a, int i) {
  return kv8_steps_before<TR>(s, a.G, i, a.unit) + (uint32_t)(i * a.start);
}

template <int TR>
__device__ __forceinline__ uint32_t kv8_units_of(const Kv8Seq& s, const Kv8AttnArgs& a, int i) {
  return kv8_steps<TR>(s, a.G, i, a.unit) + (uint32_t)a.start;
}

template <int TR>
__device__ __forceinline__ uint32_t kv8_seq_units(const Kv8Seq& s, const Kv8AttnArgs& a) {
  return s.tiles == 0 ? 0 : kv8_before<TR>(s, a, s.tiles - 1) + kv8_units_of<TR>(s, a, s.tiles - 1);
}

// NT: threads of a workgroup, a run of sequences each.
template <int NT>
struct Kv8PlanLds {
  uint4 run[NT];  // units of the wavefront's runs up to and with this one, units of this one; its one sequence's first, n
  int T[NT];      //   and T
};

// A workgroup's place among the units.
template <int TR, int NT>
struct Kv8Place {
  uint32_t per_head;   // units of one KV head
  uint32_t units;      // of all
  uint32_t share, rest;  // every range has `share` units, the first `rest` one more
  int ranges;          // workgroups with a range
  int w;               // this one's
  uint32_t u, end;     // next unit, end of the range
  int kvh, b, i;       // the tile that holds u
  Kv8Seq seq;
  uint32_t tile0, units_of;  // its first unit and its units, those of its start among them

  __device__ __forceinline__ uint32_t start(int x) const { return (uint32_t)x * share + min((uint32_t)x, rest); }
  __device__ __forceinline__ int owner(uint32_t x) const {
    const uint32_t split = rest * (share + 1);
    return (int)(x < split ? x / (share + 1) : rest + (x - split) / share);
  }

  // Up to 64 tiles of a sequence are counted in the lanes of a wavefront and added up there (one
  // division, where the closed form takes three, and its terms one after the other).
  uint32_t lane_units, lane_sum;
  __device__ __forceinline__ void scan_tiles(const Kv8AttnArgs& a) {
    const int lane = threadIdx.x & (kWave - 1);
    lane_units = lane < seq.tiles ? kv8_units_of<TR>(seq, a, lane) : 0;
    lane_sum = kv8_lane_scan(lane_units);
  }

  // False: no range for this workgroup.  `grid` workgroups, this one `index`.
  __device__ __forceinline__ bool begin(const Kv8AttnArgs& a, Kv8PlanLds<NT>& lds, int index, int grid) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int per_run = (a.r.batch + NT - 1) / NT;
    bool scanned = false;
    if (a.r.batch == 1) {
      seq = kv8_seq<TR>(a, 0);
      if (seq.tiles <= kWave) {
        scan_tiles(a);
        scanned = true;
        per_head = __builtin_amdgcn_readlane(lane_sum, kWave - 1);
      } else {
        per_head = kv8_seq_units<TR>(seq, a);
      }
    } else {
      uint32_t mine = 0;
      Kv8Seq last = {};
      for (int k = 0; k < per_run; ++k) {
        const int x = tid * per_run + k;
        if (x >= a.r.batch) break;
        last = kv8_seq<TR>(a, x);
        mine += kv8_seq_units<TR>(last, a);
      }
      const uint32_t scan = kv8_lane_scan(mine);
      lds.run[tid] = make_uint4(scan, mine, (uint32_t)last.first, (uint32_t)last.n);
      lds.T[tid] = last.T;
      __syncthreads();
      per_head = 0;
#pragma unroll
      for (int k = 0; k < NT / kWave; ++k) per_head += lds.run[k * kWave + kWave - 1].x;
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
      // the wavefront whose runs hold the unit, then the run: the first that ends behind it
      int wv = 0;
#pragma unroll
      for (int k = 0; k < NT / kWave - 1; ++k) {
        const uint32_t n = lds.run[k * kWave + kWave - 1].x;
        if (wv == k && rem >= n) {
          rem -= n;
          tile0 += n;
          wv = k + 1;
        }
      }
      wv = __builtin_amdgcn_readfirstlane(wv);
      rem = __builtin_amdgcn_readfirstlane(rem);
      const uint4 run = lds.run[wv * kWave + lane];
      const int T = lds.T[wv * kWave + lane];
      const int at = min(__popcll(__ballot(run.x <= rem)), kWave - 1);
      const uint32_t before = __builtin_amdgcn_readlane(run.x, at) - __builtin_amdgcn_readlane(run.y, at);
      rem -= before;
      tile0 += before;
      b = (wv * kWave + at) * per_run;
      if (per_run == 1) {
        seq = kv8_seq_of<TR>(a, __builtin_amdgcn_readlane(run.z, at), __builtin_amdgcn_readlane(run.w, at), __builtin_amdgcn_readlane(T, at));
      } else {
        for (;; ++b) {
          if (b >= a.r.batch) return false;  // not reached: the runs hold the unit
          seq = kv8_seq<TR>(a, b);
          const uint32_t n = kv8_seq_units<TR>(seq, a);
          if (rem < n) break;
          rem -= n;
          tile0 += n;
        }
      }
    }
    i = 0;
    if (seq.tiles > 1) {
      uint32_t before;
      if (seq.tiles <= kWave) {
        if (!scanned) scan_tiles(a);
        i = __popcll(__ballot(lane < seq.tiles && lane_sum <= rem));
        before = __builtin_amdgcn_readlane(lane_sum - lane_units, i);
      } else {  // the lanes test 64 tiles at a time
        for (int count = seq.tiles; count > 1;) {
          const int stride = (count + kWave - 1) / kWave;
          const bool at = lane * stride < count && kv8_before<TR>(seq, a, i + min(lane * stride, count - 1)) <= rem;
          const int k = __popcll(__ballot(at)) - 1;
          i += k * stride;
          count = min(stride, count - k * stride);
        }
        before = __builtin_amdgcn_readfirstlane(kv8_before<TR>(seq, a, i));
      }
      i = __builtin_amdgcn_readfirstlane(i);
      tile0 += before;
    }
    units_of = kv8_units_of<TR>(seq, a, i);
    return true;
  }

  // Steps s0 .. s1 - 1 of the tile's `steps` are this range's; false: none, the range ends in its start.
  __device__ __forceinline__ bool part(const Kv8AttnArgs& a, int& s0, int& s1, int& steps) const {
    steps = (int)kv8_steps<TR>(seq, a.G, i, 0);
    const int lo = max((int)(u - tile0) - a.start, 0), hi = (int)min(end - tile0, units_of) - a.start;
    s0 = lo << a.unit;
    s1 = min(hi << a.unit, steps);
    return lo < hi;
  }
  // The range with the tile's first step, how many ranges have steps of it, and whether the first one's
  // part is its second (it began with the end of another tile).
  __device__ __forceinline__ int first_range(const Kv8AttnArgs& a) const { return owner(tile0 + (uint32_t)a.start); }
  __device__ __forceinline__ int parts(const Kv8AttnArgs& a) const { return owner(tile0 + units_of - 1) - first_range(a) + 1; }
  __device__ __forceinline__ int second_part(const Kv8AttnArgs& a) const { return start(first_range(a)) < tile0 ? 1 : 0; }

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
    units_of = kv8_units_of<TR>(seq, a, i);
    return true;
  }
};

}  // namespace sdv
