// Moving what the caches hold: whole page blocks of every layer (both caches), and the tokens of an accepted path (kv8).
#include "sdv_kv8.h"

namespace sdv {

// ---------------------------------------------------------------------------- whole blocks
struct CopyArgs {
  const uint8_t* from[3];  // K, V, scales
  uint8_t* to[3];
  int bytes[3];            // of a block, multiples of 16
  int from_blocks, to_blocks;
  const int32_t *src, *dst;
  int n;
};

// A wavefront copies one block of one layer, its three parts as one run of 16-byte pieces, kCopyBatch of them a lane in
// flight.  Bound by the memory: 3001 blocks of 24 layers (627 MB both ways) 102 us, 6.1 TB/s; 32 of them 4.5 us.
constexpr int kCopyWaves = 4, kCopyBatch = 8;

__global__ __launch_bounds__(kCopyWaves * kWave) void copy_blocks_kernel(CopyArgs a) {
  const int pair = (int)blockIdx.x * kCopyWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (pair >= a.n) return;
  const int lane = threadIdx.x & (kWave - 1), layer = blockIdx.y;
  const int s = __builtin_amdgcn_readfirstlane(a.src[pair]), d = __builtin_amdgcn_readfirstlane(a.dst[pair]);
  if (s < 0 || s >= a.from_blocks || d < 0 || d >= a.to_blocks) return;
  const int64_t from = (int64_t)layer * a.from_blocks + s, to = (int64_t)layer * a.to_blocks + d;
  const uint8_t* const f[3] = {a.from[0] + from * a.bytes[0], a.from[1] + from * a.bytes[1], a.from[2] + from * a.bytes[2]};
  uint8_t* const t[3] = {a.to[0] + to * a.bytes[0], a.to[1] + to * a.bytes[1], a.to[2] + to * a.bytes[2]};
  const int e0 = a.bytes[0], e1 = e0 + a.bytes[1], end = e1 + a.bytes[2];
  for (int at = lane * 16; at < end; at += kCopyBatch * kWave * 16) {
    uint4 w[kCopyBatch];
#pragma unroll
    for (int i = 0; i < kCopyBatch; ++i) {
      const int o = at + i * kWave * 16;
      if (o < end) w[i] = load_stream16(o < e0 ? f[0] + o : o < e1 ? f[1] + (o - e0) : f[2] + (o - e1));
    }
#pragma unroll
    for (int i = 0; i < kCopyBatch; ++i) {
      const int o = at + i * kWave * 16;
      if (o < end)
        __builtin_nontemporal_store(u32x4_t{w[i].x, w[i].y, w[i].z, w[i].w},
                                    reinterpret_cast<u32x4_t*>(o < e0 ? t[0] + o : o < e1 ? t[1] + (o - e0) : t[2] + (o - e1)));
    }
  }
}

// ---------------------------------------------------------------------------- the tokens of an accepted path
struct KeepArgs {
  Kv8Rows r;  // cu: where each sequence's entries of `kept` lie, r.total of them
  const int32_t *kept, *starts;
  uint8_t *k, *v;
  float* s;
  int64_t k_layer, v_layer, s_layer;  // elements between layers
  int kv_heads;
};

constexpr int kKeepTokens = 64;
template <int D>
constexpr int kKeepThreads = 2 * D;

// A workgroup moves the tokens of one sequence, KV head and layer: 64 at a time, all of them read before the first is
// written.  Destinations lie in order, so that with ascending entries (each at least its own index) a later batch reads
// nothing that an earlier one has written.
//
// A token's V is one byte of every row of its page, so that it moves D / 4 times its bytes (whole cache lines) and a call
// is bound by those and by its chain of loads (entries, pages, codes): the paths of 8 trees of 24 (2 KV heads of 128, 28 layers)
// 4.3 us in a graph, of 48 trees of 64 (2 of 64, 24 layers) 7.3.  Two tokens' V at a time: with 256 threads for 64 dimensions
// too the latter take 7.8, with 128 for 128 the former 4.9.  With the loads of tokens that stay done too, so that eight are under
// way without a condition: 4.9, 10.8.
template <int D>
__global__ __launch_bounds__(kKeepThreads<D>) void kv8_keep_kernel(KeepArgs a) {
  constexpr int T = kKeepThreads<D>;
  __shared__ __align__(16) uint8_t lds_k[kKeepTokens][D], lds_v[kKeepTokens][D];
  __shared__ float lds_s[kKeepTokens][2];
  __shared__ int from[kKeepTokens], to[kKeepTokens];  // slots, -1: none
  const int tid = threadIdx.x, b = blockIdx.x, kvh = blockIdx.y;
  int first, n;
  kv8_rows(a.r, b, first, n);
  if (n == 0) return;
  const int start = a.starts[b];
  uint8_t* const k = a.k + blockIdx.z * a.k_layer;
  uint8_t* const v = a.v + blockIdx.z * a.v_layer;
  float* const s = a.s + blockIdx.z * a.s_layer;
  const auto slot = [&](int64_t pos) {
    if (pos < 0 || pos >= (int64_t)a.r.max_blocks * kBlock) return -1;
    const int id = kv8_block(a.r, b, (int)pos >> 4);
    return id < 0 ? -1 : id * kBlock + ((int)pos & 15);
  };
  const auto page = [&](int slot) { return (int64_t)(slot >> 4) * a.kv_heads + kvh; };

  for (int base = 0; base < n; base += kKeepTokens) {
    const int m = min(n - base, kKeepTokens);
    if (tid < m) {
      const int x = slot((int64_t)start + a.kept[first + base + tid]), y = slot((int64_t)start + base + tid);
      const bool move = x >= 0 && y >= 0 && x != y;
      from[tid] = move ? x : -1;
      to[tid] = move ? y : -1;
    }
    __syncthreads();
#pragma unroll 2
    for (int e = tid; e < m * (D / 16); e += T) {
      const int i = e / (D / 16), c = e % (D / 16), x = from[i];
      if (x >= 0)
        *reinterpret_cast<uint4*>(&lds_k[i][16 * c]) = *reinterpret_cast<const uint4*>(k + page(x) * (kBlock * D) + (x >> 2 & 3) * (4 * D) + c * 64 + (x & 3) * 16);
    }
#pragma unroll 4
    for (int e = tid; e < m * D; e += T) {
      const int i = e / D, d = e % D, x = from[i];
      if (x >= 0) lds_v[i][d] = v[page(x) * (kBlock * D) + d * kBlock + (x & 15)];
    }
    for (int e = tid; e < 2 * m; e += T) {
      const int x = from[e >> 1];
      if (x >= 0) lds_s[e >> 1][e & 1] = s[page(x) * (2 * kBlock) + (e & 1) * kBlock + (x & 15)];
    }
    __syncthreads();
#pragma unroll 2
    for (int e = tid; e < m * (D / 16); e += T) {
      const int i = e / (D / 16), c = e % (D / 16), y = to[i];
      if (y >= 0)
        *reinterpret_cast<uint4*>(k + page(y) * (kBlock * D) + (y >> 2 & 3) * (4 * D) + c * 64 + (y & 3) * 16) = *reinterpret_cast<const uint4*>(&lds_k[i][16 * c]);
    }
#pragma unroll 4
    for (int e = tid; e < m * D; e += T) {
      const int i = e / D, d = e % D, y = to[i];
      if (y >= 0) v[page(y) * (kBlock * D) + d * kBlock + (y & 15)] = lds_v[i][d];
    }
    for (int e = tid; e < 2 * m; e += T) {
      const int y = to[e >> 1];
      if (y >= 0) s[page(y) * (2 * kBlock) + (e & 1) * kBlock + (y & 15)] = lds_s[e >> 1][e & 1];
    }
    __syncthreads();  // the LDS arrays; and a later batch's reads stand behind this one's writes
  }
}

}  // namespace sdv

using namespace sdv;

extern "C" int sdv_copy_blocks(const void* k_from, const void* v_from, const float* s_from, int32_t from_blocks, void* k_to, void* v_to,
                               float* s_to, int32_t to_blocks, int64_t k_bytes, int64_t v_bytes, int64_t s_bytes, int32_t num_layers,
                               const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  if (!k_from || !v_from || !s_from || !k_to || !v_to || !s_to || !src || !dst) return SDV_ERR_NULL;
  if (from_blocks <= 0 || to_blocks <= 0 || num_layers <= 0 || num_layers > 65535 || n < 0) return SDV_ERR_SHAPE;
  if (k_bytes <= 0 || v_bytes <= 0 || s_bytes <= 0 || k_bytes + v_bytes + s_bytes > (1 << 29)) return SDV_ERR_SHAPE;
  if (k_bytes % 16 || v_bytes % 16 || s_bytes % 16 || !aligned(k_from, 16) || !aligned(v_from, 16) || !aligned(s_from, 16) ||
      !aligned(k_to, 16) || !aligned(v_to, 16) || !aligned(s_to, 16) || !aligned(src, 4) || !aligned(dst, 4))
    return SDV_ERR_ALIGN;
  if (n == 0) return SDV_OK;
  CopyArgs a = {{static_cast<const uint8_t*>(k_from), static_cast<const uint8_t*>(v_from), reinterpret_cast<const uint8_t*>(s_from)},
                {static_cast<uint8_t*>(k_to), static_cast<uint8_t*>(v_to), reinterpret_cast<uint8_t*>(s_to)},
                {(int)k_bytes, (int)v_bytes, (int)s_bytes}, from_blocks, to_blocks, src, dst, n};
  constexpr int most = 1 << 25;  // pairs of a launch, which has fewer than 2^32 threads along x
  for (int64_t first = 0; first < n; first += most) {
    a.src = src + first;
    a.dst = dst + first;
    a.n = (int)(n - first < most ? n - first : most);
    hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)((a.n + kCopyWaves - 1) / kCopyWaves), (unsigned)num_layers),
                       dim3(kCopyWaves * kWave), 0, static_cast<hipStream_t>(stream), a);
  }
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}

extern "C" int sdv_kv8_keep(void* k_pages, void* v_pages, float* scales, int32_t num_blocks, int64_t k_layer_stride,
                            int64_t v_layer_stride, int64_t s_layer_stride, int32_t num_layers, const int32_t* block_table,
                            int32_t max_blocks_per_seq, const int32_t* cu_kept, const int32_t* kept, int32_t total_kept,
                            const int32_t* starts, int32_t batch, int32_t kv_heads, int32_t head_dim, void* stream) {
  if (!k_pages || !v_pages || !scales || !block_table || !cu_kept || !kept || !starts) return SDV_ERR_NULL;
  if (num_blocks <= 0 || num_blocks > INT32_MAX / kBlock || max_blocks_per_seq <= 0 || max_blocks_per_seq > INT32_MAX / kBlock ||
      batch <= 0 || kv_heads <= 0 || kv_heads > 65535 || num_layers <= 0 || num_layers > 65535 || total_kept < 0)
    return SDV_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return SDV_ERR_UNSUPPORTED;
  const int64_t codes = (int64_t)num_blocks * kv_heads * kBlock * head_dim, of_scales = (int64_t)num_blocks * kv_heads * 2 * kBlock;
  if (num_layers > 1 && (k_layer_stride < codes || v_layer_stride < codes || s_layer_stride < of_scales)) return SDV_ERR_SHAPE;
  if (!aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(scales, 16) || k_layer_stride % 16 || v_layer_stride % 16 ||
      s_layer_stride % 4 || !aligned(block_table, 4) || !aligned(cu_kept, 4) || !aligned(kept, 4) || !aligned(starts, 4))
    return SDV_ERR_ALIGN;
  if (total_kept == 0) return SDV_OK;
  KeepArgs a = {{cu_kept, block_table, max_blocks_per_seq, num_blocks, batch, total_kept}, kept, starts,
                static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages), scales, k_layer_stride, v_layer_stride,
                s_layer_stride, kv_heads};
  hipStream_t s = static_cast<hipStream_t>(stream);
  constexpr int most = 1 << 23;  // sequences of a launch, which has fewer than 2^32 threads along x
  for (int64_t first = 0; first < batch; first += most) {
    a.r.cu = cu_kept + first;
    a.r.table = block_table + first * max_blocks_per_seq;
    a.r.batch = (int)(batch - first < most ? batch - first : most);
    a.starts = starts + first;
    const dim3 grid((unsigned)a.r.batch, (unsigned)kv_heads, (unsigned)num_layers);
    if (head_dim == 128)
      hipLaunchKernelGGL((kv8_keep_kernel<128>), grid, dim3(kKeepThreads<128>), 0, s, a);
    else
      hipLaunchKernelGGL((kv8_keep_kernel<64>), grid, dim3(kKeepThreads<64>), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? SDV_OK : SDV_ERR_HIP;
}
