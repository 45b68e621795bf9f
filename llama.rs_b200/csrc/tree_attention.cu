// tree_attention.cu -- attention of the nodes of token trees over a paged KV
// cache (lrs_tree_attention).
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "common.h"
#include "device_common.cuh"
#include "kv.cuh"

namespace lrs {
namespace {

// Four values of row r, columns c.. of a cache tile.
template <int HD, int DT>
__device__ __forceinline__ float4 tile4(const uint8_t* tile, bool is_v, int r, int c) {
  if constexpr (DT == LRS_KV_F32) {
    return *reinterpret_cast<const float4*>(tile + ((size_t)r * HD + c) * 4);
  } else if constexpr (DT == LRS_KV_BF16) {
    const uint2 u = *reinterpret_cast<const uint2*>(tile + ((size_t)r * HD + c) * 2);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u),
                       __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
  } else {
    float x[4];
    const float d = __half2float(*reinterpret_cast<const __half*>(
        tile + (is_v ? q8_v_scale(HD, r, c / 32) : q8_k_scale(HD, r, c / 32))));
    for (int j = 0; j < 4; j++)
      x[j] = d * (float)(int8_t)tile[is_v ? q8_v_code(HD, r, c + j) : q8_k_code(r, c + j)];
    return make_float4(x[0], x[1], x[2], x[3]);
  }
}

// One warp per (node, query head): 32 positions at a time, a lane dots one K
// row with q; the running maximum and sum of the softmax; then the lanes share
// the columns of V.
template <int HD, int DT>
__global__ void __launch_bounds__(128) tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  __shared__ float qs[4][HD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nh = a.c.heads * a.group;
  const long long item = (long long)blockIdx.x * 4 + warp;
  const int node = (int)(item / nh), head = (int)(item % nh);
  if (node >= a.n_nodes) return;
  // the node's tree: the last one that starts at or before it
  int t = -1;
  for (int i = lane; i < a.n_trees; i += 32)
    if (a.start[i] <= node && node < a.start[i + 1]) t = i;
  t = __reduce_max_sync(0xffffffffu, t);
  if (t < 0) return;
  const int s = a.start[t], n = a.start[t + 1] - s, ctx = a.ctx[t], seq = a.seq[t];
  if (n > a.max_nodes || ctx < 0 || (long long)ctx + n > a.max_len || s < 0 || a.start[t + 1] > a.n_nodes) {
    if (lane == 0) atomicExch(a.c.err, kErrCacheIndex);
    return;
  }
  const int i = node - s, len = ctx + n;
  const unsigned long long mask = a.mask ? a.mask[node] : (i == 63 ? ~0ull : (2ull << i) - 1);
  float* q = qs[warp];
  for (int c = lane; c < HD; c += 32) q[c] = a.q[(size_t)node * a.q_ld + (size_t)head * HD + c] * a.scale;
  __syncwarp();
  constexpr size_t TILE = kv_tile_bytes(DT, HD);
  const int kvh = head / a.group;
  constexpr int W = HD / 32;
  float m = -INFINITY, l = 0.0f, o[W] = {};
  for (int p0 = 0; p0 < len; p0 += 32) {
    const int p = p0 + lane;
    const int page = kv_page(a.c, seq, p0);
    if (page < 0) return;
    const bool seen = p < ctx || (p < len && (mask >> (p - ctx) & 1));
    const uint8_t* kt = a.c.k + ((size_t)page * a.c.heads + kvh) * TILE;
    const uint8_t* vt = a.c.v + ((size_t)page * a.c.heads + kvh) * TILE;
    float sc = -INFINITY;
    if (seen) {
      sc = 0.0f;
      for (int c = 0; c < HD; c += 4) {
        const float4 k = tile4<HD, DT>(kt, false, p & (kPageSize - 1), c);
        sc = fmaf(k.x, q[c], fmaf(k.y, q[c + 1], fmaf(k.z, q[c + 2], fmaf(k.w, q[c + 3], sc))));
      }
    }
    float mx = sc;
    for (int w = 16; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    const unsigned live = __ballot_sync(0xffffffffu, seen);
    if (!live) continue;
    const float mn = fmaxf(m, mx);
    const float f = m == -INFINITY ? 0.0f : expf(m - mn);
    const float pr = seen ? expf(sc - mn) : 0.0f;
    float sum = pr;
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    l = l * f + sum;
    m = mn;
    for (int w = 0; w < W; w++) o[w] *= f;
    for (int j = 0; j < 32; j++) {
      if (!(live >> j & 1)) continue;
      const float pj = __shfl_sync(0xffffffffu, pr, j);
      const int r = (p0 + j) & (kPageSize - 1);
      if constexpr (W == 4) {
        const float4 v = tile4<HD, DT>(vt, true, r, lane * 4);
        o[0] = fmaf(pj, v.x, o[0]), o[1] = fmaf(pj, v.y, o[1]);
        o[2] = fmaf(pj, v.z, o[2]), o[3] = fmaf(pj, v.w, o[3]);
      } else {
        const float4 v = tile4<HD, DT>(vt, true, r, lane / 2 * 4);
        o[0] = fmaf(pj, lane & 1 ? v.z : v.x, o[0]);
        o[1] = fmaf(pj, lane & 1 ? v.w : v.y, o[1]);
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int w = 0; w < W; w++)
    a.out[(size_t)node * a.out_ld + (size_t)head * HD + lane * W + w] = o[w] * inv;
}

}  // namespace

size_t tree_attention_workspace_bytes(const TreeArgs&, int, int) { return 0; }

cudaError_t launch_tree_attention(const TreeArgs& a, uint32_t dtype, int hd, int, cudaStream_t st) {
  const long long items = (long long)a.n_nodes * a.c.heads * a.group;
  const unsigned grid = (unsigned)((items + 3) / 4);
  if (hd == 128) {
    if (dtype == LRS_KV_F32) tree_attention_kernel<128, LRS_KV_F32><<<grid, 128, 0, st>>>(a);
    else if (dtype == LRS_KV_BF16) tree_attention_kernel<128, LRS_KV_BF16><<<grid, 128, 0, st>>>(a);
    else tree_attention_kernel<128, LRS_KV_Q8_0><<<grid, 128, 0, st>>>(a);
  } else {
    if (dtype == LRS_KV_F32) tree_attention_kernel<64, LRS_KV_F32><<<grid, 128, 0, st>>>(a);
    else if (dtype == LRS_KV_BF16) tree_attention_kernel<64, LRS_KV_BF16><<<grid, 128, 0, st>>>(a);
    else tree_attention_kernel<64, LRS_KV_Q8_0><<<grid, 128, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace lrs
