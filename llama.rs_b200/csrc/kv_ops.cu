// kv_ops.cu -- writing, reading back and compacting the paged KV cache in its
// own type, and the C entry points of these operators and of the tree
// attention (tree_attention.cu).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "common.h"
#include "device_common.cuh"
#include "internal.h"
#include "kv.cuh"

namespace lrs {
namespace {

constexpr int kStoreWarps = 4;
constexpr int kStoreRows = 32;  // most rows a CTA of the store kernel

__device__ __forceinline__ float4 load4(const float* p, bool vec) {
  if (vec) return *reinterpret_cast<const float4*>(p);
  return make_float4(p[0], p[1], p[2], p[3]);
}

// The Q8_0 code of x under inv = 1 / d (quantize_block_q8_0, src/quant.rs:650-662:
// f32 product, round half away from zero, clamp; NaN, which 0 * inf gives for
// blocks of f32 subnormals, becomes 0).
__device__ __forceinline__ uint32_t q8_code(float x, float inv) {
  const float r = roundf(__fmul_rn(x, inv));
  const int i = r != r ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
  return (uint32_t)i & 0xffu;
}
// Eight codes of a block whose products are finite and below 127.5: the sum with
// 1.5 * 2^23 rounds a product to the nearest integer, ties to even.  False if one
// is an exact tie, which goes away from zero (q8_code).
__device__ __forceinline__ bool q8_codes(const float (&x)[8], float inv, uint32_t (&w)[2]) {
  constexpr float kMagic = 12582912.0f;
  float off = 0.0f;
#pragma unroll
  for (int h = 0; h < 2; h++) {
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      // (scalar products: a packed one may be fused into the sums below)
      const float2 y = make_float2(__fmul_rn(x[4 * h + i], inv), __fmul_rn(x[4 * h + i + 1], inv));
      const float2 s = add2(y, make_float2(kMagic, kMagic));
      const float2 r = add2(s, make_float2(-kMagic, -kMagic));
      const float2 d = add2(y, make_float2(-r.x, -r.y));
      off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
      t[i] = __float_as_uint(s.x), t[i + 1] = __float_as_uint(s.y);
    }
    w[h] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
  }
  return off < 0.5f;
}

// Rows [blockIdx.x * rows, + rows) of K (blockIdx.z = 0) or V (1) of head
// blockIdx.y.  The rows' cells are looked up once, one row a thread; then a lane
// owns eight consecutive columns, and a warp has kBatch rows' loads under way
// before it encodes the first.  Q8_0: four lanes share a block's maximum by shuffles (as
// integers: a NaN or a value past the limit shows there and takes the block to the
// slow form).  V interleaves four positions per word, so the codes of the
// CTA's rows meet in shared memory and leave as 16-byte stores wherever four
// consecutive rows are four aligned positions of one slot, and as single bytes
// elsewhere (a decode step's rows, the ends of a run): byte stores never touch a
// neighbouring position.
// 65,536 rows of 4 heads x 128, L2 flushed before: into f32 93 us and bf16 70 us, both 5.8
// TB/s of what is read and written and near DRAM's rate; into q8_0 86 us, 4.0 TB/s, bound
// by the encoding's instructions (the schedulers issue in 74 of 100 cycles, DRAM is at
// 48 %).  A decode step's rows are the launch and the lookups (5 us together with the load).
constexpr int kBatch = 2;

template <int HD, int DT>
__global__ void __launch_bounds__(32 * kStoreWarps)
    kv_store_kernel(const __grid_constant__ KvStoreArgs a, int rows, bool vec) {
  constexpr int LPR = HD / 8, RPW = 32 / LPR;  // lanes a row, rows a warp
  __shared__ uint2 codes[kStoreRows][LPR];
  __shared__ int row_page[kStoreRows], row_seq[kStoreRows], row_pos[kStoreRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const long long i0 = (long long)blockIdx.x * rows;
  const int cnt = (int)min((long long)rows, a.n - i0);
  const float* src = (is_v ? a.v : a.k) + (size_t)i0 * a.ld + (size_t)head * HD;
  uint8_t* pool = is_v ? a.c.v : a.c.k;
  constexpr size_t TILE = kv_tile_bytes(DT, HD);
  const int ln = lane % LPR, col = ln * 8;
  constexpr int kStep = kStoreWarps * RPW;  // rows that the warps take at once
  float4 f[kBatch][2];
  auto load = [&](int r0) {
#pragma unroll
    for (int b = 0; b < kBatch; b++) {
      const int r = r0 + b * kStep;
#pragma unroll
      for (int h = 0; h < 2; h++)
        f[b][h] = r < cnt ? load4(src + (size_t)r * a.ld + col + h * 4, vec) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
  };
  const int mine = warp * RPW + lane / LPR;
  load(mine);
  if (threadIdx.x < cnt) {
    const int seq = a.seq[i0 + threadIdx.x], pos = a.pos[i0 + threadIdx.x];
    row_seq[threadIdx.x] = seq;
    row_pos[threadIdx.x] = pos;
    row_page[threadIdx.x] = kv_page(a.c, seq, pos);
  }
  __syncthreads();
  for (int r0 = mine; r0 - mine < cnt; r0 += kBatch * kStep) {
    if (r0 != mine) load(r0);
#pragma unroll
    for (int bt = 0; bt < kBatch; bt++) {
      const int r = r0 + bt * kStep;
      const bool live = r < cnt;
      const int page = live ? row_page[r] : -1, pr = live ? row_pos[r] & (kPageSize - 1) : 0;
      float x[8] = {f[bt][0].x, f[bt][0].y, f[bt][0].z, f[bt][0].w, f[bt][1].x, f[bt][1].y, f[bt][1].z, f[bt][1].w};
      uint8_t* tile = pool + ((size_t)max(page, 0) * a.c.heads + head) * TILE;
      if constexpr (DT == LRS_KV_F32) {
        if (page >= 0) {
          float4* o = reinterpret_cast<float4*>(tile + ((size_t)pr * HD + col) * 4);
          o[0] = f[bt][0];
          o[1] = f[bt][1];
        }
      } else if constexpr (DT == LRS_KV_BF16) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&p);
        }
        if (page >= 0)
          *reinterpret_cast<uint4*>(tile + ((size_t)pr * HD + col) * 2) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        int mb = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) mb = max(mb, __float_as_int(x[i]) & 0x7fffffff);
        mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
        mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 2));
        float m = __int_as_float(mb);
        // the block of ordinary values: none past the limit, 1 / d finite
        const bool plain = mb <= __float_as_int(kQ8Limit) && (mb == 0 || m > 1e-30f);
        if (!plain) {
          float mx = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; i++) {
            x[i] = x[i] != x[i] ? 0.0f : fminf(fmaxf(x[i], -kQ8Limit), kQ8Limit);
            mx = fmaxf(mx, fabsf(x[i]));
          }
          const uint32_t four = 0xfu << (lane & 28);  // the block's lanes are here together
          mx = fmaxf(mx, __shfl_xor_sync(four, mx, 1));
          m = fmaxf(mx, __shfl_xor_sync(four, mx, 2));
        }
        const float d = __fdiv_rn(m, 127.0f);
        const float inv = d == 0.0f ? 0.0f : __fdiv_rn(1.0f, d);
        uint32_t w[2];
        if (!q8_codes(x, inv, w) || !plain) {
          w[0] = w[1] = 0;
#pragma unroll
          for (int i = 0; i < 8; i++) w[i / 4] |= q8_code(x[i], inv) << (8 * (i % 4));
        }
        if (page >= 0) {
          if ((lane & 3) == 0)
            *reinterpret_cast<__half*>(tile + (is_v ? q8_v_scale(HD, pr, col / 32) : q8_k_scale(HD, pr, col / 32))) =
                __float2half_rn(d);
          if (!is_v) *reinterpret_cast<uint2*>(tile + q8_k_code(pr, col)) = make_uint2(w[0], w[1]);
        }
        if (is_v && live) codes[r][ln] = make_uint2(w[0], w[1]);
      }
    }
  }
  if constexpr (DT == LRS_KV_Q8_0) {
    if (!is_v) return;
    __syncthreads();
    for (int r = mine; r < cnt; r += kStep) {
      if (row_page[r] < 0) continue;
      const int pos = row_pos[r], g = r - (pos & 3);  // first row of the aligned group
      bool full = g >= 0 && g + 3 < cnt;
      for (int i = 0; i < 4 && full; i++)
        full = row_seq[g + i] == row_seq[r] && row_pos[g + i] == (pos & ~3) + i;
      if (full && g != r) continue;  // row g writes the group
      const int pr = pos & (kPageSize - 1);
      uint8_t* tile = pool + ((size_t)row_page[r] * a.c.heads + head) * TILE;
#pragma unroll
      for (int h = 0; h < 2; h++) {  // four columns each
        const int c4 = col + 4 * h;
        if (full) {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; i++) w[i] = h ? codes[g + i][ln].y : codes[g + i][ln].x;
          const uint32_t a0 = __byte_perm(w[0], w[1], 0x5140), a1 = __byte_perm(w[2], w[3], 0x5140);
          const uint32_t b0 = __byte_perm(w[0], w[1], 0x7362), b1 = __byte_perm(w[2], w[3], 0x7362);
          *reinterpret_cast<uint4*>(tile + q8_v_code(HD, pr, c4)) =
              make_uint4(__byte_perm(a0, a1, 0x5410), __byte_perm(a0, a1, 0x7632),
                         __byte_perm(b0, b1, 0x5410), __byte_perm(b0, b1, 0x7632));
        } else {
          const uint32_t w = h ? codes[r][ln].y : codes[r][ln].x;
#pragma unroll
          for (int i = 0; i < 4; i++) tile[q8_v_code(HD, pr, c4 + i)] = (uint8_t)(w >> (8 * i));
        }
      }
    }
  }
}

// The inverse.  A CTA has kLoadRows consecutive rows of K or V, all heads: the
// rows' cells are looked up once; then a thread takes four columns of a (row, head)
// at a time, kLoadBatch of them under way together, neighbouring threads writing
// neighbouring heads of a row.  The lines that four positions share (V codes, K's
// 16-byte chunks) come from L2 once.  65,536 rows of 4 heads x 128, L2 flushed before:
// from f32 92 us, 5.8 TB/s, near DRAM's rate; from q8_0 82 us, 4.2 TB/s, bound by
// instructions (66 of 100 cycles issue, DRAM 45 %); from bf16 94 us, 4.3 TB/s, waiting for
// its loads (15 of a warp's 23 cycles an instruction), of 8 bytes a lane where f32's are 16.
constexpr int kLoadRows = 32, kLoadThreads = 256, kLoadBatch = 4;

template <int HD, int DT>
__global__ void __launch_bounds__(kLoadThreads)
    kv_load_kernel(const __grid_constant__ KvLoadArgs a, int rows, bool vec) {
  constexpr int LPR = HD / 4, kStep = kLoadThreads / LPR;  // (row, head) pairs at once
  __shared__ int row_page[kLoadRows], row_in[kLoadRows];
  const bool is_v = blockIdx.y != 0;
  float* dst = is_v ? a.v : a.k;
  const long long i0 = (long long)blockIdx.x * rows;
  const int cnt = (int)min((long long)rows, a.n - i0);
  if (!dst) return;
  if (threadIdx.x < cnt) {
    const int pos = a.pos[i0 + threadIdx.x];
    row_page[threadIdx.x] = kv_page(a.c, a.seq[i0 + threadIdx.x], pos);
    row_in[threadIdx.x] = pos & (kPageSize - 1);
  }
  __syncthreads();
  constexpr size_t TILE = kv_tile_bytes(DT, HD);
  const uint8_t* pool = is_v ? a.c.v : a.c.k;
  const int heads = a.c.heads, col = (threadIdx.x % LPR) * 4;
  int row = threadIdx.x / LPR / heads, head = threadIdx.x / LPR % heads;
  while (row < cnt) {
    uint4 raw[kLoadBatch];
    __half d[kLoadBatch];
    int in[kLoadBatch];
    float* out[kLoadBatch];  // null: no such row
#pragma unroll
    for (int b = 0; b < kLoadBatch; b++) {
      out[b] = nullptr;
      if (row < cnt && row_page[row] >= 0) {
        const int pr = row_in[row];
        const uint8_t* t = pool + ((size_t)row_page[row] * heads + head) * TILE;
        in[b] = pr;
        out[b] = dst + (size_t)(i0 + row) * a.ld + (size_t)head * HD + col;
        if constexpr (DT == LRS_KV_F32) {
          raw[b] = *reinterpret_cast<const uint4*>(t + ((size_t)pr * HD + col) * 4);
        } else if constexpr (DT == LRS_KV_BF16) {
          const uint2 u = *reinterpret_cast<const uint2*>(t + ((size_t)pr * HD + col) * 2);
          raw[b] = make_uint4(u.x << 16, u.x & 0xffff0000u, u.y << 16, u.y & 0xffff0000u);
        } else if (is_v) {
          raw[b] = *reinterpret_cast<const uint4*>(t + q8_v_code(HD, pr & ~3, col));
          d[b] = *reinterpret_cast<const __half*>(t + q8_v_scale(HD, pr, col / 32));
        } else {
          raw[b].x = *reinterpret_cast<const uint32_t*>(t + q8_k_code(pr, col));
          d[b] = *reinterpret_cast<const __half*>(t + q8_k_scale(HD, pr, col / 32));
        }
      }
      for (head += kStep; head >= heads; head -= heads) row++;
    }
#pragma unroll
    for (int b = 0; b < kLoadBatch; b++) {
      if (!out[b]) continue;
      uint4 v = raw[b];
      if constexpr (DT == LRS_KV_Q8_0) {
        const float f = __half2float(d[b]);
        // K: the four bytes of a word; V: byte (position % 4) of four words
        uint32_t w = v.x;
        if (is_v) {
          const uint32_t at = in[b] & 3, sel = at | (at + 4) << 4;
          w = __byte_perm(__byte_perm(v.x, v.y, sel), __byte_perm(v.z, v.w, sel), 0x5410);
        }
        v = make_uint4(__float_as_uint(__fmul_rn(f, (float)(int8_t)w)),
                       __float_as_uint(__fmul_rn(f, (float)(int8_t)(w >> 8))),
                       __float_as_uint(__fmul_rn(f, (float)(int8_t)(w >> 16))),
                       __float_as_uint(__fmul_rn(f, (float)(int8_t)(w >> 24))));
      }
      if (vec) {
        __stcs(reinterpret_cast<uint4*>(out[b]), v);
      } else {
        out[b][0] = __uint_as_float(v.x), out[b][1] = __uint_as_float(v.y);
        out[b][2] = __uint_as_float(v.z), out[b][3] = __uint_as_float(v.w);
      }
    }
  }
}

// ---- accept ---------------------------------------------------------------
constexpr int kAcceptCaches = 128;  // pools in one launch's parameters

struct AcceptArgs {
  KvView c;  // pools unused
  uint8_t* k[kAcceptCaches];
  uint8_t* v[kAcceptCaches];
  int n_caches;
  const int* seq;
  const int* ctx;
  const int* start;
  const int* nodes;
  int n_trees, n_nodes;
};

// One warp moves the path's rows of one (tree, cache, head, K or V).  The path
// ascends, so row j's target ctx + j is at or below its source and below every
// later source: rows move in chunks, each chunk read whole before it is
// written, and no chunk overwrites a row that a later one reads.  Bound by the chain
// of lookups and by DRAM: 28 bf16 caches x 64 trees, 4 heads x 128, 12 nodes drafted:
// 14 us, a warp to each (tree, cache, head, K or V).  One warp for a tree's lookups and
// several caches took as long.
template <int HD, int DT>
__global__ void __launch_bounds__(128) kv_accept_kernel(const __grid_constant__ AcceptArgs a) {
  const int lane = threadIdx.x & 31;
  long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const bool is_v = item & 1;
  item >>= 1;
  const int head = (int)(item % a.c.heads);
  item /= a.c.heads;
  const int cache = (int)(item % a.n_caches), t = (int)(item / a.n_caches);
  if (t >= a.n_trees) return;
  const int s = a.start[t], end = a.start[t + 1], ctx = a.ctx[t], seq = a.seq[t];
  if (s == end) return;
  // (compared, not subtracted: the difference of two arbitrary values may overflow)
  bool ok = s >= 0 && end > s && end <= a.n_nodes && end - s <= LRS_TREE_MAX_NODES && seq >= 0 &&
            seq < a.c.n_seqs && ctx >= 0 &&
            ctx <= (int)min((long long)a.c.max_pages * kPageSize, (long long)INT_MAX) - 1;
  const int n = ok ? end - s : 0;
  int node0 = -1, node1 = -1;  // of rows `lane` and `lane + 32`
  if (ok) {
    if (lane < n) node0 = a.nodes[s + lane];
    if (lane + 32 < n) node1 = a.nodes[s + lane + 32];
  }
  const int prev0 = __shfl_up_sync(0xffffffffu, node0, 1), top0 = __shfl_sync(0xffffffffu, node0, 31);
  int prev1 = __shfl_up_sync(0xffffffffu, node1, 1);
  if (lane == 0) prev1 = top0;
  if (lane < n) ok = ok && node0 >= 0 && node0 < LRS_TREE_MAX_NODES && (lane == 0 || node0 > prev0);
  if (lane + 32 < n) ok = ok && node1 < LRS_TREE_MAX_NODES && node1 > prev1;
  ok = __all_sync(0xffffffffu, ok);
  int page0 = -1, page1 = -1;  // of ctx, and of the page after it
  if (ok) {
    const int last = __reduce_max_sync(0xffffffffu, max(node0, node1));
    page0 = kv_page(a.c, seq, ctx);
    ok = page0 >= 0;
    if (ok && ctx % kPageSize + last >= kPageSize) {
      page1 = kv_page(a.c, seq, ctx - ctx % kPageSize + kPageSize);
      ok = page1 >= 0;
    }
  }
  if (!ok) {
    if (lane == 0) atomicMax(a.c.err, kErrCacheIndex);
    return;
  }
  uint8_t* pool = is_v ? a.v[cache] : a.k[cache];
  constexpr size_t TILE = kv_tile_bytes(DT, HD);
  // row at `off` positions past ctx: its tile and its row in the page
  auto cell = [&](int off, int* r) {
    const int p = ctx % kPageSize + off;
    *r = p & (kPageSize - 1);
    return pool + ((size_t)(p < kPageSize ? page0 : page1) * a.c.heads + head) * TILE;
  };
  auto node_of = [&](int j) {
    const int lo = __shfl_sync(0xffffffffu, node0, j & 31), hi = __shfl_sync(0xffffffffu, node1, j & 31);
    return j < 32 ? lo : hi;
  };
  if constexpr (DT != LRS_KV_Q8_0) {
    constexpr int ROWB = HD * (DT == LRS_KV_BF16 ? 2 : 4), VPR = ROWB / 16;  // vectors a row
    constexpr int CH = 8;                                                    // vectors a lane
    for (int v0 = 0; v0 < n * VPR; v0 += 32 * CH) {
      uint4 x[CH];
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int e = v0 + 32 * c + lane, j = min(e / VPR, n - 1);
        int r;
        const uint8_t* t0 = cell(node_of(j), &r);
        if (e < n * VPR) x[c] = *reinterpret_cast<const uint4*>(t0 + (size_t)r * ROWB + e % VPR * 16);
      }
      __syncwarp();
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int e = v0 + 32 * c + lane;
        int r;
        uint8_t* t1 = cell(e / VPR, &r);
        if (e < n * VPR) *reinterpret_cast<uint4*>(t1 + (size_t)r * ROWB + e % VPR * 16) = x[c];
      }
      __syncwarp();
    }
  } else {
    constexpr int WPR = HD / 4, BPR = HD / 32;  // words of codes, scales of a row
    constexpr int CH = 8;
    for (int v0 = 0; v0 < n * WPR; v0 += 32 * CH) {
      uint32_t x[CH];
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int e = v0 + 32 * c + lane, j = min(e / WPR, n - 1), col = e % WPR * 4;
        int r;
        const uint8_t* t0 = cell(node_of(j), &r);
        if (e < n * WPR) {
          if (is_v) {
            x[c] = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) x[c] |= (uint32_t)t0[q8_v_code(HD, r, col + i)] << (8 * i);
          } else {
            x[c] = *reinterpret_cast<const uint32_t*>(t0 + q8_k_code(r, col));
          }
        }
      }
      __syncwarp();
#pragma unroll
      for (int c = 0; c < CH; c++) {
        const int e = v0 + 32 * c + lane, col = e % WPR * 4;
        int r;
        uint8_t* t1 = cell(e / WPR, &r);
        if (e < n * WPR) {
          if (is_v) {
#pragma unroll
            for (int i = 0; i < 4; i++) t1[q8_v_code(HD, r, col + i)] = (uint8_t)(x[c] >> (8 * i));
          } else {
            *reinterpret_cast<uint32_t*>(t1 + q8_k_code(r, col)) = x[c];
          }
        }
      }
      __syncwarp();
    }
    for (int v0 = 0; v0 < n * BPR; v0 += 32) {  // the scales: whole rows per pass
      const int e = v0 + lane, j = min(e / BPR, n - 1), b = e % BPR;
      int r;
      const uint8_t* t0 = cell(node_of(j), &r);
      uint16_t d = 0;
      if (e < n * BPR)
        d = *reinterpret_cast<const uint16_t*>(t0 + (is_v ? q8_v_scale(HD, r, b) : q8_k_scale(HD, r, b)));
      __syncwarp();
      uint8_t* t1 = cell(j, &r);
      if (e < n * BPR)
        *reinterpret_cast<uint16_t*>(t1 + (is_v ? q8_v_scale(HD, r, b) : q8_k_scale(HD, r, b))) = d;
      __syncwarp();
    }
  }
}

// Calls f<HD, DT>() of the cache's head_dim and type.
#define LRS_KV_DISPATCH(hd, dtype, CALL)                                      \
  do {                                                                        \
    if ((hd) == 128) {                                                        \
      if ((dtype) == LRS_KV_F32) { CALL(128, LRS_KV_F32); }                   \
      else if ((dtype) == LRS_KV_BF16) { CALL(128, LRS_KV_BF16); }            \
      else { CALL(128, LRS_KV_Q8_0); }                                        \
    } else {                                                                  \
      if ((dtype) == LRS_KV_F32) { CALL(64, LRS_KV_F32); }                    \
      else if ((dtype) == LRS_KV_BF16) { CALL(64, LRS_KV_BF16); }             \
      else { CALL(64, LRS_KV_Q8_0); }                                         \
    }                                                                         \
  } while (0)

}  // namespace

cudaError_t launch_kv_store(const KvStoreArgs& a, uint32_t dtype, int hd, int sms, cudaStream_t st) {
  // few rows: four a CTA, so that the step's rows spread over the SMs (64 rows stored
  // and loaded: 12.9 us against 16.6 with 32; 65,536 rows: 395 us with four, 158 with 32)
  const long long big = (a.n + kStoreRows - 1) / kStoreRows * a.c.heads * 2;
  const int rows = big >= 4ll * sms ? kStoreRows : 4;
  const bool vec = a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.k) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
  const dim3 grid((unsigned)((a.n + rows - 1) / rows), a.c.heads, 2);
#define LRS_CALL(HD, DT) kv_store_kernel<HD, DT><<<grid, 32 * kStoreWarps, 0, st>>>(a, rows, vec)
  LRS_KV_DISPATCH(hd, dtype, LRS_CALL);
#undef LRS_CALL
  return cudaGetLastError();
}

cudaError_t launch_kv_load(const KvLoadArgs& a, uint32_t dtype, int hd, int sms, cudaStream_t st) {
  // few rows: fewer a CTA, so that they spread over the SMs (65,536 rows: 139 us with
  // four, 77 with 32)
  const long long big = (a.n + kLoadRows - 1) / kLoadRows * 2;
  const int rows = big >= 4ll * sms ? kLoadRows : 4;
  const bool vec = a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.k) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(a.v) % 16 == 0;
  const dim3 grid((unsigned)((a.n + rows - 1) / rows), 2);
#define LRS_CALL(HD, DT) kv_load_kernel<HD, DT><<<grid, kLoadThreads, 0, st>>>(a, rows, vec)
  LRS_KV_DISPATCH(hd, dtype, LRS_CALL);
#undef LRS_CALL
  return cudaGetLastError();
}

}  // namespace lrs

using namespace lrs;

namespace {

// The backend's device for the length of a call.
class OnDevice {
 public:
  explicit OnDevice(int device) {
    err = cudaGetDevice(&was_);
    if (err == cudaSuccess && was_ != device) {
      err = cudaSetDevice(device);
      moved_ = err == cudaSuccess;
    }
  }
  ~OnDevice() {
    if (moved_) cudaSetDevice(was_);
  }
  cudaError_t err;

 private:
  int was_ = 0;
  bool moved_ = false;
};

int32_t cuda_status(cudaError_t e, const char* what) {
  return e == cudaSuccess ? (int32_t)LRS_OK
                          : fail(LRS_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

KvView view_of(const lrs_kv_cache& c, int* err) {
  return KvView{static_cast<uint8_t*>(c.k_pool), static_cast<uint8_t*>(c.v_pool), c.pages,
                (int)c.n_pages, (int)c.n_seqs, (int)c.max_pages, (int)c.kv_heads, err};
}

// A device array of T, or null.
template <typename T>
bool aligned(const T* p) {
  return reinterpret_cast<uintptr_t>(p) % sizeof(T) == 0;
}
int32_t unaligned(const char* what) {
  return fail(LRS_ERR_INVALID, std::string(what) + ": an array is not aligned to its values");
}

// `n` rows `ld` floats apart lie in the address space (a negative stride of a
// language with signed sizes arrives as one that does not).
bool stride_fits(size_t n, size_t ld) { return n == 0 || ld <= ((size_t)1 << 45) / n; }
int32_t bad_stride(const char* what, size_t ld) {
  return fail(LRS_ERR_INVALID, std::string(what) + ": rows " + std::to_string(ld) + " values apart exceed the address space");
}

int32_t check_rows(const lrs_kv_cache* c, size_t n, size_t* ld, const char* what) {
  int32_t rc = lrs_kv_check(c, nullptr);
  if (rc) return rc;
  const size_t width = (size_t)c->kv_heads * c->head_dim;
  if (*ld == 0) *ld = width;
  if (*ld < width)
    return fail(LRS_ERR_INVALID, std::string(what) + ": row stride " + std::to_string(*ld) +
                                     " is below the row's " + std::to_string(width) + " values");
  if (n > (size_t)INT_MAX) return fail(LRS_ERR_INVALID, std::string(what) + ": too many rows");
  if (!stride_fits(n, *ld)) return bad_stride(what, *ld);
  return LRS_OK;
}

int32_t check_trees(const lrs_kv_cache* c, const lrs_tree_batch* t, uint32_t n_heads) {
  int32_t rc = lrs_kv_check(c, nullptr);
  if (rc) return rc;
  if (!t) return fail(LRS_ERR_INVALID, "null tree batch");
  if (n_heads == 0 || n_heads % c->kv_heads)
    return fail(LRS_ERR_INVALID, "n_heads must be a positive multiple of kv_heads");
  if (n_heads / c->kv_heads > 64)
    return fail(LRS_ERR_UNSUPPORTED, "tree attention supports up to 64 query heads per KV head");
  if (t->n_trees == 0 || t->n_nodes == 0) return LRS_OK;
  if (!t->seq || !t->ctx || !t->start) return fail(LRS_ERR_INVALID, "null tree array");
  if (t->max_nodes == 0 || t->max_nodes > LRS_TREE_MAX_NODES)
    return fail(LRS_ERR_INVALID, "max_nodes must be in 1..=" + std::to_string(LRS_TREE_MAX_NODES));
  if (!aligned(t->seq) || !aligned(t->ctx) || !aligned(t->start) || !aligned(t->mask)) return unaligned("tree batch");
  if (t->max_len == 0 || t->max_len > (uint64_t)c->max_pages * LRS_KV_PAGE)
    return fail(LRS_ERR_INVALID, "max_len " + std::to_string(t->max_len) +
                                     " is outside the slots' " + std::to_string(c->max_pages) + " pages");
  // the kernels number the batch's tiles (128 positions by 16 rows at least) and
  // the positions of whole tiles in int32
  const uint64_t rows = ((uint64_t)t->max_nodes * (n_heads / c->kv_heads) + 15) / 16,
                 tiles = ((uint64_t)t->max_len + 127) / 128;
  if (t->n_trees > 65535u || t->n_nodes > (1u << 24) || t->max_len > (uint32_t)INT_MAX - 128u ||
      rows * tiles > (uint64_t)INT_MAX / ((uint64_t)t->n_trees * c->kv_heads))
    return fail(LRS_ERR_UNSUPPORTED, "too many trees, nodes or positions");
  return LRS_OK;
}

TreeArgs tree_args(const lrs_kv_cache& c, const lrs_tree_batch& t, uint32_t n_heads, int* err) {
  TreeArgs a{};
  a.c = view_of(c, err);
  a.seq = t.seq;
  a.ctx = t.ctx;
  a.start = t.start;
  a.mask = reinterpret_cast<const unsigned long long*>(t.mask);
  a.n_trees = (int)t.n_trees;
  a.n_nodes = (int)t.n_nodes;
  a.max_nodes = (int)t.max_nodes;
  a.max_len = (int)t.max_len;
  a.group = (int)(n_heads / c.kv_heads);
  return a;
}

}  // namespace

int32_t lrs::kv_accept(lrs_backend* be, const lrs_kv_cache* caches, size_t n_caches, const int32_t* d_seq,
                       const int32_t* d_ctx, const int32_t* d_start, const int32_t* d_nodes, size_t n_trees,
                       size_t n_nodes, int err_word, void* stream) {
  if (n_caches && !caches) return fail(LRS_ERR_INVALID, "null cache");
  int32_t rc;
  for (size_t i = 0; i < n_caches; i++) {
    if ((rc = lrs_kv_check(&caches[i], nullptr))) return rc;
    const lrs_kv_cache &x = caches[i], &y = caches[0];
    if (x.pages != y.pages || x.n_pages != y.n_pages || x.n_seqs != y.n_seqs ||
        x.max_pages != y.max_pages || x.kv_heads != y.kv_heads || x.head_dim != y.head_dim ||
        x.kv_dtype != y.kv_dtype)
      return fail(LRS_ERR_INVALID, "lrs_kv_accept: the caches may differ in their pools only");
  }
  if (n_trees > (size_t)INT_MAX || n_nodes > (size_t)INT_MAX)
    return fail(LRS_ERR_INVALID, "lrs_kv_accept: too many trees or nodes");
  if (n_caches == 0 || n_trees == 0 || n_nodes == 0) return LRS_OK;
  // a pool named twice would be compacted by two warps at once
  for (size_t i = 0; i < n_caches; i++)
    for (size_t j = 0; j <= i; j++)
      if ((j < i && (caches[i].k_pool == caches[j].k_pool || caches[i].v_pool == caches[j].v_pool)) ||
          caches[i].k_pool == caches[j].v_pool || caches[i].v_pool == caches[j].k_pool)
        return fail(LRS_ERR_INVALID, "lrs_kv_accept: a pool is named twice");
  if (!be || !d_seq || !d_ctx || !d_start || !d_nodes) return fail(LRS_ERR_INVALID, "null argument");
  if (!aligned(d_seq) || !aligned(d_ctx) || !aligned(d_start) || !aligned(d_nodes)) return unaligned("lrs_kv_accept");
  const size_t per_cache = n_trees * caches[0].kv_heads * 2;
  if (per_cache > (size_t)INT_MAX) return fail(LRS_ERR_INVALID, "lrs_kv_accept: too many trees or nodes");
  OnDevice on(be->device);
  if (on.err != cudaSuccess) return cuda_status(on.err, "cudaSetDevice");
  cudaStream_t st = stream ? (cudaStream_t)stream : be->stream;
  const size_t most = std::max<size_t>(1, std::min<size_t>(kAcceptCaches, (size_t)INT_MAX / per_cache));
  for (size_t c0 = 0; c0 < n_caches; c0 += most) {
    AcceptArgs a{};
    a.c = view_of(caches[0], be->d_err + err_word);
    a.n_caches = (int)std::min(most, n_caches - c0);
    for (int i = 0; i < a.n_caches; i++) {
      a.k[i] = static_cast<uint8_t*>(caches[c0 + i].k_pool);
      a.v[i] = static_cast<uint8_t*>(caches[c0 + i].v_pool);
    }
    a.seq = d_seq;
    a.ctx = d_ctx;
    a.start = d_start;
    a.nodes = d_nodes;
    a.n_trees = (int)n_trees;
    a.n_nodes = (int)n_nodes;
    const unsigned grid = (unsigned)((per_cache * a.n_caches + 3) / 4);
#define LRS_CALL(HD, DT) kv_accept_kernel<HD, DT><<<grid, 128, 0, st>>>(a)
    LRS_KV_DISPATCH(caches[0].head_dim, caches[0].kv_dtype, LRS_CALL);
#undef LRS_CALL
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_status(e, "lrs_kv_accept");
  }
  return LRS_OK;
}

extern "C" {

lrs_status lrs_kv_check(const lrs_kv_cache* c, size_t* tile_bytes) try {
  if (!c) return fail(LRS_ERR_INVALID, "null cache");
  if (c->kv_dtype > LRS_KV_Q8_0)
    return fail(LRS_ERR_UNSUPPORTED, "unknown KV cache type " + std::to_string(c->kv_dtype));
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(LRS_ERR_UNSUPPORTED, "the KV cache operators support head_dim 64 or 128");
  if (!c->n_pages || !c->n_seqs || !c->max_pages || !c->kv_heads)
    return fail(LRS_ERR_INVALID, "KV cache: pages, slots and heads must be non-zero");
  // positions and page numbers are int32 on the device; heads are a grid dimension
  if (c->n_pages > (uint32_t)INT_MAX || c->n_seqs > (uint32_t)INT_MAX ||
      c->max_pages > (uint32_t)INT_MAX / LRS_KV_PAGE || c->kv_heads > 65535u)
    return fail(LRS_ERR_INVALID, "KV cache: too many pages, slots or heads");
  if (!c->k_pool || !c->v_pool || !c->pages) return fail(LRS_ERR_INVALID, "KV cache: null pool or page table");
  if (reinterpret_cast<uintptr_t>(c->k_pool) % 16 || reinterpret_cast<uintptr_t>(c->v_pool) % 16)
    return fail(LRS_ERR_INVALID, "KV cache: pools must be 16-byte aligned");
  if (!aligned(c->pages)) return unaligned("KV cache");
  if (tile_bytes) *tile_bytes = kv_tile_bytes(c->kv_dtype, (int)c->head_dim);
  return LRS_OK;
} catch (...) {
  return lrs::status_of_current_exception();
}

lrs_status lrs_kv_store(lrs_backend* be, const lrs_kv_cache* c, const int32_t* d_seq,
                        const int32_t* d_pos, size_t n, const float* d_k, const float* d_v,
                        size_t ld, void* stream) try {
  int32_t rc = check_rows(c, n, &ld, "lrs_kv_store");
  if (rc) return rc;
  if (n == 0) return LRS_OK;
  if (!be || !d_seq || !d_pos || !d_k || !d_v) return fail(LRS_ERR_INVALID, "null argument");
  if (!aligned(d_seq) || !aligned(d_pos) || !aligned(d_k) || !aligned(d_v)) return unaligned("lrs_kv_store");
  OnDevice on(be->device);
  if (on.err != cudaSuccess) return cuda_status(on.err, "cudaSetDevice");
  KvStoreArgs a{view_of(*c, be->d_err + kErrQueued), d_seq, d_pos, (long long)n, d_k, d_v, (long long)ld};
  return cuda_status(launch_kv_store(a, c->kv_dtype, (int)c->head_dim, be->sms,
                                     stream ? (cudaStream_t)stream : be->stream),
                     "lrs_kv_store");
} catch (...) {
  return lrs::status_of_current_exception();
}

lrs_status lrs_kv_load(lrs_backend* be, const lrs_kv_cache* c, const int32_t* d_seq,
                       const int32_t* d_pos, size_t n, float* d_k, float* d_v, size_t ld,
                       void* stream) try {
  int32_t rc = check_rows(c, n, &ld, "lrs_kv_load");
  if (rc) return rc;
  if (n == 0 || (!d_k && !d_v)) return LRS_OK;
  if (!be || !d_seq || !d_pos) return fail(LRS_ERR_INVALID, "null argument");
  if (!aligned(d_seq) || !aligned(d_pos) || !aligned(d_k) || !aligned(d_v)) return unaligned("lrs_kv_load");
  OnDevice on(be->device);
  if (on.err != cudaSuccess) return cuda_status(on.err, "cudaSetDevice");
  KvLoadArgs a{view_of(*c, be->d_err + kErrQueued), d_seq, d_pos, (long long)n, d_k, d_v, (long long)ld};
  return cuda_status(launch_kv_load(a, c->kv_dtype, (int)c->head_dim, be->sms,
                                    stream ? (cudaStream_t)stream : be->stream),
                     "lrs_kv_load");
} catch (...) {
  return lrs::status_of_current_exception();
}

lrs_status lrs_kv_accept(lrs_backend* be, const lrs_kv_cache* caches, size_t n_caches,
                         const int32_t* d_seq, const int32_t* d_ctx, const int32_t* d_start,
                         const int32_t* d_nodes, size_t n_trees, size_t n_nodes, void* stream) try {
  return kv_accept(be, caches, n_caches, d_seq, d_ctx, d_start, d_nodes, n_trees, n_nodes,
                   kErrQueued, stream);
} catch (...) {
  return lrs::status_of_current_exception();
}

lrs_status lrs_tree_attention_workspace(const lrs_backend* be, const lrs_kv_cache* c,
                                        const lrs_tree_batch* t, uint32_t n_heads, size_t* bytes) try {
  int32_t rc = check_trees(c, t, n_heads);
  if (rc) return rc;
  if (!bytes) return fail(LRS_ERR_INVALID, "null argument");
  if (!be) return fail(LRS_ERR_INVALID, "null backend");
  *bytes = tree_attention_workspace_bytes(tree_args(*c, *t, n_heads, nullptr), (int)c->head_dim, be->sms);
  return LRS_OK;
} catch (...) {
  return lrs::status_of_current_exception();
}

lrs_status lrs_tree_attention(lrs_backend* be, const lrs_kv_cache* c, const lrs_tree_batch* t,
                              const float* d_q, size_t q_ld, float* d_out, size_t out_ld,
                              uint32_t n_heads, float scale, void* d_workspace,
                              size_t workspace_bytes, void* stream) try {
  int32_t rc = check_trees(c, t, n_heads);
  if (rc) return rc;
  const size_t width = (size_t)n_heads * c->head_dim;
  if (q_ld == 0) q_ld = width;
  if (out_ld == 0) out_ld = width;
  if (q_ld < width || out_ld < width)
    return fail(LRS_ERR_INVALID, "lrs_tree_attention: row stride below the row's " + std::to_string(width) + " values");
  if (!stride_fits(t->n_nodes, std::max(q_ld, out_ld))) return bad_stride("lrs_tree_attention", std::max(q_ld, out_ld));
  if (!std::isfinite(scale)) return fail(LRS_ERR_INVALID, "lrs_tree_attention: scale must be finite");
  if (t->n_trees == 0 || t->n_nodes == 0) return LRS_OK;
  // (a row is read before any CTA writes it only where both have the same place)
  if (d_q && d_out == d_q && q_ld != out_ld)
    return fail(LRS_ERR_INVALID, "lrs_tree_attention: out that is q must have q's row stride");
  if (!be || !d_q || !d_out) return fail(LRS_ERR_INVALID, "null argument");
  if (!aligned(d_q) || !aligned(d_out)) return unaligned("lrs_tree_attention");
  TreeArgs a = tree_args(*c, *t, n_heads, be->d_err + kErrQueued);
  const size_t need = tree_attention_workspace_bytes(a, (int)c->head_dim, be->sms);
  if (workspace_bytes < need || (need && !d_workspace))
    return fail(LRS_ERR_INVALID, "lrs_tree_attention: workspace of " + std::to_string(workspace_bytes) +
                                     " bytes, needs " + std::to_string(need));
  if (reinterpret_cast<uintptr_t>(d_workspace) % 16)
    return fail(LRS_ERR_INVALID, "lrs_tree_attention: the workspace must be 16-byte aligned");
  OnDevice on(be->device);
  if (on.err != cudaSuccess) return cuda_status(on.err, "cudaSetDevice");
  a.q = d_q;
  a.out = d_out;
  a.q_ld = (long long)q_ld;
  a.out_ld = (long long)out_ld;
  a.scale = scale;
  a.workspace = d_workspace;
  return cuda_status(launch_tree_attention(a, c->kv_dtype, (int)c->head_dim, be->sms,
                                           stream ? (cudaStream_t)stream : be->stream),
                     "lrs_tree_attention");
} catch (...) {
  return lrs::status_of_current_exception();
}

}  // extern "C"
