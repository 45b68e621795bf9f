// tree_attention.cu -- attention of the nodes of token trees over a paged KV
// cache (lrs_tree_attention), on the 5th-generation tensor cores.
//
// out[i][h] = sum_p softmax_p(scale q[i][h].K[p]) V[p] over the committed
// positions of the node's slot and the nodes of its mask.  The query heads of
// one KV head and the nodes of one tree share every K/V row, so they form the
// rows (node, head) of one product: at 7 heads and 8 nodes 56 rows a row of K.
//
// Both products are transposed, so that the 128 lanes of an MMA are always
// full, whatever the number of rows (they are its N, 16..64):
//   S[position][row] = K[128 positions][hd] . q^T     (A = K, B = q)
//   O[column][row]   = V^T[hd][128 positions] . P     (A = V^T, B = P)
// The A operands live in tensor memory: the decoding warps write the values of
// the cache there (a lane is a position of K, a column of V), so a tile passes
// shared memory once, as raw cache bytes.
//
// Arithmetic.  The products are exact and accumulate in f32: each operand is a
// sum of 16-bit terms, of which the products that matter at 2^-22 are taken.
//   Q8_0  d * code = hi + lo in f16, exactly (hi = rn(d code), lo its error:
//         an fma, representable since d code is a multiple of 2^-24 below
//         65504); q and P split into f16 hi + lo (22 bits): 3 products.
//   BF16  K and V as they are; q and P in 3 bf16 terms (24 bits): 3 products.
//   F32   3 bf16 terms on both sides: 6 products.
// q carries scale * log2(e) and, for f16, a power of two per row; scores are in
// base 2.  A tile's O is read out and added in registers with round-to-nearest
// (a tensor core's own sum over a long context would truncate at every step).
//
// The softmax keeps a running maximum per row that moves only when a score
// exceeds it by 2^8: P = 2^(s - m + 7) stays below 2^15, inside f16, and the
// sums hold 2^-25 of the largest weight.  A lane is a position, so the test is
// one comparison per score and one vote; the cross-lane maximum and the
// rescaling of O run only in the tiles that raise it (the first one, mostly).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "common.h"
#include "device_common.cuh"
#include "gemv.cuh"
#include "kv.cuh"

namespace lrs {
namespace {

constexpr int kTilePos = 128;   // positions of a tile: the lanes of an MMA
constexpr int kMaxRows = 64;    // rows (node, head) of a CTA's unit
constexpr int kTaThreads = 576; // four groups of four warps, the copies' warp, the MMAs' warp
constexpr float kShift = 7.0f;  // P = 2^(s - m + kShift)
constexpr float kLimit = 15.0f; // largest exponent of P before the maximum moves
constexpr float kUnset = -3e38f;

template <int HD, int DT, int NR>
struct TaShape {
  static constexpr int kA = DT == LRS_KV_F32 ? 3 : DT == LRS_KV_BF16 ? 1 : 2;  // terms of K, V
  static constexpr int kB = DT == LRS_KV_Q8_0 ? 2 : 3;                        // terms of q, P
  static constexpr bool kF16 = DT == LRS_KV_Q8_0;
  static constexpr int kProducts = DT == LRS_KV_F32 ? 6 : 3;
  // tensor memory columns
  static constexpr int kTmK = 0, kTmV = kTmK + kA * HD / 2, kTmS = kTmV + kA * kTilePos / 2;
  static constexpr int kNS = kTmS + 3 * NR <= 512 ? 2 : 1;  // score buffers
  static constexpr int kTmO = kTmS + kNS * NR;
  static constexpr int kTmCols = kTmO + NR <= 256 ? 256 : 512;
  static_assert(kTmO + NR <= 512, "tensor memory");
  // raw tiles: K rows of f32 / bf16 padded by 16 bytes against bank conflicts
  static constexpr int kSlotPos = DT == LRS_KV_F32 ? 32 : 64;
  static constexpr int kSlots = kTilePos / kSlotPos;  // slots a tile
  static constexpr int kRowK = DT == LRS_KV_F32 ? HD * 4 + 16 : HD * 2 + 16;
  static constexpr int kTileB = (int)kv_tile_bytes(DT, HD);
  static constexpr int kSlotK = DT == LRS_KV_Q8_0 ? kTileB : kSlotPos * kRowK;
  static constexpr int kSlotV = kTileB / (kPageSize / kSlotPos);
  // shared memory
  static constexpr int kQTerm = NR * HD * 2, kPTerm = NR * kTilePos * 2;
  static constexpr int kOffQ = 0, kOffP = kB * kQTerm, kOffRow = kOffP + kB * kPTerm;
  static constexpr int kOffRing = kOffRow + 5120;
  // a K slot has one reader, or two that read one tile's halves: whole tiles of
  // slots keep a slot's readers the same, so that none misses one of its phases
  static constexpr int kRoom = 226 * 1024 - kOffRing;
  static constexpr int kRing0 = (kRoom / (kSlotK + kSlotV) + kSlots - 1) / kSlots * kSlots;
  static constexpr int kRingK = kRing0 > 8 ? 8 : kRing0;
  static constexpr int kRingV0 = (kRoom - kRingK * kSlotK) / kSlotV;
  static constexpr int kRingV = kRingV0 > 8 ? 8 : kRingV0;
  static constexpr int kOffV = kOffRing + kRingK * kSlotK;
  static constexpr int kSmem = kOffV + kRingV * kSlotV;
  static_assert(kRingK % kSlots == 0 && kRingV >= 2 && kSlotK % 16 == 0 && kSlotV % 16 == 0, "ring");
};

// The part of shared memory that is not operands (kOffRow).
struct TaShared {
  unsigned long long mask[2][kMaxRows];  // per unit parity: the row's node mask
  long long out[2][kMaxRows];            // offset of the row's output, -1 = no row
  float fin_m[2][kMaxRows], fin_l[2][kMaxRows];
  unsigned vbad[2][4][2];                // nodes whose V is not finite, per warp that reads V
  float c[kMaxRows], m[kMaxRows];        // score factor, maximum - kShift
  float f[2][kMaxRows];                  // rescaling of the earlier tiles, per tile parity
  int moved[2];
  int fail[2];  // a softmax warp's wait gave up, per tile parity
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8];
  uint64_t ak_full, ak_empty, av_full, q_full, p_full, pv_done, o_empty, drain;
  uint64_t s_full[2], s_empty[2], u_full[2], u_empty[2];
  int abort;
  uint32_t tmem;
  // the schedule
  long long first, last;  // this CTA's tiles
  int tree, unit, tile;   // of `first`
  long long unit0;        // first tile of that unit
  int active;
};
static_assert(sizeof(TaShared) <= 5120, "shared state");

__device__ __forceinline__ void ta_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ta_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void ta_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void ta_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}
// D[tmem] (+)= A[tmem] . B[shared]
__device__ __forceinline__ void ta_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ uint64_t ta_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// kind::f16 instruction: f32 D, M = 128, N = n; f16 or bf16 operands, B K-major or N-major.
__device__ __forceinline__ uint32_t ta_idesc(bool f16, bool b_n_major, int n) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)b_n_major << 16) |
         ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void ta_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ta_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void ta_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float ta_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Barrier of the 128 threads of a warp group; ORs a flag.
__device__ __forceinline__ bool ta_group_or(int id, bool flag) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n bar.red.or.pred q, %1, 128, p;\n"
      " selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)flag)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void ta_group_sync(int id) {
  asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory");
}

// A wait that gives up after a bounded number of polls, or when another role did.
__device__ __forceinline__ bool ta_wait(TaShared& sh, uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kSpinLimit >> 4; i++) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 63 && *reinterpret_cast<volatile int*>(&sh.abort)) return false;
  }
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
  return false;
}

// Two f32 values as `TERMS` 16-bit pairs whose sum they are (to 2^-22, 2^-24).
template <bool F16, int TERMS>
__device__ __forceinline__ void ta_split(float a, float b, uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; i++) {
    if constexpr (F16) {
      const __half2 h = __floats2half2_rn(a, b);
      t[i] = *reinterpret_cast<const uint32_t*>(&h);
      if (i + 1 < TERMS) a -= __low2float(h), b -= __high2float(h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      t[i] = *reinterpret_cast<const uint32_t*>(&h);
      if (i + 1 < TERMS) a -= __uint_as_float(t[i] << 16), b -= __uint_as_float(t[i] & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ uint32_t ta_h2(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 ta_u2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// d * code of four int8 codes as exact f16 hi + lo pairs; d01, d23: their scales.
__device__ __forceinline__ void ta_q8(uint32_t w, __half2 d01, __half2 d23, uint32_t (&hi)[2],
                                      uint32_t (&lo)[2]) {
  const uint32_t u = w ^ 0x80808080u;  // code + 128
  const __half2 bias = ta_u2(0x64806480u);  // 1024 + 128
  const __half2 c01 = __hsub2(ta_u2(__byte_perm(u, 0x64646464u, 0x4140)), bias);
  const __half2 c23 = __hsub2(ta_u2(__byte_perm(u, 0x64646464u, 0x4342)), bias);
  const __half2 h01 = __hmul2(d01, c01), h23 = __hmul2(d23, c23);
  hi[0] = ta_h2(h01), hi[1] = ta_h2(h23);
  lo[0] = ta_h2(__hfma2(d01, c01, __hneg2(h01)));
  lo[1] = ta_h2(__hfma2(d23, c23, __hneg2(h23)));
}

// Tree t's nodes and lengths; false (and the error word) if out of range.
struct TaTree {
  int s, n, ctx, len, seq, chunks, tiles;  // chunks of rows, tiles of a chunk
  __device__ __forceinline__ bool load(const TreeArgs& a, int t, int nr) {
    s = a.start[t];
    n = a.start[t + 1] - s;
    ctx = a.ctx[t];
    seq = a.seq[t];
    chunks = tiles = 0;
    if (s < 0 || n < 0 || (long long)s + n > a.n_nodes || n > a.max_nodes || ctx < 0 ||
        (long long)ctx + n > a.max_len || seq < 0 || seq >= a.c.n_seqs) {
      atomicExch(a.c.err, kErrCacheIndex);
      return false;
    }
    len = ctx + n;
    if (n == 0) return true;
    chunks = (n * a.group + nr - 1) / nr;
    tiles = (len + kTilePos - 1) / kTilePos;
    return true;
  }
  __device__ __forceinline__ long long total(const TreeArgs& a) const {
    return (long long)tiles * chunks * a.c.heads;
  }
};

// Partial results: [2 * CTAs] segments of [kMaxRows] (m, l) and [NR][HD] sums.
struct TaDesc {
  int nseg;  // segments of the unit whose second one starts this CTA; 0 = none
  int kvh, row0, rows, s;
};
template <int HD, int NR>
__host__ __device__ constexpr size_t ta_seg_floats() {
  return 2 * NR + (size_t)NR * HD;
}

// The units (tree, KV head, chunk of rows) of a CTA, tile range by tile range.
struct TaIter {
  int tree, unit, tile;  // next unit, its first tile here
  long long left;        // tiles left
  TaTree t;
  int t0, t1, index;     // the current unit's tiles, its number in this CTA
  int kvh, row0, rows;
  bool loaded;
  __device__ __forceinline__ void begin(const TaShared& sh) {
    tree = sh.tree;
    unit = sh.unit;
    tile = sh.tile;
    left = sh.last - sh.first;
    index = -1;
    loaded = false;
  }
  __device__ __forceinline__ bool next(const TreeArgs& a, int nr) {
    if (left <= 0) return false;
    while (!loaded || unit >= t.chunks * a.c.heads) {
      if (loaded) tree++, unit = 0;
      if (tree >= a.n_trees) return false;  // the arrays changed under the kernel
      t.load(a, tree, nr);
      loaded = true;
    }
    kvh = unit / t.chunks;
    // rows of a chunk: an even share, in whole steps of the MMA's N
    const int all = t.n * a.group, share = ((all + t.chunks - 1) / t.chunks + 15) & ~15;
    row0 = (unit % t.chunks) * share;
    rows = max(0, min(share, all - row0));
    t0 = tile;
    t1 = (int)min((long long)t.tiles, t0 + left);
    left -= t1 - t0;
    index++;
    unit++;
    tile = 0;
    return true;
  }
};

template <int HD, int DT, int NR>
__global__ void __launch_bounds__(kTaThreads, 1)
    tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  using S = TaShape<HD, DT, NR>;
  constexpr int kA = S::kA, kB = S::kB;
  constexpr bool kF16 = S::kF16;
  constexpr int kWarpsD = HD / 32;  // warps that own columns of V
  extern __shared__ __align__(128) uint8_t smem[];
  TaShared& sh = *reinterpret_cast<TaShared*>(smem + S::kOffRow);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float* segs = static_cast<float*>(a.workspace);

  // ---- the schedule: every CTA finds its share of all tiles ----
  {
    __shared__ long long wsum[kTaThreads / 32];
    const int per = (a.n_trees + kTaThreads - 1) / kTaThreads;
    long long mine = 0;
    for (int i = 0; i < per; i++) {
      const int t = tid * per + i;
      TaTree tr;
      if (t < a.n_trees && tr.load(a, t, NR)) mine += tr.total(a);
    }
    long long incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) wsum[warp] = incl;
    if (tid == 0) sh.active = 0;
    __syncthreads();
    long long before = incl - mine, total = 0;
    for (int w = 0; w < kTaThreads / 32; w++) {
      if (w < warp) before += wsum[w];
      total += wsum[w];
    }
    const long long ctas = min((long long)gridDim.x, total), c = blockIdx.x;
    if (c < ctas) {
      const long long first = total * c / ctas, last = total * (c + 1) / ctas;
      if (before <= first && first < before + mine) {  // the thread that holds the first tile's tree
        long long at = before;
        for (int i = 0; i < per; i++) {
          TaTree tr;
          const int t = tid * per + i;
          if (t >= a.n_trees || !tr.load(a, t, NR)) continue;
          if (first < at + tr.total(a)) {
            sh.tree = t;
            sh.unit = (int)((first - at) / tr.tiles);
            sh.tile = (int)((first - at) % tr.tiles);
            sh.unit0 = at + (long long)sh.unit * tr.tiles;
            sh.first = first;
            sh.last = last;
            sh.active = 1;
            // this CTA starts inside a unit: the first such CTA describes it
            TaDesc d{};
            if (sh.tile > 0 && total * (c - 1) / ctas <= sh.unit0) {
              const long long end = sh.unit0 + tr.tiles;
              d.nseg = 2;
              while (total * (c + d.nseg - 1) / ctas < end) d.nseg++;
              const int all = tr.n * a.group, share = ((all + tr.chunks - 1) / tr.chunks + 15) & ~15;
              d.kvh = sh.unit / tr.chunks;
              d.row0 = (sh.unit % tr.chunks) * share;
              d.rows = max(0, min(share, all - d.row0));
              d.s = tr.s;
            }
            reinterpret_cast<TaDesc*>(a.workspace)[c] = d;
            break;
          }
          at += tr.total(a);
        }
      }
    } else if (tid == 0) {
      TaDesc d{};
      reinterpret_cast<TaDesc*>(a.workspace)[c] = d;
    }
    segs = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + gridDim.x * sizeof(TaDesc));
  }
  if (tid == 0) {
    for (int i = 0; i < 8; i++) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], S::kSlotPos / 32);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], kWarpsD);
    }
    mbar_init(&sh.ak_full, 4);
    mbar_init(&sh.ak_empty, 1);
    mbar_init(&sh.av_full, kWarpsD);
    mbar_init(&sh.q_full, 4);
    mbar_init(&sh.p_full, 4);
    mbar_init(&sh.pv_done, 1);
    mbar_init(&sh.o_empty, kWarpsD);
    mbar_init(&sh.drain, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_empty[i], 4);
      mbar_init(&sh.u_full[i], 4);
      mbar_init(&sh.u_empty[i], kWarpsD);
      sh.fail[i] = 0;
    }
    sh.abort = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  if (!sh.active) return;
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sh.tmem)),
                 "r"((uint32_t)S::kTmCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  ta_fence_before();
  __syncthreads();
  ta_fence_after();
  const uint32_t tmem = sh.tmem;
  const uint32_t sbase = smem_u32(smem);
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;  // this warp's lanes of tensor memory
  TaIter it;
  it.begin(sh);
  bool ok = true;

  if (warp < 4) {
    // ---- K: a lane is a position; its row into tensor memory ----
    uint32_t tile = 0;
    while (ok && it.next(a, NR)) {
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        const uint32_t n = tile * S::kSlots + (warp * 32) / S::kSlotPos, slot = n % S::kRingK;
        ok = ta_wait(sh, &sh.k_full[slot], (n / S::kRingK) & 1);
        if (ok && tile > 0) ok = ta_wait(sh, &sh.ak_empty, (tile - 1) & 1);
        if (!ok) break;
        ta_fence_after();
        const uint8_t* raw = smem + S::kOffRing + slot * S::kSlotK;
        const int r = (warp * 32 + lane) % S::kSlotPos;
        if constexpr (DT == LRS_KV_Q8_0) {
          __half d[HD / 32];
#pragma unroll
          for (int b = 0; b < HD / 32; b++)
            d[b] = *reinterpret_cast<const __half*>(raw + q8_k_scale(HD, r, b));
#pragma unroll
          for (int b = 0; b < HD / 32; b++) {  // a block: 16 columns of hi, 16 of lo
            uint32_t hi[16], lo[16];
            const __half2 d2 = __half2half2(d[b]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const uint4 w4 = *reinterpret_cast<const uint4*>(raw + q8_k_code(r, b * 32 + h * 16));
              const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
              for (int i = 0; i < 4; i++) {
                uint32_t x[2], y[2];
                ta_q8(w[i], d2, d2, x, y);
                hi[h * 8 + i * 2] = x[0], hi[h * 8 + i * 2 + 1] = x[1];
                lo[h * 8 + i * 2] = y[0], lo[h * 8 + i * 2 + 1] = y[1];
              }
            }
            ta_st16(tmem + lanes + S::kTmK + b * 16, hi);
            ta_st16(tmem + lanes + S::kTmK + HD / 2 + b * 16, lo);
          }
        } else {
          const uint8_t* row = raw + r * S::kRowK;
#pragma unroll
          for (int b = 0; b < HD / 32; b++) {  // 32 values: 16 columns a term
            uint32_t x[kA][16];
            if constexpr (DT == LRS_KV_BF16) {
#pragma unroll
              for (int i = 0; i < 4; i++) {
                const uint4 w = *reinterpret_cast<const uint4*>(row + b * 64 + i * 16);
                x[0][i * 4] = w.x, x[0][i * 4 + 1] = w.y, x[0][i * 4 + 2] = w.z, x[0][i * 4 + 3] = w.w;
              }
            } else {
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const float4 f = *reinterpret_cast<const float4*>(row + b * 128 + i * 16);
                uint32_t y[kA];
                ta_split<false, kA>(f.x, f.y, y);
#pragma unroll
                for (int k = 0; k < kA; k++) x[k][i * 2] = y[k];
                ta_split<false, kA>(f.z, f.w, y);
#pragma unroll
                for (int k = 0; k < kA; k++) x[k][i * 2 + 1] = y[k];
              }
            }
#pragma unroll
            for (int k = 0; k < kA; k++)
              ta_st16(tmem + lanes + S::kTmK + k * HD / 2 + b * 16, x[k]);
          }
        }
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.k_empty[slot]);
        ta_wait_st();
        ta_fence_before();
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.ak_full);
      }
    }
  } else if (warp < 8) {
    // ---- V: a lane is a column of the head; positions along its row ----
    const int w = warp - 4, h = w * 32 + lane;
    uint32_t tile = 0;
    while (w < kWarpsD && ok && it.next(a, NR)) {
      // the words of the unit before last have been read
      if (it.index >= 2) ok = ta_wait(sh, &sh.u_empty[it.index & 1], ((it.index >> 1) - 1) & 1);
      unsigned* vbad = sh.vbad[it.index & 1][w];
      if (lane < 2) vbad[lane] = 0;
      __syncwarp();
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        if (tile > 0) ok = ta_wait(sh, &sh.pv_done, (tile - 1) & 1);
        ta_fence_after();
        const bool tail = (t + 1) * kTilePos > it.t.ctx;  // holds nodes, or positions past the end
#pragma unroll 1
        for (int k = 0; k < S::kSlots && ok; k++) {
          const uint32_t n = tile * S::kSlots + k, slot = n % S::kRingV;
          ok = ta_wait(sh, &sh.v_full[slot], (n / S::kRingV) & 1);
          if (!ok) break;
          const uint8_t* raw = smem + S::kOffV + slot * S::kSlotV;
          const int p0 = t * kTilePos + k * S::kSlotPos;
          const uint32_t col = tmem + lanes + S::kTmV + k * (S::kSlotPos / 2);
#pragma unroll
          for (int g = 0; g < S::kSlotPos / 32; g++) {  // 32 positions: 16 columns a term
            uint32_t x[kA][16];
            if constexpr (DT == LRS_KV_Q8_0) {
#pragma unroll
              for (int i = 0; i < 8; i++) {
                const int r = g * 32 + i * 4;
                uint2 dd = *reinterpret_cast<const uint2*>(raw + q8_v_scale(HD, r, w));
                if (tail) {
#pragma unroll
                  for (int j = 0; j < 4; j++) {
                    uint32_t& d = j < 2 ? dd.x : dd.y;
                    const uint32_t keep = j & 1 ? 0x0000ffffu : 0xffff0000u, bits = d & ~keep;
                    const int p = p0 + r + j;
                    const bool bad = (bits & (j & 1 ? 0x7c000000u : 0x7c00u)) == (j & 1 ? 0x7c000000u : 0x7c00u);
                    if (p >= it.t.len || (bad && p >= it.t.ctx)) {
                      d &= keep;
                      if (p < it.t.len && lane == 0)
                        atomicOr(&vbad[(p - it.t.ctx) >> 5], 1u << ((p - it.t.ctx) & 31));
                    }
                  }
                }
                const uint32_t cw = *reinterpret_cast<const uint32_t*>(raw + q8_v_code(HD, r, h));
                uint32_t hi[2], lo[2];
                ta_q8(cw, ta_u2(dd.x), ta_u2(dd.y), hi, lo);
                x[0][i * 2] = hi[0], x[0][i * 2 + 1] = hi[1];
                x[1][i * 2] = lo[0], x[1][i * 2 + 1] = lo[1];
              }
            } else {
#pragma unroll
              for (int i = 0; i < 16; i++) {
                float f[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                  const int r = g * 32 + i * 2 + j, p = p0 + r;
                  f[j] = DT == LRS_KV_BF16
                             ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(raw)[r * HD + h] << 16)
                             : reinterpret_cast<const float*>(raw)[r * HD + h];
                  if (tail) {
                    const bool bad = (__float_as_uint(f[j]) & 0x7f800000u) == 0x7f800000u;
                    if (p >= it.t.len || (bad && p >= it.t.ctx)) {
                      f[j] = 0.0f;
                      if (p < it.t.len)
                        atomicOr(&vbad[(p - it.t.ctx) >> 5], 1u << ((p - it.t.ctx) & 31));
                    }
                  }
                }
                uint32_t y[kA];
                ta_split<false, kA>(f[0], f[1], y);
#pragma unroll
                for (int q = 0; q < kA; q++) x[q][i] = y[q];
              }
            }
#pragma unroll
            for (int q = 0; q < kA; q++) ta_st16(col + q * (kTilePos / 2) + g * 16, x[q]);
          }
          __syncwarp();
          if (lane == 0) ta_arrive(&sh.v_empty[slot]);
        }
        if (!ok) break;
        ta_wait_st();
        ta_fence_before();
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.av_full);
      }
    }
  } else if (warp < 12) {
    // ---- q, and the softmax: a lane is a position ----
    const int w = warp - 8, gt = tid - 256;
    constexpr int kBar = 1;
    float l[NR];
    uint32_t tile = 0;
    bool left = false;
    // the four warps meet at barriers: one whose wait gave up goes on (on stale
    // data, in bounds) to the next vote, where they leave together
    while (!left && it.next(a, NR)) {
      const int u = it.index & 1;
      if (it.index >= 2) ok = ok && ta_wait(sh, &sh.u_empty[u], ((it.index >> 1) - 1) & 1);
      const int rows = it.rows, steps = (rows + 15) >> 4;  // MMA rows in steps of 16
      if (gt < NR) {
        const int row = it.row0 + gt, node = row / a.group, g = row % a.group;
        const bool live = gt < rows;
        sh.out[u][gt] = live ? (long long)(it.t.s + node) * a.out_ld + (long long)(it.kvh * a.group + g) * HD : -1;
        unsigned long long m = 0;
        if (live) {
          m = a.mask ? a.mask[it.t.s + node] : (node == 63 ? ~0ull : (2ull << node) - 1);
          if (it.t.n < 64) m &= (1ull << it.t.n) - 1;
        }
        sh.mask[u][gt] = m;
        sh.m[gt] = kUnset;
      }
      // q * scale * log2(e) in terms, K-major core matrices: a warp takes 8 rows,
      // a lane 8 columns of one at a time
      const float qs = a.scale * 1.44269504088896f;
      const bool vec = a.q_ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
      for (int g8 = w; g8 < 2 * steps; g8 += 4) {
        const int gr = g8 * 8 + (lane & 7), row = it.row0 + gr;
        const float* src = a.q + (size_t)(it.t.s + row / a.group) * a.q_ld +
                           (size_t)(it.kvh * a.group + row % a.group) * HD;
        float x[HD / 32][8];
        float mx = 0.0f;
#pragma unroll
        for (int j = 0; j < HD / 32; j++) {
          const int c = (j * 4 + (lane >> 3)) * 8;
#pragma unroll
          for (int e = 0; e < 8; e++) x[j][e] = 0.0f;
          if (gr < rows) {
            if (vec) {
              const float4 f0 = *reinterpret_cast<const float4*>(src + c), f1 = *reinterpret_cast<const float4*>(src + c + 4);
              x[j][0] = f0.x, x[j][1] = f0.y, x[j][2] = f0.z, x[j][3] = f0.w;
              x[j][4] = f1.x, x[j][5] = f1.y, x[j][6] = f1.z, x[j][7] = f1.w;
            } else {
#pragma unroll
              for (int e = 0; e < 8; e++) x[j][e] = src[c + e];
            }
          }
#pragma unroll
          for (int e = 0; e < 8; e++) {
            x[j][e] *= qs;
            mx = fmaxf(mx, fabsf(x[j][e]));
          }
        }
        int ex = 0;
        if constexpr (kF16) {  // the row's largest magnitude to [2^10, 2^11)
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          if (mx > 0.0f && mx < INFINITY) {
            frexpf(mx, &ex);
            ex -= 11;
          }
        }
        if (lane < 8) sh.c[gr] = ldexpf(1.0f, ex);
#pragma unroll
        for (int j = 0; j < HD / 32; j++) {
          uint32_t y[kB][4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float f0 = x[j][2 * e], f1 = x[j][2 * e + 1];
            if constexpr (kF16) f0 = ldexpf(f0, -ex), f1 = ldexpf(f1, -ex);
            uint32_t z[kB];
            ta_split<kF16, kB>(f0, f1, z);
#pragma unroll
            for (int k = 0; k < kB; k++) y[k][e] = z[k];
          }
          uint8_t* dst = smem + S::kOffQ + g8 * (HD / 8 * 128) + (j * 4 + (lane >> 3)) * 128 + (lane & 7) * 16;
#pragma unroll
          for (int k = 0; k < kB; k++)
            *reinterpret_cast<uint4*>(dst + k * S::kQTerm) = make_uint4(y[k][0], y[k][1], y[k][2], y[k][3]);
        }
      }
      fence_proxy_async();
      ta_group_sync(kBar);
      if (lane == 0) ta_arrive(&sh.q_full);
#pragma unroll
      for (int r = 0; r < NR; r++) l[r] = 0.0f;
      for (int t = it.t0; t < it.t1; t++, tile++) {
        const int sb = tile % S::kNS, par = tile & 1;
        ok = ok && ta_wait(sh, &sh.s_full[sb], (tile / S::kNS) & 1);
        if (!ok) sh.fail[par] = 1;
        ta_fence_after();
        const uint32_t st = tmem + lanes + S::kTmS + sb * NR;
        const int p = t * kTilePos + w * 32 + lane;
        const bool full = (t + 1) * kTilePos <= it.t.ctx;
        // whether row r sees this lane's position
        const int node = p - it.t.ctx;
        auto seen = [&](int r) {
          return full || node < 0 || (p < it.t.len && (sh.mask[u][r] >> node & 1));
        };
        // does a score exceed its row's maximum by more than the margin?
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < NR / 16; c++) {
          if (c >= steps) break;
          float s[16];
          ta_ld16(st + c * 16, s);
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int r = c * 16 + i;
            const float d = fmaf(s[i], sh.c[r], -sh.m[r]);
            if (seen(r)) top = fmaxf(top, d);
          }
        }
        const bool move = ta_group_or(kBar, top > kLimit);
        left = *reinterpret_cast<volatile int*>(&sh.fail[par]) != 0;
        if (left) break;
        // the last tile's product has read P, and its O, f and moved may be overwritten
        if (tile > 0) ok = ok && ta_wait(sh, &sh.pv_done, (tile - 1) & 1);
        if (move) {
          // the rows' maxima over the tile: 16 rows by 32 lanes to a row a lane pair
          float* red = reinterpret_cast<float*>(smem + S::kOffP);
#pragma unroll
          for (int c = 0; c < NR / 16; c++) {
            if (c >= steps) break;
            float s[16];
            ta_ld16(st + c * 16, s);
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const int r = c * 16 + i;
              s[i] = seen(r) ? s[i] * sh.c[r] : kUnset;
            }
            int row = c * 16;
#pragma unroll
            for (int wd = 16, nn = 8; wd >= 2; wd >>= 1, nn >>= 1) {
              const bool up = lane & wd;
#pragma unroll
              for (int i = 0; i < 8; i++) {
                if (i < nn) {
                  const float send = up ? s[i] : s[i + nn], keep = up ? s[i + nn] : s[i];
                  s[i] = fmaxf(keep, __shfl_xor_sync(0xffffffffu, send, wd));
                }
              }
              if (up) row += nn;
            }
            s[0] = fmaxf(s[0], __shfl_xor_sync(0xffffffffu, s[0], 1));
            if (!(lane & 1)) red[w * NR + row] = s[0];
          }
          ta_group_sync(kBar);
          if (gt < steps * 16) {
            const float was = sh.m[gt];
            float mx = fmaxf(fmaxf(red[gt], red[NR + gt]), fmaxf(red[2 * NR + gt], red[3 * NR + gt]));
            mx = mx > kUnset ? fmaxf(was, mx - kShift) : was;
            sh.f[par][gt] = was == kUnset ? 0.0f : ta_exp2(was - mx);
            sh.m[gt] = mx;
          }
          if (gt == 0) sh.moved[par] = 1;
          ta_group_sync(kBar);
#pragma unroll
          for (int r = 0; r < NR; r++)
            if (r < steps * 16) l[r] *= sh.f[par][r];
        } else {
          if (gt == 0) sh.moved[par] = 0;
        }
        // P = 2^(s - m + 7), its terms N-major: a lane writes 8 rows at once
#pragma unroll
        for (int c = 0; c < NR / 16; c++) {
          if (c >= steps) break;
          float s[16];
          ta_ld16(st + c * 16, s);
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const int r = c * 16 + i;
            s[i] = ta_exp2(fmaf(s[i], sh.c[r], -sh.m[r]));
            if (!seen(r)) s[i] = 0.0f;
            l[r] += s[i];
          }
#pragma unroll
          for (int g = 0; g < 2; g++) {
            uint32_t y[kB][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              uint32_t z[kB];
              ta_split<kF16, kB>(s[g * 8 + 2 * e], s[g * 8 + 2 * e + 1], z);
#pragma unroll
              for (int k = 0; k < kB; k++) y[k][e] = z[k];
            }
            const int pp = w * 32 + lane;
            uint8_t* dst = smem + S::kOffP + (pp >> 3) * (NR * 16) + (c * 2 + g) * 128 + (pp & 7) * 16;
#pragma unroll
            for (int k = 0; k < kB; k++)
              *reinterpret_cast<uint4*>(dst + k * S::kPTerm) = make_uint4(y[k][0], y[k][1], y[k][2], y[k][3]);
          }
        }
        ta_fence_before();
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          ta_arrive(&sh.s_empty[sb]);
          ta_arrive(&sh.p_full);
        }
      }
      if (left) break;
      // the rows' sums over the lanes: NR rows by 32 lanes to NR / 32 rows a lane
      {
        int row = 0;
#pragma unroll
        for (int wd = 16, nn = NR / 2; wd >= 1; wd >>= 1, nn >>= 1) {
          if (nn >= 1) {
            const bool up = lane & wd;
#pragma unroll
            for (int i = 0; i < NR / 2; i++) {
              if (i < nn) {
                const float send = up ? l[i] : l[i + nn], keep = up ? l[i + nn] : l[i];
                l[i] = keep + __shfl_xor_sync(0xffffffffu, send, wd);
              }
            }
            if (up) row += nn;
          } else {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], wd);
          }
        }
        constexpr int kKeep = NR >= 32 ? NR / 32 : 1;
        // fin_l as [4 warps] partials would need room: add them one warp at a time
        for (int k = 0; k < 4; k++) {
          if (k == w && (NR >= 32 || !(lane & 1))) {
#pragma unroll
            for (int i = 0; i < kKeep; i++)
              sh.fin_l[u][row + i] = (k ? sh.fin_l[u][row + i] : 0.0f) + l[i];
          }
          ta_group_sync(kBar);
        }
        if (gt < NR) sh.fin_m[u][gt] = sh.m[gt];
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.u_full[u]);
      }
    }
  } else if (warp < 16) {
    // ---- O: a lane is a column; sums of the tiles' products in registers ----
    const int w = warp - 12, h = w * 32 + lane;
    uint32_t tile = 0;
    while (w < kWarpsD && ok && it.next(a, NR)) {
      const int u = it.index & 1, steps = (it.rows + 15) >> 4;
      float o[NR];
#pragma unroll
      for (int r = 0; r < NR; r++) o[r] = 0.0f;
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        ok = ta_wait(sh, &sh.pv_done, tile & 1);
        if (!ok) break;
        ta_fence_after();
        const int par = tile & 1;
        const bool moved = sh.moved[par] != 0;
#pragma unroll
        for (int c = 0; c < NR / 16; c++) {
          if (c >= steps) break;
          float x[16];
          ta_ld16(tmem + lanes + S::kTmO + c * 16, x);
          if (moved) {
#pragma unroll
            for (int i = 0; i < 16; i++) o[c * 16 + i] = fmaf(o[c * 16 + i], sh.f[par][c * 16 + i], x[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; i++) o[c * 16 + i] += x[i];
          }
        }
        ta_fence_before();
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.o_empty);
      }
      if (!ok) break;
      ok = ta_wait(sh, &sh.u_full[u], (it.index >> 1) & 1);
      if (!ok) break;
      unsigned long long vbad = 0;
#pragma unroll
      for (int i = 0; i < kWarpsD; i++) vbad |= sh.vbad[u][i][0] | (unsigned long long)sh.vbad[u][i][1] << 32;
      const bool whole = it.t0 == 0 && it.t1 == it.t.tiles;
      float* seg = segs + (size_t)(2 * blockIdx.x + (it.t0 == 0)) * ta_seg_floats<HD, NR>();
#pragma unroll
      for (int r = 0; r < NR; r++) {
        const long long at = sh.out[u][r];
        if (at >= 0) {
          const float lr = sh.fin_l[u][r];
          float x = o[r];
          if (sh.mask[u][r] & vbad) x = __int_as_float(0x7fc00000);
          if (whole) {
            a.out[at + h] = lr == 0.0f ? 0.0f : x / lr;
          } else {
            if (w == 0 && lane == 0) seg[2 * r] = sh.fin_m[u][r], seg[2 * r + 1] = lr;
            seg[2 * NR + r * HD + h] = x;
          }
        }
      }
      __syncwarp();
      if (lane == 0) ta_arrive(&sh.u_empty[u]);
    }
  } else if (warp == 16) {
    // ---- copies: raw K and V tiles of the pages ----
    const uint64_t pol = evict_first_policy();
    uint32_t n = 0, nk = 0, nv = 0;  // the slot, K and V slots issued
    while (ok && it.next(a, NR)) {
      const int used = (it.t.len + kPageSize - 1) / kPageSize;  // the slot's pages that hold positions
      for (int t = it.t0; t < it.t1 && ok; t++) {
        for (int k = 0; k < S::kSlots && ok; k++, n++) {
          const uint32_t ks = n % S::kRingK, vs = n % S::kRingV;
          const int p = t * kTilePos + k * S::kSlotPos;
          int page = -1;
          if (p / kPageSize < used) page = kv_page(a.c, it.t.seq, p);
          const size_t off = ((size_t)max(page, 0) * a.c.heads + it.kvh) * S::kTileB;
          uint8_t* kd = smem + S::kOffRing + ks * S::kSlotK;
          uint8_t* vd = smem + S::kOffV + vs * S::kSlotV;
          constexpr int kPart = S::kTileB / (kPageSize / S::kSlotPos);  // bytes of the slot's rows
          const size_t part = off + (size_t)(p % kPageSize / S::kSlotPos) * kPart;
          if (n >= S::kRingK) ok = ta_wait(sh, &sh.k_empty[ks], ((n / S::kRingK) - 1) & 1);
          if (!ok) break;
          if (page < 0) {
            if (lane == 0) ta_arrive(&sh.k_full[ks]);
          } else {
            if (lane == 0) mbar_expect_tx(&sh.k_full[ks], kPart);
            __syncwarp();
            if constexpr (DT == LRS_KV_Q8_0) {
              if (lane == 0) tma_load_1d(kd, a.c.k + part, kPart, &sh.k_full[ks], pol);
            } else {
              constexpr int kRow = kPart / S::kSlotPos;
              for (int r = lane; r < S::kSlotPos; r += 32)
                tma_load_1d(kd + r * S::kRowK, a.c.k + part + (size_t)r * kRow, kRow, &sh.k_full[ks], pol);
            }
          }
          nk = n + 1;
          if (n >= S::kRingV) ok = ta_wait(sh, &sh.v_empty[vs], ((n / S::kRingV) - 1) & 1);
          if (!ok) break;
          if (lane == 0) {
            if (page < 0) {
              ta_arrive(&sh.v_full[vs]);
            } else {
              mbar_expect_tx(&sh.v_full[vs], kPart);
              tma_load_1d(vd, a.c.v + part, kPart, &sh.v_full[vs], pol);
            }
          }
          nv = n + 1;
        }
      }
    }
    // copies in flight land before shared memory goes away (they may outlive
    // their readers only when a wait gave up)
    if (!ok) {
      auto land = [&](uint64_t* full, uint32_t ring, uint32_t issued) {
        for (uint32_t i = issued > ring ? issued - ring : 0; i < issued; i++)
          for (uint32_t j = 0; j < kSpinLimit >> 4 && !mbar_try_wait(&full[i % ring], (i / ring) & 1); j++) {
          }
      };
      land(sh.k_full, S::kRingK, nk);
      land(sh.v_full, S::kRingV, nv);
    }
  } else if (lane == 0) {
    // ---- MMAs ----
    constexpr int kPa[6] = {kA - 1, kA == 3 ? 1 : 0, 0, 1, 0, 0};  // terms of the products, small ones first
    constexpr int kPb[6] = {0, kA == 3 ? 1 : kB == 2 ? 1 : 1, kA == 3 ? 2 : 0, 0, 1, 0};
    constexpr int kPaB[3] = {0, 0, 0}, kPbB[3] = {2, 1, 0};  // one term of A
    auto term_a = [&](int i) { return kA == 1 ? kPaB[i % 3] : kPa[i]; };
    auto term_b = [&](int i) { return kA == 1 ? kPbB[i % 3] : kPb[i]; };
    uint32_t tile = 0, qk = 0;
    auto qk_tile = [&](int steps) {  // scores of tile `qk`
      const int sb = qk % S::kNS;
      bool good = ta_wait(sh, &sh.ak_full, qk & 1);
      if (good && qk >= S::kNS) good = ta_wait(sh, &sh.s_empty[sb], ((qk / S::kNS) - 1) & 1);
      if (!good) return false;
      ta_fence_after();
      const uint32_t d = tmem + S::kTmS + sb * NR, idesc = ta_idesc(kF16, false, steps * 16);
#pragma unroll
      for (int i = 0; i < S::kProducts; i++)
#pragma unroll
        for (int k = 0; k < HD / 16; k++)
          ta_mma(d, tmem + S::kTmK + term_a(i) * (HD / 2) + k * 8,
                 ta_desc(sbase + S::kOffQ + term_b(i) * S::kQTerm + k * 256, 128, HD / 8 * 128), idesc,
                 (i | k) != 0);
      ta_commit(&sh.ak_empty);
      ta_commit(&sh.s_full[sb]);
      qk++;
      return true;
    };
    while (ok && it.next(a, NR)) {
      const int steps = (it.rows + 15) >> 4;
      ok = ta_wait(sh, &sh.q_full, it.index & 1) && qk_tile(steps);
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        if (t + 1 < it.t1) ok = qk_tile(steps);
        ok = ok && ta_wait(sh, &sh.av_full, tile & 1) && ta_wait(sh, &sh.p_full, tile & 1);
        if (ok && tile > 0) ok = ta_wait(sh, &sh.o_empty, (tile - 1) & 1);
        if (!ok) break;
        ta_fence_after();
        const uint32_t d = tmem + S::kTmO, idesc = ta_idesc(kF16, true, steps * 16);
#pragma unroll
        for (int i = 0; i < S::kProducts; i++)
#pragma unroll
          for (int k = 0; k < kTilePos / 16; k++)
            ta_mma(d, tmem + S::kTmV + term_a(i) * (kTilePos / 2) + k * 8,
                   ta_desc(sbase + S::kOffP + term_b(i) * S::kPTerm + k * 2 * (NR * 16), NR * 16, 128), idesc,
                   (i | k) != 0);
        ta_commit(&sh.pv_done);
      }
    }
    if (!ok) {  // MMAs in flight end before their memory goes away
      ta_commit(&sh.drain);
      for (uint32_t j = 0; j < kSpinLimit >> 4; j++)
        if (mbar_try_wait(&sh.drain, 0)) break;
    }
  }
  if (!ok) atomicExch(a.c.err, LRS_ERR_DEVICE_TIMEOUT);
  ta_fence_before();
  __syncthreads();
  if (warp == 17) {
    ta_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"((uint32_t)S::kTmCols)
                 : "memory");
  }
}

// Merges the segments of the units that several CTAs share: block (c, y) the
// unit that CTA c is the second one of, rows y, y + gridDim.y, ...
template <int HD, int NR>
__global__ void __launch_bounds__(HD) tree_combine_kernel(const __grid_constant__ TreeArgs a, int ctas) {
  pdl_wait();
  const int c = blockIdx.x + 1, h = threadIdx.x;
  const TaDesc d = reinterpret_cast<const TaDesc*>(a.workspace)[c];
  const float* segs = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + ctas * sizeof(TaDesc));
  for (int r = blockIdx.y; d.nseg > 0 && r < d.rows; r += gridDim.y) {
    auto seg = [&](int i) {
      return segs + (size_t)(i == 0 ? 2 * (c - 1) + 1 : 2 * (c + i - 1)) * ta_seg_floats<HD, NR>();
    };
    float m = kUnset;
    for (int i = 0; i < d.nseg; i++) m = fmaxf(m, seg(i)[2 * r]);
    float l = 0.0f, o = 0.0f;
    for (int i = 0; i < d.nseg; i++) {
      const float* s = seg(i);
      const float f = s[2 * r] == kUnset ? 0.0f : exp2f(s[2 * r] - m);
      if (s[2 * r] == kUnset) continue;
      l = fmaf(s[2 * r + 1], f, l);
      o = fmaf(s[2 * NR + r * HD + h], f, o);
    }
    const int row = d.row0 + r;
    a.out[(size_t)(d.s + row / a.group) * a.out_ld +
          ((size_t)d.kvh * a.group + row % a.group) * HD + h] = l == 0.0f ? 0.0f : o / l;
  }
}

// Rows a unit: the smallest of 16, 32, 64 that holds a tree's rows.
int unit_rows(const TreeArgs& a) {
  const int rows = a.max_nodes * a.group;
  return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

int grid_ctas(const TreeArgs& a, int sms) {
  const int nr = unit_rows(a);
  const long long units = (long long)a.n_trees * a.c.heads * ((a.max_nodes * a.group + nr - 1) / nr);
  return (int)std::min<long long>(sms, units * ((a.max_len + kTilePos - 1) / kTilePos));
}

template <int HD, int DT, int NR>
cudaError_t launch(const TreeArgs& a, int sms, cudaStream_t st) {
  using S = TaShape<HD, DT, NR>;
  static std::atomic<uint64_t> attr{0};
  cudaError_t e = set_smem_once(attr, (const void*)tree_attention_kernel<HD, DT, NR>, S::kSmem);
  if (e != cudaSuccess) return e;
  const int ctas = grid_ctas(a, sms);
  tree_attention_kernel<HD, DT, NR><<<ctas, kTaThreads, S::kSmem, st>>>(a);
  e = cudaGetLastError();
  // units of one tile are never shared
  if (e != cudaSuccess || ctas < 2 || a.max_len <= kTilePos) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas - 1, NR / 4);
  cfg.blockDim = dim3(HD);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_combine_kernel<HD, NR>, a, ctas);
}

template <int HD, int DT>
cudaError_t launch_rows(const TreeArgs& a, int sms, cudaStream_t st) {
  switch (unit_rows(a)) {
    case 16: return launch<HD, DT, 16>(a, sms, st);
    case 32: return launch<HD, DT, 32>(a, sms, st);
    default: return launch<HD, DT, 64>(a, sms, st);
  }
}

}  // namespace

size_t tree_attention_workspace_bytes(const TreeArgs& a, int hd, int sms) {
  if (a.n_trees == 0 || a.n_nodes == 0) return 0;
  const size_t nr = unit_rows(a);
  return (size_t)grid_ctas(a, sms) * (sizeof(TaDesc) + 2 * 4 * (2 * nr + nr * hd)) + 16;
}

cudaError_t launch_tree_attention(const TreeArgs& a, uint32_t dtype, int hd, int sms,
                                  cudaStream_t st) {
  if (hd == 128) {
    if (dtype == LRS_KV_F32) return launch_rows<128, LRS_KV_F32>(a, sms, st);
    if (dtype == LRS_KV_BF16) return launch_rows<128, LRS_KV_BF16>(a, sms, st);
    return launch_rows<128, LRS_KV_Q8_0>(a, sms, st);
  }
  if (dtype == LRS_KV_F32) return launch_rows<64, LRS_KV_F32>(a, sms, st);
  if (dtype == LRS_KV_BF16) return launch_rows<64, LRS_KV_BF16>(a, sms, st);
  return launch_rows<64, LRS_KV_Q8_0>(a, sms, st);
}

}  // namespace lrs
