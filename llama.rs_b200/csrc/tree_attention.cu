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
// A CTA is a pipeline of roles (TaShape): two copy warps bring a tile's raw pages in by
// bulk copies; four warps decode K, four (eight) V; the softmax has a group of four
// warps per 16 rows, a lane being a position, so that a row's statistics need the
// other lanes only when its maximum moves; four warps keep the sums of O, a lane being
// a column; one warp issues the MMAs.  The tiles of all trees are one list that the
// CTAs share evenly, whatever the trees' lengths; what a unit (the rows of one tree,
// KV head and chunk) has in several CTAs leaves as (maximum, sum, O) segments, which
// tree_combine_kernel merges.
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
//
// What bounds it.  64 trees of 8 nodes on 2,100 to 4,100 positions, q8_0, 4 KV heads
// of 7 queries, 128 wide: 114 us (104 back to back), 2.0 TB/s of the cache's bytes and 0.53
// PFLOP/s of the three products; 4 trees of 64 nodes on 7,200 to 8,200: 114 us, 0.75 PFLOP/s.
// A tile takes some 3,000 clocks, of which the tensor pipe needs 1,536 and the copies, at DRAM's
// rate, 1,476; the schedulers issue in 65 of 100 clocks.  So the bound is the instructions
// of decoding (a lane's 128 values of K or V take some 450) and of the softmax, whose
// warps make 8 to 12 clocks an instruction beside one another.  A CTA spends some 15,000
// clocks before its first product (the schedule, cold instruction fetches, q) and after
// its last one: small calls are that and the launch (5 nodes on 100 positions, bf16, 12.3
// us; a decode step of 64 sequences at 700 to 1,100, q8_0, 35 us).  bf16 and f32 caches,
// which need less decoding or more bytes, take longer (64 x 8 in bf16 228 us, 32 x 8 in f32
// 151): their warps mostly wait (the schedulers issue in 27 and 35 of 100 cycles, DRAM is at
// 22 and 36 %, the tensor pipe at 14 and 24 %).
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
constexpr float kShift = 7.0f;  // P = 2^(s - m + kShift)
constexpr float kLimit = 15.0f; // largest exponent of P before the maximum moves
constexpr float kUnset = -3e38f;
constexpr int kSmemMost = 226 * 1024, kSharedBytes = 8192;

template <int HD, int DT, int NR>
struct TaShape {
  static constexpr int kA = DT == LRS_KV_F32 ? 3 : DT == LRS_KV_BF16 ? 1 : 2;  // terms of K, V
  static constexpr int kB = DT == LRS_KV_Q8_0 ? 2 : 3;                        // terms of q, P
  static constexpr bool kF16 = DT == LRS_KV_Q8_0;
  // Groups of four warps: K, V (up to 32 rows two, half of the positions each: they took
  // 9 % off a decode step of 64 sequences; at 64 rows the threads are spent), the
  // softmax (16 rows each: groups of 32 took the same time at 64 rows, and would be half
  // idle below), O; then a warp each for K's copies, V's and the MMAs.
  static constexpr int kSG = NR / 16, kVG = NR == 64 ? 1 : 2;
  static constexpr int kWarpV = 4, kWarpS = kWarpV + 4 * kVG, kWarpO = kWarpS + 4 * kSG;
  static constexpr int kWarpCopyK = kWarpO + 4, kWarpCopyV = kWarpCopyK + 1, kWarpMma = kWarpCopyV + 1;
  static constexpr int kThreads = 32 * (kWarpMma + 1);
  // Registers a thread: at launch, K and V, the softmax, O (increases beyond what
  // the others gave would wait for good).
  static constexpr int kRegs = NR == 64 ? 64 : NR == 32 ? 72 : 80;
  static constexpr int kRegsKV = NR == 64 ? 48 : 64, kRegsS = NR == 16 ? 80 : 64;
  static constexpr int kRegsO = 96;
  static_assert((1 + kVG) * kRegsKV + kSG * kRegsS + kRegsO <= (2 + kVG + kSG) * kRegs, "registers");
  static_assert(kRegsS <= kRegs && kRegsKV <= kRegs && kRegsO > kRegs, "the roles' changes of registers");
  static constexpr int kProducts = DT == LRS_KV_F32 ? 6 : 3;
  // tensor memory columns: V is double-buffered where it fits
  static constexpr int kVCols = kA * kTilePos / 2;
  static constexpr int kTmK = 0, kTmV = kTmK + kA * HD / 2;
  static constexpr int kNV = kTmV + 2 * kVCols + 2 * NR <= 512 ? 2 : 1;
  static constexpr int kTmS = kTmV + kNV * kVCols, kTmO = kTmS + NR;
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
  static constexpr int kQTerm = NR * HD * 2, kPTerm = NR * kTilePos * 2, kPBuf = kB * kPTerm;
  static constexpr int kOffQ = 0, kOffP = kB * kQTerm;
  // P is double-buffered where two tiles of slots remain beside it
  static constexpr int kNP =
      kOffP + 2 * kPBuf + kSharedBytes + 2 * kSlots * (kSlotK + kSlotV) <= kSmemMost ? 2 : 1;
  static constexpr int kOffRow = kOffP + kNP * kPBuf;
  static constexpr int kOffRing = kOffRow + kSharedBytes;
  // where a tile's slots have different readers, whole tiles of slots keep a
  // slot's readers the same, so that none misses one of its phases
  static constexpr int kRoom = kSmemMost - kOffRing;
  static constexpr int kTiles = kRoom / (kSlots * (kSlotK + kSlotV));
  static constexpr int kRing0 = kVG == 2 ? kTiles * kSlots : (kRoom / (kSlotK + kSlotV) + kSlots - 1) / kSlots * kSlots;
  static constexpr int kRingK = kRing0 > 8 ? 8 : kRing0;
  static constexpr int kRingV0 = kVG == 2 ? kRingK : (kRoom - kRingK * kSlotK) / kSlotV;
  static constexpr int kRingV = kRingV0 > 8 ? 8 : kRingV0;
  static constexpr int kOffV = kOffRing + kRingK * kSlotK;
  static constexpr int kSmem = kOffV + kRingV * kSlotV;
  static_assert(kRingK % kSlots == 0 && kRingK >= kSlots && kRingV >= 2 && kSmem <= kSmemMost &&
                kSlotK % 16 == 0 && kSlotV % 16 == 0, "ring");
};

// The part of shared memory that is not operands (kOffRow).
// A unit: the rows of one (tree, KV head, chunk of rows) and its tiles here.
struct TaUnit {
  int t0, t1, tiles;  // tiles t0..t1 of `tiles`; t1 = 0 ends the list
  int ctx, len, s, n, kvh, row0, rows, seq;
};
constexpr int kUnits = 4;  // units announced ahead

struct TaShared {
  float c[kUnits][kMaxRows];             // score factor, per unit
  float nm[kMaxRows];                    // kShift - maximum (0 before the row has one)
  float f[4][kMaxRows];                  // rescaling of the earlier tiles, per tile
  float red[4][4][16];                  // a softmax group's warps meet here
  float top[kMaxRows];                  // a row's maximum - kShift, kUnset before it has one
  float fin[2][kMaxRows];                // per unit parity: the factor of a row's output
  unsigned long long mask[2][kMaxRows];  // the row's node mask
  uint32_t vis[4][LRS_TREE_MAX_NODES];   // rows of a softmax group that see a node
  alignas(16) float* out[2][kMaxRows];   // the row's output
  unsigned vbad[2][8][2];                // nodes whose V is not finite, per warp that reads V
  alignas(16) int moved[4][4];  // per tile and softmax group
  TaUnit unit[kUnits];
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8];
  // Phases count tiles (of pv_*: every second one).  Before the MMA warp issues a
  // product it makes one wait for all that the product needs, as each costs it some
  // 200 clocks: qk_go, K's first half of the columns here and the last scores read
  // (k_rest: the other half); pv_go, V and P here and the last sums read.
  uint64_t qk_go, k_rest, k_half, s_full;  // k_half: the first half's scores are done
  uint64_t pv_go[2], pv_done[2], drain;
  uint64_t u_full[2], u_empty[2];
  uint64_t unit_full[kUnits], unit_empty[kUnits];
  int abort;
  uint32_t tmem;
  // the schedule
  int first, last;              // this CTA's tiles
  int tree, unit0, tile;        // of `first`: tree, unit of the tree, tile of the unit
  int active;
};
static_assert(sizeof(TaShared) <= kSharedBytes, "shared state");

__device__ __forceinline__ void ta_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ta_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void ta_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// The warp issues these converged, one lane elected: addresses stay in uniform registers.
__device__ __forceinline__ void ta_commit(uint32_t bar, uint32_t elected) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar),
      "r"(elected)
      : "memory");
}
// Four steps of K of D[tmem] (+)= A[tmem] . B[shared]; B advances by `step` (in 16 bytes).
__device__ __forceinline__ void ta_mma4(uint32_t d, uint32_t a, uint64_t b, uint32_t step, uint32_t idesc,
                                        bool accumulate, uint32_t elected) {
  asm volatile(
      "{\n .reg .pred p, q, t;\n .reg .b32 a1, a2, a3;\n .reg .b64 s, b1, b2, b3;\n"
      " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n setp.eq.b32 t, 0, 0;\n"
      " cvt.u64.u32 s, %6;\n add.u64 b1, %2, s;\n add.u64 b2, b1, s;\n add.u64 b3, b2, s;\n"
      " add.u32 a1, %1, 8;\n add.u32 a2, %1, 16;\n add.u32 a3, %1, 24;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(elected), "r"(step)
      : "memory");
}
__device__ __forceinline__ void ta_mma2(uint32_t d, uint32_t a, uint64_t b, uint32_t step, uint32_t idesc,
                                        bool accumulate, uint32_t elected) {
  asm volatile(
      "{\n .reg .pred p, q, t;\n .reg .b32 a1;\n .reg .b64 s, b1;\n"
      " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n setp.eq.b32 t, 0, 0;\n"
      " cvt.u64.u32 s, %6;\n add.u64 b1, %2, s;\n add.u32 a1, %1, 8;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(elected), "r"(step)
      : "memory");
}
__device__ __forceinline__ uint32_t ta_elect() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(e));
  return e;
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
__device__ __forceinline__ void ta_ld16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}
// The loaded registers may be used after this: it names them, so that no use moves above it.
template <int N>
__device__ __forceinline__ void ta_wait_ld(float (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; i++) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void ta_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void ta_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ float ta_max(float x) {  // over the warp's lanes
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
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

template <int N>
__device__ __forceinline__ void ta_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void ta_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// Tests a barrier's phase; an incomplete one suspends the warp for a while.
__device__ __forceinline__ bool ta_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// A run of tests by a whole warp, as few instructions as waiting warps may take from
// the others; the lanes agree on the result.
__device__ __forceinline__ bool ta_try_many(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, 2048;\n"
      "AGAIN:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " vote.sync.all.pred p, p, 0xffffffff;\n @p bra DONE;\n"
      " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n @q bra AGAIN;\n"
      "DONE:\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
constexpr uint32_t kPolls = 1u << 20;
// A whole warp's wait, which gives up after a bounded number of polls, or when
// another role did: its lanes go on together either way.
__device__ __forceinline__ bool ta_wait(TaShared& sh, uint64_t* bar, uint32_t parity) {
  const uint32_t at = smem_u32(bar);
#pragma unroll 1
  for (uint32_t i = 0; i < kPolls / 2048; i++) {
    if (ta_try_many(at, parity)) return true;
    if (__any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(&sh.abort))) return false;
  }
  *reinterpret_cast<volatile int*>(&sh.abort) = 1;
  return false;
}
// Waits for the product of P and V of this CTA's tile `tile`.
__device__ __forceinline__ bool wait_pv(TaShared& sh, uint32_t tile) {
  return ta_wait(sh, &sh.pv_done[tile & 1], tile >> 1 & 1);
}
// A position in a ring of N barriers and the parity of its current pass.
template <int N>
struct TaRing {
  uint32_t at = 0, parity = 0;
  __device__ __forceinline__ void step(uint32_t by = 1) {
    at += by;
    if (at >= N) at -= N, parity ^= 1;
  }
};

// Two f32 values as `TERMS` 16-bit pairs whose sum they are (to 2^-22, 2^-24).  LARGE: up
// to f32's largest, which round to bf16's infinity: there the first term is bf16's largest
// value and the second one the rest (an infinity leaves an infinity and a NaN).
template <bool F16, int TERMS, bool LARGE = false>
__device__ __forceinline__ void ta_split(float2 v, uint32_t (&t)[TERMS]) {
#pragma unroll
  for (int i = 0; i < TERMS; i++) {
    if constexpr (F16) {
      const __half2 h = __floats2half2_rn(v.x, v.y);
      t[i] = *reinterpret_cast<const uint32_t*>(&h);
      if (i + 1 < TERMS) v = add2(v, make_float2(-__low2float(h), -__high2float(h)));
    } else {
      if (LARGE && i == 0) {
        asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(t[i]) : "f"(v.y), "f"(v.x));
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
        t[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      if (i + 1 < TERMS)
        v = add2(v, make_float2(-__uint_as_float(t[i] << 16), -__uint_as_float(t[i] & 0xffff0000u)));
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
    const int end = a.start[t + 1];  // (compared with s first: the difference may overflow)
    ctx = a.ctx[t];
    seq = a.seq[t];
    chunks = tiles = n = 0;
    if (s == end) return true;  // no nodes: nothing else of it is looked at (padded batches)
    if (s < 0 || end < s || end > a.n_nodes || end - s > a.max_nodes || ctx < 0 || ctx > a.max_len ||
        end - s > a.max_len - ctx || seq < 0 || seq >= a.c.n_seqs) {
      atomicMax(a.c.err, kErrCacheIndex);
      return false;
    }
    n = end - s;
    len = ctx + n;
    chunks = (n * a.group + nr - 1) / nr;
    tiles = (len + kTilePos - 1) / kTilePos;
    return true;
  }
  // rows of a chunk: an even share, in whole steps of the MMA's N
  __device__ __forceinline__ int share(const TreeArgs& a) const {
    return ((n * a.group + chunks - 1) / chunks + 15) & ~15;
  }
  __device__ __forceinline__ int total(const TreeArgs& a) const { return tiles * chunks * a.c.heads; }
};

// Partial results: [2 * CTAs] segments of [NR] (m, l) and [NR][HD] sums.
struct TaDesc {
  int nseg;  // segments of the unit whose second one starts this CTA; 0 = none
  int kvh, row0, rows, s;
};
template <int HD, int NR>
__host__ __device__ constexpr size_t ta_seg_floats() {
  return 2 * NR + (size_t)NR * HD;
}

// The units as a warp takes them from the list.
struct TaFeed {
  TaUnit u;
  int index = -1;  // number of the unit in this CTA
  // False at the end of the list, or (ok = false) when the wait gave up.
  __device__ __forceinline__ bool next(TaShared& sh, int lane, bool& ok) {
    index++;
    const int at = index % kUnits;
    ok = ok && ta_wait(sh, &sh.unit_full[at], index / kUnits & 1);
    if (!ok) return false;
    u = sh.unit[at];
    __syncwarp();
    if (lane == 0) ta_arrive(&sh.unit_empty[at]);
    return u.t1 > 0;
  }
};

// The last tile's positions of V past the end, and nodes with a value that is not
// finite, become zeros (their weight may be a zero that must stay one); the
// nodes are noted.  A warp mends its own columns of the raw slot.
template <int HD, int DT, int POS>
__device__ __forceinline__ void mend_v(uint8_t* raw, int w, int lane, int p0, int ctx, int len, unsigned* vbad) {
  if constexpr (DT == LRS_KV_Q8_0) {
    uint16_t* d = reinterpret_cast<uint16_t*>(raw + q8_v_scale(HD, 0, w));
#pragma unroll 1
    for (int r = lane; r < POS; r += 32) {
      const int p = p0 + r;
      const bool bad = p >= ctx && (d[r] & 0x7c00) == 0x7c00;
      if (p >= len || bad) {
        d[r] = 0;
        if (p < len) atomicOr(&vbad[(p - ctx) >> 5], 1u << ((p - ctx) & 31));
      }
    }
  } else {
    const int h = w * 32 + lane;
#pragma unroll 1
    for (int r = max(0, ctx - p0); r < POS; r++) {
      const int p = p0 + r;
      uint16_t* b = reinterpret_cast<uint16_t*>(raw) + r * HD + h;
      uint32_t* f = reinterpret_cast<uint32_t*>(raw) + r * HD + h;
      const bool bad = DT == LRS_KV_BF16 ? (*b & 0x7f80) == 0x7f80 : (*f & 0x7f800000u) == 0x7f800000u;
      if (p >= len || bad) {
        if (DT == LRS_KV_BF16) *b = 0;
        else *f = 0;
        if (p < len) atomicOr(&vbad[(p - ctx) >> 5], 1u << ((p - ctx) & 31));
      }
    }
  }
  fence_proxy_async();  // the slot is refilled by copies later
  __syncwarp();
}

// Half of the columns of a position's K into tensor memory: lane = position, row r of the slot.
template <int HD, int DT, int NR>
__device__ __forceinline__ void decode_k(const uint8_t* raw, uint32_t at, int r, int half) {
  using S = TaShape<HD, DT, NR>;
  constexpr int kSteps = HD / 32;  // of 16 values: 8 columns a term
  at += half * kSteps * 8;
  if constexpr (DT == LRS_KV_Q8_0) {
    const uint8_t* code = raw + q8_k_code(r, half * kSteps * 16);
    const uint8_t* scale = raw + q8_k_scale(HD, r, half * kSteps / 2);
    uint4 w4 = *reinterpret_cast<const uint4*>(code);
    __half d1 = *reinterpret_cast<const __half*>(scale);
    // (two steps a turn: one took 5 % longer over the whole kernel, four no less)
#pragma unroll 2
    for (int b = 0; b < kSteps; b++) {  // the next step's words are under way
      uint32_t hi[8], lo[8];
      const __half2 d2 = __half2half2(d1);
      const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t x[2], y[2];
        ta_q8(w[i], d2, d2, x, y);
        hi[i * 2] = x[0], hi[i * 2 + 1] = x[1];
        lo[i * 2] = y[0], lo[i * 2 + 1] = y[1];
      }
      if (b + 1 < kSteps) {
        w4 = *reinterpret_cast<const uint4*>(code + (b + 1) * kPageSize * 16);
        d1 = *reinterpret_cast<const __half*>(scale + ((b + 1) >> 1) * 2);
      }
      ta_st8(at + b * 8, hi);
      ta_st8(at + HD / 2 + b * 8, lo);
    }
  } else {
    const uint8_t* row = raw + r * S::kRowK + half * kSteps * (DT == LRS_KV_BF16 ? 32 : 64);
#pragma unroll 1
    for (int b = 0; b < kSteps; b++) {
      uint32_t x[S::kA][8];
      if constexpr (DT == LRS_KV_BF16) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const uint4 w = *reinterpret_cast<const uint4*>(row + b * 32 + i * 16);
          x[0][i * 4] = w.x, x[0][i * 4 + 1] = w.y, x[0][i * 4 + 2] = w.z, x[0][i * 4 + 3] = w.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float4 f = *reinterpret_cast<const float4*>(row + b * 64 + i * 16);
          uint32_t y[S::kA];
          ta_split<false, S::kA, true>(make_float2(f.x, f.y), y);
#pragma unroll
          for (int k = 0; k < S::kA; k++) x[k][i * 2] = y[k];
          ta_split<false, S::kA, true>(make_float2(f.z, f.w), y);
#pragma unroll
          for (int k = 0; k < S::kA; k++) x[k][i * 2 + 1] = y[k];
        }
      }
#pragma unroll
      for (int k = 0; k < S::kA; k++) ta_st8(at + k * HD / 2 + b * 8, x[k]);
    }
  }
}

// A slot's positions of V into tensor memory: lane = column of the head.
template <int HD, int DT, int NR>
__device__ __forceinline__ void decode_v(const uint8_t* raw, uint32_t col, int w, int lane) {
  using S = TaShape<HD, DT, NR>;
  const int h = w * 32 + lane;
  if constexpr (DT == LRS_KV_Q8_0) {
    // 16 positions a step (8 columns a term); the next step's words are under way
    const uint8_t* code = raw + q8_v_code(HD, 0, h);
    const uint8_t* scale = raw + q8_v_scale(HD, 0, w);
    uint32_t cw[4];
    uint4 d8[2];
    auto fetch = [&](int g) {
#pragma unroll
      for (int i = 0; i < 4; i++) cw[i] = *reinterpret_cast<const uint32_t*>(code + (g * 4 + i) * HD * 4);
#pragma unroll
      for (int i = 0; i < 2; i++) d8[i] = *reinterpret_cast<const uint4*>(scale + g * 32 + i * 16);
    };
    fetch(0);
#pragma unroll 1
    for (int g = 0; g < S::kSlotPos / 16; g++) {
      uint32_t x[2][8];
      const uint32_t d[8] = {d8[0].x, d8[0].y, d8[0].z, d8[0].w, d8[1].x, d8[1].y, d8[1].z, d8[1].w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t hi[2], lo[2];
        ta_q8(cw[i], ta_u2(d[2 * i]), ta_u2(d[2 * i + 1]), hi, lo);
        x[0][i * 2] = hi[0], x[0][i * 2 + 1] = hi[1];
        x[1][i * 2] = lo[0], x[1][i * 2 + 1] = lo[1];
      }
      if (g + 1 < S::kSlotPos / 16) fetch(g + 1);
#pragma unroll
      for (int q = 0; q < 2; q++) ta_st8(col + q * (kTilePos / 2) + g * 8, x[q]);
    }
  } else {
#pragma unroll 1
    for (int g = 0; g < S::kSlotPos / 16; g++) {  // 16 positions: 8 columns a term
      uint32_t x[S::kA][8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int r = g * 16 + i * 2;
        if constexpr (DT == LRS_KV_BF16) {
          const uint16_t* b = reinterpret_cast<const uint16_t*>(raw) + r * HD + h;
          x[0][i] = (uint32_t)b[0] | (uint32_t)b[HD] << 16;
        } else {
          const float* f = reinterpret_cast<const float*>(raw) + r * HD + h;
          uint32_t y[S::kA];
          ta_split<false, S::kA, true>(make_float2(f[0], f[HD]), y);
#pragma unroll
          for (int q = 0; q < S::kA; q++) x[q][i] = y[q];
        }
      }
#pragma unroll
      for (int q = 0; q < S::kA; q++) ta_st8(col + q * (kTilePos / 2) + g * 8, x[q]);
    }
  }
}

// The scores of 16 rows of this lane's position as exponents of P:
// c * s - maximum + kShift (c is 1 but for f16), -inf where the row does not see it.
template <bool SCALED>
__device__ __forceinline__ void ta_exponents(float (&s)[16], const float* c, const float* nm, uint32_t vis) {
#pragma unroll
  for (int r = 0; r < 16; r += 4) {
    const float4 mm = *reinterpret_cast<const float4*>(nm + r);
    float2 x = make_float2(s[r], s[r + 1]), y = make_float2(s[r + 2], s[r + 3]);
    if constexpr (SCALED) {
      const float4 cc = *reinterpret_cast<const float4*>(c + r);
      x = fma2(x, make_float2(cc.x, cc.y), make_float2(mm.x, mm.y));
      y = fma2(y, make_float2(cc.z, cc.w), make_float2(mm.z, mm.w));
    } else {
      x = add2(x, make_float2(mm.x, mm.y));
      y = add2(y, make_float2(mm.z, mm.w));
    }
    s[r] = x.x, s[r + 1] = x.y, s[r + 2] = y.x, s[r + 3] = y.y;
  }
  if (__builtin_expect(vis != 0xffffu, 0)) {
#pragma unroll
    for (int r = 0; r < 16; r++)
      if (!(vis >> r & 1)) s[r] = -INFINITY;
  }
}

// q * scale * log2(e) of a unit's rows in terms, K-major core matrices: a warp
// takes 8 rows, a lane 8 columns of one at a time.  For f16 terms a power of two
// brings a row's largest magnitude to [2^10, 2^11); c is its inverse.
template <int HD, int DT, int NR>
__device__ __forceinline__ void load_q(const TreeArgs& a, const TaUnit& it, uint8_t* smem, float* c,
                                       int w, int lane) {
  using S = TaShape<HD, DT, NR>;
  const float qs = a.scale * 1.44269504088896f;
  const bool vec = a.q_ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
  const int groups = 2 * ((it.rows + 15) >> 4);
#pragma unroll 1
  for (int g8 = w; g8 < groups; g8 += 4) {
    const int gr = g8 * 8 + (lane & 7), row = it.row0 + gr, node = row / a.group;
    const float* src = a.q + (size_t)(it.s + node) * a.q_ld +
                       (size_t)(it.kvh * a.group + row - node * a.group) * HD + (lane >> 3) * 8;
    float x[HD / 32][8];
    if (gr >= it.rows) {
#pragma unroll
      for (int j = 0; j < HD / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[j][e] = 0.0f;
    } else if (vec) {
#pragma unroll
      for (int j = 0; j < HD / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const float4 f = *reinterpret_cast<const float4*>(src + j * 32 + e);
          x[j][e] = f.x, x[j][e + 1] = f.y, x[j][e + 2] = f.z, x[j][e + 3] = f.w;
        }
    } else {
#pragma unroll
      for (int j = 0; j < HD / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) x[j][e] = src[j * 32 + e];
    }
    // f16: times 2^k, k of the row's largest magnitude; the power may pass f32's
    // range, so up to 2^60 of it goes with the scale and the rest on its own
    float f0 = qs, f1 = 1.0f, down = 1.0f;
    if constexpr (S::kF16) {
      float mx = 0.0f;
#pragma unroll
      for (int j = 0; j < HD / 32; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[j][e]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16)) * fabsf(qs);
      const int e = (int)(__float_as_uint(mx) >> 23);
      if (mx > 0.0f && e < 255) {
        const int k = 137 - e, k0 = max(-60, min(60, k));
        f0 = qs * __uint_as_float((uint32_t)(127 + k0) << 23);
        f1 = ldexpf(1.0f, k - k0);
        down = ldexpf(1.0f, -k);
      }
    }
    if (lane < 8) c[gr] = down;
#pragma unroll
    for (int j = 0; j < HD / 32; j++) {
      uint32_t y[S::kB][4];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        float2 v = mul2(make_float2(x[j][2 * e], x[j][2 * e + 1]), make_float2(f0, f0));
        if constexpr (S::kF16) v = mul2(v, make_float2(f1, f1));
        uint32_t z[S::kB];
        ta_split<S::kF16, S::kB, true>(v, z);
#pragma unroll
        for (int k = 0; k < S::kB; k++) y[k][e] = z[k];
      }
      uint8_t* dst = smem + S::kOffQ + g8 * (HD / 8 * 128) + (j * 4 + (lane >> 3)) * 128 + (lane & 7) * 16;
#pragma unroll
      for (int k = 0; k < S::kB; k++)
        *reinterpret_cast<uint4*>(dst + k * S::kQTerm) = make_uint4(y[k][0], y[k][1], y[k][2], y[k][3]);
    }
  }
}

// The copies of K's or V's raw tiles into their ring, by one warp each: they take
// turns of some 100 instructions a slot, at a pace of 10 clocks and more beside the other
// warps (one warp for both was what f32 caches waited for: 8 trees of 13 nodes on 1,550 to 2,050
// positions took 54 us, now 42).
template <int HD, int DT, int NR, bool V>
struct TaCopy {
  using S = TaShape<HD, DT, NR>;
  static constexpr int kRing = V ? S::kRingV : S::kRingK, kSlot = V ? S::kSlotV : S::kSlotK;
  static constexpr int kPart = S::kTileB / (kPageSize / S::kSlotPos);  // bytes of a slot's rows
  uint64_t pol = evict_first_policy();
  uint32_t issued = 0;
  TaRing<kRing> ring;
  // The tiles of a unit; false if a wait gave up.
  __device__ __forceinline__ bool unit(const TreeArgs& a, TaShared& sh, uint8_t* smem, const TaUnit& un, int lane) {
    const uint8_t* pool = (V ? a.c.v : a.c.k) + (size_t)un.kvh * S::kTileB;
    const size_t page_bytes = (size_t)a.c.heads * S::kTileB;
    const int used = (un.len + kPageSize - 1) / kPageSize;  // the slot's pages that hold positions
    int ids = -1;                                           // a lane holds one of 32 pages
    const int first = un.t0 * S::kSlots, end = un.t1 * S::kSlots;
#pragma unroll 1
    for (int k = first; k < end; k++) {  // slots of kSlotPos positions
      const int pg = k * S::kSlotPos / kPageSize, at32 = (pg - first * S::kSlotPos / kPageSize) & 31;
      if (at32 == 0 && k * S::kSlotPos % kPageSize == 0)
        ids = pg + lane < used ? kv_page(a.c, un.seq, (pg + lane) * kPageSize) : -1;
      const int page = __shfl_sync(0xffffffffu, ids, at32);
      const uint32_t at = ring.at;
      uint64_t* full = V ? &sh.v_full[at] : &sh.k_full[at];
      if (issued >= (uint32_t)kRing && !ta_wait(sh, V ? &sh.v_empty[at] : &sh.k_empty[at], ring.parity ^ 1)) return false;
      ring.step();
      issued++;
      uint8_t* dst = smem + (V ? S::kOffV : S::kOffRing) + at * kSlot;
      const uint8_t* src = pool + max(page, 0) * page_bytes + k * S::kSlotPos % kPageSize / S::kSlotPos * kPart;
      if (page < 0) {
        if (lane == 0) ta_arrive(full);
      } else if (V || DT == LRS_KV_Q8_0) {
        if (lane == 0) {
          mbar_expect_tx(full, kPart);
          tma_load_1d(dst, src, kPart, full, pol);
        }
      } else {
        if (lane == 0) mbar_expect_tx(full, kPart);
        __syncwarp();
        constexpr int kRow = kPart / S::kSlotPos;
        for (int r = lane; r < S::kSlotPos; r += 32) tma_load_1d(dst + r * S::kRowK, src + r * kRow, kRow, full, pol);
      }
    }
    return true;
  }
  // Copies in flight land before shared memory goes away (they may outlive their
  // readers only when a wait gave up).
  __device__ __forceinline__ void land(TaShared& sh) {
    for (uint32_t i = issued > kRing ? issued - kRing : 0; i < issued; i++)
      for (uint32_t j = 0; j < kPolls && !ta_try_wait(smem_u32(V ? &sh.v_full[i % kRing] : &sh.k_full[i % kRing]),
                                                       (i / kRing) & 1); j++) {
      }
  }
};

template <int HD, int DT, int NR>
__global__ void __launch_bounds__(TaShape<HD, DT, NR>::kThreads, 1)
    tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  using S = TaShape<HD, DT, NR>;
  constexpr int kA = S::kA;
  constexpr bool kF16 = S::kF16;
  constexpr int kWarpsD = HD / 32;  // warps that own columns of V
  extern __shared__ __align__(128) uint8_t smem[];
  TaShared& sh = *reinterpret_cast<TaShared*>(smem + S::kOffRow);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  float* segs = static_cast<float*>(a.workspace);

  // barriers and tensor memory, beside the schedule
  if (tid == 32) {
#pragma unroll 1
    for (int i = 0; i < 8; i++) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], S::kSlotPos / 32);
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], kWarpsD);
    }
    mbar_init(&sh.qk_go, 4 + 4 * S::kSG);
    mbar_init(&sh.k_rest, 4);
    mbar_init(&sh.k_half, 1);
    mbar_init(&sh.s_full, 1);
    mbar_init(&sh.drain, 1);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.pv_go[i], 4 * S::kSG + (S::kVG + 1) * kWarpsD);
      mbar_init(&sh.pv_done[i], 1);
      mbar_init(&sh.u_full[i], 4 * S::kSG);
      mbar_init(&sh.u_empty[i], kWarpsD);
    }
#pragma unroll 1
    for (int i = 0; i < kUnits; i++) {
      mbar_init(&sh.unit_full[i], 1);
      mbar_init(&sh.unit_empty[i], 4 + 4 * S::kSG + (S::kVG + 1) * kWarpsD + 2);  // the warps that take units
    }
    sh.abort = 0;
    fence_barrier_init();
  }
  if (warp == S::kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sh.tmem)),
                 "r"((uint32_t)S::kTmCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---- the schedule: every CTA finds its share of all tiles ----
  {
    __shared__ int wsum[S::kThreads / 32];
    const int per = (a.n_trees + S::kThreads - 1) / S::kThreads;
    int mine = 0;
    TaTree tr;
#pragma unroll 1
    for (int i = 0; i < per; i++) {
      const int t = tid * per + i;
      if (t < a.n_trees && tr.load(a, t, NR)) mine += tr.total(a);
    }
    int incl = mine;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) wsum[warp] = incl;
    if (tid == 0) sh.active = 0;
    __syncthreads();
    int sums = lane < S::kThreads / 32 ? wsum[lane] : 0;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sums, o);
      if (lane >= o) sums += x;
    }
    const int total = __shfl_sync(0xffffffffu, sums, 31);
    const int before = __shfl_sync(0xffffffffu, sums, max(warp - 1, 0)) * (warp > 0) + incl - mine;
    const int ctas = min((int)gridDim.x, total), c = blockIdx.x;
    TaDesc d{};
    if (c < ctas) {
      // CTA i starts at tile i * (total / ctas) + i * (total % ctas) / ctas
      const unsigned quot = (unsigned)total / (unsigned)ctas, rem = (unsigned)total % (unsigned)ctas;
      auto start = [&](int i) { return (int)(quot * i + i * rem / (unsigned)ctas); };
      const int first = start(c);
      if (before <= first && first < before + mine) {  // the thread that holds the first tile's tree
        int at = before;
#pragma unroll 1
        for (int i = 0; i < per; i++) {
          const int t = tid * per + i;
          if (t >= a.n_trees || (per > 1 && !tr.load(a, t, NR))) continue;
          if (first < at + tr.total(a)) {
            const int unit = (first - at) / tr.tiles, unit0 = at + unit * tr.tiles;
            sh.tree = t;
            sh.unit0 = unit;
            sh.tile = first - unit0;
            sh.first = first;
            sh.last = start(c + 1);
            sh.active = 1;
            // this CTA starts inside a unit: the first such CTA describes it
            if (first > unit0 && start(c - 1) <= unit0) {
              d.nseg = 2;
#pragma unroll 1
              while (start(c + d.nseg - 1) < unit0 + tr.tiles) d.nseg++;
              const int share = tr.share(a);
              d.kvh = unit / tr.chunks;
              d.row0 = (unit % tr.chunks) * share;
              d.rows = min(share, tr.n * a.group - d.row0);
              d.s = tr.s;
            }
            reinterpret_cast<TaDesc*>(a.workspace)[c] = d;
            break;
          }
          at += tr.total(a);
        }
      }
    } else if (tid == 0) {
      reinterpret_cast<TaDesc*>(a.workspace)[c] = d;
    }
    segs = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + gridDim.x * sizeof(TaDesc));
  }
  ta_fence_before();
  __syncthreads();
  ta_fence_after();
  pdl_launch_dependents();
  const uint32_t tmem = __shfl_sync(0xffffffffu, sh.tmem, 0);
  const uint32_t sbase = smem_u32(smem);
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;  // this warp's lanes of tensor memory
  TaFeed feed;
  const TaUnit& it = feed.u;
  bool ok = true;
  if (!sh.active) {
    if (warp == S::kWarpMma)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                   "r"((uint32_t)S::kTmCols)
                   : "memory");
    return;
  }

  if (warp < S::kWarpV) {
    // ---- K: a lane is a position; its row into tensor memory ----
    if constexpr (S::kRegsKV < S::kRegs) ta_regs_dec<S::kRegsKV>();
    uint32_t tile = 0;
    TaRing<S::kRingK> ring;
    ring.at = warp * 32 / S::kSlotPos;
    while (feed.next(sh, lane, ok)) {
      // the last unit's scores are done with q and its factors
      if (tile > 0) ok = ta_wait(sh, &sh.s_full, (tile - 1) & 1);
      if (!ok) break;
      load_q<HD, DT, NR>(a, it, smem, sh.c[feed.index % kUnits], warp, lane);
      fence_proxy_async();
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        const uint32_t slot = ring.at;
        ok = ta_wait(sh, &sh.k_full[slot], ring.parity);
        ring.step(S::kSlots);
        const uint8_t* raw = smem + S::kOffRing + slot * S::kSlotK;
        const int r = (warp * 32 + lane) % S::kSlotPos;
#pragma unroll 1
        for (int half = 0; half < 2; half++) {
          if (ok && tile > 0) ok = ta_wait(sh, half ? &sh.s_full : &sh.k_half, (tile - 1) & 1);
          if (!ok) break;
          ta_fence_after();
          decode_k<HD, DT, NR>(raw, tmem + lanes + S::kTmK, r, half);
          __syncwarp();
          if (half && lane == 0) ta_arrive(&sh.k_empty[slot]);
          ta_wait_st();
          ta_fence_before();
          __syncwarp();
          if (lane == 0) ta_arrive(half ? &sh.k_rest : &sh.qk_go);
        }
      }
    }
  } else if (warp < S::kWarpS) {
    // ---- V: a lane is a column of the head; positions along its row ----
    if constexpr (S::kRegsKV < S::kRegs) ta_regs_dec<S::kRegsKV>();
    const int w = warp & 3, vg = (warp - S::kWarpV) >> 2;
    constexpr int kMine = S::kSlots / S::kVG;  // slots of a tile
    uint32_t tile = 0;
    TaRing<S::kRingV> ring;
    ring.at = vg * kMine;
    while (w < kWarpsD && feed.next(sh, lane, ok)) {
      // the words of the unit before last have been read
      const int par = feed.index & 1;
      if (feed.index >= 2) ok = ta_wait(sh, &sh.u_empty[par], ((feed.index >> 1) - 1) & 1);
      unsigned* vbad = sh.vbad[par][vg * 4 + w];
      if (lane < 2) vbad[lane] = 0;
      __syncwarp();
#pragma unroll 1
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        const uint32_t vb = tile % S::kNV;
        if (tile >= S::kNV) ok = wait_pv(sh, tile - S::kNV);
        ta_fence_after();
#pragma unroll 1
        for (int k = vg * kMine; k < (vg + 1) * kMine && ok; k++) {
          const uint32_t slot = ring.at;
          ok = ta_wait(sh, &sh.v_full[slot], ring.parity);
          ring.step(k + 1 == (vg + 1) * kMine ? S::kSlots - kMine + 1 : 1);
          if (!ok) break;
          uint8_t* raw = smem + S::kOffV + slot * S::kSlotV;
          const int p0 = t * kTilePos + k * S::kSlotPos;
          if (__builtin_expect(p0 + S::kSlotPos > it.ctx, 0))  // holds nodes, or positions past the end
            mend_v<HD, DT, S::kSlotPos>(raw, w, lane, p0, it.ctx, it.len, vbad);
          decode_v<HD, DT, NR>(raw, tmem + lanes + S::kTmV + vb * S::kVCols + k * (S::kSlotPos / 2), w, lane);
          __syncwarp();
          if (lane == 0) ta_arrive(&sh.v_empty[slot]);
        }
        if (!ok) break;
        ta_wait_st();
        ta_fence_before();
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.pv_go[tile & 1]);
      }
    }
  } else if (warp < S::kWarpO) {
    // ---- the softmax: a lane is a position, a group of four warps 16 of the rows ----
    if constexpr (S::kRegsS < S::kRegs) ta_regs_dec<S::kRegsS>();
    const int grp = (warp - S::kWarpS) >> 2, w = warp & 3, gt = w * 32 + lane, bar = 1 + grp;
    const int base = grp * 16, my = base + gt;  // threads 0..15 keep a row each
    float* nm = sh.nm + base;
    float2 l[8];
    uint32_t tile = 0;
    if (lane == 0) ta_arrive(&sh.qk_go);  // no scores before the first tile's
    // the four warps meet at barriers: one whose wait gave up goes on (without
    // waits, on stale data, in bounds) to the next unit's, where they leave together
    for (;;) {
      const bool more = feed.next(sh, lane, ok);
      const int u = feed.index & 1;
      const float* c = sh.c[feed.index % kUnits] + base;
      const bool whole = it.t0 == 0 && it.t1 == it.tiles, idle = base >= it.rows;  // idle: no rows here
      float* seg = segs + (size_t)(2 * blockIdx.x + (it.t0 == 0)) * ta_seg_floats<HD, NR>();
      if (more && feed.index >= 2) ok = ok && ta_wait(sh, &sh.u_empty[u], ((feed.index >> 1) - 1) & 1);
      if (more && gt < 16) {
        unsigned long long row_mask = 0;
        float* my_out = nullptr;
        if (my < it.rows) {
          const int row = it.row0 + my, node = row / a.group, g = row - node * a.group;
          my_out = whole ? a.out + (size_t)(it.s + node) * a.out_ld + (size_t)(it.kvh * a.group + g) * HD
                         : seg + 2 * NR + my * HD;
          row_mask = a.mask ? a.mask[it.s + node] : (node == 63 ? ~0ull : (2ull << node) - 1);
          if (it.n < 64) row_mask &= (1ull << it.n) - 1;
        }
        sh.mask[u][my] = row_mask;
        sh.out[u][my] = my_out;
        sh.top[my] = kUnset;
        nm[gt] = 0.0f;
      }
      if (ta_group_or(bar, !more || !ok)) break;
#pragma unroll
      for (int r = 0; r < 8; r++) l[r] = make_float2(0.0f, 0.0f);
      bool masks = false, unset = true;  // unset: a row may have no maximum yet
#pragma unroll 1
      for (int t = it.t0; t < it.t1; t++, tile++) {
        uint32_t vis = 0xffffu;  // rows that see this lane's position
        if (__builtin_expect((t + 1) * kTilePos > it.ctx, 0)) {
          if (!masks) {  // the rows that see each node, from the nodes that each row sees
            masks = true;
            const unsigned long long row_mask = sh.mask[u][base + (lane & 15)];
#pragma unroll 1
            for (int j = w; j < it.n; j += 4) {
              const uint32_t v = __ballot_sync(0xffffffffu, lane < 16 && (row_mask >> j & 1));
              if (lane == 0) sh.vis[grp][j] = v;
            }
            ta_group_sync(bar);
          }
          const int p = t * kTilePos + w * 32 + lane;
          if (p >= it.ctx) vis = p < it.len ? sh.vis[grp][p - it.ctx] : 0;
        }
        ok = ok && ta_wait(sh, &sh.s_full, tile & 1);
        ta_fence_after();
        float s[16];
        float* f = sh.f[tile & 3] + base;
        ta_ld16(tmem + lanes + S::kTmS + base, s);
        ta_wait_ld(s);
        ta_fence_before();
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.qk_go);  // the next tile's scores may come
        ta_exponents<kF16>(s, c, nm, vis);
        // does a score exceed its row's maximum by more than the margin?
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; r++) top = fmaxf(top, s[r]);
        const bool move = ta_group_or(bar, !idle && (unset || top > kLimit));
        if (__builtin_expect(move, 0)) {
          // the rows' largest exponents over the tile, to kShift
          float mx = -INFINITY;
#pragma unroll
          for (int r = 0; r < 16; r++) {
            const float v = ta_max(s[r]);
            if (lane == r) mx = v;
          }
          if (lane < 16) sh.red[grp][w][lane] = mx;
          ta_group_sync(bar);
          bool none = false;
          if (gt < 16) {
            const float old = sh.top[my];
            mx = fmaxf(fmaxf(sh.red[grp][0][gt], sh.red[grp][1][gt]), fmaxf(sh.red[grp][2][gt], sh.red[grp][3][gt]));
            // a row without a maximum takes the tile's, the others a larger one
            float by = old == kUnset ? mx - kShift : fmaxf(mx - kShift, 0.0f);
            if (!(mx > -INFINITY)) by = 0.0f;
            f[gt] = old == kUnset ? 0.0f : ta_exp2(-by);
            sh.red[grp][0][gt] = -by;
            const float now = mx > -INFINITY ? (old == kUnset ? 0.0f : old) + by : old;
            none = now == kUnset;
            sh.top[my] = now;
            nm[gt] = none ? 0.0f : -now;
          }
          unset = ta_group_or(bar, none);
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const float2 g = *reinterpret_cast<const float2*>(f + r);
            const float2 d = add2(make_float2(s[r], s[r + 1]), *reinterpret_cast<const float2*>(&sh.red[grp][0][r]));
            s[r] = d.x, s[r + 1] = d.y;
            l[r / 2].x *= g.x, l[r / 2].y *= g.y;
          }
        }
        if (gt == 0) sh.moved[tile & 3][grp] = move;
        // P in terms, N-major (a lane writes 8 rows at once), and the row sums
        const uint32_t pb = tile % S::kNP;
        // (of two buffers the older product had ended before these scores came)
        if (S::kNP == 1 && tile >= 1) ok = ok && wait_pv(sh, tile - 1);
        const int pp = w * 32 + lane;
        uint8_t* dst = smem + S::kOffP + pb * S::kPBuf + (pp >> 3) * (NR * 16) + (pp & 7) * 16 + base * 16;
        if (!idle) {
#pragma unroll
          for (int k = 0; k < 2; k++) {
            uint32_t y[S::kB][4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int r = k * 8 + e * 2;
              const float2 x = make_float2(ta_exp2(s[r]), ta_exp2(s[r + 1]));
              l[r / 2] = add2(l[r / 2], x);
              uint32_t z[S::kB];
              ta_split<kF16, S::kB>(x, z);
#pragma unroll
              for (int q = 0; q < S::kB; q++) y[q][e] = z[q];
            }
#pragma unroll
            for (int q = 0; q < S::kB; q++)
              *reinterpret_cast<uint4*>(dst + q * S::kPTerm + k * 128) =
                  make_uint4(y[q][0], y[q][1], y[q][2], y[q][3]);
          }
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.pv_go[tile & 1]);
      }
      // (the sums take the place of the last tile's shifts, which the other warps may
      // still be reading where it moved a maximum)
      ta_group_sync(bar);
      // the rows' sums over the lanes: 16 rows by 32 lanes to a row a lane pair
      float* lf = reinterpret_cast<float*>(l);
      int row = 0;
#pragma unroll
      for (int wd = 16, nn = 8; wd >= 2; wd >>= 1, nn >>= 1) {
        const bool up = lane & wd;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (i < nn) {
            const float send = up ? lf[i] : lf[i + nn], keep = up ? lf[i + nn] : lf[i];
            lf[i] = keep + __shfl_xor_sync(0xffffffffu, send, wd);
          }
        }
        if (up) row += nn;
      }
      lf[0] += __shfl_xor_sync(0xffffffffu, lf[0], 1);
      if (!(lane & 1)) sh.red[grp][w][row] = lf[0];
      ta_group_sync(bar);
      if (gt < 16) {
        const float sum = (sh.red[grp][0][gt] + sh.red[grp][1][gt]) + (sh.red[grp][2][gt] + sh.red[grp][3][gt]);
        // zeros for a row that sees nothing; one whose scores are all -inf or NaN gets NaN
        const bool nothing = it.ctx == 0 && sh.mask[u][my] == 0;
        sh.fin[u][my] = !whole ? 1.0f : nothing ? 0.0f : 1.0f / sum;
        if (!whole && my < it.rows) seg[2 * my] = sh.top[my], seg[2 * my + 1] = sum;
      }
      __syncwarp();
      if (lane == 0) ta_arrive(&sh.u_full[u]);
      ta_group_sync(bar);  // red is free again
    }
  } else if (warp < S::kWarpCopyK) {
    // ---- O: a lane is a column; sums of the tiles' products in registers ----
    ta_regs_inc<S::kRegsO>();
    const int w = warp - S::kWarpO, h = w * 32 + lane;
    uint32_t tile = 0;
    if (w < kWarpsD && lane == 0) ta_arrive(&sh.pv_go[0]);  // no sums before the first tile's
    while (w < kWarpsD && feed.next(sh, lane, ok)) {
      const int u = feed.index & 1, steps = (it.rows + 15) >> 4;
      float o[NR];
#pragma unroll
      for (int r = 0; r < NR; r++) o[r] = 0.0f;
#pragma unroll 1
      for (int t = it.t0; t < it.t1 && ok; t++, tile++) {
        ok = wait_pv(sh, tile);
        if (!ok) break;
        ta_fence_after();
        const int4 moved = *reinterpret_cast<const int4*>(sh.moved[tile & 3]);
        const float* f = sh.f[tile & 3];
#pragma unroll
        for (int c = 0; c < NR / 16; c++) {
          if (c >= steps) break;
          if (__builtin_expect(c == 0 ? moved.x : c == 1 ? moved.y : c == 2 ? moved.z : moved.w, 0)) {
#pragma unroll
            for (int i = 0; i < 16; i++) o[c * 16 + i] *= f[c * 16 + i];
          }
          float x[16];
          ta_ld16(tmem + lanes + S::kTmO + c * 16, x);
          ta_wait_ld(x);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float2 y = add2(make_float2(o[c * 16 + i], o[c * 16 + i + 1]), make_float2(x[i], x[i + 1]));
            o[c * 16 + i] = y.x, o[c * 16 + i + 1] = y.y;
          }
        }
        ta_fence_before();
        __syncwarp();
        if (lane == 0) ta_arrive(&sh.pv_go[(tile + 1) & 1]);
      }
      if (!ok) break;
      ok = ta_wait(sh, &sh.u_full[u], (feed.index >> 1) & 1);
      if (!ok) break;
      unsigned long long vbad = 0;
#pragma unroll
      for (int i = 0; i < kWarpsD; i++)
#pragma unroll
        for (int g = 0; g < S::kVG; g++)
          vbad |= sh.vbad[u][g * 4 + i][0] | (unsigned long long)sh.vbad[u][g * 4 + i][1] << 32;
      if (__builtin_expect(vbad != 0, 0)) {  // (the four warps write the same)
#pragma unroll 1
        for (int r = lane; r < NR; r += 32)
          if (sh.mask[u][r] & vbad) sh.fin[u][r] = __int_as_float(0x7fc00000);
        __syncwarp();
      }
#pragma unroll
      for (int r = 0; r < NR; r += 2) {
        if (r % 16 == 0 && r >= it.rows) break;
        const float2 f = *reinterpret_cast<const float2*>(&sh.fin[u][r]);
        const ulonglong2 at = *reinterpret_cast<const ulonglong2*>(&sh.out[u][r]);
        if (r < it.rows) reinterpret_cast<float*>(at.x)[h] = o[r] * f.x;
        if (r + 1 < it.rows) reinterpret_cast<float*>(at.y)[h] = o[r + 1] * f.y;
      }
      __syncwarp();
      if (lane == 0) ta_arrive(&sh.u_empty[u]);
    }
  } else if (warp == S::kWarpCopyK) {
    // ---- K's copies, and the list of units ----
    TaCopy<HD, DT, NR, false> copy;
    TaRing<kUnits> list;
    TaTree tr;
    int tree = sh.tree, unit = sh.unit0, tile = sh.tile, left = sh.last - sh.first;
    bool loaded = false;
#pragma unroll 1
    for (uint32_t index = 0; ok; index++) {
      // the next unit (the last entry of the list is empty)
      while (left > 0 && (!loaded || unit >= tr.chunks * a.c.heads)) {
        if (loaded) tree++, unit = 0;
        if (tree >= a.n_trees) left = 0;  // the arrays changed under the kernel
        else tr.load(a, tree, NR);
        loaded = true;
      }
      TaUnit un{};
      if (left > 0) {
        const int share = tr.share(a);
        un.t0 = tile, un.t1 = min(tr.tiles, tile + left), un.tiles = tr.tiles;
        un.ctx = tr.ctx, un.len = tr.len, un.s = tr.s, un.n = tr.n, un.seq = tr.seq;
        un.kvh = unit / tr.chunks;
        un.row0 = unit % tr.chunks * share;
        un.rows = min(share, tr.n * a.group - un.row0);
        left -= un.t1 - un.t0;
        unit++;
        tile = 0;
      }
      if (index >= kUnits) ok = ta_wait(sh, &sh.unit_empty[list.at], list.parity ^ 1);
      if (!ok) break;
      if (lane == 0) {
        sh.unit[list.at] = un;
        ta_arrive(&sh.unit_full[list.at]);
      }
      list.step();
      if (un.t1 == 0) break;
      ok = copy.unit(a, sh, smem, un, lane);
    }
    if (!ok) copy.land(sh);
  } else if (warp == S::kWarpCopyV) {
    // ---- V's copies ----
    TaCopy<HD, DT, NR, true> copy;
    while (ok && feed.next(sh, lane, ok)) ok = copy.unit(a, sh, smem, it, lane);
    if (!ok) copy.land(sh);
  } else {
    // ---- MMAs ----
    const uint32_t el = ta_elect();
    const uint32_t bar0 = smem_u32(&sh);
    auto bar_at = [&](const uint64_t* b) {
      return bar0 + (uint32_t)(reinterpret_cast<const uint8_t*>(b) - reinterpret_cast<const uint8_t*>(&sh));
    };
    // the products' terms (a | b << 4, four bits each), small ones first
    constexpr uint64_t kTerms = kA == 3   ? 0x001001201102ull
                                : kA == 2 ? 0x000000001001ull
                                          : 0x000000001020ull;
    const uint64_t qdesc = ta_desc(sbase + S::kOffQ, 128, HD / 8 * 128);
    const uint64_t pdesc = ta_desc(sbase + S::kOffP, NR * 16, 128);
    uint32_t tile = 0, qk = 0;  // products issued
    while (feed.next(sh, lane, ok)) {
      const int steps = NR == 16 ? 1 : (__shfl_sync(0xffffffffu, it.rows, 0) + 15) >> 4;
      const int tiles = __shfl_sync(0xffffffffu, it.t1 - it.t0, 0);
#pragma unroll 1
      for (int t = 0; t <= tiles && ok; t++) {
        if (t < tiles) {  // scores of tile t
          const uint32_t d = tmem + S::kTmS, idesc = ta_idesc(kF16, false, steps * 16);
#pragma unroll
          for (int half = 0; half < 2; half++) {
            ok = ok && ta_wait(sh, half ? &sh.k_rest : &sh.qk_go, qk & 1);
            if (!ok) break;
            ta_fence_after();
#pragma unroll
            for (int i = 0; i < S::kProducts; i++) {
              const uint32_t ta = (uint32_t)(kTerms >> (8 * i)) & 15, tb = (uint32_t)(kTerms >> (8 * i + 4)) & 15;
              const uint32_t ah = tmem + S::kTmK + ta * (HD / 2) + half * (HD / 4);
              const uint64_t qh = qdesc + tb * (S::kQTerm >> 4) + half * (HD / 2);
              if constexpr (HD == 128) ta_mma4(d, ah, qh, 16, idesc, (half | i) != 0, el);
              else ta_mma2(d, ah, qh, 16, idesc, (half | i) != 0, el);
            }
            ta_commit(bar_at(half ? &sh.s_full : &sh.k_half), el);
          }
          if (!ok) break;
          qk++;
        }
        if (t > 0) {  // values of the tile before it
          const uint32_t vb = tile % S::kNV, pb = tile % S::kNP;
          ok = ta_wait(sh, &sh.pv_go[tile & 1], tile >> 1 & 1);
          if (!ok) break;
          ta_fence_after();
          const uint32_t d = tmem + S::kTmO, idesc = ta_idesc(kF16, true, steps * 16);
          const uint32_t av = tmem + S::kTmV + vb * S::kVCols;
          const uint64_t pd = pdesc + (uint64_t)(pb * (S::kPBuf >> 4));
#pragma unroll
          for (int i = 0; i < S::kProducts; i++) {
            const uint32_t ta = (uint32_t)(kTerms >> (8 * i)) & 15, tb = (uint32_t)(kTerms >> (8 * i + 4)) & 15;
            const uint32_t at = av + ta * (kTilePos / 2);
            const uint64_t pt = pd + tb * (S::kPTerm >> 4);
            ta_mma4(d, at, pt, 2 * NR, idesc, i != 0, el);
            ta_mma4(d, at + 32, pt + 8 * NR, 2 * NR, idesc, true, el);
          }
          ta_commit(bar_at(&sh.pv_done[tile & 1]), el);
          tile++;
        }
      }
    }
    if (!ok) {  // MMAs in flight end before their memory goes away
      ta_commit(bar_at(&sh.drain), el);
      for (uint32_t j = 0; j < kPolls && !ta_try_wait(smem_u32(&sh.drain), 0); j++) {
      }
    }
  }
  if (!ok) atomicMax(a.c.err, LRS_ERR_DEVICE_TIMEOUT);
  ta_fence_before();
  __syncthreads();
  if (warp == S::kWarpMma) {
    ta_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"((uint32_t)S::kTmCols)
                 : "memory");
  }
}

// Merges the segments of the units that several CTAs share: block (c, y) rows
// 4 y .. 4 y + 3 of the unit that CTA c is the second one of.  A segment in which a row
// has no maximum (kUnset) saw nothing of the row's, or scores that are all -inf or NaN: its
// sums are 0 or NaN, and are added like the others', so that NaN stays.  Units of several
// tiles have committed positions, so that no row here sees nothing at all.
template <int HD, int NR>
__global__ void __launch_bounds__(HD * 4) tree_combine_kernel(const __grid_constant__ TreeArgs a, int ctas) {
  pdl_wait();
  const int c = blockIdx.x + 1, h = threadIdx.x % HD, r = blockIdx.y * 4 + threadIdx.x / HD;
  const TaDesc d = reinterpret_cast<const TaDesc*>(a.workspace)[c];
  if (d.nseg == 0 || r >= d.rows) return;
  constexpr size_t kSeg = ta_seg_floats<HD, NR>();
  const float* segs = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + ctas * sizeof(TaDesc));
  // the first segment ends CTA c - 1, the others start CTAs c, c + 1, ...
  const float* first = segs + (2 * (size_t)(c - 1) + 1) * kSeg;
  const float* next = segs + 2 * (size_t)c * kSeg;
  float m = first[2 * r], l = first[2 * r + 1], o = first[2 * NR + r * HD + h];
#pragma unroll 4
  for (int i = 1; i < d.nseg; i++, next += 2 * kSeg) {
    const float mi = next[2 * r], li = next[2 * r + 1], oi = next[2 * NR + r * HD + h];
    const float top = fmaxf(m, mi), f = exp2f(m - top), g = exp2f(mi - top);
    l = l * f + li * g;
    o = o * f + oi * g;
    m = top;
  }
  const int row = d.row0 + r;
  a.out[(size_t)(d.s + row / a.group) * a.out_ld + ((size_t)d.kvh * a.group + row % a.group) * HD + h] =
      o / l;
}

long long tiles_of(const TreeArgs& a, int nr) {
  return (long long)a.n_trees * a.c.heads * ((a.max_nodes * a.group + nr - 1) / nr) *
         ((a.max_len + kTilePos - 1) / kTilePos);
}

// Rows a unit: 16 while that gives a CTA two tiles at most, as the 16-row kernel starts
// and ends sooner; else the smallest of 16, 32, 64 that holds a tree's rows, as each unit
// decodes K and V for itself.  Measured back to back with 16 / 32 / 64 rows, 4 KV heads x 7
// x 128: q8_0, 8 nodes on 1,100 positions 14.5 / 14.5 / 18.3 us, 5 on 3,000 17.6 / 18.6 /
// 20.7 us, 64 trees of one node on 700 to 1,100 35 / 37 / 41 us, but 64 of 8 on 2,100 to
// 4,100 216 / 145 / 104 us; bf16, 64 of one 76 / 76 / 80 us, 64 of 8 695 / 395 / 224 us; f32,
// 2 x 6 x 128, 8 of 13 on 1,500 to 2,050 64 / 43 / 43 us.
int unit_rows(const TreeArgs& a, int sms) {
  const int rows = a.max_nodes * a.group;
  return rows <= 16 || tiles_of(a, 16) <= 2ll * sms ? 16 : rows <= 32 ? 32 : 64;
}

int grid_ctas(const TreeArgs& a, int sms) {
  return (int)std::min<long long>(sms, tiles_of(a, unit_rows(a, sms)));
}

template <int HD, int DT, int NR>
cudaError_t launch(const TreeArgs& a, int sms, cudaStream_t st) {
  using S = TaShape<HD, DT, NR>;
  static std::atomic<uint64_t> attr{0};
  cudaError_t e = set_smem_once(attr, (const void*)tree_attention_kernel<HD, DT, NR>, S::kSmem);
  if (e != cudaSuccess) return e;
  const int ctas = grid_ctas(a, sms);
  tree_attention_kernel<HD, DT, NR><<<ctas, S::kThreads, S::kSmem, st>>>(a);
  e = cudaGetLastError();
  // units of one tile are never shared
  if (e != cudaSuccess || ctas < 2 || a.max_len <= kTilePos) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas - 1, NR / 4);
  cfg.blockDim = dim3(HD * 4);
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
  switch (unit_rows(a, sms)) {
    case 16: return launch<HD, DT, 16>(a, sms, st);
    case 32: return launch<HD, DT, 32>(a, sms, st);
    default: return launch<HD, DT, 64>(a, sms, st);
  }
}

}  // namespace

size_t tree_attention_workspace_bytes(const TreeArgs& a, int hd, int sms) {
  if (a.n_trees == 0 || a.n_nodes == 0) return 0;
  const size_t nr = unit_rows(a, sms);
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
