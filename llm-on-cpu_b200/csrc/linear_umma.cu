// linear_umma.cu — dense INT4 products of tens of tokens on the 5th-generation
// tensor cores (tcgen05.mma): weights times bf16 activations, exact products,
// fp32 sums.
//
// A CTA holds 128 weight rows (eight 16-row tiles of the packed stream, see
// linear.cu) against up to 64 tokens over a share of K, in steps of 128 k.  The
// A operand starts from q - zp (GPTQ: q - 8, and z + 8 s times the group's
// activation sums xs is added beside), an exact integer of four bits.  The scale
// belongs to a row and a group:
//
//   groups of 128 k: an accumulator in TMEM per step, drained while the next are
//     computed,  acc[row][t] += s[row, g] * P[row][t]  (GPTQ: + (z + 8 s) * xs);
//   smaller groups: (q - zp) * s, 4 x 11 bits, as the exact sum of two bf16
//     operands, hi + lo.  With s = s_hi + s_lo (8 + 3 bits) hi = (q - zp) * s_hi
//     rounded, and lo = (q - zp) * s_lo + ((q - zp) * s_hi - hi) has at most 8
//     bits: three packed instructions per pair of weights and twice the MMAs, but
//     no scale is left to apply, so an accumulator takes two steps.  The zeros are
//     a product like the others, in six more columns of A and B per group: z + 8 s
//     and xs, three bf16 terms (24 bits) each, the six largest of their products.
//     A drain per group of 32 instead took 51 us at T = 37, 4101 x 7264 with zeros,
//     and the zeros added in the drain 28.7 us, against 18.1.
//     Two steps per drain, not four: the tensor core's sums are truncated, and
//     four steps' err by 8e-7 of the output's norm at K = 16384, two steps' by 6e-7.
//
//   TMEM   accumulators of 64 columns, one per issuer (4; small groups 2), then
//          the A slots: 4 of 64 columns (128 rows x 128 k, bf16 pairs), or 3 of
//          hi and lo
//   shared memory: B slots (N tokens x 128 k, K-major, 128-byte swizzle, and the
//          zeros' columns), the weight blocks and scales as they are stored, the
//          activation sums of 16 steps or the zeros' columns of A
//
//   warps 0..3    an elected lane issues the MMAs of the steps j % 4 == warp (an MMA
//                 costs its issuing thread 75 to 100 cycles); small groups: two warps
//   warp  4       activations by TMA (unaligned ones: warps 6, 7 with plain loads)
//   warp  5       weights: a bulk copy per tile and block of two steps, blocks ahead
//   warps 6, 7    GPTQ: the group sums of what landed (mma.sync with ones and zeros)
//   warps 8..15   dequantisers, thread = weight row = TMEM lane, even and odd steps
//   warps 16..23  drain, one lane quadrant and half of the columns each
//
// Loads through registers or cp.async were the bound before: an SM got 15 bytes per
// clock of activations that all CTAs read (T = 64, 11008 x 4096: 22.8 us, now 19.2;
// groups of 32: 42.4, now 26.0).  Now it is the instructions of 24 warps, of which a
// step of 128 k costs 0.45 us, 0.6 with small groups; groups of 128 wait for the
// drain, small groups for the dequantisers and, with zeros, the sums.
//
// K splits over the CTAs of a cluster; their partial sums meet in distributed
// shared memory and are added in rank order.  Every wait is bounded; one that
// gives up sets the handle's error word (llmoc_int4_linear_status) and every role
// drains and exits.
//
// Why the parity waits are sound.  A waiter looks at every phase of a barrier before
// the next can complete, and an arrival comes after the phase before is complete.
// The rings of the weights, activations and accumulators give both, as a slot and
// its barriers turn together (a dequantising or drain warp waits for each weight
// block, also for a first one of which it needs no step).  `full` and `empty` do
// not belong to a slot but turn by steps, kSteps of them, since all that holds the
// four warps of a group and the two groups of dequantisers together is the wait for
// `empty` of step j - kASlots.  With 3 A slots it says that the other group was
// through with step j - 3, so that j - 6 is complete, and while a warp is at step j
// the other group completes no step beyond j + 1: 6 entries.  (With 4, as many as
// B slots, a warp could arrive for step j while one beside it had not for j - 4, and
// the MMAs read unwritten rows; and a group late at its wait for step j - 3 missed
// it once j + 1 was complete, which has the same parity.)  With 4 A slots it is a
// wait for the warp's own group: a warp at step j knows that all of them are through
// with j - 4, and so with j - 6.  tests/test_umma_waits.py walks the interleavings.
// Sums of step j are overwritten by step j + 16's, whose activations have landed
// only after the MMAs of step j + 10 completed; their issuer had waited until every
// drain warp gave back step j + 6's accumulator, which each does after it is
// through with step j.
#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

#include "ops.cuh"
#include "umma_dev.cuh"

namespace llmoc {

namespace {

constexpr int kUCols = 64;   // most tokens of a CTA
constexpr int kUSide = 16;   // slots of activation sums (groups of 128)
constexpr int kULinThreads = 24 * 32;

template <int FL, bool AWQ>
struct UCfg {
  static constexpr bool kSplit = FL < 4;             // the scale in the A operand, as two bf16 terms
  static constexpr bool kSums = !AWQ;                // activation sums are needed
  static constexpr bool kZCols = kSums && kSplit;    // zeros as more columns of A, the sums as more of B
  static constexpr int kGs = 4 / FL;                 // scale groups per step
  static constexpr int kAcc = kSplit ? 2 : 4;        // accumulators, each an issuer's
  static constexpr int kHold = kSplit ? 2 : 1;       // steps added up in an accumulator between drains
  static constexpr int kASlots = kSplit ? 3 : 4;     // A slots
  static constexpr int kACols = kSplit ? 128 : 64;   // TMEM columns of one
  static constexpr int kXSlots = kZCols ? 4 : 6;     // B slots
  static constexpr int kSteps = 6;                   // entries of the barrier rings `full` and `empty`
  static constexpr int kRing = kZCols ? 3 : 6;       // blocks of weights, two steps each
  static constexpr int kBB = lin_block_bytes(FL, !AWQ);
  static constexpr int kParts = kZCols ? 3 : 2;      // 64-wide parts of a B slot
  static constexpr int kSideBytes = kZCols ? kASlots * 16384 : kSums ? kUSide * kUCols * 4 : 0;
  static constexpr int smem(int n) { return 1024 + kXSlots * kParts * n * 128 + kSideBytes + kRing * 8 * kBB; }
  static_assert(kAcc * 64 + kASlots * kACols <= 512, "TMEM");
  static_assert(smem(kUCols) <= 226 * 1024, "shared memory");
  static_assert(kXSlots <= kSteps && kSteps == 6 && (kASlots == 3 || kASlots == 4), "the turns argued above");
};

struct UPlan {
  int N;       // tokens of a CTA, a multiple of 16
  int c;       // CTAs of a cluster, splitting K
  int steps;   // 128-wide steps of K
  int tma;     // the activations come by TMA
};

__device__ __forceinline__ uint32_t nib16(uint32_t w) {  // (16 + q_lo, 16 + q_hi) as bf16
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(0x00780078u), "r"(0x41804180u));
  return d;
}
__device__ __forceinline__ uint32_t bf2_sub(uint32_t x, uint32_t y) {
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// two fp32 sums at once
__device__ __forceinline__ uint64_t f2_pack(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ float2 f2_unpack(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t x, uint64_t y) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  return d;
}
__device__ __forceinline__ uint32_t bf2_pack(float lo, float hi) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// v = v0 + v1 + v2 in bf16 terms, 24 bits: returned as their rounded values
struct Terms {
  float v0, v1, v2;
};
__device__ __forceinline__ Terms bf16_terms(float v) {
  Terms r;
  r.v0 = __bfloat162float(__float2bfloat16_rn(v));
  r.v1 = __bfloat162float(__float2bfloat16_rn(v - r.v0));
  r.v2 = v - r.v0 - r.v1;
  return r;
}
// D[tmem] += A[smem] * B[smem]^T over K = 16 * ks
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, int ks) {
  for (int i = 0; i < ks; ++i)
    asm volatile("tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, 1;" ::"r"(d), "l"(da + 2 * i), "l"(db + 2 * i),
                 "r"(idesc));
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// d += a b of m16n8k16
__device__ __forceinline__ void mma_sum(float (&d)[4], const uint32_t (&a)[4], uint32_t b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%8}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b));
}
__device__ __forceinline__ void u_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// tcgen05.st of 16 columns of this warp's lane quadrant
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ uint32_t bf2_mul(uint32_t x, uint32_t y) {
  const __nv_bfloat162 r =
      __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf2_fma(uint32_t x, uint32_t y, uint32_t z) {
  const __nv_bfloat162 r =
      __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y),
              *reinterpret_cast<const __nv_bfloat162*>(&z));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf2_fms(uint32_t x, uint32_t y, uint32_t z) {  // x y - z
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y),
                                   __hneg2(*reinterpret_cast<const __nv_bfloat162*>(&z)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t bf2_dup(float f) {
  const __nv_bfloat162 r = __float2bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&r);
}

// C columns of this warp's lane quadrant
template <int C>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float (&v)[C]) {
  if constexpr (C == 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
  else
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(p));
  return p != 0;
}

template <int FL, bool AWQ>
__global__ void __launch_bounds__(kULinThreads, 1)
    k_lin_umma(const LinArgs a, const UPlan p, const __grid_constant__ CUtensorMap xmap) {
  using C = UCfg<FL, AWQ>;
  constexpr bool kSplit = C::kSplit, kSums = C::kSums, kZCols = C::kZCols;
  constexpr int kGs = C::kGs, kBB = C::kBB, kAcc = C::kAcc, kASlots = C::kASlots, kXSlots = C::kXSlots, kRing = C::kRing,
                kSteps = C::kSteps;
  constexpr int kGrp = 8 / FL;  // groups per block of the stream
  extern __shared__ __align__(1024) unsigned char usm[];
  __shared__ __align__(8) uint64_t xFull[kXSlots], full[kSteps], empty[kSteps], wFull[kRing], wEmpty[kRing], accFull[4],
      accEmpty[4], done[4];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;
  const int half_bytes = p.N * 128, slot_bytes = half_bytes * C::kParts;  // 64-wide parts of a B slot
  unsigned char* ringB = usm + ((1024 - (su32(usm) & 1023)) & 1023);
  unsigned char* side = ringB + kXSlots * slot_bytes;
  unsigned char* ringZ = side;                         // small groups: [kASlots][128 rows][128 bytes]
  float* xs = reinterpret_cast<float*>(side);          // groups of 128: [kUSide][kUCols]
  unsigned char* ringW = side + C::kSideBytes;         // [kRing][8 tiles][kBB]
  auto warp_wait = [&](uint64_t* b, uint32_t par) {  // by a whole warp
    return __all_sync(0xffffffffu, mb_wait(b, par, &abort_flag)) != 0;
  };
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, quad = warp & 3;
  const int rank = blockIdx.x % p.c, unit = blockIdx.x / p.c, tok0 = blockIdx.y * kUCols;
  const int j0 = p.steps * rank / p.c, n = p.steps * (rank + 1) / p.c - j0;  // this CTA's steps
  const int b0 = j0 >> 1, nblk = ((j0 + n + 1) >> 1) - b0;                   // and blocks of the stream
  const size_t tile_bytes = (size_t)a.nb * kBB;
  // the steps after which an accumulator is drained: every kHold-th of its issuer's,
  // the issuers' in turn, and its last
  auto drained = [&](int j) { return !kSplit || (j / kAcc + j) % C::kHold == 0 || j + kAcc >= n; };
  const int halves = p.N > 16 ? 2 : 1;  // drain warps per quadrant with columns
  if (threadIdx.x == 0) {
    for (int s = 0; s < kXSlots; ++s) mb_init(&xFull[s], 1);
    for (int s = 0; s < kSteps; ++s) {
      mb_init(&full[s], 4 + (p.tma && !kSums ? 0 : 2));  // four dequantising warps, the activation warps
      mb_init(&empty[s], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mb_init(&wFull[i], 1);
      mb_init(&wEmpty[i], 8 + (kSplit ? 0 : 4 * halves));  // the dequantising warps, the drain warps
    }
    for (int i = 0; i < kAcc; ++i) {
      mb_init(&accFull[i], 1);
      mb_init(&accEmpty[i], 4 * halves);
      mb_init(&done[i], 1);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&tmem_base)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;
  bool ok = true;
  auto load_block = [&](int i) {  // by the weight warp: lanes 0..7, a tile each
    const int slot = i % kRing;
    if (lane == 0) mb_expect(&wFull[slot], 8 * kBB);
    __syncwarp();
    if (lane < 8)
      bulk_g2s(su32(ringW) + (slot * 8 + lane) * kBB,
               a.q + (size_t)min(unit * 8 + lane, a.mt - 1) * tile_bytes + (size_t)(b0 + i) * kBB, kBB, &wFull[slot]);
  };
  if (warp == 5)  // the weights do not depend on the previous kernel
    for (int i = 0; i < kRing && i < nblk; ++i) load_block(i);
  grid_dep_wait();
  grid_dep_release();
  float* red = reinterpret_cast<float*>(ringB);  // sums [column][row], over the B slots
  const int h2 = (warp - 16) >> 2;                            // drain: column half
  const int colw = ((p.N + 31) >> 5) << 4;                    // columns of half 0
  const int cbeg = h2 * colw, ncol = min(p.N - cbeg, colw);  // this warp's columns (16 or 32, or none)

  if (warp < 4) {
    if (warp < kAcc && elect_one()) {
      const uint32_t idesc = instr_desc(128, p.N);
      const uint32_t half = (uint32_t)half_bytes >> 4;  // descriptor units to the next 64 k
      const uint64_t dB0 = smem_desc(su32(ringB)), dZ = smem_desc(su32(ringZ));
      const uint32_t dacc = tmem + warp * 64;
      bool fresh = true;  // the next MMAs start a new sum
      uint32_t drains = 0;
      for (int j = warp; j < n; j += kAcc) {
        const int slot = j % kXSlots, step = j % kSteps;
        const uint32_t ta = tmem + kAcc * 64 + j % kASlots * C::kACols;
        const uint64_t dB = dB0 + slot * (slot_bytes >> 4);
        // the step's operands, and the accumulator's last sum drained
        if ((p.tma && !kSums && !mb_wait(&xFull[slot], j / kXSlots & 1, &abort_flag)) ||
            !mb_wait(&full[step], j / kSteps & 1, &abort_flag) ||
            (fresh && drains && !mb_wait(&accEmpty[warp], (drains - 1) & 1, &abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        umma_ts_k64(dacc, ta, dB, idesc, !fresh);
        umma_ts_k64(dacc, ta + 32, dB + half, idesc, 1);
        if (kSplit) {
          umma_ts_k64(dacc, ta + 64, dB, idesc, 1);
          umma_ts_k64(dacc, ta + 96, dB + half, idesc, 1);
        }
        if (kZCols) umma_ss(dacc, dZ + j % kASlots * 1024, dB + 2 * half, idesc, kGs / 2);
        fresh = drained(j);
        if (fresh) {
          umma_commit(&accFull[warp]);
          ++drains;
        }
        umma_commit(&empty[step]);
      }
      // every MMA this thread issued has completed once its `done` fires
      umma_commit(&done[warp]);
      const long long t0 = clock64();
      while (!mb_try(&done[warp], 0))
        if (clock64() - t0 > kWaitCycles) {
          ok = false;
          break;
        }
    }
    __syncwarp();
  } else if (warp == 4) {
    if (p.tma && lane == 0) {
      int j = 0;
      for (; j < n; ++j) {
        const int slot = j % kXSlots;
        if (j >= kXSlots && !mb_wait(&empty[(j - kXSlots) % kSteps], (j - kXSlots) / kSteps & 1, &abort_flag)) {
          ok = false;
          break;
        }
        mb_expect(&xFull[slot], 2 * half_bytes);
        const uint32_t dst = su32(ringB) + slot * slot_bytes;
        tma_load_2d(dst, &xmap, (j0 + j) * 128, tok0, &xFull[slot]);
        tma_load_2d(dst + half_bytes, &xmap, (j0 + j) * 128 + 64, tok0, &xFull[slot]);
      }
      if (!ok) drain_ring(xFull, kXSlots, j, 0, 1);  // no copy is in flight when the CTA leaves
    }
    __syncwarp();
  } else if (warp == 5) {
    int i = min(kRing, nblk);
    for (; i < nblk; ++i) {
      if (!warp_wait(&wEmpty[i % kRing], (i / kRing - 1) & 1)) {
        ok = false;
        break;
      }
      load_block(i);
    }
    if (!ok) drain_ring(wFull, kRing, i, 0, 1);
  } else if (warp < 8) {
    // activations of 32 tokens: loaded here where TMA cannot, and their group sums
    const int aw = warp - 6, g = lane >> 2, t = lane & 3, pc = lane & 15;
    // The sums come from mma.sync: 16 tokens times a B that is one in the columns of
    // the group at hand, so that lane (g, t) ends with tokens g and g + 8 of group q
    constexpr int kDup = 4 / kGs;  // lanes with the same sums: they write in turn
    const int q = t / kDup;
    const int row0[2] = {32 * aw, 32 * aw + (32 * aw + 16 < p.N ? 16 : 0)};  // twice 16 tokens, or the same ones
    auto sums = [&](int j) {
      const uint32_t slot = su32(ringB) + j % kXSlots * slot_bytes;
      float d[2][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 64 k: 16-byte pieces 2 k, 2 k + 1
        uint32_t x[2][4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            ldmatrix4(slot + (row0[r] + (lane & 15)) * 128 + h * half_bytes + (((2 * k + (lane >> 4)) ^ (lane & 7)) << 4),
                      x[r][k]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int r = 0; r < 2; ++r) mma_sum(d[r], x[r][k], (4 * h + k) / (2 * FL) == g / (2 * kDup) ? 0x3F803F80u : 0u);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (kDup > 1 && (t & 1) != (c & 1)) continue;
        const float x = d[c >> 1][2 * (c & 1)];
        const int row = row0[c >> 1] + g + 8 * (c & 1);
        if (kZCols) {
          const Terms m = bf16_terms(x);
          const uint32_t w[3] = {bf2_pack(m.v0, m.v1), bf2_pack(m.v2, m.v0), bf2_pack(m.v1, m.v0)};
#pragma unroll
          for (int c = 0; c < 3; ++c) {
            const int wi = 3 * q + c;
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(slot + 2 * half_bytes + row * 128 +
                                                         (((wi >> 2) ^ (row & 7)) << 4) + (wi & 3) * 4),
                         "r"(w[c])
                         : "memory");
          }
        } else {
          xs[(j & (kUSide - 1)) * kUCols + row] = x;
        }
      }
    };
    if (kZCols)  // columns past the last group's stay zero
      for (int s = 0; s < kXSlots; ++s)
        for (int i = lane; i < 32 * 8 && 32 * aw + (i >> 3) < p.N; i += 32)
          asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(su32(ringB) + s * slot_bytes + 2 * half_bytes +
                                                                        32 * aw * 128 + i * 16),
                       "r"(0)
                       : "memory");
    if (!p.tma || kSums)
      for (int j = 0; j < n; ++j) {
        const int slot = j % kXSlots;
        if (p.tma) {
          ok = warp_wait(&xFull[slot], j / kXSlots & 1);
        } else {
          ok = j < kXSlots || warp_wait(&empty[(j - kXSlots) % kSteps], (j - kXSlots) / kSteps & 1);
          const int k = (j0 + j) * 128 + pc * 8;
          for (int i = lane >> 4; ok && i < 32 && 32 * aw + i < p.N; i += 2) {
            const int r = 32 * aw + i;
            uint32_t w[4] = {0, 0, 0, 0};
            if (tok0 + r < a.T && k < a.K) {
              const unsigned short* u = reinterpret_cast<const unsigned short*>(a.X + (long long)(tok0 + r) * a.ldx + k);
#pragma unroll
              for (int c = 0; c < 4; ++c) w[c] = u[2 * c] | ((uint32_t)u[2 * c + 1] << 16);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(su32(ringB) + slot * slot_bytes +
                                                                          (pc >> 3) * half_bytes + r * 128 +
                                                                          (((pc ^ r) & 7) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
        }
        if (!ok) break;
        __syncwarp();
        if (kSums && 32 * aw < p.N) sums(j);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mb_arrive(&full[j % kSteps]);
      }
  } else if (warp < 16) {
    // the words of this thread's row: 8 bytes of each 16 of its pair of rows' 64 in
    // every chunk of its tile, conflict-free
    const int dg = (warp - 8) >> 2, g = lane & 7, hi = (lane >> 3) & 1, row = quad * 32 + lane;  // dg: even or odd steps
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16) + kAcc * 64;
    const uint32_t zp2 = (0x4180u + ((AWQ ? (uint32_t)a.zp : 8u) << 3)) * 0x10001u;  // 16 + zp, zp < 16
    uint32_t woff[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) woff[t] = (2 * quad + (lane >> 4)) * kBB + (g * 4 + (t ^ (g >> 1))) * 16 + hi * 8;
    if (dg == 1 && (j0 & 1)) {  // the first block holds no step of this group
      ok = warp_wait(&wFull[0], 0);
      if (lane == 0) mb_arrive(&wEmpty[0]);
    }
    for (int j = dg; j < n && ok; j += 2) {
      const int bi = ((j0 + j) >> 1) - b0, slot = bi % kRing, odd = (j0 + j) & 1;
      if (j >= kASlots) {  // the A slot's last MMAs
        const int o = j - kASlots;
        if (!warp_wait(&empty[o % kSteps], o / kSteps & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      if (!warp_wait(&wFull[slot], (bi / kRing) & 1)) {
        ok = false;
        break;
      }
      const unsigned char* wb = ringW + slot * 8 * kBB;
      const uint32_t ta = tl + j % kASlots * C::kACols;
      uint32_t shi[kGs], slo[kGs];  // the groups' scales as pairs of two bf16 terms
      if (kSplit) {
        uint32_t zw[16];  // three bf16 terms of z + 8 s against three of the sum: six columns a group
#pragma unroll
        for (int c = 0; c < 16; ++c) zw[c] = 0;
#pragma unroll
        for (int c = 0; c < kGs; ++c) {
          const unsigned char* sp = wb + (row >> 4) * kBB + 2048 + (odd * kGs + c) * 32 + g * 4 + hi * 2;
          const float f = __half2float(*reinterpret_cast<const __half*>(sp));
          shi[c] = bf2_dup(f);
          slo[c] = bf2_dup(f - __uint_as_float(shi[c] << 16));
          if (kZCols) {
            const Terms m = bf16_terms(fmaf(8.f, f, __half2float(*reinterpret_cast<const __half*>(sp + kGrp * 32))));
            zw[3 * c] = bf2_pack(m.v0, m.v0), zw[3 * c + 1] = bf2_pack(m.v0, m.v1), zw[3 * c + 2] = bf2_pack(m.v1, m.v2);
          }
        }
        if (kZCols) {
          const uint32_t zp = su32(ringZ) + j % kASlots * 16384 + row * 128;
#pragma unroll
          for (int c = 0; c < kGs; ++c)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(zp + ((c ^ (row & 7)) << 4)), "r"(zw[4 * c]),
                         "r"(zw[4 * c + 1]), "r"(zw[4 * c + 2]), "r"(zw[4 * c + 3])
                         : "memory");
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint2 raw[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) raw[t] = *reinterpret_cast<const uint2*>(wb + (odd * 2 + h) * 512 + woff[t]);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t r[16], lo[16];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t w = kb ? raw[t].y : raw[t].x;  // k = 32 kb + 8 t + {0..7}
#pragma unroll
            for (int c = 0; c < 4; ++c) r[4 * t + c] = bf2_sub(nib16(__funnelshift_r(w, w, 4 * c)), zp2);
          }
          if (kSplit) {
            const uint32_t sh = shi[kGs == 4 ? 2 * h + kb : h], sl = slo[kGs == 4 ? 2 * h + kb : h];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const uint32_t q = r[c];
              r[c] = bf2_mul(q, sh);
              lo[c] = bf2_fma(q, sl, bf2_fms(q, sh, r[c]));
            }
            tmem_st16(ta + 64 + 32 * h + 16 * kb, lo);
          }
          tmem_st16(ta + 32 * h + 16 * kb, r);
        }
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      if (kZCols) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mb_arrive(&full[j % kSteps]);
        mb_arrive(&wEmpty[slot]);
      }
    }
  } else if (ncol > 0) {
    const uint32_t tq = tmem + ((uint32_t)(quad * 32) << 16) + cbeg;
    const int row = quad * 32 + lane;
    uint64_t acc[16];  // pairs of columns
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0;
    int slot = 0, wpar = 0;  // the weight block's place and parity
    uint32_t phase = 0;  // bit w: parity of accumulator w's next drain
    // cols: this warp's columns, as a constant
    auto drain = [&](auto cols) {
      constexpr int kC = decltype(cols)::value;
      for (int j = 0; j < n; ++j) {
        if (!drained(j)) continue;
        const int buf = j % kAcc;
        float f = 1.f, zf = 0.f;  // the row's scale, and z + 8 s
        if (!kSplit) {
          const int odd = (j0 + j) & 1;
          if (!(odd && j) && !warp_wait(&wFull[slot], wpar)) {  // once a block
            ok = false;
            break;
          }
          // pair (g, g + 8) of the row's tile
          const unsigned char* sp =
              ringW + (slot * 8 + (row >> 4)) * kBB + 2048 + odd * 32 + (row & 7) * 4 + ((row >> 3) & 1) * 2;
          f = __half2float(*reinterpret_cast<const __half*>(sp));
          if (kSums) zf = fmaf(8.f, f, __half2float(*reinterpret_cast<const __half*>(sp + kGrp * 32)));
          if (odd || j == n - 1) {
            __syncwarp();
            if (lane == 0) mb_arrive(&wEmpty[slot]);
            if (++slot == kRing) slot = 0, wpar ^= 1;
          }
        }
        if (!warp_wait(&accFull[buf], (phase >> buf) & 1)) {
          ok = false;
          break;
        }
        phase ^= 1u << buf;
        tc_fence_after();
        float v[kC];
        tmem_ld<kC>(tq + buf * 64, v);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mb_arrive(&accEmpty[buf]);
        if (kSplit) {
#pragma unroll
          for (int c = 0; c < kC; c += 2) acc[c >> 1] = f2_add(acc[c >> 1], f2_pack(v[c], v[c + 1]));
        } else {
          const uint64_t s = f2_pack(f, f);
#pragma unroll
          for (int c = 0; c < kC; c += 2) acc[c >> 1] = f2_fma(s, f2_pack(v[c], v[c + 1]), acc[c >> 1]);
          if (kSums) {
            const uint64_t z = f2_pack(zf, zf);
            const float* x = xs + (j & (kUSide - 1)) * kUCols + cbeg;
#pragma unroll
            for (int c = 0; c < kC; c += 4) {
              const float4 xv = *reinterpret_cast<const float4*>(x + c);
              acc[c >> 1] = f2_fma(z, f2_pack(xv.x, xv.y), acc[c >> 1]);
              acc[(c >> 1) + 1] = f2_fma(z, f2_pack(xv.z, xv.w), acc[(c >> 1) + 1]);
            }
          }
        }
      }
    };
    if (ncol > 16)
      drain(std::integral_constant<int, 32>{});
    else
      drain(std::integral_constant<int, 16>{});
    // this warp has seen every MMA of the CTA complete: the B slots are free
#pragma unroll
    for (int c = 0; c < 16; ++c)
      if (2 * c < ncol) {
        const float2 v = f2_unpack(acc[c]);
        red[(cbeg + 2 * c) * 128 + row] = v.x;
        red[(cbeg + 2 * c + 1) * 128 + row] = v.y;
      }
  }
  if (!ok && a.err) atomicOr(a.err, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if (p.c > 1) u_cluster_sync();
  const uint32_t local = su32(red);
  // a thread stores two rows for every 12 c-th token
  constexpr int per = kULinThreads / 64;
  const int cols = min(p.N, a.T - tok0), row = 2 * (threadIdx.x & 63), m = unit * 128 + row;
  int col = (threadIdx.x >> 6) + rank * per;
  if (m < a.M && col < cols) {
    const bool two = m + 1 < a.M;
    const int es = a.y_f32 ? 4 : 2;
    char* y = reinterpret_cast<char*>(a.Y) + ((long long)(tok0 + col) * a.ldy + m) * es;
    const __nv_bfloat16* r = a.R + (a.R ? (long long)(tok0 + col) * a.ldr + m : 0);
#pragma unroll 1
    for (; col < cols; col += per * p.c, y += per * p.c * a.ldy * es, r += per * p.c * a.ldr) {
      float2 v = make_float2(0.f, 0.f);
      if (a.R) {
        v.x = __bfloat162float(r[0]);
        if (two) v.y = __bfloat162float(r[1]);
      }
      float2 s = make_float2(0.f, 0.f);
      if (p.c == 1) {
        s = *reinterpret_cast<const float2*>(red + col * 128 + row);
      } else {
        float2 w[8];  // the ranks' parts, all on their way at once
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          w[q] = make_float2(0.f, 0.f);
          if (q < p.c) {
            uint32_t at;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local + (col * 128 + row) * 4), "r"(q));
            asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(w[q].x), "=f"(w[q].y) : "r"(at) : "memory");
          }
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) s.x += w[q].x, s.y += w[q].y;
      }
      v.x += s.x, v.y += s.y;
      if (a.y_vec && two) {
        if (a.y_f32)
          *reinterpret_cast<float2*>(y) = v;
        else
          *reinterpret_cast<__nv_bfloat162*>(y) = __float22bfloat162_rn(v);
      } else if (a.y_f32) {
        reinterpret_cast<float*>(y)[0] = v.x;
        if (two) reinterpret_cast<float*>(y)[1] = v.y;
      } else {
        reinterpret_cast<__nv_bfloat16*>(y)[0] = __float2bfloat16_rn(v.x);
        if (two) reinterpret_cast<__nv_bfloat16*>(y)[1] = __float2bfloat16_rn(v.y);
      }
    }
  }
  if (p.c > 1) u_cluster_sync();  // no CTA leaves while another reads its partial sums
}

template <int FL, bool AWQ>
cudaError_t launch_u(const LinArgs& a, cudaStream_t st) {
  UPlan p{};
  const int ntb = (a.T + kUCols - 1) / kUCols;
  p.N = std::min(kUCols, (a.T + 15) / 16 * 16);
  p.steps = (a.K + 127) / 128;
  const long long units = (long long)((a.mt + 7) / 8) * ntb;
  // CTAs per cluster: the fewest rounds x (steps + what a CTA costs besides,
  // about ten steps)
  long long cost = -1;
  for (int c = 1; c <= 8 && c <= p.steps; ++c) {
    const int at_once = cluster_ctas(c);
    const long long now = (units * c + at_once - 1) / at_once * ((p.steps + c - 1) / c + 10);
    if (cost < 0 || now < cost) cost = now, p.c = c;
  }
  const int smem = UCfg<FL, AWQ>::smem(p.N);
  constexpr int most = UCfg<FL, AWQ>::smem(kUCols);
  CUtensorMap xmap{};
  p.tma = a.x_vec && b_tensor_map(&xmap, a.X, a.K, a.T, a.ldx, p.N);
  const auto kernel = k_lin_umma<FL, AWQ>;
  static std::atomic<bool> attr[64];  // by device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr[dev].store(true, std::memory_order_relaxed);
  }
  const long long gx = (long long)((a.mt + 7) / 8) * p.c;
  if (gx > 0x7FFFFFFFll || ntb > 65535) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)gx, (unsigned)ntb);
  cfg.blockDim = dim3(kULinThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)p.c;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.c > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, p, xmap);
}

}  // namespace

cudaError_t launch_linear_umma(const LinArgs& a, int fl, bool awq, cudaStream_t st) {
  switch (fl) {
    case 1: return awq ? launch_u<1, true>(a, st) : launch_u<1, false>(a, st);
    case 2: return awq ? launch_u<2, true>(a, st) : launch_u<2, false>(a, st);
    default: return awq ? launch_u<4, true>(a, st) : launch_u<4, false>(a, st);
  }
}

}  // namespace llmoc
