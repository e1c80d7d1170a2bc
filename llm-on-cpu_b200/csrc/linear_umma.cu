// linear_umma.cu — dense INT4 products of tens of tokens on the 5th-generation
// tensor cores (tcgen05.mma): exact integers times bf16 activations, fp32 group
// sums, the group's scale applied to its fp32 sum.
//
// A CTA holds 128 weight rows (eight 16-row tiles of the packed stream, see
// linear.cu) against up to 64 tokens over a share of K, in steps of 128 k.  The
// A operand is q - zp (GPTQ: q - 8, and z + 8 s times the group's activation
// sums xs is added beside), an exact integer of four bits.  The scale belongs to
// a row and a group:
//
//   groups of 128 k: an accumulator in TMEM per step, drained while the next are
//     computed,  acc[row][t] += s[row, g] * P[row][t];
//   smaller groups: (q - zp) * s, 4 x 11 bits, as the exact sum of two bf16
//     operands, hi + lo.  With s = s_hi + s_lo (8 + 3 bits) hi = (q - zp) * s_hi
//     rounded, and lo = (q - zp) * s_lo + ((q - zp) * s_hi - hi) has at most 8
//     bits: three packed instructions per pair of weights and twice the MMAs, but
//     one drain per step.  A drain per group of 32 took twice the time (T = 37,
//     4101 x 7264 with zeros: 51 us against 28.7 us): each waits in turn for
//     its MMAs, its load and the accumulator's next use.
//
//   TMEM   [0, 256)          accumulators: one of 64 columns per issuer
//          [256, 512)        A slots: 4 of 64 columns (128 rows x 128 k, bf16 pairs), or
//                            2 of hi and lo
//   shared memory: B slots (4 x N tokens x 128 k, K-major, 128-byte swizzle),
//   and the activation sums and scales of 16 steps, which the drain reads after
//   it has given the accumulator back.
//
//   warps 0..3    lane 0 issues the MMAs of the steps j % 4 == warp (an MMA costs
//                 its issuing thread about 100 cycles, so four issue in turn)
//   warps 4..7    activations: 16-byte cp.async into the swizzled slot up to two
//                 steps ahead, the group sums from what landed, the scales
//   warps 8..15   dequantisers, thread = weight row = TMEM lane, even and odd
//                 steps; the words of two steps on are in flight in registers
//   warps 16..23  drain, one lane quadrant and half of the columns each, step by step
//
// K splits over the CTAs of a cluster; their partial sums meet in distributed
// shared memory and are added in rank order.  Every wait is bounded; one that
// gives up sets the handle's error word (llmoc_int4_linear_status) and every role
// drains and exits.
//
// Why the parity waits are sound: each barrier's waiter (an issuer for its full,
// acc-empty and slot barriers; a dequantising warp and a loader warp for a slot's
// empty barrier; a drain warp for an accumulator's full barrier) waits for
// every phase of it in order, and is at most one phase ahead of it.  Sums and
// scales of step j are overwritten by step j + 16, whose loader has seen the MMAs
// of step j + 12 complete; their issuer had waited until every drain warp gave
// back step j + 8's accumulator, which each does after it is through with step j.
#include <algorithm>
#include <string>

#include "ops.cuh"
#include "umma_dev.cuh"

namespace llmoc {

namespace {

constexpr int kUSteps = 4;   // A and B slots
constexpr int kUSide = 16;   // slots of sums and scales
constexpr int kUCols = 64;   // most tokens of a CTA
constexpr int kULinThreads = 24 * 32;

struct UPlan {
  int N;       // tokens of a CTA, a multiple of 16
  int c;       // CTAs of a cluster, splitting K
  int steps;   // 128-wide steps of K
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
__device__ __forceinline__ uint4 ld_words(const char* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
__device__ __forceinline__ uint32_t bf2_dup(float f) {
  const __nv_bfloat162 r = __float2bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <int FL, bool AWQ>
__global__ void __launch_bounds__(kULinThreads, 1) k_lin_umma(const LinArgs a, const UPlan p) {
  constexpr int kBB = lin_block_bytes(FL, !AWQ);
  constexpr bool kSplit = FL < 4;           // the scale in the A operand, as two bf16 terms
  constexpr int kGs = 4 / FL;               // scale groups per step
  constexpr int kASlots = kSplit ? 2 : 4;
  constexpr int kGrp = 8 / FL;  // groups per block of the stream
  extern __shared__ __align__(1024) unsigned char usm[];
  __shared__ __align__(8) uint64_t full[kUSteps], empty[kUSteps], accFull[4], accEmpty[4], done[4];
  __shared__ uint32_t tmem_base;
  __shared__ volatile int abort_flag;
  unsigned char* ringB = usm + ((1024 - (su32(usm) & 1023)) & 1023);
  float* xs = reinterpret_cast<float*>(ringB + kUSteps * p.N * 256);     // [kUSide][kGs][kUCols]
  __half* sc = reinterpret_cast<__half*>(xs + kUSide * kGs * kUCols);  // [kUSide][8 tiles][kGs][8 pairs]
  __half* zr = sc + kUSide * kGs * 128;                                // the same (GPTQ)
  auto warp_wait = [&](uint64_t* b, uint32_t par) {  // by a whole warp
    return __all_sync(0xffffffffu, mb_wait(b, par, &abort_flag)) != 0;
  };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = warp & 3;
  const int rank = blockIdx.x % p.c, unit = blockIdx.x / p.c, tok0 = blockIdx.y * kUCols;
  const int j0 = p.steps * rank / p.c, n = p.steps * (rank + 1) / p.c - j0;  // this CTA's steps
  constexpr bool kSums = !AWQ;
  const int slot_bytes = p.N * 256;                                          // two 64-wide halves
  const size_t tile_bytes = (size_t)a.nb * kBB;
  const int halves = p.N > 16 ? 2 : 1;  // drain warps per quadrant with columns
  // word pieces of this dequantiser's row: 64 bytes of every chunk of its tile
  const bool deq = warp >= 8 && warp < 16;
  const int r16 = lane & 15, hi = r16 >> 3;
  const char* wsrc = a.q + (size_t)min(unit * 8 + 2 * quad + (lane >> 4), a.mt - 1) * tile_bytes + (r16 & 7) * 64;
  uint4 raw[2][4];
  auto fetch = [&](int h, int j) {  // half h of step j
    const char* src = wsrc + (size_t)(j >> 1) * kBB + ((j & 1) * 2 + h) * 512;
#pragma unroll
    for (int t = 0; t < 4; ++t) raw[h][t] = ld_words(src + t * 16);
  };
  unsigned short sraw[kGs];
  auto fetch_scales = [&](int j) {
    const char* src = wsrc - (r16 & 7) * 60 + hi * 2 + (size_t)(j >> 1) * kBB + 2048 + (j & 1) * (kGs * 32);
#pragma unroll
    for (int q = 0; q < kGs; ++q) sraw[q] = __ldg(reinterpret_cast<const unsigned short*>(src + q * 32));
  };
  const int dg = (warp - 8) >> 2;  // even or odd steps
  if (deq && dg < n) {  // the weights do not depend on the previous kernel
    if (kSplit) fetch_scales(j0 + dg);
    fetch(0, j0 + dg);
    fetch(1, j0 + dg);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kUSteps; ++s) {
      mb_init(&full[s], 8);  // four dequantising warps, four loader warps
      mb_init(&empty[s], 1);
    }
    for (int i = 0; i < 4; ++i) {
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
  grid_dep_wait();
  grid_dep_release();
  bool ok = true;
  float* red = reinterpret_cast<float*>(ringB);  // partial sums [column][row], over the B slots
  auto store = [&](int row, int tok, float v) {
    if (row >= a.M || tok >= a.T) return;
    if (a.R) v += __bfloat162float(a.R[(long long)tok * a.ldr + row]);
    if (a.y_f32)
      reinterpret_cast<float*>(a.Y)[(long long)tok * a.ldy + row] = v;
    else
      reinterpret_cast<__nv_bfloat16*>(a.Y)[(long long)tok * a.ldy + row] = __float2bfloat16_rn(v);
  };
  const int h2 = (warp - 16) >> 2;                            // drain: column half
  const int colw = ((p.N + 31) >> 5) << 4;                    // columns of half 0
  const int cbeg = h2 * colw, ncol = min(p.N - cbeg, colw);  // this warp's columns (16 or 32, or none)

  if (warp < 4) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc(128, p.N);
      const uint64_t dB = smem_desc(su32(ringB) + warp * slot_bytes);
      const uint32_t half = (uint32_t)(p.N * 128) >> 4;  // descriptor units to the second 64 k
      const uint32_t dacc = tmem + warp * 64;
      for (int j = warp; j < n; j += 4) {
        const uint32_t ta = tmem + 256 + (j % kASlots) * (256 / kASlots);
        // the step's operands, and the accumulator's last use drained
        if (!mb_wait(&full[warp], (j >> 2) & 1, &abort_flag) ||
            (j >= 4 && !mb_wait(&accEmpty[warp], ((j >> 2) - 1) & 1, &abort_flag))) {
          ok = false;
          break;
        }
        tc_fence_after();
        umma_ts_k64(dacc, ta, dB, idesc, 0);
        umma_ts_k64(dacc, ta + 32, dB + half, idesc, 1);
        if (kSplit) {
          umma_ts_k64(dacc, ta + 64, dB, idesc, 1);
          umma_ts_k64(dacc, ta + 96, dB + half, idesc, 1);
        }
        umma_commit(&accFull[warp]);
        umma_commit(&empty[warp]);
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
  } else if (warp < 8) {
    const int lt = threadIdx.x - 128;  // 0..127
    // thread's 16-byte pieces of a step: piece pc of rows r0, r0 + 8, ... (p.N / 8 of them)
    const int pieces = p.N >> 3, pc = lt & 15, r0 = lt >> 4;
    const uint32_t place = su32(ringB) + (pc >> 3) * (p.N * 128) + r0 * 128 + (((pc & 7) ^ r0) << 4);  // + 1024 a piece
    const __nv_bfloat16* xsrc = a.X + (long long)(tok0 + r0) * a.ldx + pc * 8;
    auto issue = [&](int j) {
      const uint32_t dst = place + (j & 3) * slot_bytes;
      if (lt < 16 * kGs) {  // the scales: kGs * 32 bytes of each tile
        const int tile = lt / (2 * kGs), part = lt % (2 * kGs), g = j0 + j;
        const char* src = a.q + (size_t)min(unit * 8 + tile, a.mt - 1) * tile_bytes + (size_t)(g >> 1) * kBB + 2048 +
                          (g & 1) * (kGs * 32) + part * 16;
        const uint32_t to = su32(sc) + (j & (kUSide - 1)) * (kGs * 256) + lt * 16;
        cp_async16(to, src, 16);
        if (!AWQ) cp_async16(to + kUSide * kGs * 256, src + kGrp * 32, 16);
      }
      const int k = (j0 + j) * 128;
      const bool kin = k + pc * 8 < a.K;
      if (a.x_vec) {
        const __nv_bfloat16* src = xsrc + k;
        const int rows = kin ? a.T - tok0 - r0 : 0;  // piece i lies in the batch: i * 8 < rows
#pragma unroll
        for (int i = 0; i < kUCols / 8; ++i) {
          if (i < pieces) cp_async16(dst + i * 1024, i * 8 < rows ? src : a.X, i * 8 < rows ? 16 : 0);
          src += 8 * a.ldx;
        }
      } else {
        for (int i = 0; i < pieces; ++i) {
          uint32_t w[4] = {0, 0, 0, 0};
          if (kin && tok0 + r0 + i * 8 < a.T) {
            const unsigned short* u = reinterpret_cast<const unsigned short*>(xsrc + k + i * 8 * a.ldx);
#pragma unroll
            for (int q = 0; q < 4; ++q) w[q] = u[2 * q] | ((uint32_t)u[2 * q + 1] << 16);
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + i * 1024), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                       "r"(w[3])
                       : "memory");
        }
      }
    };
    auto publish = [&](int j) {  // a step that has landed
      if constexpr (kSums) {
      const uint32_t src = place + (j & 3) * slot_bytes;
      float* to = xs + ((j & (kUSide - 1)) * kGs + pc / (4 * FL)) * kUCols + r0;
      float v[kUCols / 8];
#pragma unroll
      for (int i = 0; i < kUCols / 8; ++i) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (i < pieces)
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                       : "r"(src + i * 1024)
                       : "memory");
        v[i] = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[i] += __uint_as_float(w[q] << 16) + __uint_as_float(w[q] & 0xFFFF0000u);
      }
#pragma unroll
      for (int o = 1; o < 4 * FL; o <<= 1)
#pragma unroll
        for (int i = 0; i < kUCols / 8; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      if ((pc & (4 * FL - 1)) == 0)
#pragma unroll
        for (int i = 0; i < kUCols / 8; ++i)
          if (i < pieces) to[i * 8] = v[i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mb_arrive(&full[j & 3]);
    };
    int pub = 0;  // next step to publish
    for (int j = 0; j < n; ++j) {
      const int s = j & 3;
      // what has landed is published before any wait
      if (j >= kUSteps && !__all_sync(0xffffffffu, mb_try(&empty[s], ((j >> 2) - 1) & 1))) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        while (pub < j) publish(pub++);
        if (!warp_wait(&empty[s], ((j >> 2) - 1) & 1)) {
          ok = false;
          break;
        }
      }
      issue(j);
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (j - pub == 2) {
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        publish(pub++);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    while (ok && pub < n) publish(pub++);
  } else if (deq) {
    const uint32_t tl = tmem + ((uint32_t)(quad * 32) << 16) + 256;
    const uint32_t rot = 4 * hi, zp2 = (0x4180u + ((AWQ ? (uint32_t)a.zp : 8u) << 3)) * 0x10001u;  // 16 + zp, zp < 16
    for (int j = dg; j < n && ok; j += 2) {
      if (j >= kASlots) {  // the slot's last MMAs
        const int o = j - kASlots;
        if (!warp_wait(&empty[o & 3], (o >> 2) & 1)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      const uint32_t ta = tl + (j % kASlots) * (256 / kASlots);
      uint32_t shi[kGs], slo[kGs];  // the groups' scales as pairs of two bf16 terms
      if (kSplit) {
#pragma unroll
        for (int q = 0; q < kGs; ++q) {
          const float f = __half2float(__ushort_as_half(sraw[q]));
          shi[q] = bf2_dup(f);
          slo[q] = bf2_dup(f - __uint_as_float(shi[q] << 16));
        }
        if (j + 2 < n) fetch_scales(j0 + j + 2);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t r[16], lo[16];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {  // word (kb, kt): k = 32 kb + 8 t + 4 kt + {0..3}
              const uint4& u = raw[h][t];
              const uint32_t w = kb ? (kt ? u.w : u.z) : (kt ? u.y : u.x);
              const uint32_t v = __funnelshift_r(w, w, rot);
              const int col = 4 * t + 2 * kt;
              r[col] = nib16(v);
              r[col + 1] = nib16(__funnelshift_r(v, v, 8));
              r[col] = bf2_sub(r[col], zp2);
              r[col + 1] = bf2_sub(r[col + 1], zp2);
            }
          }
          if (kSplit) {
            const uint32_t hi = shi[kGs == 4 ? 2 * h + kb : h], sl = slo[kGs == 4 ? 2 * h + kb : h];
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const uint32_t q = r[c];
              r[c] = bf2_mul(q, hi);
              lo[c] = bf2_fma(q, sl, bf2_fma(q, hi, r[c] ^ 0x80008000u));
            }
            tmem_st16(ta + 64 + 32 * h + 16 * kb, lo);
          }
          tmem_st16(ta + 32 * h + 16 * kb, r);
        }
        if (j + 2 < n) fetch(h, j0 + j + 2);
      }
      asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mb_arrive(&full[j & 3]);
    }
  } else if (ncol > 0) {
    const uint32_t tq = tmem + ((uint32_t)(quad * 32) << 16) + cbeg;
    const int row = quad * 32 + lane;
    float acc[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = 0.f;
    // The columns come in two halves of 16; a half's load is in flight while the
    // one before it is added, across steps.
    uint32_t lo[16], up[16];
    ok = warp_wait(&accFull[0], 0);
    tc_fence_after();
    if (ok) tmem_ld16_issue(tq, lo);
    for (int j = 0; ok && j < n; ++j) {
      const int side = j & (kUSide - 1), buf = j & 3;
      // pair (g, g + 8) of the row's tile in the step's first scale group
      const int si = (side * 8 + (row >> 4)) * kGs * 16 + (row & 7) * 2 + ((row >> 3) & 1);
      const float s = kSplit ? 1.f : __half2float(sc[si]);
      const float* x = xs + side * kGs * kUCols + cbeg;
      auto add = [&](const uint32_t (&v)[16], int c0) {
#pragma unroll
        for (int c = 0; c < 16; ++c)
          acc[c0 + c] = kSplit ? acc[c0 + c] + __uint_as_float(v[c]) : fmaf(s, __uint_as_float(v[c]), acc[c0 + c]);
        if (kSums)
#pragma unroll
          for (int q = 0; q < kGs; ++q) {
            const int sq = si + q * 16;
            const float z = fmaf(8.f, __half2float(sc[sq]), __half2float(zr[sq]));
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              const float4 xv = *reinterpret_cast<const float4*>(x + q * kUCols + c0 + c);
              acc[c0 + c] = fmaf(z, xv.x, acc[c0 + c]), acc[c0 + c + 1] = fmaf(z, xv.y, acc[c0 + c + 1]);
              acc[c0 + c + 2] = fmaf(z, xv.z, acc[c0 + c + 2]), acc[c0 + c + 3] = fmaf(z, xv.w, acc[c0 + c + 3]);
            }
          }
      };
      tmem_ld16_wait(lo);
      if (ncol > 16) {
        tmem_ld16_issue(tq + buf * 64 + 16, up);
        add(lo, 0);
        tmem_ld16_wait(up);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mb_arrive(&accEmpty[buf]);
      if (ncol <= 16) {
#pragma unroll
        for (int c = 0; c < 16; ++c) up[c] = lo[c];
      }
      if (j + 1 < n) {
        const int nb = (j + 1) & 3;
        ok = warp_wait(&accFull[nb], ((j + 1) >> 2) & 1);
        tc_fence_after();
        if (ok) tmem_ld16_issue(tq + nb * 64, lo);
      }
      if (ncol > 16)
        add(up, 16);
      else
        add(up, 0);
    }
    // this warp has seen every MMA of the CTA complete: the B slots are free
    if (p.c > 1) {
#pragma unroll
      for (int c = 0; c < 32; ++c)
        if (c < ncol) red[(cbeg + c) * 128 + row] = acc[c];
    } else {
      const int m = unit * 128 + row, left = m < a.M ? min(ncol, a.T - tok0 - cbeg) : 0;
      if (a.R) {
        const __nv_bfloat16* r = a.R + (long long)(tok0 + cbeg) * a.ldr + m;
#pragma unroll
        for (int c = 0; c < 32; ++c, r += a.ldr)
          if (c < left) acc[c] += __bfloat162float(*r);
      }
      if (a.y_f32) {
        float* y = reinterpret_cast<float*>(a.Y) + (long long)(tok0 + cbeg) * a.ldy + m;
#pragma unroll
        for (int c = 0; c < 32; ++c, y += a.ldy)
          if (c < left) *y = acc[c];
      } else {
        __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(a.Y) + (long long)(tok0 + cbeg) * a.ldy + m;
#pragma unroll
        for (int c = 0; c < 32; ++c, y += a.ldy)
          if (c < left) *y = __float2bfloat16_rn(acc[c]);
      }
    }
  }
  if (!ok && a.err) atomicOr(a.err, 1);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
  if (p.c == 1) return;
  u_cluster_sync();
  const uint32_t local = su32(red);
  const int cols = min(p.N, a.T - tok0);
  for (int e = threadIdx.x + rank * kULinThreads; e < cols * 128; e += kULinThreads * p.c) {
    float v = 0.f;
    for (int q = 0; q < p.c; ++q) {
      uint32_t at;
      float w;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local + e * 4), "r"(q));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(w) : "r"(at) : "memory");
      v += w;
    }
    store(unit * 128 + (e & 127), tok0 + (e >> 7), v);
  }
  u_cluster_sync();  // no CTA leaves while another reads its partial sums
}

template <int FL, bool AWQ>
cudaError_t launch_u(const LinArgs& a, cudaStream_t st) {
  UPlan p{};
  const int ntb = (a.T + kUCols - 1) / kUCols;
  p.N = std::min(kUCols, (a.T + 15) / 16 * 16);
  p.steps = (a.K + 127) / 128;
  const long long units = (long long)((a.mt + 7) / 8) * ntb;
  // CTAs per cluster: the fewest rounds x (steps + what a CTA costs besides,
  // about ten steps); a cluster's CTAs share a GPC, which leaves some SMs over
  static const int resident[9] = {0, 148, 148, 138, 136, 130, 126, 126, 128};
  long long cost = -1;
  for (int c = 1; c <= 8 && c <= p.steps; ++c) {
    const long long now = (units * c + resident[c] - 1) / resident[c] * ((p.steps + c - 1) / c + 10);
    if (cost < 0 || now < cost) cost = now, p.c = c;
  }
  constexpr int side = kUSide * (4 / FL) * (kUCols * 4 + 128 * 2 * (AWQ ? 1 : 2));
  const int smem = kUSteps * p.N * 256 + side + 1024;
  constexpr int most = kUSteps * kUCols * 256 + side + 1024;
  static_assert(most <= 227 * 1024, "shared memory");
  const auto kernel = k_lin_umma<FL, AWQ>;
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr[dev] = true;
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
  return cudaLaunchKernelEx(&cfg, kernel, a, p);
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
