// linear.cu — dense INT4 products on device-resident weights,
//
//     Y[t, m] = sum_g s[m, g] * sum_{k in g} (q[m, k] - zp) * X[t, k]  (+ R[t, m])
//
// (GPTQ: + z[m, g] * sum_{k in g} X[t, k] with zp = 0), the matrix-vector and
// small-batch products of a decode step.  What bounds them is reading the
// weights once: M * K / 2 bytes.
//
// Weights are packed for this kernel (k_lin_pack): per 16-row tile a stream of
// blocks of 256 k, each four 512-byte chunks of words (64 k: lane (g, t)'s 16
// bytes at 64 g + 16 (t xor g / 2), two words of row g, then two of row g + 8, a
// word the 8 k from 8 t of one of the chunk's two 32 k), then the block's scales
// (and zeros) as fp16 pairs of rows (g, g + 8).  Groups that are other multiples of 32, 64 or 128 repeat their
// scale, so a block holds 8, 4 or 2 groups of 32, 64 or 128.
//
// Work.  A warp owns a tile against NT * 8 tokens over a slice of K.  The
// 16 warps of a CTA take 16 / ksw tiles and split K ksw ways; a cluster
// of c CTAs splits K c ways more.  With c = ksw = 1 a CTA walks tile groups
// (persistent) and its warps never meet; otherwise the partial sums meet in
// (distributed) shared memory and are added in slice order, so no workspace is
// needed and the bits do not depend on timing.
//
// The stream runs through a ring in shared memory per warp, filled by one bulk
// copy per block and tile as soon as a place has been read, across tile ends, so
// up to 8 blocks (17 to 20 KB) of a warp are on their way.  Loads into a ring of
// registers brought 15 to 18 bytes per clock and SM at most and took the issue
// slots that dequantisation needs (248320 x 2048, T = 8: 57.1 us, now 55.0; groups
// of 32: 77.8, now 61.6; 11008 x 4096, T = 8: 16.0, now 12.4).  One CTA per SM, so
// that the activations are staged once.
//
// What bounds it now: with T = 1 at 248320 x 2048 52.5 us are 4.97 TB/s; with the
// shifts of the dequantisation left out (and wrong results) the same kernel takes
// 41.5 us, the rate of a plain copy.  Three of four register pairs need one, they
// run at half rate, and a product by a power of two in their place is slower.
//
// Dequantisation.  A word holds eight nibbles, pair j of them (one per 16-bit
// half) at bits 3 + 4j: rotated right by 4j and merged into 0x4180 it is the
// bf16 pair 16 + q, exact, two instructions per pair and no subtraction.  With
// P = sum (16 + q) x from mma.m16n8k16 (exact products, fp32 sums) and the
// group's activation sum xs, the group adds s * (P - (16 + zp) * xs), or
// s * (P - 16 xs) + z * xs.  The offset 16 (the smallest power of two above
// the nibbles) keeps the cancellation to a factor of about five; 128, which
// needs no positioned nibbles, would lose five bits.
//
// Activations are staged once per CTA and K slab in shared memory in B fragment
// order (lane (g, t): token g, 8 consecutive k from 8 t), one conflict-free
// 16-byte load per 32 k and 8 tokens, with the group sums beside them.  One
// token is stored once and read as all eight columns.
#include <algorithm>
#include <atomic>
#include <string>

#include "ops.cuh"
#include "umma_dev.cuh"

namespace llmoc {

namespace {

constexpr int kLinWarps = 16, kLinWarpsLog = 4;
constexpr int kLinThreads = kLinWarps * 32;
constexpr int kRingMax = 8;      // places of a warp's ring at most
constexpr uint32_t kOffset = 16;  // A elements are kOffset + q

__device__ __forceinline__ float2 pair_f32(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ uint32_t nib_pair(uint32_t w) {  // (16 + q_lo, 16 + q_hi) as bf16
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(0x00780078u), "r"(0x41804180u));
  return d;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Every CTA of the cluster arrives and waits; shared-memory writes before it
// are visible to the cluster's CTAs after it.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// *p of the cluster's CTA `rank`
__device__ __forceinline__ float ld_cluster(const float* p, int rank) {
  uint32_t at;
  float v;
  const uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(local), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

struct LinPlan {
  int lk;     // log2 of ksw, the warps of a CTA that split K
  int lc;     // log2 of c, the CTAs of a cluster that split K
  int units;  // tile groups (of 16 / ksw tiles)
  int bps;    // blocks of 256 k per staged slab
  int nslab;  // slabs of a CTA's share of K
  int ring;   // places of a warp's ring, each a block of its tile
};

// FL: 32-wide blocks per scale group (1, 2, 4); TP: token rows staged (1, or
// NT * 8).
template <int FL, bool AWQ, int NT, int TP>
__global__ void __launch_bounds__(kLinThreads, 1) k_linear(const LinArgs a, const LinPlan p) {
  constexpr int kBB = lin_block_bytes(FL, !AWQ);
  constexpr int kGrp = 8 / FL;                  // scale groups per block
  constexpr int kCols = NT * 8, kColLd = 16 + 4;
  constexpr int kXW = TP * 4;                   // 16-byte pieces per 32 k
  extern __shared__ __align__(128) char lsm[];  // [warp][ring][kBB]: the weights as they are stored
  __shared__ __align__(8) uint64_t landed[kLinWarps][kRingMax];
  __shared__ volatile int abort_flag;
  uint4* sx = reinterpret_cast<uint4*>(lsm + kLinWarps * p.ring * kBB);  // [slab's 32-blocks][kXW]: B fragments
  float* xs = reinterpret_cast<float*>(sx + (size_t)p.bps * 8 * kXW);  // [slab's groups][TP]: activation sums
  float* red = xs + (size_t)p.bps * kGrp * TP;                         // [warp][col][row]: partial sums
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int c = 1 << p.lc, ksw = 1 << p.lk, lr = kLinWarpsLog - p.lk;  // lr: log2 of the CTA's tile groups
  const int rank = blockIdx.x & (c - 1), ncl = gridDim.x >> p.lc;
  const int tok0 = blockIdx.y * kCols;
  const int wt = warp & ((1 << lr) - 1), wk = warp >> lr;
  const int p0 = a.nb * rank >> p.lc, p1 = a.nb * (rank + 1) >> p.lc;  // nb < 2^23
  const int nslab = p.nslab;

  // segment (unit, slab) of this warp: its first block within the slab, its
  // blocks and their address
  struct Seg {
    const char* q;
    int b0, nb;
  };
  const size_t tile_bytes = (size_t)a.nb * kBB;
  auto seg_of = [&](int unit, int slab) {
    Seg s;
    const int s0 = p0 + slab * p.bps, n = max(0, min(p1, s0 + p.bps) - s0);
    const int tile = (unit << lr) + wt;
    s.b0 = n * wk >> p.lk;
    s.nb = tile < a.mt && unit < p.units ? (n * (wk + 1) >> p.lk) - s.b0 : 0;
    s.q = a.q + (size_t)min(tile, a.mt - 1) * tile_bytes + (size_t)(s0 + s.b0) * kBB;
    return s;
  };
  const int lq = (g * 4 + (t ^ ((g >> 1) & 3))) * 16, ls = 2048 + g * 4;
  char* ring = lsm + warp * p.ring * kBB;
  uint64_t* bar = landed[warp];
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < p.ring; ++i) mb_init(&bar[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // the next block to fetch: the segments in the order of use
  int iunit = blockIdx.x >> p.lc, islab = 0, ib = 0, islot = 0;
  uint32_t issued = 0;
  bool bad = false;
  Seg is = seg_of(iunit, 0);
  auto fetch = [&]() {  // into the next place, which is free
    while (iunit < p.units && ib >= is.nb) {
      if (++islab == p.nslab) islab = 0, iunit += ncl;
      is = seg_of(iunit, islab), ib = 0;
    }
    if (iunit >= p.units || bad) return;
    if (lane == 0) {
      mb_expect(&bar[islot], kBB);
      bulk_g2s(su32(ring + islot * kBB), is.q + (size_t)ib * kBB, kBB, &bar[islot]);
    }
    ++ib, ++issued;
    if (++islot == p.ring) islot = 0;
  };
  for (int i = 0; i < p.ring; ++i) fetch();  // the weights do not depend on the previous kernel
  int slot = 0, par = 0;

  int unit = blockIdx.x >> p.lc, slab = 0;
  Seg cur = seg_of(unit, 0);
  grid_dep_wait();
  grid_dep_release();

  float acc[NT][4], part[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = part[n][i] = 0.f;
  const float zoff = AWQ ? -(float)(kOffset + a.zp) : -(float)kOffset;
  const uint4* xl = sx + (TP == 1 ? t : lane);
  const float* xsl = xs + (TP == 1 ? 0 : 2 * t);

  auto flush = [&](const float* xg, const char* w) {  // xg: the group's sums, w: its scale pairs
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float2 x;
      if (TP == 1)
        x.x = x.y = *xg;
      else
        x = *reinterpret_cast<const float2*>(xg + n * 8);
      const float2 sf = pair_f32(*reinterpret_cast<const uint32_t*>(w));
      float (&o)[4] = acc[n];
      float (&q)[4] = part[n];
      if (!AWQ) {
        const float2 zf = pair_f32(*reinterpret_cast<const uint32_t*>(w + kGrp * 32));
        o[0] = fmaf(zf.x, x.x, o[0]), o[1] = fmaf(zf.x, x.y, o[1]);
        o[2] = fmaf(zf.y, x.x, o[2]), o[3] = fmaf(zf.y, x.y, o[3]);
      }
      o[0] = fmaf(sf.x, fmaf(zoff, x.x, q[0]), o[0]), o[1] = fmaf(sf.x, fmaf(zoff, x.y, q[1]), o[1]);
      o[2] = fmaf(sf.y, fmaf(zoff, x.x, q[2]), o[2]), o[3] = fmaf(sf.y, fmaf(zoff, x.y, q[3]), o[3]);
      q[0] = q[1] = q[2] = q[3] = 0.f;
    }
  };

  // one slab of activations: rows tok0 .., blocks [s0, s0 + bps); zeros past T and K
  auto stage = [&](int s0, int s1) {
    const int np = (s1 - s0) * 32;  // 16-byte pieces of a row; a warp's 32 lie in one row
    int row = 0;
    for (int pc = threadIdx.x;; pc += kLinThreads) {
      while (pc >= np && row < TP) pc -= np, ++row;
      if (row >= TP) break;
      const int tok = tok0 + row, k = s0 * 256 + pc * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (tok < a.T && k < a.K) {
        const __nv_bfloat16* src = a.X + (long long)tok * a.ldx + k;
        if (a.x_vec) {
          v = *reinterpret_cast<const uint4*>(src);
        } else {
          const unsigned short* u = reinterpret_cast<const unsigned short*>(src);
          v.x = u[0] | ((uint32_t)u[1] << 16), v.y = u[2] | ((uint32_t)u[3] << 16);
          v.z = u[4] | ((uint32_t)u[5] << 16), v.w = u[6] | ((uint32_t)u[7] << 16);
        }
      }
      const uint32_t wd[4] = {v.x, v.y, v.z, v.w};
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) s += __uint_as_float(wd[i] << 16) + __uint_as_float(wd[i] & 0xFFFF0000u);
#pragma unroll
      for (int o = 1; o < 4 * FL; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      sx[(size_t)(pc >> 2) * kXW + (row >> 3) * 32 + (row & 7) * 4 + (pc & 3)] = v;
      if ((pc & (4 * FL - 1)) == 0) xs[(pc / (4 * FL)) * TP + row] = s;
    }
  };

  auto store = [&](int row, int tok, float v) {
    if (row >= a.M || tok >= a.T) return;
    if (a.R) v += __bfloat162float(a.R[(long long)tok * a.ldr + row]);
    if (a.y_f32)
      reinterpret_cast<float*>(a.Y)[(long long)tok * a.ldy + row] = v;
    else
      reinterpret_cast<__nv_bfloat16*>(a.Y)[(long long)tok * a.ldy + row] = __float2bfloat16_rn(v);
  };

  bool staged = false;
  while (unit < p.units) {  // the same for all CTAs of a cluster
    if (!staged || nslab > 1) {
      const int s0 = p0 + slab * p.bps;
      if (staged) __syncthreads();  // the slab before is read no more
      stage(s0, min(p1, s0 + p.bps));
      __syncthreads();
      staged = true;
    }
    const int nslab1 = slab + 1 < nslab ? slab + 1 : 0, nunit = nslab1 ? unit : unit + ncl;
    const Seg nxt = seg_of(nunit, nslab1);
    const uint4* xb = xl + (size_t)cur.b0 * 8 * kXW;
    const float* xg = xsl + cur.b0 * kGrp * TP;
    for (int b = 0; b < cur.nb; ++b) {
      if (!__all_sync(0xffffffffu, mb_wait(&bar[slot], par, &abort_flag))) bad = true;
      const char* wb = ring + slot * kBB;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(wb + lq + i * 512);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint4 x[NT];
#pragma unroll
          for (int n = 0; n < NT; ++n) x[n] = xb[(2 * i + kb) * kXW + n * 32];
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            uint32_t f[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {  // rows g and g + 8, k in two halves
              const uint32_t v = (h & 1) ? (kb ? w.w : w.z) : (kb ? w.y : w.x);
              f[h] = nib_pair(__funnelshift_r(v, v, 4 * (2 * kt + (h >> 1))));
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(part[n], f, kt ? x[n].z : x[n].x, kt ? x[n].w : x[n].y);
          }
          if ((2 * i + kb) % FL == FL - 1) {
            const int gi = (2 * i + kb) / FL;
            flush(xg + gi * TP, wb + ls + gi * 32);
          }
        }
      }
      xb += 8 * kXW;
      xg += kGrp * TP;
      __syncwarp();  // the place has been read
      fetch();
      if (++slot == p.ring) slot = 0, par ^= 1;
    }
    cur = nxt;
    if (nslab1 == 0) {  // the unit's last slab
      if (p.lk == 0 && p.lc == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            store(((unit << lr) + wt) * 16 + g + (i >> 1) * 8, tok0 + n * 8 + 2 * t + (i & 1), acc[n][i]);
      } else {
        // partial sums of the K slices, added in slice order (warps, then ranks); such
        // a grid has a cluster per unit, so the buffer is written once
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            red[(warp * kCols + n * 8 + 2 * t + (i & 1)) * kColLd + g + (i >> 1) * 8] = acc[n][i];
        __syncthreads();
        const int lrows = lr + 4;
        const int cols = min(kCols, a.T - tok0);
        auto at = [&](int e) {  // the sum of the first warp of row e's tile
          const int row = e & ((1 << lrows) - 1), col = e >> lrows;
          return red + ((row >> 4) * kCols + col) * kColLd + (row & 15);
        };
        for (int e = threadIdx.x; e < cols << lrows; e += kLinThreads) {
          float* p0 = at(e);
          float v = 0.f;
          for (int s = 0; s < ksw; ++s) v += p0[(s << lr) * kCols * kColLd];
          if (c > 1)
            *p0 = v;
          else
            store((unit << lrows) + (e & ((1 << lrows) - 1)), tok0 + (e >> lrows), v);
        }
        if (c > 1) {
          cluster_sync();
          for (int e = threadIdx.x + rank * kLinThreads; e < cols << lrows; e += kLinThreads << p.lc) {
            const float* p0 = at(e);
            float w[8];  // the ranks' sums, all on their way at once
#pragma unroll
            for (int q = 0; q < 8; ++q) w[q] = q < c ? ld_cluster(p0, q) : 0.f;
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q) v += w[q];
            store((unit << lrows) + (e & ((1 << lrows) - 1)), tok0 + (e >> lrows), v);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
    }
    unit = nunit;
    slab = nslab1;
  }
  if (bad) {
    if (a.err && lane == 0) atomicOr(a.err, 1);
    drain_ring(bar, p.ring, issued, 0, 1);  // no copy is in flight when the CTA leaves
  }
  if (c > 1) cluster_sync();  // no CTA leaves while another reads its partial sums
}

constexpr int kLinSmemMax = 224 * 1024;  // one CTA per SM

template <int FL, bool AWQ, int NT, int TP>
cudaError_t launch_shape(const LinArgs& a, cudaStream_t st) {
  LinPlan p{};
  const int ntb = (a.T + NT * 8 - 1) / (NT * 8);
  // K is split as long as every CTA stays resident at once (one per SM) and a
  // warp keeps a block: inside the CTA while its activations stay below half of
  // its weights, then over a cluster, then inside the CTA at any price.  A second
  // round of CTAs costs more than the shorter slices give (T = 8, 11008 x 4096 with
  // half as large CTAs: 17.5 us in two rounds, 16.0 us in one).
  int ksw = 1, c = 1;
  auto fits = [&](int w, int k) {
    const int rbt = kLinWarps / w;
    return (long long)((a.mt + rbt - 1) / rbt) * ntb * k <= cluster_ctas(k) && a.nb >= w * k;
  };
  while (ksw < kLinWarps && TP * ksw * 2 <= 16 && fits(2 * ksw, c)) ksw *= 2, ++p.lk;
  while (c < 8 && fits(ksw, 2 * c)) c *= 2, ++p.lc;
  while (ksw < kLinWarps && fits(2 * ksw, c)) ksw *= 2, ++p.lk;
  const int rbt = kLinWarps / ksw;
  p.units = (a.mt + rbt - 1) / rbt;
  const bool split = ksw > 1 || c > 1;
  const int red = split ? kLinWarps * NT * 8 * (16 + 4) * 4 : 0;
  const int per_block = TP * 4 * 8 * 16 + 8 / FL * TP * 4;
  const int share = (a.nb + c - 1) / c;
  // the activations get what leaves two places of each warp's ring, the ring the rest
  constexpr int place = kLinWarps * lin_block_bytes(FL, !AWQ);
  p.bps = std::max(1, std::min(share, (kLinSmemMax - red - 2 * place) / per_block));
  p.nslab = (share + p.bps - 1) / p.bps;
  const int ncl = !split ? std::min(p.units, std::max(1, 148 / ntb)) : p.units;
  const long long mine = (long long)((p.units + ncl - 1) / ncl) * ((share + ksw - 1) / ksw);  // a warp's blocks at most
  p.ring = (int)std::min<long long>(std::min(kRingMax, (kLinSmemMax - red - p.bps * per_block) / place), mine);
  static_assert(2 * place + kLinWarps * NT * 8 * (16 + 4) * 4 + TP * 4 * 8 * 16 + 8 / FL * TP * 4 <= kLinSmemMax, "");
  const int smem = p.ring * place + p.bps * per_block + red;
  const auto kernel = k_linear<FL, AWQ, NT, TP>;
  static std::atomic<bool> attr[64];  // by device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmemMax);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr[dev].store(true, std::memory_order_relaxed);
  }
  const long long gx = ncl * (long long)c;
  if (gx > 0x7FFFFFFFll || ntb > 65535) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)gx, (unsigned)ntb);
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)c;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = c > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, p);
}

template <int FL, bool AWQ>
cudaError_t launch_fl(const LinArgs& a, cudaStream_t st) {
  if (a.T == 1) return launch_shape<FL, AWQ, 1, 1>(a, st);
  if (a.T <= 8) return launch_shape<FL, AWQ, 1, 8>(a, st);
  return launch_shape<FL, AWQ, 2, 16>(a, st);
}

// One 32-bit word of the stream per thread: words of a block (rows past M and
// columns past K are 0, which zero activations meet), then its scale pairs.
__global__ void k_lin_pack(const LinPack a) {
  const int bw = lin_block_bytes(a.fl, a.gptq) / 4, grp = 8 / a.fl;
  const size_t n = (size_t)((a.M + 15) / 16) * a.nb * bw;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
    const int in = (int)(i % bw);
    const size_t tb = i / bw;
    const int b = (int)(tb % a.nb);
    const long long r0 = (long long)(tb / a.nb) * 16;
    uint32_t v = 0;
    if (in < 512) {
      const int wd = in & 3, g = (in >> 4) & 7, t = ((in >> 2) & 3) ^ ((g >> 1) & 3);
      const int k = b * 256 + (in >> 7) * 64 + (wd & 1) * 32 + t * 8;
      const long long row = r0 + g + 8 * (wd >> 1);
      for (int e = 0; e < 8; ++e) {
        if (row >= a.M || k + e >= a.K) continue;
        const uint32_t byte = a.q[(size_t)row * (a.K / 2) + ((k + e) >> 1)];
        const uint32_t nib = e & 1 ? byte >> 4 : byte & 15;
        v |= nib << (4 * ((e & 1) * 4 + (e >> 1)));
      }
      v = __funnelshift_l(v, v, 3);
    } else {
      const int s = in - 512, z = s / (8 * grp), gi = s / 8 % grp, g = s % 8;
      const int k = b * 256 + gi * a.fl * 32;
      const uint16_t* src = z ? a.z : a.s;
      for (int h = 0; h < 2; ++h) {
        const long long row = r0 + g + 8 * h;
        if (row < a.M && k < a.K && src) v |= (uint32_t)src[(size_t)row * a.ng + k / a.gs] << (16 * h);
      }
    }
    a.out[i] = v;
  }
}

}  // namespace

int cluster_ctas(int c) {
  static std::atomic<int> known[64][9];  // by device; 0: not asked yet
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& at = known[dev & 63][c];
  int n = dev < 64 ? at.load(std::memory_order_relaxed) : 0;
  if (n) return n;
  const auto kernel = k_linear<4, true, 1, 1>;  // any kernel with one CTA an SM
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)c);
  cfg.blockDim = dim3(kLinThreads);
  cfg.dynamicSmemBytes = kLinSmemMax;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (c == 1) {
    n = 148;
  } else if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmemMax) != cudaSuccess ||
             cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 100 / c * c;  // what any device has
  } else {
    n *= c;
  }
  if (dev < 64) at.store(n, std::memory_order_relaxed);
  return n;
}

cudaError_t launch_lin_pack(const LinPack& a, cudaStream_t st) {
  k_lin_pack<<<148 * 8, 256, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_linear(const LinArgs& a, int fl, bool awq, cudaStream_t st) {
  // mma.sync needs the weights dequantised once per 16 tokens, tcgen05's CTAs take
  // 64 tokens against 128 rows.  From 17 tokens on the latter is faster up to some
  // 100000 rows, and always from 33 (T = 24, groups of 128: 4096 x 4096 8.5 against
  // 10.6 us, 60000 x 4096 67 against 80, 100000 x 2048 61.2 against 59.4, 248320 x
  // 2048 142 against 130); from 9 tokens on while its tiles need about one round of
  // CTAs, half that with small groups (T = 16, K = 4096: 4096 rows 8.0 against 15.6
  // us, 11008 rows 14.8 against 16.5, 30000 rows 30.3 against 29.3; groups of 32: 4096
  // rows 10.2 against 16.9, 11008 rows 23.8 against 19.2).
  const int tiles = (a.mt + 7) / 8;
  const bool umma = a.T > 32 || (a.T > 16 && tiles <= 768) || (a.T > 8 && tiles <= (fl == 4 ? 148 : 64));
  if (umma && (!awq || a.zp < 16)) return launch_linear_umma(a, fl, awq, st);
  switch (fl) {
    case 1: return awq ? launch_fl<1, true>(a, st) : launch_fl<1, false>(a, st);
    case 2: return awq ? launch_fl<2, true>(a, st) : launch_fl<2, false>(a, st);
    default: return awq ? launch_fl<4, true>(a, st) : launch_fl<4, false>(a, st);
  }
}

}  // namespace llmoc
