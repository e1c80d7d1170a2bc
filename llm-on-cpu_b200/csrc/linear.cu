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
// word the 8 k from 8 t of one of the chunk's two 32 k) followed by the block's scales (and zeros) as fp16 pairs of rows
// (g, g + 8).  Groups that are other multiples of 32, 64 or 128 repeat their
// scale, so a block holds 8, 4 or 2 groups of 32, 64 or 128.
//
// Work.  A warp owns RT tiles against NT * 8 tokens over a slice of K.  The
// eight warps of a CTA take 8 / ksw tile groups and split K ksw ways; a cluster
// of c CTAs splits K c ways more.  With c = ksw = 1 a CTA walks tile groups
// (persistent) and its warps never meet; otherwise the partial sums meet in
// (distributed) shared memory and are added in slice order, so no workspace is
// needed and the bits do not depend on timing.
//
// The stream runs through a ring of registers, 4 KB per warp: a chunk is one
// coalesced 16-byte load per lane, reissued for the place 8 / RT chunks further
// on as soon as it is consumed, across tile ends.
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
#include <string>

#include "ops.cuh"

namespace llmoc {

namespace {

constexpr int kLinWarps = 8;
constexpr int kLinThreads = kLinWarps * 32;
constexpr uint32_t kOffset = 16;  // A elements are kOffset + q

__device__ __forceinline__ uint4 ld_stream(const char* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_pair(const char* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
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
// *p of the cluster's CTA `rank` (c = 1: of this CTA)
__device__ __forceinline__ float ld_cluster(const float* p, int rank, int c) {
  if (c == 1) return *p;
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
  int units;  // tile groups (8 / ksw warps x RT tiles)
  int bps;    // blocks of 256 k per staged slab
  int nslab;  // slabs of a CTA's share of K
};

// FL: 32-wide blocks per scale group (1, 2, 4); TP: token rows staged (1, or
// NT * 8).
template <int FL, bool AWQ, int NT, int RT, int TP>
__global__ void __launch_bounds__(kLinThreads, 2) k_linear(const LinArgs a, const LinPlan p) {
  constexpr int kBB = lin_block_bytes(FL, !AWQ);
  constexpr int GB = 2 / RT;                    // blocks in flight per tile
  constexpr int kGrp = 8 / FL;                  // scale groups per block
  constexpr int kRows = RT * 16, kCols = NT * 8, kColLd = kRows + 4;
  constexpr int kXW = TP * 4;                   // 16-byte pieces per 32 k
  extern __shared__ __align__(16) uint4 sx[];   // [slab's 32-blocks][kXW]: B fragments
  float* xs = reinterpret_cast<float*>(sx + (size_t)p.bps * 8 * kXW);  // [slab's groups][TP]: activation sums
  float* red = xs + (size_t)p.bps * kGrp * TP;                         // [warp][col][row]: partial sums
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int c = 1 << p.lc, ksw = 1 << p.lk, lr = 3 - p.lk;  // lr: log2 of the CTA's tile groups
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
    const int tile = ((unit << lr) + wt) * RT;
    s.b0 = n * wk >> p.lk;
    s.nb = tile < a.mt && unit < p.units ? (n * (wk + 1) >> p.lk) - s.b0 : 0;
    s.q = a.q + (size_t)min(tile, a.mt - 1) * tile_bytes + (size_t)(s0 + s.b0) * kBB;
    return s;
  };
  uint4 qw[GB][4][RT];
  uint32_t sw[GB][kGrp][RT], zw[GB][kGrp][RT];
  // a tile past the end reads the last one again; its rows are not stored
  auto tile_off = [&](int r, int unit) { return r && ((unit << lr) + wt) * RT + r < a.mt ? tile_bytes : 0; };
  const int lq = (g * 4 + (t ^ ((g >> 1) & 3))) * 16, ls = 2048 + g * 4;

  int unit = blockIdx.x >> p.lc, slab = 0;
  Seg cur = seg_of(unit, 0);
#pragma unroll
  for (int j = 0; j < GB; ++j)  // the weights do not depend on the previous kernel
    if (j < cur.nb)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const char* q = cur.q + tile_off(r, unit) + j * kBB;
#pragma unroll
        for (int i = 0; i < 4; ++i) qw[j][i][r] = ld_stream(q + lq + i * 512);
#pragma unroll
        for (int i = 0; i < kGrp; ++i) {
          sw[j][i][r] = ld_pair(q + ls + i * 32);
          if (!AWQ) zw[j][i][r] = ld_pair(q + ls + (kGrp + i) * 32);
        }
      }
  grid_dep_wait();
  grid_dep_release();

  float acc[RT][NT][4], part[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = part[r][n][i] = 0.f;
  const float zoff = AWQ ? -(float)(kOffset + a.zp) : -(float)kOffset;
  const uint4* xl = sx + (TP == 1 ? t : lane);
  const float* xsl = xs + (TP == 1 ? 0 : 2 * t);

  auto flush = [&](const float* xg, const uint32_t (&s)[RT], const uint32_t (&z)[RT]) {  // xg: the group's sums
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float2 x;
      if (TP == 1)
        x.x = x.y = *xg;
      else
        x = *reinterpret_cast<const float2*>(xg + n * 8);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float2 sf = pair_f32(s[r]);
        float (&o)[4] = acc[r][n];
        float (&q)[4] = part[r][n];
        if (!AWQ) {
          const float2 zf = pair_f32(z[r]);
          o[0] = fmaf(zf.x, x.x, o[0]), o[1] = fmaf(zf.x, x.y, o[1]);
          o[2] = fmaf(zf.y, x.x, o[2]), o[3] = fmaf(zf.y, x.y, o[3]);
        }
        o[0] = fmaf(sf.x, fmaf(zoff, x.x, q[0]), o[0]), o[1] = fmaf(sf.x, fmaf(zoff, x.y, q[1]), o[1]);
        o[2] = fmaf(sf.y, fmaf(zoff, x.x, q[2]), o[2]), o[3] = fmaf(sf.y, fmaf(zoff, x.y, q[3]), o[3]);
        q[0] = q[1] = q[2] = q[3] = 0.f;
      }
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
    for (int b = 0; b < cur.nb || b == 0; b += GB) {
      const bool last = b + GB >= cur.nb;
      const char* src = last ? nxt.q : cur.q + (size_t)(b + GB) * kBB;
      const int left = last ? nxt.nb : cur.nb - b - GB;  // blocks to fetch from src
      const size_t off = RT > 1 ? tile_off(1, last ? nunit : unit) : 0;
#pragma unroll
      for (int j = 0; j < GB; ++j) {
        const bool more = j < left;
        const char* sq = src + j * kBB;
        if (b + j < cur.nb) {  // uniform over the warp
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t w[RT][4];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              w[r][0] = qw[j][i][r].x, w[r][1] = qw[j][i][r].y, w[r][2] = qw[j][i][r].z, w[r][3] = qw[j][i][r].w;
              if (more) qw[j][i][r] = ld_stream(sq + (r ? off : 0) + lq + i * 512);
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
              uint4 x[NT];
#pragma unroll
              for (int n = 0; n < NT; ++n) x[n] = xb[(2 * i + kb) * kXW + n * 32];
#pragma unroll
              for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                  uint32_t f[4];
#pragma unroll
                  for (int h = 0; h < 4; ++h) {  // rows g and g + 8, k in two halves
                    const uint32_t v = w[r][(h & 1) * 2 + kb];
                    f[h] = nib_pair(__funnelshift_r(v, v, 4 * (2 * kt + (h >> 1))));
                  }
#pragma unroll
                  for (int n = 0; n < NT; ++n) mma16816(part[r][n], f, kt ? x[n].z : x[n].x, kt ? x[n].w : x[n].y);
                }
              if ((2 * i + kb) % FL == FL - 1) {
                const int gi = (2 * i + kb) / FL;
                flush(xg + gi * TP, sw[j][gi], zw[j][gi]);
                if (more)
#pragma unroll
                  for (int r = 0; r < RT; ++r) {
                    sw[j][gi][r] = ld_pair(sq + (r ? off : 0) + ls + gi * 32);
                    if (!AWQ) zw[j][gi][r] = ld_pair(sq + (r ? off : 0) + ls + (kGrp + gi) * 32);
                  }
              }
            }
          }
          xb += 8 * kXW;
          xg += kGrp * TP;
        } else if (more) {
#pragma unroll
          for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int i = 0; i < 4; ++i) qw[j][i][r] = ld_stream(sq + (r ? off : 0) + lq + i * 512);
#pragma unroll
            for (int i = 0; i < kGrp; ++i) {
              sw[j][i][r] = ld_pair(sq + (r ? off : 0) + ls + i * 32);
              if (!AWQ) zw[j][i][r] = ld_pair(sq + (r ? off : 0) + ls + (kGrp + i) * 32);
            }
          }
        }
      }
    }
    cur = nxt;
    if (nslab1 == 0) {  // the unit's last slab
      if (p.lk == 0 && p.lc == 0) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              store((((unit << lr) + wt) * RT + r) * 16 + g + (i >> 1) * 8, tok0 + n * 8 + 2 * t + (i & 1), acc[r][n][i]);
      } else {
        // partial sums of the K slices, added in slice order (rank, then warp);
        // such a grid has a cluster per unit, so the buffer is written once
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              red[(warp * kCols + n * 8 + 2 * t + (i & 1)) * kColLd + r * 16 + g + (i >> 1) * 8] = acc[r][n][i];
        if (c > 1)
          cluster_sync();
        else
          __syncthreads();
        constexpr int kLrow = RT == 1 ? 4 : 5;  // log2 of kRows
        const int lrows = lr + kLrow, step = kLinThreads << p.lc;
        const int cols = min(kCols, a.T - tok0);
        for (int e = threadIdx.x + rank * kLinThreads; e < cols << lrows; e += step) {
          const int row = e & ((1 << lrows) - 1), col = e >> lrows, w0 = row >> kLrow;
          const float* at = red + (w0 * kCols + col) * kColLd + (row & (kRows - 1));
          float v = 0.f;
          for (int q = 0; q < c; ++q)
            for (int s = 0; s < ksw; ++s) v += ld_cluster(at + (s << lr) * kCols * kColLd, q, c);
          store((unit << lrows) + row, tok0 + col, v);
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.f;
    }
    unit = nunit;
    slab = nslab1;
  }
  if (c > 1) cluster_sync();  // no CTA leaves while another reads its partial sums
}

constexpr int kLinSmemMax = 100 * 1024;  // two CTAs per SM

template <int FL, bool AWQ, int NT, int RT, int TP>
cudaError_t launch_shape(const LinArgs& a, cudaStream_t st) {
  LinPlan p{};
  const int ntb = (a.T + NT * 8 - 1) / (NT * 8);
  const int tg = (a.mt + RT - 1) / RT;
  // K is split as long as every CTA stays resident at once (two per SM) and a
  // warp keeps a block: inside the CTA while its activations stay below half of
  // its weights, then over a cluster, then inside the CTA at any price.  A second
  // round of CTAs costs more than the shorter slices give (T = 8, 11008 x 4096:
  // 344 CTAs 17.5 us, 172 CTAs 10.3 us).
  int ksw = 1, c = 1;
  auto fits = [&](int w, int k) {
    const int rbt = kLinWarps / w;
    return (long long)((tg + rbt - 1) / rbt) * ntb * k <= 2 * 148 && a.nb >= w * k;
  };
  while (ksw < kLinWarps && TP * ksw * 2 <= 16 * RT && fits(2 * ksw, c)) ksw *= 2, ++p.lk;
  while (c < 8 && fits(ksw, 2 * c)) c *= 2, ++p.lc;
  while (ksw < kLinWarps && fits(2 * ksw, c)) ksw *= 2, ++p.lk;
  const int rbt = kLinWarps / ksw;
  p.units = (tg + rbt - 1) / rbt;
  const bool split = ksw > 1 || c > 1;
  const int red = split ? kLinWarps * NT * 8 * (RT * 16 + 4) * 4 : 0;
  const int per_block = TP * 4 * 8 * 16 + 8 / FL * TP * 4;
  const int share = (a.nb + c - 1) / c;
  p.bps = std::max(1, std::min(share, (kLinSmemMax - red) / per_block));
  p.nslab = (share + p.bps - 1) / p.bps;
  const int smem = p.bps * per_block + red;
  const auto kernel = k_linear<FL, AWQ, NT, RT, TP>;
  static bool attr[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmemMax);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr[dev] = true;
  }
  const long long gx = (split ? p.units : std::min(p.units, std::max(1, 148 * 2 / ntb))) * (long long)c;
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
  if (a.T == 1) return launch_shape<FL, AWQ, 1, 1, 1>(a, st);
  if (a.T <= 8) return launch_shape<FL, AWQ, 1, 1, 8>(a, st);
  return launch_shape<FL, AWQ, 2, 2, 16>(a, st);
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

cudaError_t launch_lin_pack(const LinPack& a, cudaStream_t st) {
  k_lin_pack<<<148 * 8, 256, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_linear(const LinArgs& a, int fl, bool awq, cudaStream_t st) {
  // From 17 tokens on mma.sync, which needs the weights dequantised once per 16
  // tokens, is slower on every shape measured (K = 4096; T = 24, groups of 128:
  // 9.9 against 35 us at 4096 rows, 87 against 88 at 60000); at 16 tokens it is
  // faster for wide matrices and small groups (52 against 81 us at 60000 rows, 60
  // against 154 with groups of 32) and about equal otherwise.
  if (a.T > 16 && (!awq || a.zp < 16)) return launch_linear_umma(a, fl, awq, st);
  switch (fl) {
    case 1: return awq ? launch_fl<1, true>(a, st) : launch_fl<1, false>(a, st);
    case 2: return awq ? launch_fl<2, true>(a, st) : launch_fl<2, false>(a, st);
    default: return awq ? launch_fl<4, true>(a, st) : launch_fl<4, false>(a, st);
  }
}

}  // namespace llmoc
