// linear.cu — dense INT4 products on device-resident weights,
//
//     Y[t, m] = sum_g s[m, g] * sum_{k in g} (q[m, k] - zp) * X[t, k]  (+ R[t, m])
//
// (GPTQ: + z[m, g] * sum_{k in g} X[t, k] with zp = 0), the matrix-vector and
// small-batch products of a decode step.  What bounds them is reading the
// weights once: M * K / 2 bytes.
//
// One warp owns RT 16-row tiles of W, a block of NT * 8 tokens and a slice of
// K.  It streams its weights through a ring of kRing 512-byte chunks held in
// registers: a chunk (16 rows x 64 k) is one coalesced 16-byte load per lane,
// reissued for the chunk kRing further on as soon as it is consumed, so every
// warp keeps kRing * 512 bytes in flight.  A word's eight nibbles become the
// bf16 A fragments of one mma.m16n8k16 (128 + q by one lop3 per pair, then an
// exact subtraction of 128 + zp), so products and group sums are exact up to
// the tensor core's fp32 accumulation; each group's fp32 partial is scaled on
// the accumulator.  Activations are the B fragments, read by 16-byte loads
// that hit L1 after their first use on an SM.
#include <algorithm>
#include <string>

#include "ops.cuh"

namespace llmoc {

namespace {

constexpr int kLinWarps = 8;
constexpr int kLinThreads = kLinWarps * 32;

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t nib_pair(uint32_t w) {  // (128 + q_lo, 128 + q_hi) as bf16
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(w), "r"(0x000F000Fu), "r"(0x43004300u));
  return d;
}
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r =
      __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight consecutive activations of one token as four bf16 pairs.
__device__ __forceinline__ uint4 load_x(const __nv_bfloat16* p, bool ok, int vec) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (ok) {
    if (vec) {
      v = __ldg(reinterpret_cast<const uint4*>(p));
    } else {
      const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
      v.x = __ldg(u) | ((uint32_t)__ldg(u + 1) << 16);
      v.y = __ldg(u + 2) | ((uint32_t)__ldg(u + 3) << 16);
      v.z = __ldg(u + 4) | ((uint32_t)__ldg(u + 5) << 16);
      v.w = __ldg(u + 6) | ((uint32_t)__ldg(u + 7) << 16);
    }
  }
  return v;
}

// GSB: 32-wide blocks per scale group: 1, 2 or 4, or 0 for any other multiple
// (then each block is scaled on its own).
template <int GSB, bool AWQ, int NT, int RT>
__global__ void __launch_bounds__(kLinThreads, 2) k_linear(const LinArgs a) {
  constexpr int kRing = 8 / RT;
  constexpr int kGpc = GSB == 2 || GSB == 4 ? 1 : 2;  // scale pairs fetched per 64-wide chunk
  constexpr int kRows = RT * 16, kCols = NT * 8, kColLd = kRows + 4;
  __shared__ float red[kLinWarps][kCols * kColLd];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tb = blockIdx.x % a.ntb;
  const int ks = a.ks, upc = kLinWarps / ks;
  const int u0 = (blockIdx.x / a.ntb) * upc;            // first unit of the CTA
  const int unit = u0 + warp / ks, sl = warp % ks;
  const int nu = (a.mt + RT - 1) / RT;
  int c0 = 0, c1 = 0;
  if (unit < nu) {  // slices of whole chunk pairs (a group of 128 never straddles two)
    const int pairs = (a.Kc + 1) >> 1;
    c0 = min(a.Kc, 2 * (int)((long long)pairs * sl / ks));
    c1 = min(a.Kc, 2 * (int)((long long)pairs * (sl + 1) / ks));
  }
  int tile[RT];
  const uint4* qp[RT];
  const __half2* sp[RT];
  const __half2* zp[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {  // a tile past the end repeats the last one; its rows are not stored
    tile[r] = min(unit * RT + r, a.mt - 1);
    qp[r] = a.q + (size_t)tile[r] * a.Kc * 32 + piece_slot(lane);
    sp[r] = a.s + (size_t)tile[r] * a.ng * 8 + g;
    zp[r] = AWQ ? nullptr : a.z + (size_t)tile[r] * a.ng * 8 + g;
  }
  // scale group of block kb of chunk c
  const int gsb = a.gs >> 5;
  auto grp = [&](int c, int kb) { return GSB == 4 ? c >> 1 : GSB == 2 ? c : GSB == 1 ? 2 * c + kb : (2 * c + kb) / gsb; };
  auto ld_s = [&](const __half2* p, int c, int kb) { return __ldg(p + (size_t)min(grp(c, kb), a.ng - 1) * 8); };

  uint4 qw[kRing][RT];
  __half2 sw[kRing][RT][kGpc], zw[kRing][RT][kGpc];
  auto fetch = [&](int i, int c) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      qw[i][r] = ld_stream(qp[r] + (size_t)c * 32);
#pragma unroll
      for (int kb = 0; kb < kGpc; ++kb) {
        sw[i][r][kb] = ld_s(sp[r], c, kb);
        if (!AWQ) zw[i][r][kb] = ld_s(zp[r], c, kb);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < kRing; ++i)
    if (c0 + i < c1) fetch(i, c0 + i);  // weights do not depend on the previous kernel
  grid_dep_wait();
  grid_dep_release();

  float acc[RT][NT][4], part[RT][NT][4], xs[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xs[n][i] = 0.f;
#pragma unroll
      for (int r = 0; r < RT; ++r) acc[r][n][i] = part[r][n][i] = 0.f;
    }
  }
  const uint32_t zoff = AWQ ? (0x4300u + (uint32_t)a.zp) * 0x10001u : 0x43004300u;  // 128 + zp, exact below 256
  const int tok0 = tb * kCols + g;
  const __nv_bfloat16* xp = a.X + (long long)tok0 * a.ldx + 8 * t;

  auto flush = [&](const __half2 (&s)[RT], const __half2 (&z)[RT]) {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float2 sf = __half22float2(s[r]);
      float2 zf = make_float2(0.f, 0.f);
      if (!AWQ) zf = __half22float2(z[r]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[r][n][0] = fmaf(sf.x, part[r][n][0], acc[r][n][0]);
        acc[r][n][1] = fmaf(sf.x, part[r][n][1], acc[r][n][1]);
        acc[r][n][2] = fmaf(sf.y, part[r][n][2], acc[r][n][2]);
        acc[r][n][3] = fmaf(sf.y, part[r][n][3], acc[r][n][3]);
        if (!AWQ) {
          acc[r][n][0] = fmaf(zf.x, xs[n][0], acc[r][n][0]);
          acc[r][n][1] = fmaf(zf.x, xs[n][1], acc[r][n][1]);
          acc[r][n][2] = fmaf(zf.y, xs[n][0], acc[r][n][2]);
          acc[r][n][3] = fmaf(zf.y, xs[n][1], acc[r][n][3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) part[r][n][i] = 0.f;
      }
    }
    if (!AWQ) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) xs[n][i] = 0.f;
    }
  };

  for (int cb = c0; cb < c1; cb += kRing) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) {
      const int c = cb + i;
      if (c >= c1) break;  // uniform over the warp
      uint32_t w[RT][4];
      __half2 s[kGpc][RT], z[kGpc][RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        w[r][0] = qw[i][r].x, w[r][1] = qw[i][r].y, w[r][2] = qw[i][r].z, w[r][3] = qw[i][r].w;
#pragma unroll
        for (int kb = 0; kb < kGpc; ++kb) {
          s[kb][r] = sw[i][r][kb];
          if (!AWQ) z[kb][r] = zw[i][r][kb];
        }
      }
      if (c + kRing < c1) fetch(i, c + kRing);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int k = c * 64 + kb * 32;
        uint4 x[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
          x[n] = load_x(xp + (long long)n * 8 * a.ldx + k, tok0 + n * 8 < a.T && k < a.K, a.x_vec);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          if (!AWQ) {
            const uint32_t ones[4] = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(xs[n], ones, kt ? x[n].z : x[n].x, kt ? x[n].w : x[n].y);
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            const uint32_t v = w[r][kb * 2 + kt];
            uint32_t f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = sub2(nib_pair(v >> (4 * j)), zoff);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(part[r][n], f, kt ? x[n].z : x[n].x, kt ? x[n].w : x[n].y);
          }
        }
        if (kGpc == 2) flush(s[kb], z[kb]);
      }
      if (GSB == 2 || (GSB == 4 && ((c & 1) || c + 1 == c1))) flush(s[0], z[0]);
    }
  }

  auto store = [&](int row, int tok, float v) {
    if (row >= a.M || tok >= a.T) return;
    if (a.R) v += __bfloat162float(a.R[(long long)tok * a.ldr + row]);
    if (a.y_f32)
      reinterpret_cast<float*>(a.Y)[(long long)tok * a.ldy + row] = v;
    else
      reinterpret_cast<__nv_bfloat16*>(a.Y)[(long long)tok * a.ldy + row] = __float2bfloat16_rn(v);
  };
  // partial sums of the K slices meet in shared memory and are added in slice order
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[warp][(n * 8 + 2 * t + (i & 1)) * kColLd + r * 16 + g + (i >> 1) * 8] = acc[r][n][i];
  __syncthreads();
  const int rows_cta = upc * kRows;
  for (int e = threadIdx.x; e < rows_cta * kCols; e += kLinThreads) {
    const int row = e % rows_cta, col = e / rows_cta, w0 = row / kRows * ks;
    float v = 0.f;
    for (int s = 0; s < ks; ++s) v += red[w0 + s][col * kColLd + row % kRows];
    store(u0 * kRows + row, tb * kCols + col, v);
  }
}

template <int GSB, bool AWQ>
cudaError_t launch_gs(LinArgs a, cudaStream_t st) {
  const int nt = a.T <= 8 ? 1 : a.T <= 16 ? 2 : 4;
  const int rt = nt == 1 ? 1 : 2;
  a.ntb = (a.T + nt * 8 - 1) / (nt * 8);
  const int units = (a.mt + rt - 1) / rt;
  // K split: as few warps per tile as give the machine 16 warps per SM
  int ks = 1;
  while (ks < kLinWarps && (long long)units * a.ntb * ks < 148 * 16 && a.Kc >= 4 * ks) ks *= 2;
  a.ks = ks;
  const int upc = kLinWarps / ks;
  const dim3 grid((unsigned)((long long)((units + upc - 1) / upc) * a.ntb));
  if (nt == 1) return launch_pdl(k_linear<GSB, AWQ, 1, 1>, grid, dim3(kLinThreads), 0, st, a);
  if (nt == 2) return launch_pdl(k_linear<GSB, AWQ, 2, 2>, grid, dim3(kLinThreads), 0, st, a);
  return launch_pdl(k_linear<GSB, AWQ, 4, 2>, grid, dim3(kLinThreads), 0, st, a);
}

__global__ void k_pair_rows(uint16_t* s, size_t n) {
  const size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  uint16_t v[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) v[r] = s[i * 16 + r];
#pragma unroll
  for (int r = 0; r < 16; ++r) s[i * 16 + (r & 7) * 2 + (r >> 3)] = v[r];
}

}  // namespace

cudaError_t launch_pair_rows(uint16_t* s, size_t n, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  k_pair_rows<<<(unsigned)((n + 255) / 256), 256, 0, st>>>(s, n);
  return cudaGetLastError();
}

cudaError_t launch_linear(const LinArgs& a, bool awq, cudaStream_t st) {
  switch (a.gs) {
    case 32: return awq ? launch_gs<1, true>(a, st) : launch_gs<1, false>(a, st);
    case 64: return awq ? launch_gs<2, true>(a, st) : launch_gs<2, false>(a, st);
    case 128: return awq ? launch_gs<4, true>(a, st) : launch_gs<4, false>(a, st);
    default: return awq ? launch_gs<0, true>(a, st) : launch_gs<0, false>(a, st);
  }
}

}  // namespace llmoc
