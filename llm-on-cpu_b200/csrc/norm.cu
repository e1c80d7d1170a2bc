// norm.cu — what stands between two blocks of a decoder, in one pass over the
// rows:
//
//     u  = post(block)                      post: none, RMS norm or layer norm
//     r' = residual_scale * residual + block_scale * act(gate) * u
//     n  = pre(r')                          the norm before the next block
//
// RMS norm: x * rsqrt(mean(x^2) + eps) * w; layer norm: (x - mean) *
// rsqrt(mean((x - mean)^2) + eps) * w + b.  r' is stored rounded to the
// residual's type, n is computed from the unrounded r'; everything in between
// is fp32.
//
// It is bound by HBM (each operand read once, each result written once) and,
// for few rows, by the launch and the chain load -> reduce -> reduce -> store.
// A group of G threads holds a whole row in registers, so both norms need no
// second read; the variance of a layer norm is the centred sum over those
// registers.  8192 x 4096 bf16 rows with a gate per token take 44.7 us, 6.0 TB/s,
// 0.93 of a plain copy's rate; 129 x 5001 with an fp32 residual, whose odd width
// allows single columns only, 7.5 us; one row of 2048 2.1 us.  Rows copied ahead in
// bulk by CTAs that stay (59.6 us) were slower than more CTAs in flight.
#include <algorithm>
#include <cfloat>
#include <string>

#include "../../include/llmoc_b200.h"
#include "ops.cuh"

namespace llmoc {

namespace {

// Eight consecutive values as fp32 by 16-byte loads.
__device__ __forceinline__ void load8(const void* p, long long i, int f32, float (&v)[8]) {
  if (f32) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(w[k] << 16);
      v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
    }
  }
}
__device__ __forceinline__ void store8(void* p, long long i, int f32, const float (&v)[8]) {
  if (f32) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
__device__ __forceinline__ float load1(const void* p, long long i, int f32) {
  return f32 ? reinterpret_cast<const float*>(p)[i] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
// Sum over the G threads of a row, in a fixed order; every thread gets it.
template <int G>
__device__ __forceinline__ float row_sum(float v, float* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (G > 32) {
    constexpr int W = G / 32;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) v += sh[w];
  }
  return v;
}

// threads of a CTA: a row's, or four rows of one warp
constexpr int norm_threads(int G) { return G > 32 ? G : 128; }

// How a thread holds its columns of an operand: eight neighbours per 16-byte
// access (kVec), all of them bf16 and kept packed until used (kBf16), or columns
// G apart (kScalar).
enum { kScalar = 0, kVec = 1, kBf16 = 2 };

template <int MODE, int VPT>
struct Held {
  float v[8 * VPT];
};
template <int VPT>
struct Held<kBf16, VPT> {
  uint4 v[VPT];
};

// HOLD: every operand of a row is requested before the first reduction, so a row
// waits for memory once.  Without, the weights are fetched where they are used,
// which leaves registers for more rows per SM.
template <int G, int VPT, int MODE, bool HOLD>
__global__ void __launch_bounds__(norm_threads(G), (MODE == kBf16 || !HOLD) && VPT <= 2 ? 1024 / norm_threads(G) : 1)
    k_norm(const __grid_constant__ NormArgs a) {
  constexpr int N = 8 * VPT;
  using Row = Held<MODE, VPT>;
  __shared__ float sh[8][32];  // one slice per reduction of a row: no second barrier between two of them
  const int tid = G > 32 ? threadIdx.x : threadIdx.x & 31;
  const int row = G > 32 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
  grid_dep_wait();
  grid_dep_release();
  if (row >= a.T) return;  // whole warps, and only where no barrier follows (G == 32)
  const int H = a.H;
  const float inv = 1.f / (float)H;
  auto col = [&](int j) { return MODE != kScalar ? ((j >> 3) * G + tid) * 8 + (j & 7) : j * G + tid; };
  auto inside = [&](int j) { return MODE != kScalar ? ((j >> 3) * G + tid) * 8 < H : j * G + tid < H; };
  // columns past H are held as 0
  auto fetch = [&](const void* p, long long off, int f32, Row& r) {
    if constexpr (MODE == kBf16) {
#pragma unroll
      for (int q = 0; q < VPT; ++q)
        r.v[q] = inside(q * 8) ? *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p) + off + col(q * 8))
                               : make_uint4(0, 0, 0, 0);
    } else if constexpr (MODE == kVec) {
#pragma unroll
      for (int q = 0; q < VPT; ++q) {
        float x[8] = {};
        if (inside(q * 8)) load8(p, off + col(q * 8), f32, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) r.v[q * 8 + k] = x[k];
      }
    } else if (f32) {
      const float* src = reinterpret_cast<const float*>(p) + off + tid;
#pragma unroll
      for (int j = 0; j < N; ++j) r.v[j] = inside(j) ? src[j * G] : 0.f;
    } else {
      const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(p) + off + tid;
#pragma unroll
      for (int j = 0; j < N; ++j) r.v[j] = inside(j) ? __bfloat162float(src[j * G]) : 0.f;
    }
  };
  auto at = [&](const Row& r, int j) {
    if constexpr (MODE == kBf16) {
      const uint4& u = r.v[j >> 3];
      const uint32_t w = (j & 7) < 2 ? u.x : (j & 7) < 4 ? u.y : (j & 7) < 6 ? u.z : u.w;
      return __uint_as_float(j & 1 ? w & 0xFFFF0000u : w << 16);
    } else {
      return r.v[j];
    }
  };
  auto store = [&](void* p, long long off, int f32, const float (&v)[N]) {
    if (MODE != kScalar) {
#pragma unroll
      for (int q = 0; q < VPT; ++q) {
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = v[q * 8 + k];
        if (inside(q * 8)) store8(p, off + col(q * 8), MODE == kBf16 ? 0 : f32, x);
      }
    } else if (f32) {
      float* dst = reinterpret_cast<float*>(p) + off + tid;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (inside(j)) dst[j * G] = v[j];
    } else {
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(p) + off + tid;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (inside(j)) dst[j * G] = __float2bfloat16_rn(v[j]);
    }
  };
  // x = norm(x); `si` picks the reductions' shared slices.  Sums that leave
  // fp32's range (squares of values above about 1e17) are formed again from
  // x * 2^-80, which is exact and drops out of the quotient; eps, far below an
  // ulp of such sums, becomes any small value that keeps 0 / 0 out.
  auto normed = [&](float (&x)[N], int kind, const void* w, const void* b, Row& hw, Row& hb, int si) {
    float eps = a.eps;
    bool shrunk = false;
    auto shrink = [&]() {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= 0x1p-80f;
      eps = 1e-30f;
      shrunk = true;
    };
    auto sum = [&](int i) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) s += x[j];
      return row_sum<G>(s, sh[i]);
    };
    auto squares = [&](int i) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < N; ++j) s = fmaf(x[j], x[j], s);
      return row_sum<G>(s, sh[i]);
    };
    if (kind == LLMOC_NORM_LAYER) {
      float s = sum(si);
      if (!(fabsf(s) <= FLT_MAX)) {  // the same for all threads of the row
        shrink();
        s = sum(si + 1);
      }
      const float mean = s * inv;
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = inside(j) ? x[j] - mean : 0.f;
    }
    float q = squares(si + 2);
    if (!(q <= FLT_MAX) && !shrunk) {
      shrink();
      q = squares(si + 3);
    }
    const float rs = rsqrtf(q * inv + eps);
    if (w) {
      if (!HOLD) fetch(w, 0, a.w_f32, hw);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = x[j] * rs * (at(hw, j) + a.w_off);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= rs;
    }
    if (b) {
      if (!HOLD) fetch(b, 0, a.w_f32, hb);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] += at(hb, j);
    }
  };
  auto act = [&](float v) { return a.gate_sigmoid ? 1.f / (1.f + expf(-v)) : v; };

  const bool post = a.block && a.post != LLMOC_NORM_NONE, pre = a.out && a.pre != LLMOC_NORM_NONE;
  Row hx, hr, hg, pw, pb, qw, qb;
  if (a.block) fetch(a.block, row * a.ld_block, a.block_f32, hx);
  if (a.res) fetch(a.res, row * a.ld_res, a.res_f32, hr);
  float g1 = 0.f;
  if (a.gate && a.gate_col == 0) g1 = load1(a.gate, row * a.gate_row, a.gate_f32);
  if (HOLD) {
    if (a.gate && a.gate_col) fetch(a.gate, row * a.gate_row, a.gate_f32, hg);
    if (post && a.post_w) fetch(a.post_w, 0, a.w_f32, pw);
    if (post && a.post_b) fetch(a.post_b, 0, a.w_f32, pb);
    if (pre && a.pre_w) fetch(a.pre_w, 0, a.w_f32, qw);
    if (pre && a.pre_b) fetch(a.pre_b, 0, a.w_f32, qb);
  }
  float r[N];
  if (a.block) {
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = at(hx, j);
    if (post) normed(x, a.post, a.post_w, a.post_b, pw, pb, 0);
    float scale = a.block_scale;
    if (a.gate) {
      if (a.gate_col == 0) {  // one value a row
        scale *= act(g1);
      } else {
        if (!HOLD) fetch(a.gate, row * a.gate_row, a.gate_f32, hg);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= act(at(hg, j));
      }
    }
    if (a.res) {
#pragma unroll
      for (int j = 0; j < N; ++j) r[j] = fmaf(scale, x[j], a.res_scale * at(hr, j));
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) r[j] = scale * x[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = a.res_scale * at(hr, j);
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (!inside(j)) r[j] = 0.f;
  if (a.res_out) store(a.res_out, row * a.ld_res_out, a.res_f32, r);
  if (a.out) {
    if (pre) normed(r, a.pre, a.pre_w, a.pre_b, qw, qb, 4);
    store(a.out, row * a.ld_out, a.out_f32, r);
  }
}

// every operand read or written in rows is bf16
bool all_bf16(const NormArgs& a) {
  return !(a.block && a.block_f32) && !((a.res || a.res_out) && a.res_f32) && !(a.out && a.out_f32) &&
         !((a.post_w || a.post_b || a.pre_w || a.pre_b) && a.w_f32) && !(a.gate && a.gate_col && a.gate_f32);
}

template <int G, int VPT, bool HOLD>
cudaError_t launch_held(const NormArgs& a, cudaStream_t st) {
  const dim3 block(norm_threads(G));
  const dim3 grid((unsigned)(G > 32 ? a.T : (a.T + 3) / 4));
  if (!a.vec) return launch_pdl(k_norm<G, VPT, kScalar, HOLD>, grid, block, 0, st, a);
  if (all_bf16(a)) return launch_pdl(k_norm<G, VPT, kBf16, VPT < 4>, grid, block, 0, st, a);
  return launch_pdl(k_norm<G, VPT, kVec, HOLD>, grid, block, 0, st, a);
}

// Up to two rows per SM the chain of one row decides, and its operands are all
// held (packed bf16 ones are, in any case); more rows want more of them
// resident.
template <int G, int VPT>
cudaError_t launch_g(const NormArgs& a, cudaStream_t st) {
  if constexpr (VPT < 4)
    if (a.T <= 2 * 148) return launch_held<G, VPT, true>(a, st);
  return launch_held<G, VPT, false>(a, st);
}

}  // namespace

cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  const bool few = !a.vec && a.T <= 2 * 148;  // single-column accesses: fewer of them a thread
  if (a.H <= 256) return launch_g<32, 1>(a, st);
  // Many rows of bf16: more columns a thread leave fewer threads to meet in a
  // row's reductions and as many bytes in flight per SM.  16 columns from two rows
  // per SM on (1000 x 2048 5.2 -> 4.5 us, 8192 x 512 15.9 -> 8.9), 32 columns of
  // wide rows from 1024 rows on (8192 x 4096 53.5 -> 44.6, 4096 x 8192 62 -> 47.5,
  // 8192 x 2048 27.4 -> 24.4; 500 x 4096 4.8 -> 5.1 without that rule).  64 columns
  // are slower again (48.5 us at 8192 x 4096).  Mixed types unpack into twice the
  // registers and lose by it (fp32 residual, 8192 x 4096: 92 -> 138 us).
  if (a.vec && a.T > 2 * 148 && all_bf16(a)) {
    const bool wide = a.T > 1024;
    if (a.H <= 512) return launch_g<32, 2>(a, st);
    if (a.H <= 1024) return launch_g<64, 2>(a, st);
    if (a.H <= 2048) return wide ? launch_g<64, 4>(a, st) : launch_g<128, 2>(a, st);
    if (a.H <= 4096 && wide) return launch_g<128, 4>(a, st);
    if (a.H <= 8192 && wide) return launch_g<256, 4>(a, st);
  }
  if (a.H <= 1024) return launch_g<128, 1>(a, st);
  if (a.H <= 2048) return launch_g<256, 1>(a, st);
  if (a.H <= 4096) return few ? launch_g<512, 1>(a, st) : launch_g<256, 2>(a, st);
  if (a.H <= 8192) return few ? launch_g<1024, 1>(a, st) : launch_g<512, 2>(a, st);
  return launch_g<512, 4>(a, st);
}

}  // namespace llmoc
