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
// registers.
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
__device__ __forceinline__ void store1(void* p, long long i, int f32, float v) {
  if (f32)
    reinterpret_cast<float*>(p)[i] = v;
  else
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
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

constexpr int kNormMinThreads = 128;  // rows of one warp share a CTA of four

// VEC: eight consecutive columns per 16-byte access; else columns G apart.
template <int G, int VPT, bool VEC>
__global__ void __launch_bounds__(G > kNormMinThreads ? G : kNormMinThreads) k_norm(const NormArgs a) {
  constexpr int N = 8 * VPT;
  __shared__ float sh[8][32];  // one slice per reduction of a row: no second barrier between two of them
  const int tid = G > 32 ? threadIdx.x : threadIdx.x & 31;
  const int row = G > 32 ? blockIdx.x : blockIdx.x * (kNormMinThreads / 32) + (threadIdx.x >> 5);
  grid_dep_wait();
  grid_dep_release();
  if (row >= a.T) return;  // whole warps, and only where no barrier follows (G == 32)
  const int H = a.H;
  const float inv = 1.f / (float)H;
  // column of value j
  auto col = [&](int j) { return VEC ? ((j >> 3) * G + tid) * 8 + (j & 7) : j * G + tid; };
  auto load = [&](const void* p, long long off, int f32, float (&v)[N], float fill) {
    if (VEC) {
#pragma unroll
      for (int q = 0; q < VPT; ++q) {
        float x[8];
        const int c = (q * G + tid) * 8;
        if (c < H) load8(p, off + c, f32, x);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[q * 8 + k] = c < H ? x[k] : fill;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = col(j) < H ? load1(p, off + col(j), f32) : fill;
    }
  };
  auto store = [&](void* p, long long off, int f32, const float (&v)[N]) {
    if (VEC) {
#pragma unroll
      for (int q = 0; q < VPT; ++q) {
        const int c = (q * G + tid) * 8;
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = v[q * 8 + k];
        if (c < H) store8(p, off + c, f32, x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (col(j) < H) store1(p, off + col(j), f32, v[j]);
    }
  };
  // x = norm(x); `at` picks the reductions' shared slices.  Sums that leave
  // fp32's range (squares of values above about 1e17) are formed again from
  // x * 2^-80, which is exact and drops out of the quotient; eps, far below an
  // ulp of such sums, becomes any small value that keeps 0 / 0 out.
  auto normed = [&](float (&x)[N], int kind, const void* w, const void* b, int at) {
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
      float s = sum(at);
      if (!(fabsf(s) <= FLT_MAX)) {  // the same for all threads of the row
        shrink();
        s = sum(at + 1);
      }
      const float mean = s * inv;
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = col(j) < H ? x[j] - mean : 0.f;
    }
    float q = squares(at + 2);
    if (!(q <= FLT_MAX) && !shrunk) {
      shrink();
      q = squares(at + 3);
    }
    const float rs = rsqrtf(q * inv + eps);
    float v[N];
    if (w) {
      load(w, 0, a.w_f32, v, 0.f);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = x[j] * rs * (v[j] + a.w_off);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] *= rs;
    }
    if (b) {
      load(b, 0, a.w_f32, v, 0.f);
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] += v[j];
    }
  };

  auto act = [&](float v) { return a.gate_sigmoid ? 1.f / (1.f + expf(-v)) : v; };
  float r[N];
  if (a.res)
    load(a.res, row * a.ld_res, a.res_f32, r, 0.f);
  else
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = 0.f;
  if (a.block) {
    float x[N];
    load(a.block, row * a.ld_block, a.block_f32, x, 0.f);
    if (a.post != LLMOC_NORM_NONE) normed(x, a.post, a.post_w, a.post_b, 0);
    if (a.gate) {
      float gt[N];
      const long long off = row * a.gate_row;
      if (a.gate_col == 0) {  // one value a row
        const float one = act(load1(a.gate, off, a.gate_f32));
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= one;
      } else {
        load(a.gate, off, a.gate_f32, gt, 0.f);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] *= act(gt[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] = fmaf(a.block_scale, x[j], a.res_scale * r[j]);
  } else if (a.res_scale != 1.f) {
#pragma unroll
    for (int j = 0; j < N; ++j) r[j] *= a.res_scale;
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (col(j) >= H) r[j] = 0.f;
  if (a.res_out) store(a.res_out, row * a.ld_res_out, a.res_f32, r);
  if (a.out) {
    if (a.pre != LLMOC_NORM_NONE) normed(r, a.pre, a.pre_w, a.pre_b, 4);
    store(a.out, row * a.ld_out, a.out_f32, r);
  }
}

template <int G, int VPT>
cudaError_t launch_g(const NormArgs& a, cudaStream_t st) {
  const dim3 block(std::max(G, kNormMinThreads));
  const dim3 grid((unsigned)(G > 32 ? a.T : (a.T + 3) / 4));
  return a.vec ? launch_pdl(k_norm<G, VPT, true>, grid, block, 0, st, a)
               : launch_pdl(k_norm<G, VPT, false>, grid, block, 0, st, a);
}

}  // namespace

cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  if (a.H <= 256) return launch_g<32, 1>(a, st);
  if (a.H <= 1024) return launch_g<128, 1>(a, st);
  if (a.H <= 2048) return launch_g<256, 1>(a, st);
  if (a.H <= 4096) return launch_g<256, 2>(a, st);
  if (a.H <= 8192) return launch_g<512, 2>(a, st);
  return launch_g<512, 4>(a, st);
}

}  // namespace llmoc
