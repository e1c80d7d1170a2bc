// beam.cu — one step of beam search on the device: the selection over beams
// and vocabulary, and the reordering of the beams' states.
//
// Selection.  With l = logits of a beam (non-finite values masked),
//     cand[w, v] = scores[w] + l[w, v] - (max l + log sum exp(l - max l)),
// the n_out best of a sequence's beams x vocab candidates, ordered by value,
// then beam, then token.  A finished beam has the one candidate (eos, its
// score); a beam with a non-finite score has none.  It is bound by reading the
// logits once.
//
//   k_beam_rows   one CTA per (row, vocabulary slice), which it reads once, a
//                 warp in tiles of 64 bytes a lane: the slice's max and sum of
//                 exponentials, and its n_out best logits.  A lower bound of the
//                 n_out-th best comes from maxima of disjoint sets of elements:
//                 the n_out-th largest of the 256 threads' first maxima, then
//                 the smallest of at least n_out thread groups' running maxima.
//                 What reaches the bound goes to a shared list and is ranked by
//                 counting.  A slice with more such elements than the list holds
//                 (adversarial values, many ties) finds its exact n_out-th best
//                 by bisection, on the values' codes and then on the index.
//   k_beam_merge  one CTA per sequence: each beam's log-sum from its slices,
//                 summed in fp64 (candidates of different beams are compared by
//                 it), and the best of the slices' lists, 2048 entries at a time:
//                 a bound, what reaches it, ranked by counting.
//
// What bounds it (graph replay): 32 sequences x 8 beams x 248320 bf16 logits take
// 44.4 us, 2.9 TB/s.  No unit is busy all of that time: the instructions, some 390 a
// scheduler for a warp's 1024 elements, fill 21 us (the exponentials' unit 17 of
// them), the bytes 20.  A fifth of the time an SM has no warp (the launch, the last
// CTAs); in the rest a scheduler issues in 61 % of the cycles, since 512 CTAs on 592
// places leave it six warps, each of which waits ten cycles per instruction: fixed
// latencies 2.3, loads 1.4, barriers 1.0, instruction fetch and branches 1.1, its
// turn 1.4.  With a fifth of the beams finished (the time is the same) it issues in
// 54 %, and SMs differ by much.  Rows copied ahead in bulk were 3 % slower, and CTAs
// gathered on the live rows gain nothing.  8 x 4 x 131072 fp32 with 8 candidates take 15.0 us
// (1.1 TB/s), 1 x 4 x 32003 7.6 us, of which the two launches and a chain of load,
// first bound, list and merge are nearly all; the merge has 3 to 5 us of each.
//
// Order of summation is fixed by the slice and thread numbers alone, so equal
// rows get equal bits and ties resolve by index.
//
// Reordering.  dst[b, k] = src[b, parent[b, k]] for any number of tensors in
// one launch; a thread owns a column of a sequence's rows, loads it from every
// parent before it stores any, so a tensor may be reordered in place and a parent
// chosen several times is read from HBM once.  Bound by HBM: 32 tensors of 8 x 8
// rows of 256 KB take 140.4 us, 6.3 TB/s, 0.98 of a plain copy's rate.
#include <algorithm>
#include <cfloat>
#include <string>

#include "ops.cuh"

namespace llmoc {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kListMax = 512;
constexpr int kFewHits = 6;   // lanes of a tile whose elements are looked at one lane after the other
constexpr int kListCut = 64;  // list length above which the closing bound is applied once more
constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ float masked(float x) { return fabsf(x) <= FLT_MAX ? x : kNegInf; }
// order-preserving bits of a float (larger value, larger code)
__device__ __forceinline__ uint32_t order_code(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_code(uint32_t c) {
  return __uint_as_float(c & 0x80000000u ? c & 0x7FFFFFFFu : ~c);
}
// a before b in the order "larger value, then smaller index"
__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

// exp(x - m) as 2^(x * kLog2e - log2_ref(m)): the rounding of the constant and
// of the product drop out of the log-sum, which the merge corrects (log_sum).
// Every sum and every change of reference goes by the same rounded product: an
// unrounded one in its place (a contracted multiply-add) is off by 2^-24 of the
// logits' own size.
constexpr float kLog2e = 1.44269504f;
__device__ __forceinline__ float log2_ref(float m) { return __fmul_rn(m, kLog2e); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// At kScaleMax the rounding of the product is up to 16, a factor of 2^16 that the
// sum can bear; above it exp(x - m) is 2^((x - m) * kLog2e), relative to m itself.
// Logits of which one lies above it and one below are at least 32 apart: what such
// a change of reference carries over is below 2^16 e^-32 of the sum, and not
// corrected for.
constexpr float kScaleMax = 0x1p28f;
// the factor from a sum relative to m to one relative to n
__device__ __forceinline__ float rescale(float m, float n) {
  return exp2_fast(fabsf(m) <= kScaleMax && fabsf(n) <= kScaleMax ? __fsub_rn(log2_ref(m), log2_ref(n)) : (m - n) * kLog2e);
}
// log sum exp of a row whose largest value is m, from that sum relative to m
__device__ __forceinline__ double log_sum(float m, double s) {
  if (fabsf(m) > kScaleMax) return (double)m + log(s);
  const float c = log2_ref(m);
  return (double)m + log(s) + ((double)c - (double)m * (double)kLog2e) * 0.69314718055994531;
}

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %4};\n mov.b64 z, {%5, %5};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// A load that stays where it is written (a plain one sinks to its first use,
// a tile later, and waits there).
__device__ __forceinline__ uint4 ld_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ float logit_at(const BeamArgs& a, long long i) {
  return masked(a.f32 ? __ldg(reinterpret_cast<const float*>(a.logits) + i)
                      : bf16_bits_to_f32(__ldg(reinterpret_cast<const unsigned short*>(a.logits) + i)));
}

// By one warp: v[0] = a lower bound of the k-th largest (k <= 256) of the 256
// order codes v, its upper 16 bits (all of a bf16's code).  Eight codes a lane,
// two bits a step.
__device__ __forceinline__ void kth_of_256(uint32_t* v, int k, int lane) {
  uint32_t c[8], kth = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = v[i * 32 + lane];
#pragma unroll 1
  for (int bit = 30; bit >= 16; bit -= 2) {  // two bits a step: three counts, of at most 256 each, in one sum
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (uint32_t d = 1; d < 4; ++d) n += c[i] >= (kth | d << bit) ? 1u << (10 * (d - 1)) : 0u;
    n = __reduce_add_sync(0xffffffffu, n);
    uint32_t most = 0;
#pragma unroll
    for (uint32_t d = 1; d < 4; ++d)
      if ((int)(n >> (10 * (d - 1)) & 1023) >= k) most = d;
    kth |= most << bit;
  }
  if (lane == 0) v[0] = kth;
}

// The slice's n_out best where more elements reach the bound than the list
// holds (long ties, adversarial orders): the n_out-th best value by bisection on
// the order codes (none needed when the maximum itself repeats that often),
// then, among the elements equal to it, the last index that still belongs.
// Reads the slice again for each step.
__device__ __noinline__ int bisect_slice(const BeamArgs& a, long long base, int v0, int v1, float m, float* best_v,
                                         int* best_i, int* sh_i, int* sh_cnt) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, k = a.n_out;
  auto count = [&](auto&& in) {  // elements for which in(value, index), over the CTA
    int mine = 0;
    for (int c = v0 + tid; c < v1; c += kRowThreads) {
      const float v = logit_at(a, base + c);
      mine += v > kNegInf && in(v, c);
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    __syncthreads();
    if (lane == 0) sh_i[warp] = mine;
    __syncthreads();
    int tot = 0;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) tot += sh_i[w];
    return tot;
  };
  uint32_t kth = order_code(m);  // largest code that at least k elements reach
  if (count([&](float v, int) { return order_code(v) >= kth; }) < k) {
    kth = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = kth | (1u << bit);
      if (count([&](float v, int) { return order_code(v) >= t; }) >= k) kth = t;
    }
  }
  const int above = count([&](float v, int) { return order_code(v) > kth; });
  int lo = v0, hi = v1 - 1;  // the smallest index up to which k - above equal ones lie
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (count([&](float v, int c) { return order_code(v) == kth && c <= mid; }) >= k - above)
      hi = mid;
    else
      lo = mid + 1;
  }
  __syncthreads();
  if (tid == 0) *sh_cnt = 0;
  __syncthreads();
  for (int c = v0 + tid; c < v1; c += kRowThreads) {
    const float v = logit_at(a, base + c);
    const uint32_t code = order_code(v);
    if (v > kNegInf && (code > kth || (code == kth && c <= lo))) {
      const int at = atomicAdd(sh_cnt, 1);  // k of them
      if (at < kListMax) best_v[at] = v, best_i[at] = c;
    }
  }
  __syncthreads();
  return min(*sh_cnt, kListMax);
}

// A CTA's slice is eight warps' shares of whole tiles; a tile is 32 lanes x Q
// pieces of eight neighbours (64 bytes a lane, in registers, each piece refilled
// for the next tile as soon as it is used).  The warps run freely: each
// publishes the maxima of its groups of 2^p lanes (at least n_out groups over
// the CTA) and takes the smallest published one as its bound; an old value only
// makes the bound weaker.  A lane's exponentials are summed relative to `ref`,
// its first maximum, which moves only when a logit exceeds it by more than
// kRefSlack.
//
// What is rare, a tile with a NaN, +inf or values above kScaleMax, goes through one rolled loop that
// reads the logits again and masks them (`careful`).  So the loop that runs hot
// stays small: inlined per piece, these cases doubled the time by instruction
// fetches alone.  Vocabularies of fewer
// than eight tiles (small) go through it whole, thread t taking t, t + 256, ...
//
// VEC: rows at 16-byte boundaries.  Else a piece comes by aligned 32-bit words,
// each of which holds at least one byte of the row, shifted together.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kRowThreads, 4) k_beam_rows(const __grid_constant__ BeamArgs a) {
  constexpr int Q = F32 ? 2 : 4, N = 8 * Q, kTile = 32 * N;
  constexpr int kWords = F32 ? 8 : 4;  // of a piece
  constexpr float kRefSlack = 20.f;
  __shared__ float sh_f[kRowWarps];
  __shared__ float sh_s[kRowWarps];
  __shared__ uint32_t sh_grp[kBeamMaxOut];  // order codes
  __shared__ uint32_t sh_max[kRowThreads];
  __shared__ int sh_cnt;
  __shared__ int sh_i[kRowWarps];
  __shared__ float list_v[kListMax];
  __shared__ int list_i[kListMax];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / a.splits, sl = blockIdx.x - row * a.splits, k = a.n_out;
  grid_dep_wait();
  grid_dep_release();
  const float score = a.scores[row];
  const unsigned char fin = a.fin ? a.fin[row] : 0;
  float2* cand = a.cand + ((size_t)row * a.splits + sl) * k;
  const bool small = a.vocab < kRowWarps * kTile;
  // tiles [t0, t1) of the slice, [w0, w1) of this warp
  const int tiles = (a.vocab + kTile - 1) / kTile, each = tiles / a.splits, rest = tiles - each * a.splits;
  auto cut = [&](int i) { return i * each + min(i, rest); };
  const int t0 = cut(sl), t1 = cut(sl + 1);
  const int w0 = small ? 0 : t0 + (t1 - t0) * warp / kRowWarps, w1 = small ? 1 : t0 + (t1 - t0) * (warp + 1) / kRowWarps;
  const long long base = (long long)row * a.ld;
  const char* rowp = reinterpret_cast<const char*>(a.logits) + base * (F32 ? 4 : 2);
  const bool shift = !VEC && !F32 && (reinterpret_cast<uintptr_t>(rowp) & 2);
  if (tid == 0) sh_cnt = 0;
  int p = 5;
  while ((kRowThreads >> p) < k) --p;
  const int ng = kRowThreads >> p;

  uint32_t u[Q][kWords];
  auto fetch = [&](int t, int q) {
    const int i0 = t * kTile + (q * 32 + lane) * 8;
    const char* src = rowp + (size_t)i0 * (F32 ? 4 : 2);
    if (i0 + 8 > a.vocab) {  // past the row's end: -inf
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[q][i] = F32 ? 0xFF800000u : 0xFF80FF80u;
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (i0 + e < a.vocab) {
          if (F32)
            u[q][e] = __ldg(reinterpret_cast<const uint32_t*>(src) + e);
          else
            u[q][e >> 1] = __byte_perm(u[q][e >> 1], __ldg(reinterpret_cast<const unsigned short*>(src) + e),
                                       e & 1 ? 0x5410 : 0x3254);
        }
    } else if (VEC) {
#pragma unroll
      for (int h = 0; h < kWords / 4; ++h) {
        const uint4 v = ld_once(reinterpret_cast<const uint4*>(src) + h);
        u[q][4 * h] = v.x, u[q][4 * h + 1] = v.y, u[q][4 * h + 2] = v.z, u[q][4 * h + 3] = v.w;
      }
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(src - (shift ? 2 : 0));
#pragma unroll
      for (int i = 0; i < kWords; ++i) u[q][i] = __ldg(w + i);
      if (shift) {
        const uint32_t last = __ldg(w + kWords);
#pragma unroll
        for (int i = 0; i < kWords; ++i) u[q][i] = __funnelshift_r(u[q][i], i + 1 < kWords ? u[q][i + 1] : last, 16);
      }
    }
  };
  auto value = [](const uint32_t (&w)[kWords], int e) {
    return __uint_as_float(F32 ? w[e] : e & 1 ? w[e >> 1] & 0xFFFF0000u : w[e >> 1] << 16);
  };
  // the largest logit of the lane's tile in u; NaN are passed over
  auto tile_max = [&]() {
    if (F32) {
      float v = kNegInf;
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) v = fmaxf(v, value(u[q], e));
      return v;
    }
    __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&u[0][0]);
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
      for (int i = 0; i < kWords; ++i) v = __hmax2(v, *reinterpret_cast<const __nv_bfloat162*>(&u[q][i]));
    return fmaxf(__low2float(v), __high2float(v));
  };
  // index of this lane's element j of tile t
  auto index = [&](int t, int j) {
    return small ? tid + j * kRowThreads : t * kTile + ((j >> 3) * 32 + lane) * 8 + (j & 7);
  };
  auto masked_max = [&](int t) {
    float v = kNegInf;
#pragma unroll 16
    for (int j = 0; j < N; ++j) {
      const int i = index(t, j);
      if (i < a.vocab) v = fmaxf(v, logit_at(a, base + i));
    }
    return v;
  };
  float m = kNegInf;                     // this lane's max
  float ref = kNegInf, c = 0.f, s = 0.f;  // its reference, log2_ref(ref), and sum
  float bound = kNegInf;                 // at least k elements of the slice reach it
  float shown = kNegInf;                 // the maximum published for this lane's group
  auto publish = [&]() {
    shown = m;
    for (int o = 1; o < (1 << p); o <<= 1) shown = fmaxf(shown, __shfl_xor_sync(0xffffffffu, shown, o));
    if ((lane & ((1 << p) - 1)) == 0) *const_cast<volatile uint32_t*>(&sh_grp[tid >> p]) = order_code(shown);
  };
  auto read_bound = [&]() {
    const volatile uint32_t* grp = sh_grp;
    uint32_t g = grp[lane & (ng - 1)];
    for (int i = 32; i < ng; i += 32) g = min(g, grp[i + lane]);
    bound = fmaxf(bound, from_code(__reduce_min_sync(0xffffffffu, g)));
  };
  auto move_ref = [&](float to) {
    s = s > 0.f ? s * rescale(ref, to) : 0.f;
    ref = to;
    c = log2_ref(to);
  };
  auto take = [&](float v, int i) {
    const int at = atomicAdd(&sh_cnt, 1);
    if (at < kListMax) list_v[at] = v, list_i[at] = i;
  };
  auto careful = [&](int t, bool taken) {  // maximum, sum and (not taken yet) candidates of a tile, masked
    const float tm = masked_max(t);
    m = fmaxf(m, tm);
    if (tm > ref) move_ref(tm);
#pragma unroll 16
    for (int j = 0; j < N; ++j) {
      const int i = index(t, j);
      const float v = i < a.vocab ? logit_at(a, base + i) : kNegInf;
      if (v > kNegInf) {
        s += exp2_fast(fabsf(ref) <= kScaleMax ? fmaf(v, kLog2e, -c) : (v - ref) * kLog2e);
        if (v >= bound && !taken) take(v, i);
      }
    }
  };
  if (!small && w0 < w1)
#pragma unroll
    for (int q = 0; q < Q; ++q) fetch(w0, q);
  if (!(fabsf(score) <= FLT_MAX) || fin) return;  // the merge reads nothing of such a row
  if (small) {
    m = masked_max(0);
  } else if (w0 < w1) {
    m = tile_max();
    if (!(m <= FLT_MAX)) m = masked_max(w0);
  }
  if (m > kNegInf) move_ref(m);
  publish();
  sh_max[tid] = order_code(m);
  __syncthreads();
  if (warp == 0) kth_of_256(sh_max, k, lane);
  __syncthreads();
  bound = sh_max[0] <= order_code(kNegInf) ? kNegInf : from_code(sh_max[0]);
  read_bound();
  for (int t = w0; t < w1; ++t) {
    if (!small) {
      const bool more = t + 1 < w1;
      const float tm = tile_max();
      if (tm > ref + kRefSlack && tm <= FLT_MAX) move_ref(tm);
      // a branch of the whole warp: were it each lane's own, the compiler would
      // give both sides a copy of the sums, one after the other (measured: 1.7
      // times the exponentials)
      const bool hit = tm >= bound && tm > kNegInf && tm <= FLT_MAX;
      unsigned hits = __ballot_sync(0xffffffffu, hit);
      if (__popc(hits) <= kFewHits) {
        // lane by lane, the warp looks at the lane's elements, one a thread: 0.1 us
        // where walking through them took 1.5 (32 x 8 x 248320: 46.5 -> 44.4 us)
        while (hits) {
          const int from = __ffs(hits) - 1;
          hits &= hits - 1;
          uint32_t w = 0;
#pragma unroll
          for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
              const uint32_t x = __shfl_sync(0xffffffffu, u[q][i], from);
              if (q * kWords + i == (F32 ? lane : lane >> 1)) w = x;
            }
          const float v = __uint_as_float(F32 || (lane & 1) ? (F32 ? w : w & 0xFFFF0000u) : w << 16);
          const bool in = lane < N && v >= bound && v > kNegInf;
          const unsigned all = __ballot_sync(0xffffffffu, in);
          int at = 0;
          if (lane == 0 && all) at = atomicAdd(&sh_cnt, __popc(all));
          at = __shfl_sync(0xffffffffu, at, 0) + __popc(all & ((1u << lane) - 1));
          if (in && at < kListMax) list_v[at] = v, list_i[at] = t * kTile + ((lane >> 3) * 32 + from) * 8 + (lane & 7);
        }
      } else {
#pragma unroll 1
        for (int q = 0; q < Q; ++q) {
          uint32_t w[kWords];  // u[q]
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            w[i] = u[0][i];
#pragma unroll
            for (int r = 1; r < Q; ++r) w[i] = q == r ? u[r][i] : w[i];
          }
          float wm = value(w, 0);
#pragma unroll
          for (int e = 1; e < 8; ++e) wm = fmaxf(wm, value(w, e));
          if (!__any_sync(0xffffffffu, hit && wm >= bound)) continue;
#pragma unroll 1
          for (int i = 0; i < kWords; ++i) {  // w[0] is the word at hand
#pragma unroll
            for (int h = 0; h < (F32 ? 1 : 2); ++h) {
              const float v = value(w, h);
              if (hit && v >= bound && v > kNegInf) take(v, t * kTile + (q * 32 + lane) * 8 + i * (F32 ? 1 : 2) + h);
            }
            __syncwarp();
#pragma unroll
            for (int r = 0; r + 1 < kWords; ++r) w[r] = w[r + 1];
          }
        }
      }
      float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int q = 0; q < Q; ++q) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float2 x = fma2(make_float2(value(u[q], e), value(u[q], e + 1)), kLog2e, -c);
          sum[e >> 1 & 1] = add2(sum[e >> 1 & 1], make_float2(exp2_fast(x.x), exp2_fast(x.y)));
        }
        if (more) fetch(t + 1, q);
      }
      const float ts = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      if (tm <= FLT_MAX) m = fmaxf(m, tm);
      // (a lane that has met masked logits only has no reference yet, and nothing to add)
      if (ts <= FLT_MAX && (fabsf(ref) <= kScaleMax || tm == kNegInf))
        s += ts;
      else  // a NaN, +inf (no candidates taken yet), or products that leave fp32
        careful(t, tm <= FLT_MAX);
    } else {
      careful(t, false);
    }
    __syncwarp();
    if (__any_sync(0xffffffffu, m > shown)) publish();
    read_bound();
  }
  // the slice's max and sum
  float M = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (lane == 0) sh_f[warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowWarps; ++w) M = fmaxf(M, sh_f[w]);
  s = s > 0.f ? s * rescale(ref, M) : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh_s[warp] = s;
  int n = sh_cnt;
  if (n > kListMax) {
    n = bisect_slice(a, base, t0 * kTile, min(a.vocab, t1 * kTile), M, list_v, list_i, sh_i, &sh_cnt);
  } else if (n > kListCut) {  // the last bound leaves few of a long list
    read_bound();
    constexpr int kMine = kListMax / kRowThreads;
    float v[kMine];
    int id[kMine];
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      const int i = tid + j * kRowThreads;
      v[j] = i < n ? list_v[i] : kNegInf;
      id[j] = i < n ? list_i[i] : 0;
    }
    __syncthreads();
    if (tid == 0) sh_cnt = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMine; ++j)
      if (v[j] >= bound && v[j] > kNegInf) {
        const int i = atomicAdd(&sh_cnt, 1);
        list_v[i] = v[j], list_i[i] = id[j];
      }
    __syncthreads();
    n = sh_cnt;
  } else {
    __syncthreads();
  }
  if (tid == 0) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) t += sh_s[w];
    a.stat[(size_t)row * a.splits + sl] = make_float2(M, t);
  }
  for (int i = tid; i < n; i += kRowThreads) {
    const float v = list_v[i];
    const int id = list_i[i];
    int rank = 0;
    for (int q = 0; q < n; ++q) rank += before(list_v[q], list_i[q], v, id);
    if (rank < k) cand[rank] = make_float2(v, __int_as_float(id));
  }
  for (int i = n + tid; i < k; i += kRowThreads) cand[i] = make_float2(kNegInf, __int_as_float(-1));
}

constexpr int kMergeThreads = 256;
constexpr int kMergeWarps = kMergeThreads / 32;
constexpr int kMergeFew = 64;                               // entries ranked sooner than bounded
constexpr int kMergeMine = 8;                               // entries a thread holds at a time
constexpr int kMergeChunk = kMergeMine * kMergeThreads;     // of the sequence
constexpr int kMergeKept = 2 * kBeamMaxOut;                 // most entries a cut leaves
constexpr int kMergeList = kMergeChunk + kMergeKept;        // a chunk on top of them

__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const __grid_constant__ BeamArgs a) {
  __shared__ double base[kBeamMaxBeams];  // score - log-sum of each live beam
  __shared__ int kind[kBeamMaxBeams];     // 0 no candidate, 1 live, 2 finished
  __shared__ double list_v[kMergeList];
  __shared__ long long list_i[kMergeList];  // beam, token
  __shared__ uint32_t sh_max[kMergeThreads];
  __shared__ int sh_n[2][kMergeWarps];
  __shared__ int cnt;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x, W = a.beams, S = a.splits, k = a.n_out;
  const int per = S * k, all = W * per;  // entries of a beam, of the sequence
  const float2* cand = a.cand + (size_t)b * all;
  // Twice: first on one made-up candidate, nothing read or written, while the
  // kernel before still runs, which brings in the instructions (0.2 to 0.5 us).
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const bool real = pass == 1;
    if (real) {
      grid_dep_wait();
      grid_dep_release();
    }
    if (tid == 0) cnt = 0;
    // neighbouring entries (one beam's) go to different warps; a chunk's loads are
    // all in flight at once, the first chunk's before anything else (what a beam
    // without candidates left in the workspace is read, not used)
    auto place = [&](int i) { return i * kMergeThreads + lane * kMergeWarps + warp; };
    float2 mine[kMergeMine];
    auto fetch = [&](int from) {
#pragma unroll
      for (int i = 0; i < kMergeMine; ++i) {
        if (!real) mine[i] = make_float2(tid + i ? kNegInf : 0.f, 0.f);
        if (real && from + place(i) < all) mine[i] = cand[from + place(i)];
      }
    };
    fetch(0);
    const int slices = real ? S : 0;
    const int beams = real ? W : min(W, kMergeWarps);
    for (int w = warp; w < beams; w += kMergeWarps) {  // a warp per beam: its slices in lane order
      const int row = b * W + w;
      const float2* st = a.stat + (size_t)row * S;
      float2 first = lane < slices ? st[lane] : make_float2(kNegInf, 0.f);
      if (!real && lane == 0) first = make_float2(0.f, 1.f);
      const float sc = real ? a.scores[row] : 0.f;
      int kd = fabsf(sc) <= FLT_MAX ? (real && a.fin && a.fin[row] ? 2 : 1) : 0;
      double lse = 0;
      if (kd == 1) {
        float M = first.x;
        for (int s = lane + 32; s < slices; s += 32) M = fmaxf(M, st[s].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        if (M > kNegInf) {
          // a slice's sum from its own max to the row's
          auto term = [&](const float2& v) { return v.x > kNegInf ? (double)(v.y * rescale(v.x, M)) : 0.; };
          double t = term(first);
          for (int s = lane + 32; s < slices; s += 32) t += term(st[s]);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
          lse = log_sum(M, t);
        } else {
          kd = 0;  // every token masked
        }
      }
      if (lane == 0) {
        kind[w] = kd;
        base[w] = (double)sc - lse;
      }
    }
    __syncthreads();
    // cuts the list to what reaches the upper 16 bits of its k-th value's code, or,
    // if ties leave too many, to its k best
    auto cut = [&](int n) {
      constexpr int kMine = (kMergeList + kMergeThreads - 1) / kMergeThreads;
      double v[kMine];
      long long id[kMine];
      uint32_t c[kMine], kth = 0;
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int i = tid + j * kMergeThreads;
        v[j] = i < n ? list_v[i] : -INFINITY;
        id[j] = i < n ? list_i[i] : 0;
        c[j] = i < n ? order_code(__double2float_rd(v[j])) : 0;
      }
#pragma unroll 1
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t t = kth | (1u << bit);
        int m = 0;
#pragma unroll
        for (int j = 0; j < kMine; ++j) m += c[j] >= t;
        m = __reduce_add_sync(0xffffffffu, m);
        if (lane == 0) sh_n[bit & 1][warp] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int w = 0; w < kMergeWarps; ++w) m += sh_n[bit & 1][w];
        if (m >= k) kth = t;
      }
      if (tid == 0) cnt = 0;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMine; ++j)
        if (c[j] >= kth && c[j] > 0) {
          const int at = atomicAdd(&cnt, 1);
          list_v[at] = v[j], list_i[at] = id[j];
        }
      __syncthreads();
      n = cnt;
      if (n <= kMergeKept) return;
      int rank[kMine];
#pragma unroll
      for (int j = 0; j < kMine; ++j) {
        const int i = tid + j * kMergeThreads;
        rank[j] = k;
        if (i < n) {
          v[j] = list_v[i], id[j] = list_i[i], rank[j] = 0;
          for (int q = 0; q < n; ++q) rank[j] += list_v[q] > v[j] || (list_v[q] == v[j] && list_i[q] < id[j]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kMine; ++j)
        if (rank[j] < k) list_v[rank[j]] = v[j], list_i[rank[j]] = id[j];
      if (tid == 0) cnt = k;
      __syncthreads();
    };
    double bound = -INFINITY;
    for (int from = 0; from < (real ? all : 1); from += kMergeChunk) {
      double val[kMergeMine], m = -INFINITY;
      long long pos[kMergeMine];
#pragma unroll
      for (int i = 0; i < kMergeMine; ++i) {
        val[i] = -INFINITY, pos[i] = 0;
        const int e = from + place(i);
        if (from + i * kMergeThreads < all && e < all) {  // the first for the whole CTA
          const int w = e / per;
          if (kind[w] == 1) {
            if (mine[i].x > kNegInf)
              val[i] = base[w] + (double)mine[i].x, pos[i] = (long long)w << 32 | __float_as_int(mine[i].y);
          } else if (kind[w] == 2 && e == w * per) {
            val[i] = base[w], pos[i] = (long long)w << 32 | a.eos;
          }
        }
        m = fmax(m, val[i]);
      }
      if (real && from + kMergeChunk < all) fetch(from + kMergeChunk);
      if (all > kMergeFew) {  // the k-th largest of the threads' maxima: at least k entries reach it
        sh_max[tid] = order_code(__double2float_rd(m));
        __syncthreads();
        if (warp == 0) kth_of_256(sh_max, k, lane);
        __syncthreads();
        if (sh_max[0] > order_code(kNegInf)) bound = fmax(bound, (double)from_code(sh_max[0]));
      }
#pragma unroll
      for (int i = 0; i < kMergeMine; ++i)
        if (val[i] >= bound && val[i] > -INFINITY) {
          const int at = atomicAdd(&cnt, 1);
          list_v[at] = val[i], list_i[at] = pos[i];
        }
      __syncthreads();
      const int n = cnt;
      __syncthreads();
      if (n > 2 * kMergeFew && n > k) cut(n);  // so no more than kMergeKept stay
    }
    const int n = cnt;
    for (int i = tid >> 3; i < (n + 3 & ~3); i += kMergeThreads / 8) {  // eight threads an entry
      const double v = i < n ? list_v[i] : -INFINITY;
      const long long id = i < n ? list_i[i] : 0;
      int rank = 0;
      for (int q = tid & 7; q < n; q += 8) rank += list_v[q] > v || (list_v[q] == v && list_i[q] < id);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (i < n && rank < k && real && (tid & 7) == 0) {
        const int w = (int)(id >> 32), t = (int)id, at = b * k + rank;
        a.parent[at] = w;
        a.token[at] = t;
        a.out[at] = (float)v;
        if (a.fin_out) a.fin_out[at] = kind[w] == 2 || t == a.eos;
      }
    }
    for (int i = real ? n + tid : k; i < k; i += kMergeThreads) {  // fewer candidates than asked for
      const int at = b * k + i;
      a.parent[at] = -1;
      a.token[at] = -1;
      a.out[at] = kNegInf;
      if (a.fin_out) a.fin_out[at] = 0;
    }
    __syncthreads();
  }
}

}  // namespace

// Slices of the vocabulary per row, of at least eight tiles (one a warp): the
// number that makes rounds of resident CTAs x (tiles a warp walks + what a CTA
// costs besides, about five tiles) the smallest.
static unsigned beam_tiles(int vocab, int f32) { return ((unsigned)vocab + (f32 ? 511 : 1023)) / (f32 ? 512 : 1024); }
int beam_splits(int batch, int beams, int vocab, int f32) {
  const unsigned rows = (unsigned)(batch * beams), tiles = beam_tiles(vocab, f32);
  constexpr unsigned resident = 148 * 4;
  const unsigned most = std::min(std::max(1u, tiles / kRowWarps), 2 * resident);
  unsigned best = 1;
  unsigned long long cost = ~0ull;
  for (unsigned s = 1; s <= most; ++s) {
    // no s from here on costs less than rows * s / resident x (tiles / (8 s) + 5)
    if (rows * (tiles + 5ull * kRowWarps * s) / (resident * kRowWarps) >= cost) break;
    const unsigned per = (tiles + s * kRowWarps - 1) / (s * kRowWarps);
    const unsigned long long c = ((unsigned long long)rows * s + resident - 1) / resident * (per + 5);
    if (c < cost) best = s, cost = c;
  }
  return (int)best;
}

// The most lists (rows x slices) of any batch up to the given one: more rows may
// take fewer slices in all.  From 148 (tiles / 8 + 5) rows on one slice a row is
// the cheapest (a second costs rows / 592 x 4 more, the round it may save tiles /
// 8 + 5), and the lists grow with the rows.
long long beam_lists(int batch, int beams, int vocab, int f32) {
  const long long one = 148ll * ((beam_tiles(vocab, f32) + kRowWarps - 1) / kRowWarps + 5);
  long long most = (long long)batch * beams * beam_splits(batch, beams, vocab, f32);
  for (int b = 1; b < batch && (long long)b * beams <= one; ++b)
    most = std::max(most, (long long)b * beams * beam_splits(b, beams, vocab, f32));
  return most;
}

cudaError_t launch_beam_select(const BeamArgs& a, cudaStream_t st) {
  const long long ctas = (long long)a.batch * a.beams * a.splits;
  if (ctas > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)ctas), block(kRowThreads);
  const cudaError_t e = a.f32 ? (a.vec ? launch_pdl(k_beam_rows<true, true>, grid, block, 0, st, a)
                                       : launch_pdl(k_beam_rows<true, false>, grid, block, 0, st, a))
                              : (a.vec ? launch_pdl(k_beam_rows<false, true>, grid, block, 0, st, a)
                                       : launch_pdl(k_beam_rows<false, false>, grid, block, 0, st, a));
  if (e != cudaSuccess) return e;
  return launch_pdl(k_beam_merge, dim3((unsigned)a.batch), dim3(kMergeThreads), 0, st, a);
}

namespace {

constexpr int kCopyThreads = 256;

// One column of V (1 to 16 bytes) of a sequence's rows per thread and step.
template <typename V, int K>
__device__ __forceinline__ void move_column(const char* src, char* dst, long long ss, long long ds, const int (&par)[K],
                                            int n_out) {
  V v[K];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (k < n_out && par[k] >= 0) v[k] = *reinterpret_cast<const V*>(src + par[k] * ss);
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (k < n_out && par[k] >= 0) *reinterpret_cast<V*>(dst + k * ds) = v[k];
}

template <int K>
__global__ void __launch_bounds__(kCopyThreads) k_reorder(const __grid_constant__ ReorderArgs a) {
  __shared__ int sh_par[kReorderMaxOut];
  const long long blk = blockIdx.x;
  int i = 0;
  while (i + 1 < a.n && blk >= a.first[i + 1]) ++i;
  const ReorderTensor& t = a.t[i];
  const long long in = blk - a.first[i];
  const long long per = (a.first[i + 1] - a.first[i]) / a.batch;  // blocks per sequence
  const int b = (int)(in / per);
  grid_dep_wait();
  grid_dep_release();
  if (threadIdx.x < a.n_out) {
    const int p = a.parent[b * a.n_out + threadIdx.x];
    // an in-place row that stays where it is needs no copy
    sh_par[threadIdx.x] = p < 0 || p >= a.beams || (t.src == t.dst && p == (int)threadIdx.x) ? -1 : p;
  }
  __syncthreads();
  int par[K];
#pragma unroll
  for (int k = 0; k < K; ++k) par[k] = k < a.n_out ? sh_par[k] : -1;
  const long long cols = t.seg_bytes / t.width;  // per segment; the ragged end goes byte by byte
  const long long tail = t.seg_bytes - cols * t.width;
  const long long c = (in % per) * kCopyThreads + threadIdx.x;
  const long long per_seg = cols + tail;
  if (c >= per_seg * t.n_seg) return;
  const long long seg = c / per_seg, j = c % per_seg;
  const bool whole = j < cols;
  const long long off = seg * t.seg_stride + (whole ? j * t.width : cols * t.width + (j - cols));
  const char* src = t.src + (long long)b * a.beams * t.src_stride + off;
  char* dst = t.dst + (long long)b * a.n_out * t.dst_stride + off;
  switch (whole ? t.width : 1) {
    case 16:
      if constexpr (K <= 32) move_column<uint4, K>(src, dst, t.src_stride, t.dst_stride, par, a.n_out);
      break;  // more rows would not fit the registers: the host asks for 8 bytes at most
    case 8: move_column<uint2, K>(src, dst, t.src_stride, t.dst_stride, par, a.n_out); break;
    case 4: move_column<uint32_t, K>(src, dst, t.src_stride, t.dst_stride, par, a.n_out); break;
    case 2: move_column<uint16_t, K>(src, dst, t.src_stride, t.dst_stride, par, a.n_out); break;
    default: move_column<uint8_t, K>(src, dst, t.src_stride, t.dst_stride, par, a.n_out);
  }
}

}  // namespace

cudaError_t launch_reorder(ReorderArgs& a, cudaStream_t st) {
  long long total = 0;
  for (int i = 0; i < a.n; ++i) {
    ReorderTensor& t = a.t[i];
    if (a.n_out > 32) t.width = std::min(t.width, 8);
    a.first[i] = total;
    const long long per_seg = t.seg_bytes / t.width + t.seg_bytes % t.width;
    total += (per_seg * t.n_seg + kCopyThreads - 1) / kCopyThreads * a.batch;
  }
  a.first[a.n] = total;
  if (total == 0) return cudaSuccess;
  if (total > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)total), block(kCopyThreads);
  if (a.n_out <= 4) return launch_pdl(k_reorder<4>, grid, block, 0, st, a);
  if (a.n_out <= 8) return launch_pdl(k_reorder<8>, grid, block, 0, st, a);
  if (a.n_out <= 16) return launch_pdl(k_reorder<16>, grid, block, 0, st, a);
  if (a.n_out <= 32) return launch_pdl(k_reorder<32>, grid, block, 0, st, a);
  return launch_pdl(k_reorder<64>, grid, block, 0, st, a);
}

}  // namespace llmoc
