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
//   k_beam_rows   one CTA per (row, vocabulary slice): the slice is read once
//                 into registers; the slice's max and sum of exponentials, and
//                 its n_out best logits.  A lower bound of the n_out-th best
//                 comes from the maxima of at least n_out disjoint thread
//                 groups (each holds an element at least as large as the
//                 smallest of those maxima); what reaches the bound goes to a
//                 shared list and is ranked by counting.  A slice with more
//                 such elements than the list holds (adversarial values, many
//                 ties) finds its exact n_out-th best by bisection on the
//                 (value, index) keys, which are distinct.
//   k_beam_merge  one CTA per sequence: each beam's log-sum from its slices,
//                 in fp64 (candidates of different beams are compared by it),
//                 and the best of the slices' sorted lists.
//
// Order of summation is fixed by the slice and thread numbers alone, so equal
// rows get equal bits and ties resolve by index.
//
// Reordering.  dst[b, k] = src[b, parent[b, k]] for any number of tensors in
// one launch; a thread owns a column of a sequence's rows, loads it from every
// parent before it stores any, so a tensor may be reordered in place.
#include <algorithm>
#include <cfloat>
#include <string>

#include "ops.cuh"

namespace llmoc {

namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kListMax = 512;
constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ float masked(float x) { return fabsf(x) <= FLT_MAX ? x : kNegInf; }
// order-preserving bits of a float (larger value, larger code)
__device__ __forceinline__ uint32_t order_code(float x) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long order_code64(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x == 0. ? 0. : x);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double from_code64(unsigned long long c) {
  return __longlong_as_double((long long)(c >> 63 ? c & ~(1ull << 63) : ~c));
}
// a before b in the order "larger value, then smaller index"
__device__ __forceinline__ bool before(float va, int ia, float vb, int ib) { return va > vb || (va == vb && ia < ib); }

template <int E, bool F32>
__global__ void __launch_bounds__(kRowThreads) k_beam_rows(const BeamArgs a) {
  __shared__ float sh_f[kRowWarps];
  __shared__ float sh_s[kRowWarps];
  __shared__ float sh_grp[kBeamMaxOut];
  __shared__ int sh_cnt;
  __shared__ int sh_i[kRowWarps];
  __shared__ float list_v[kListMax];
  __shared__ int list_i[kListMax];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / a.splits, sl = blockIdx.x % a.splits, k = a.n_out;
  grid_dep_wait();
  grid_dep_release();
  float2* cand = a.cand + ((size_t)row * a.splits + sl) * k;
  if (!(fabsf(a.scores[row]) <= FLT_MAX) || (a.fin && a.fin[row])) return;  // the merge reads nothing of such a row
  const int v0 = sl * a.slice, v1 = min(a.vocab, v0 + a.slice);
  // token of value j of this thread
  auto tok = [&](int j) { return a.vec ? v0 + ((j >> 3) * kRowThreads + tid) * 8 + (j & 7) : v0 + j * kRowThreads + tid; };
  float x[E];
  const long long base = (long long)row * a.ld;
  if (a.vec) {
#pragma unroll
    for (int q = 0; q < E / 8; ++q) {
      const int c = v0 + (q * kRowThreads + tid) * 8;
      if (c + 8 <= v1) {
        if (F32) {
          const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.logits) + base + c);
          const float4 u = __ldg(p), w = __ldg(p + 1);
          x[q * 8] = u.x, x[q * 8 + 1] = u.y, x[q * 8 + 2] = u.z, x[q * 8 + 3] = u.w;
          x[q * 8 + 4] = w.x, x[q * 8 + 5] = w.y, x[q * 8 + 6] = w.z, x[q * 8 + 7] = w.w;
        } else {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.logits) + base + c));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[q * 8 + 2 * e] = __uint_as_float(w[e] << 16);
            x[q * 8 + 2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[q * 8 + e] = c + e >= v1 ? kNegInf
                         : F32 ? reinterpret_cast<const float*>(a.logits)[base + c + e]
                               : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.logits)[base + c + e]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = v0 + j * kRowThreads + tid;
      x[j] = c >= v1 ? kNegInf
             : F32   ? __ldg(reinterpret_cast<const float*>(a.logits) + base + c)
                     : bf16_bits_to_f32(__ldg(reinterpret_cast<const unsigned short*>(a.logits) + base + c));
    }
  }
  float m = kNegInf;
#pragma unroll
  for (int j = 0; j < E; ++j) {
    x[j] = masked(x[j]);
    m = fmaxf(m, x[j]);
  }
  // maxima of groups of 2^p lanes, at least k groups over the CTA
  int p = 5;
  while ((kRowThreads >> p) < k) --p;
  float gm = m, wm;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float other = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = other;
    if (o < (1 << p)) gm = m;
  }
  wm = m;
  const int ng = kRowThreads >> p;
  if ((lane & ((1 << p) - 1)) == 0 && (tid >> p) < ng) sh_grp[tid >> p] = gm;
  if (lane == 0) sh_f[warp] = wm;
  if (tid == 0) sh_cnt = 0;
  __syncthreads();
  float M = sh_f[0], bound = sh_grp[0];
#pragma unroll
  for (int w = 1; w < kRowWarps; ++w) M = fmaxf(M, sh_f[w]);
  for (int i = 1; i < ng; ++i) bound = fminf(bound, sh_grp[i]);
  // sum of exponentials below the slice's max
  float s = 0.f;
  if (M > kNegInf) {
#pragma unroll
    for (int j = 0; j < E; ++j) s += __expf(x[j] - M);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh_s[warp] = s;
  // what reaches the bound
#pragma unroll
  for (int j = 0; j < E; ++j)
    if (x[j] >= bound && x[j] > kNegInf) {
      const int at = atomicAdd(&sh_cnt, 1);
      if (at < kListMax) list_v[at] = x[j], list_i[at] = tok(j);
    }
  __syncthreads();
  if (tid == 0) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < kRowWarps; ++w) t += sh_s[w];
    a.stat[(size_t)row * a.splits + sl] = make_float2(M, t);
  }
  int n = sh_cnt;
  if (n > kListMax) {
    // the k-th best key by bisection: 32 value bits, then the index (smaller first)
    uint64_t lo = 0;  // largest key with at least k elements >= it
    for (int bit = 62; bit >= 0; --bit) {
      const uint64_t c = lo | (1ull << bit);
      int mine = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const uint64_t key = ((uint64_t)order_code(x[j]) << 31) | (uint32_t)(0x7FFFFFFF - tok(j));
        mine += x[j] > kNegInf && key >= c;
      }
      mine = __reduce_add_sync(0xffffffffu, mine);
      __syncthreads();
      if (lane == 0) sh_i[warp] = mine;
      __syncthreads();
      int tot = 0;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) tot += sh_i[w];
      if (tot >= k) lo = c;
    }
    __syncthreads();
    if (tid == 0) sh_cnt = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const uint64_t key = ((uint64_t)order_code(x[j]) << 31) | (uint32_t)(0x7FFFFFFF - tok(j));
      if (x[j] > kNegInf && key >= lo) {
        const int at = atomicAdd(&sh_cnt, 1);  // k of them
        if (at < kListMax) list_v[at] = x[j], list_i[at] = tok(j);
      }
    }
    __syncthreads();
    n = min(sh_cnt, kListMax);
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
constexpr int kMergeList = 1024;

__global__ void __launch_bounds__(kMergeThreads) k_beam_merge(const BeamArgs a) {
  __shared__ double base[kBeamMaxBeams];  // score - log-sum of each live beam
  __shared__ int kind[kBeamMaxBeams];     // 0 no candidate, 1 live, 2 finished
  __shared__ double list_v[kMergeList];
  __shared__ long long list_i[kMergeList];  // beam * vocab + token
  __shared__ unsigned long long grp[kBeamMaxOut];  // order codes
  __shared__ double red_v[kMergeWarps];
  __shared__ long long red_i[kMergeWarps];
  __shared__ int cnt;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.x, W = a.beams, S = a.splits, k = a.n_out;
  grid_dep_wait();
  grid_dep_release();
  if (tid == 0) cnt = 0;
  if (tid < kBeamMaxOut) grp[tid] = 0;
  for (int w = warp; w < W; w += kMergeWarps) {  // a warp per beam: its slices in lane order
    const int row = b * W + w;
    const float sc = a.scores[row];
    int kd = fabsf(sc) <= FLT_MAX ? (a.fin && a.fin[row] ? 2 : 1) : 0;
    double lse = 0;
    if (kd == 1) {
      float M = kNegInf;
      for (int s = lane; s < S; s += 32) M = fmaxf(M, a.stat[(size_t)row * S + s].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
      if (M > kNegInf) {
        double t = 0;
        for (int s = lane; s < S; s += 32) {
          const float2 st = a.stat[(size_t)row * S + s];
          if (st.x > kNegInf) t += (double)st.y * exp((double)st.x - (double)M);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        lse = (double)M + log(t);
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
  const int lists = W * S;
  // head of list l (a slice of a beam), or of a finished beam
  auto entry = [&](int l, int j, double* v, long long* id) {
    const int w = l / S, s = l % S;
    *v = -INFINITY;
    *id = 0;
    if (kind[w] == 1) {
      const float2 c = a.cand[((size_t)(b * W + w) * S + s) * k + j];
      if (c.x > kNegInf) *v = base[w] + (double)c.x, *id = (long long)w * a.vocab + __float_as_int(c.y);
    } else if (kind[w] == 2 && s == 0 && j == 0) {
      *v = base[w], *id = (long long)w * a.vocab + a.eos;
    }
  };
  // bound: the smallest of the maxima of k groups of list heads, neighbouring
  // lists (slices of one beam) in different groups
  const int ng = min(k, lists);
  for (int l = tid; l < lists; l += kMergeThreads) {
    double v;
    long long id;
    entry(l, 0, &v, &id);
    atomicMax(&grp[l % ng], order_code64(v));
  }
  __syncthreads();
  unsigned long long lowest = grp[0];
  for (int i = 1; i < ng; ++i) lowest = min(lowest, grp[i]);
  const double bound = lists < k ? -INFINITY : from_code64(lowest);
  for (int l = tid; l < lists; l += kMergeThreads)
    for (int j = 0; j < k; ++j) {
      double v;
      long long id;
      entry(l, j, &v, &id);
      if (!(v >= bound) || v == -INFINITY) break;
      const int at = atomicAdd(&cnt, 1);
      if (at < kMergeList) list_v[at] = v, list_i[at] = id;
    }
  __syncthreads();
  int n = cnt;
  if (n > kMergeList) {
    // too many above the bound: take the best k one by one, each the best
    // after the last taken
    double pv = INFINITY;
    long long pi = -1;
    n = 0;
    for (int q = 0; q < k; ++q) {
      double bv = -INFINITY;
      long long bi = 0x7FFFFFFFFFFFFFFFll;
      for (int l = tid; l < lists; l += kMergeThreads)
        for (int j = 0; j < k; ++j) {
          double v;
          long long id;
          entry(l, j, &v, &id);
          if (v == -INFINITY) break;
          if (v < pv || (v == pv && id > pi)) {
            if (v > bv || (v == bv && id < bi)) bv = v, bi = id;
            break;  // the rest of the list comes after it
          }
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const long long oi = __shfl_xor_sync(0xffffffffu, bi, o);
        if (ov > bv || (ov == bv && oi < bi)) bv = ov, bi = oi;
      }
      __syncthreads();
      if (lane == 0) red_v[warp] = bv, red_i[warp] = bi;
      __syncthreads();
      for (int w = 0; w < kMergeWarps; ++w)
        if (red_v[w] > bv || (red_v[w] == bv && red_i[w] < bi)) bv = red_v[w], bi = red_i[w];
      if (bv == -INFINITY) break;  // uniform
      if (tid == 0) list_v[q] = bv, list_i[q] = bi;
      pv = bv, pi = bi;
      n = q + 1;
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += kMergeThreads) {
    const double v = list_v[i];
    const long long id = list_i[i];
    int rank = 0;
    for (int q = 0; q < n; ++q) rank += list_v[q] > v || (list_v[q] == v && list_i[q] < id);
    if (rank < k) {
      const int w = (int)(id / a.vocab), t = (int)(id % a.vocab), at = b * k + rank;
      a.parent[at] = w;
      a.token[at] = t;
      a.out[at] = (float)v;
      if (a.fin_out) a.fin_out[at] = kind[w] == 2 || t == a.eos;
    }
  }
  for (int i = n + tid; i < k; i += kMergeThreads) {  // fewer candidates than asked for
    const int at = b * k + i;
    a.parent[at] = -1;
    a.token[at] = -1;
    a.out[at] = kNegInf;
    if (a.fin_out) a.fin_out[at] = 0;
  }
}

}  // namespace

// Slices of the vocabulary per row: small ones while the grid leaves SMs
// idle, large ones (fewer lists to merge) otherwise.
void beam_split(int batch, int beams, int vocab, int* splits, int* slice) {
  const long long rows = (long long)batch * beams;
  int e = 32;
  while (e > 8 && rows * ((vocab + e * kRowThreads - 1) / (e * kRowThreads)) < 148 * 4) e /= 2;
  *slice = e * kRowThreads;
  *splits = (vocab + *slice - 1) / *slice;
}

cudaError_t launch_beam_select(const BeamArgs& a, cudaStream_t st) {
  const long long ctas = (long long)a.batch * a.beams * a.splits;
  if (ctas > 0x7FFFFFFFll) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)ctas), block(kRowThreads);
  cudaError_t e;
  switch (a.slice / kRowThreads) {
    case 8: e = a.f32 ? launch_pdl(k_beam_rows<8, true>, grid, block, 0, st, a)
                      : launch_pdl(k_beam_rows<8, false>, grid, block, 0, st, a); break;
    case 16: e = a.f32 ? launch_pdl(k_beam_rows<16, true>, grid, block, 0, st, a)
                       : launch_pdl(k_beam_rows<16, false>, grid, block, 0, st, a); break;
    default: e = a.f32 ? launch_pdl(k_beam_rows<32, true>, grid, block, 0, st, a)
                       : launch_pdl(k_beam_rows<32, false>, grid, block, 0, st, a);
  }
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
