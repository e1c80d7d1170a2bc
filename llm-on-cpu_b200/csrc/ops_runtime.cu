// ops_runtime.cu — host side of the operators around the MoE layer
// (include/llmoc_b200.h): argument checks, the resident weights of a dense
// INT4 product, and the calls that chain a MoE layer with the norms around it.
//
// Every check that needs no device comes before the first CUDA call, and a
// refused call launches nothing.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <string>

#include "../../include/llmoc_b200.h"
#include "kernels.cuh"
#include "ops.cuh"

using namespace llmoc;

namespace llmoc {
int layer_device(const llmoc_moe_layer* L);
int layer_hidden(const llmoc_moe_layer* L);
}  // namespace llmoc

struct llmoc_int4_linear {
  int device = 0;
  int M = 0, K = 0, nb = 0, mt = 0, zp = 7;
  int fl = 4;  // 32-wide blocks per packed scale group
  bool awq = true;
  char* arena = nullptr;
  int* err = nullptr;  // device error word, behind the stream
  size_t weight_bytes = 0;
};

namespace {

llmoc_status refuse(llmoc_status s, const std::string& msg) {
  set_last_error(msg);
  return s;
}

size_t up256(size_t v) { return (v + 255) & ~size_t(255); }

// The call's device for the scope of an entry point.
struct OnDevice {
  int prev = -1;
  bool ok = false;
  explicit OnDevice(int dev) {
    int cur = -1;
    if (cudaGetDevice(&cur) == cudaSuccess) {
      if (cur == dev) {
        ok = true;
      } else if (dev >= 0 && cudaSetDevice(dev) == cudaSuccess) {
        prev = cur;
        ok = true;
      }
    }
    if (!ok) cudaGetLastError();
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

llmoc_status no_device(const char* who, int dev) {
  return refuse(LLMOC_ERR_NO_DEVICE, std::string(who) + ": no such CUDA device: " + std::to_string(dev));
}
llmoc_status launched(cudaError_t e, const char* who, int n) {
  if (e == cudaSuccess) {
    note_launches(n);
    return LLMOC_OK;
  }
  cudaGetLastError();
  return refuse(LLMOC_ERR_CUDA, std::string(who) + ": " + cudaGetErrorString(e));
}

bool dtype_ok(int d) { return d == LLMOC_DTYPE_F32 || d == LLMOC_DTYPE_BF16; }
size_t dtype_bytes(int d) { return d == LLMOC_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// A block of `rows` rows of `width` bytes, `ld` bytes apart.
struct Rows {
  const void* p;
  long long ld, width;
  int rows;
};
// Whether two blocks of rows share a byte (rows of different strides that lie
// in one another's range count as sharing).
bool overlap(const Rows& a, const Rows& b) {
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
  const long long pa = (long long)reinterpret_cast<uintptr_t>(a.p), pb = (long long)reinterpret_cast<uintptr_t>(b.p);
  if (pa + (a.rows - 1) * a.ld + a.width <= pb || pb + (b.rows - 1) * b.ld + b.width <= pa) return false;
  if (a.rows == 1 && b.rows == 1) return true;
  if (a.ld != b.ld || a.ld <= 0) return true;
  const long long d = (((pb - pa) % a.ld) + a.ld) % a.ld;
  return d < a.width || a.ld - d < b.width;
}

bool vec_rows(const void* p, long long ld_bytes) { return !p || (aligned(p, 16) && ld_bytes % 16 == 0); }

}  // namespace

extern "C" {

// ------------------------------------------------------------ INT4 products

llmoc_status llmoc_int4_linear_create(const llmoc_int4_view* views, int n_views, int device, int on_device,
                                      llmoc_int4_linear** out) {
  const char* who = "llmoc_int4_linear_create";
  if (!out) return refuse(LLMOC_ERR_INVALID, "null out");
  *out = nullptr;
  if (!views || n_views <= 0) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": no views");
  const int K = views[0].K, gs = views[0].group_size > 0 ? views[0].group_size : 128;
  const uint32_t scheme = views[0].scheme;
  const int zp = views[0].awq_zp > 0 ? views[0].awq_zp : 7;
  if (scheme != LLMOC_SCHEME_AWQ_SYM && scheme != LLMOC_SCHEME_GPTQ_ASYM)
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": unknown INT4 scheme");
  const bool awq = scheme == LLMOC_SCHEME_AWQ_SYM;
  if (K <= 0) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": K must be positive");
  if (K % 32 || gs % 32)
    return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": K and group_size must be multiples of 32");
  if (awq && zp > 127) return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": zero point above 127");
  long long M = 0;
  for (int i = 0; i < n_views; ++i) {
    const llmoc_int4_view& v = views[i];
    const int vgs = v.group_size > 0 ? v.group_size : 128, vzp = v.awq_zp > 0 ? v.awq_zp : 7;
    if (!v.qweight || !v.scales || v.M <= 0)
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": view " + std::to_string(i) + " is empty");
    if (on_device && (!aligned(v.scales, 2) || (!awq && !aligned(v.zeros, 2))))
      return refuse(LLMOC_ERR_INVALID,
                    std::string(who) + ": view " + std::to_string(i) + ": a pointer is not aligned to its element");
    if (v.K != K || vgs != gs || v.scheme != scheme || (awq && vzp != zp))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": view " + std::to_string(i) +
                                           " differs from the first in K, group size, scheme or zero point");
    if (i + 1 < n_views && v.M % 16)
      return refuse(LLMOC_ERR_UNSUPPORTED,
                    std::string(who) + ": every view but the last needs a multiple of 16 rows");
    M += v.M;
  }
  if (M > 0x7FFFFFF0ll) return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": more than 2^31 - 16 rows");
  int ndev = 0;
  if (cudaGetDeviceCount(&ndev) != cudaSuccess || device < 0 || device >= ndev) {
    cudaGetLastError();
    return no_device(who, device);
  }
  OnDevice od(device);
  if (!od.ok) return no_device(who, device);
  for (int i = 0; i < n_views && on_device; ++i)  // the kernel that packs them would fault on pageable memory
    for (const void* p : {(const void*)views[i].qweight, (const void*)views[i].scales,
                          (const void*)(awq ? nullptr : views[i].zeros)}) {
      cudaPointerAttributes at{};
      if (!p) continue;
      if (cudaPointerGetAttributes(&at, p) != cudaSuccess) cudaGetLastError();
      if (at.type == cudaMemoryTypeUnregistered || (at.type == cudaMemoryTypeDevice && at.device != device))
        return refuse(LLMOC_ERR_INVALID, std::string(who) + ": view " + std::to_string(i) + " is not in memory of device " +
                                             std::to_string(device));
    }
  auto* L = new (std::nothrow) llmoc_int4_linear();
  if (!L) return refuse(LLMOC_ERR_NO_MEMORY, std::string(who) + ": out of memory");
  L->device = device;
  L->M = (int)M;
  L->K = K;
  L->nb = (K + 255) / 256;
  L->mt = (int)((M + 15) / 16);
  L->zp = zp;
  L->fl = gs % 128 == 0 ? 4 : gs % 64 == 0 ? 2 : 1;
  L->awq = awq;
  const int ng = (K + gs - 1) / gs;
  const size_t tile_bytes = (size_t)L->nb * lin_block_bytes(L->fl, !awq);
  L->weight_bytes = (size_t)L->mt * tile_bytes;
  cudaStream_t st = nullptr;
  void* staging = nullptr;
  llmoc_status rc = LLMOC_OK;
  auto cuda = [&](cudaError_t e, llmoc_status code) {
    if (e == cudaSuccess) return true;
    cudaGetLastError();
    rc = refuse(code, std::string(who) + ": " + cudaGetErrorString(e));
    return false;
  };
  do {
    if (!cuda(cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking), LLMOC_ERR_CUDA)) break;
    if (!cuda(cudaMalloc((void**)&L->arena, up256(L->weight_bytes) + 256), LLMOC_ERR_NO_MEMORY)) break;
    char* at = L->arena;
    L->err = (int*)(L->arena + up256(L->weight_bytes));
    if (!cuda(cudaMemsetAsync(L->err, 0, 4, st), LLMOC_ERR_CUDA)) break;
    size_t need = 0;  // staging of the largest host view
    for (int i = 0; i < n_views && !on_device; ++i) {
      const size_t n = up256((size_t)views[i].M * (K / 2)) + 2 * up256((size_t)views[i].M * ng * 2);
      need = n > need ? n : need;
    }
    if (need && !cuda(cudaMalloc(&staging, need), LLMOC_ERR_NO_MEMORY)) break;
    for (int i = 0; i < n_views && rc == LLMOC_OK; ++i) {
      const llmoc_int4_view& v = views[i];
      const size_t qsrc = (size_t)v.M * (K / 2), ssrc = (size_t)v.M * ng * 2;
      const uint16_t* vz = awq ? nullptr : v.zeros;
      LinPack ra{};
      ra.q = v.qweight;
      ra.s = v.scales;
      ra.z = vz;
      if (!on_device) {
        char* p = (char*)staging;
        if (!cuda(cudaMemcpyAsync(p, v.qweight, qsrc, cudaMemcpyHostToDevice, st), LLMOC_ERR_CUDA)) break;
        ra.q = (const uint8_t*)p;
        p += up256(qsrc);
        if (!cuda(cudaMemcpyAsync(p, v.scales, ssrc, cudaMemcpyHostToDevice, st), LLMOC_ERR_CUDA)) break;
        ra.s = (const uint16_t*)p;
        p += up256(ssrc);
        if (vz) {
          if (!cuda(cudaMemcpyAsync(p, vz, ssrc, cudaMemcpyHostToDevice, st), LLMOC_ERR_CUDA)) break;
          ra.z = (const uint16_t*)p;
        }
      }
      ra.M = v.M;
      ra.K = K;
      ra.gs = gs;
      ra.ng = ng;
      ra.nb = L->nb;
      ra.fl = L->fl;
      ra.gptq = !awq;
      ra.out = (uint32_t*)at;
      if (!cuda(launch_lin_pack(ra, st), LLMOC_ERR_CUDA)) break;
      note_launches(1);
      at += (size_t)((v.M + 15) / 16) * tile_bytes;
    }
    if (rc != LLMOC_OK) break;
    cuda(cudaStreamSynchronize(st), LLMOC_ERR_CUDA);
  } while (false);
  if (st) {
    cudaStreamSynchronize(st);
    cudaStreamDestroy(st);
  }
  if (staging) cudaFree(staging);
  if (rc != LLMOC_OK) {
    if (L->arena) cudaFree(L->arena);
    delete L;
    return rc;
  }
  *out = L;
  return LLMOC_OK;
}

void llmoc_int4_linear_destroy(llmoc_int4_linear* L) {
  if (!L) return;
  OnDevice od(L->device);
  if (od.ok && L->arena) cudaFree(L->arena);
  delete L;
}

size_t llmoc_int4_linear_weight_bytes(const llmoc_int4_linear* L) { return L ? L->weight_bytes : 0; }

llmoc_status llmoc_int4_linear_forward(const llmoc_int4_linear* L, const uint16_t* X, int64_t ldx, int T,
                                       const uint16_t* R, int64_t ldr, void* Y, int64_t ldy, int y_dtype,
                                       void* stream) {
  const char* who = "llmoc_int4_linear_forward";
  if (!L || T < 0 || !dtype_ok(y_dtype)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": bad arguments");
  if (T == 0) return LLMOC_OK;
  if (!X || !Y) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": null X or Y");
  if (ldx < L->K || ldy < L->M || (R && ldr < L->M))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a row stride is smaller than its row");
  const long long es = (long long)dtype_bytes(y_dtype);
  if (!aligned(X, 2) || !aligned(Y, (size_t)es) || !aligned(R, 2))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a pointer is not aligned to its element");
  const Rows rx{X, ldx * 2, (long long)L->K * 2, T}, ry{Y, ldy * es, L->M * es, T};
  const Rows rr{R, ldr * 2, (long long)L->M * 2, T};
  const bool in_place = (const void*)R == Y && y_dtype == LLMOC_DTYPE_BF16 && (ldr == ldy || T == 1);
  if (overlap(rx, ry) || (R && !in_place && overlap(rr, ry)))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": Y overlaps an input");
  OnDevice od(L->device);
  if (!od.ok) return no_device(who, L->device);
  LinArgs a{};
  a.q = L->arena;
  a.M = L->M;
  a.K = L->K;
  a.nb = L->nb;
  a.mt = L->mt;
  a.zp = L->zp;
  a.X = (const __nv_bfloat16*)X;
  a.ldx = ldx;
  a.T = T;
  a.R = (const __nv_bfloat16*)R;
  a.ldr = ldr;
  a.Y = Y;
  a.ldy = ldy;
  a.y_f32 = y_dtype == LLMOC_DTYPE_F32;
  a.x_vec = aligned(X, 16) && ldx % 8 == 0;
  a.y_vec = aligned(Y, a.y_f32 ? 8 : 4) && ldy % 2 == 0;
  a.err = L->err;
  return launched(launch_linear(a, L->fl, L->awq, (cudaStream_t)stream), who, 1);
}

llmoc_status llmoc_int4_linear_status(llmoc_int4_linear* L, void* stream) {
  const char* who = "llmoc_int4_linear_status";
  if (!L) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": null linear");
  OnDevice od(L->device);
  if (!od.ok) return no_device(who, L->device);
  cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing((cudaStream_t)stream, &cap) != cudaSuccess || cap != cudaStreamCaptureStatusNone) {
    cudaGetLastError();
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the stream is being captured");
  }
  int word = 0;
  cudaError_t e = cudaMemcpyAsync(&word, L->err, 4, cudaMemcpyDeviceToHost, (cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaMemsetAsync(L->err, 0, 4, (cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
  if (e != cudaSuccess) return launched(e, who, 0);
  if (word)
    return refuse(LLMOC_ERR_TIMEOUT, std::string(who) + ": a bounded device-side wait gave up; outputs are not valid");
  return LLMOC_OK;
}

// ------------------------------------------------------------------- norms

static llmoc_status check_norm(const llmoc_norm_desc* d, const char* who) {
  if (!d) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": null norm description");
  if (d->hidden <= 0) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": hidden must be positive");
  if (d->hidden > kNormMaxH)
    return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": hidden above " + std::to_string(kNormMaxH));
  for (int k : {d->post, d->pre})
    if (k != LLMOC_NORM_NONE && k != LLMOC_NORM_RMS && k != LLMOC_NORM_LAYER)
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": unknown norm");
  if (d->gate_act != LLMOC_ACT_NONE && d->gate_act != LLMOC_ACT_SIGMOID)
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": unknown gate activation");
  if (!dtype_ok(d->weight_dtype)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": unknown weight type");
  if (!(d->eps > 0.f) || !std::isfinite(d->eps))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": eps must be positive");
  for (const void* p : {d->post_weight, d->post_bias, d->pre_weight, d->pre_bias})
    if (!aligned(p, dtype_bytes(d->weight_dtype)))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a weight is not aligned to its element");
  return LLMOC_OK;
}

// checks the call and, with `run`, makes it
static llmoc_status norm_call(const llmoc_norm_desc* d, const llmoc_norm_io* io, int T, int device, void* stream,
                              bool run) {
  const char* who = "llmoc_norm_residual";
  const llmoc_status ok = check_norm(d, who);
  if (ok != LLMOC_OK) return ok;
  if (!io || T < 0) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": bad arguments");
  if (T == 0) return LLMOC_OK;
  if (!dtype_ok(io->block_dtype) || !dtype_ok(io->residual_dtype) || !dtype_ok(io->norm_dtype) ||
      !dtype_ok(io->gate_dtype))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": unknown type");
  if (!io->block && !io->residual) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": neither block nor residual");
  if (!io->residual_out && !io->norm_out) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": no output");
  const int H = d->hidden;
  const struct {
    const void* p;
    int64_t ld;
    int dt;
  } rows[4] = {{io->block, io->ld_block, io->block_dtype},
               {io->residual, io->ld_residual, io->residual_dtype},
               {io->residual_out, io->ld_residual_out, io->residual_dtype},
               {io->norm_out, io->ld_norm_out, io->norm_dtype}};
  bool vec = H % 8 == 0;
  for (const auto& r : rows) {
    if (!r.p) continue;
    if (r.ld < H) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a row stride is smaller than hidden");
    if (!aligned(r.p, dtype_bytes(r.dt)))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a pointer is not aligned to its element");
    vec = vec && vec_rows(r.p, r.ld * (long long)dtype_bytes(r.dt));
  }
  if (io->gate) {
    if (!io->block) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a gate without a block");
    if (io->gate_row_stride < 0 || (io->gate_col_stride != 0 && io->gate_col_stride != 1))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": gate strides");
    if (!aligned(io->gate, dtype_bytes(io->gate_dtype)))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the gate is not aligned to its element");
    if (io->gate_col_stride) vec = vec && vec_rows(io->gate, io->gate_row_stride * (long long)dtype_bytes(io->gate_dtype));
  }
  auto range = [&](int i) {
    const long long es = (long long)dtype_bytes(rows[i].dt);
    return Rows{rows[i].p, rows[i].ld * es, H * es, T};
  };
  for (int o = 2; o < 4; ++o)
    for (int i = 0; i < o; ++i) {
      if (!rows[o].p || !rows[i].p || !overlap(range(o), range(i))) continue;
      const bool same = rows[o].p == rows[i].p && rows[o].dt == rows[i].dt && (rows[o].ld == rows[i].ld || T == 1);
      if (i == 2 || !same)
        return refuse(LLMOC_ERR_INVALID, std::string(who) + ": an output overlaps another operand");
    }
  if (io->gate) {
    const long long es = (long long)dtype_bytes(io->gate_dtype);
    const Rows g{io->gate, io->gate_row_stride * es, (io->gate_col_stride ? H : 1) * es, io->gate_row_stride ? T : 1};
    if (overlap(g, range(2)) || overlap(g, range(3)))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": an output overlaps the gate");
  }
  for (const void* p : {d->post_weight, d->post_bias, d->pre_weight, d->pre_bias}) {
    const Rows w{p, 0, H * (long long)dtype_bytes(d->weight_dtype), 1};  // read anew for every row
    if (overlap(w, range(2)) || overlap(w, range(3)))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": an output overlaps a weight");
    vec = vec && vec_rows(p, 0);
  }
  if (!run) return LLMOC_OK;
  OnDevice od(device);
  if (!od.ok) return no_device(who, device);
  NormArgs a{};
  a.block = io->block;
  a.res = io->residual;
  a.res_out = io->residual_out;
  a.out = io->norm_out;
  a.post_w = d->post_weight;
  a.post_b = d->post_bias;
  a.pre_w = d->pre_weight;
  a.pre_b = d->pre_bias;
  a.gate = io->gate;
  a.ld_block = io->ld_block;
  a.ld_res = io->ld_residual;
  a.ld_res_out = io->ld_residual_out;
  a.ld_out = io->ld_norm_out;
  a.gate_row = io->gate_row_stride;
  a.gate_col = io->gate_col_stride;
  a.T = T;
  a.H = H;
  a.post = d->post;
  a.pre = d->pre;
  a.block_f32 = io->block_dtype == LLMOC_DTYPE_F32;
  a.res_f32 = io->residual_dtype == LLMOC_DTYPE_F32;
  a.out_f32 = io->norm_dtype == LLMOC_DTYPE_F32;
  a.w_f32 = d->weight_dtype == LLMOC_DTYPE_F32;
  a.gate_f32 = io->gate_dtype == LLMOC_DTYPE_F32;
  a.gate_sigmoid = d->gate_act == LLMOC_ACT_SIGMOID;
  a.w_off = d->weight_offset;
  a.eps = d->eps;
  a.block_scale = d->block_scale;
  a.res_scale = d->residual_scale;
  a.vec = vec;
  return launched(launch_norm(a, (cudaStream_t)stream), who, 1);
}

llmoc_status llmoc_norm_residual(const llmoc_norm_desc* d, const llmoc_norm_io* io, int T, int device, void* stream) {
  return norm_call(d, io, T, device, stream, true);
}

size_t llmoc_moe_block_workspace_bytes(const llmoc_moe_layer* layer, int max_tokens) {
  if (!layer || max_tokens < 0) return 0;
  return up256((size_t)max_tokens * layer_hidden(layer) * 2) * 2 + llmoc_moe_workspace_bytes(layer, max_tokens);
}

llmoc_status llmoc_moe_forward_block(const llmoc_moe_layer* layer, const llmoc_norm_desc* in,
                                     const llmoc_norm_desc* out, const llmoc_norm_io* io, int T, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* who = "llmoc_moe_forward_block";
  if (!layer || !io || T < 0) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": bad arguments");
  llmoc_status rc = check_norm(in, who);
  if (rc == LLMOC_OK) rc = check_norm(out, who);
  if (rc != LLMOC_OK) return rc;
  const int H = layer_hidden(layer);
  if (in->hidden != H || out->hidden != H)
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the norms' hidden is not the layer's");
  if (in->pre == LLMOC_NORM_NONE) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": no norm before the block");
  if (T == 0) return LLMOC_OK;
  if (!io->residual) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": null residual");
  if (io->residual_dtype != LLMOC_DTYPE_BF16 || (io->norm_out && io->norm_dtype != LLMOC_DTYPE_BF16))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": residual and norm_out must be bf16");
  const size_t need = llmoc_moe_block_workspace_bytes(layer, T);
  if (!workspace || workspace_bytes < need)
    return refuse(LLMOC_ERR_WORKSPACE, std::string(who) + ": workspace too small");
  if (!aligned(workspace, 16))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the workspace is not aligned to 16");
  char* x = (char*)workspace;
  char* b = x + up256((size_t)T * H * 2);
  char* ws = b + up256((size_t)T * H * 2);
  llmoc_norm_desc first = *in;
  first.post = LLMOC_NORM_NONE;
  first.block_scale = first.residual_scale = 1.f;
  llmoc_norm_io i1{};
  i1.residual = io->residual;
  i1.ld_residual = io->ld_residual;
  i1.residual_dtype = i1.norm_dtype = i1.block_dtype = i1.gate_dtype = LLMOC_DTYPE_BF16;
  i1.norm_out = x;
  i1.ld_norm_out = H;
  llmoc_norm_io i2 = *io;
  i2.block = b;
  i2.ld_block = H;
  i2.block_dtype = LLMOC_DTYPE_BF16;
  const int dev = layer_device(layer);
  rc = norm_call(out, &i2, T, dev, stream, false);  // refuse before anything runs
  if (rc != LLMOC_OK) return rc;
  const long long gs = (long long)dtype_bytes(io->gate_dtype);
  const Rows wr{workspace, (long long)need, (long long)need, 1};
  for (const Rows& r : {Rows{io->residual, io->ld_residual * 2, H * 2ll, T},
                        Rows{io->residual_out, io->ld_residual_out * 2, H * 2ll, T},
                        Rows{io->norm_out, io->ld_norm_out * 2, H * 2ll, T},
                        Rows{io->gate, io->gate_row_stride * gs, (io->gate_col_stride ? H : 1) * gs,
                             io->gate_row_stride ? T : 1}})
    if (overlap(wr, r)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the workspace overlaps an operand");
  rc = norm_call(&first, &i1, T, dev, stream, true);
  if (rc != LLMOC_OK) return rc;
  rc = llmoc_moe_forward(layer, (const uint16_t*)x, T, (uint16_t*)b, ws,
                         workspace_bytes - (size_t)(ws - (char*)workspace), stream);
  if (rc != LLMOC_OK) return rc;
  return llmoc_norm_residual(out, &i2, T, dev, stream);
}

// ------------------------------------------------------------- beam search

static llmoc_status check_beam(const llmoc_beam_desc* d, const char* who) {
  if (!d || d->batch < 0 || d->beams <= 0 || d->vocab <= 0 || d->n_out <= 0 || d->eos_token < -1 ||
      d->eos_token >= d->vocab)
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": bad description");
  if (d->beams > kBeamMaxBeams || d->n_out > kBeamMaxOut)
    return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": more than 128 beams or candidates");
  if (d->vocab > (1 << 30) || (long long)d->batch * d->beams > (1 << 24))
    return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": vocabulary or batch too large");
  return LLMOC_OK;
}

static size_t beam_bytes(const llmoc_beam_desc* d, long long lists) {
  return up256((size_t)lists * d->n_out * 8) + up256((size_t)lists * 8);
}

size_t llmoc_beam_workspace_bytes(const llmoc_beam_desc* d) {
  if (check_beam(d, "llmoc_beam_workspace_bytes") != LLMOC_OK) return 0;
  return beam_bytes(d, std::max(beam_lists(d->batch, d->beams, d->vocab, 0), beam_lists(d->batch, d->beams, d->vocab, 1)));
}

llmoc_status llmoc_beam_select(const llmoc_beam_desc* d, const void* logits, int64_t ld, int logits_dtype,
                               const float* scores, const uint8_t* finished, int32_t* parent, int32_t* token,
                               float* out_scores, uint8_t* finished_out, void* workspace, size_t workspace_bytes,
                               int device, void* stream) {
  const char* who = "llmoc_beam_select";
  const llmoc_status ok = check_beam(d, who);
  if (ok != LLMOC_OK) return ok;
  if (!dtype_ok(logits_dtype)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": unknown type");
  if (finished && d->eos_token < 0)
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": finished beams need an eos_token");
  if (d->batch == 0) return LLMOC_OK;
  if (!logits || !scores || !parent || !token || !out_scores)
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": null operand");
  if (ld < d->vocab) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": ld is smaller than vocab");
  const size_t es = dtype_bytes(logits_dtype);
  if (!aligned(logits, es) || !aligned(scores, 4) || !aligned(parent, 4) || !aligned(token, 4) ||
      !aligned(out_scores, 4))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": a pointer is not aligned to its element");
  const long long rows = (long long)d->batch * d->beams, n = (long long)d->batch * d->n_out;
  const Rows in[3] = {{logits, (long long)(ld * es), (long long)(d->vocab * es), (int)rows},
                      {scores, rows * 4, rows * 4, 1},
                      {finished, rows, rows, 1}};
  const Rows outs[4] = {{parent, n * 4, n * 4, 1}, {token, n * 4, n * 4, 1}, {out_scores, n * 4, n * 4, 1},
                        {finished_out, n, n, 1}};
  for (int o = 0; o < 4; ++o) {
    for (int i = 0; i < 3; ++i)
      if (overlap(outs[o], in[i]))
        return refuse(LLMOC_ERR_INVALID, std::string(who) + ": an output overlaps an input");
    for (int i = 0; i < o; ++i)
      if (overlap(outs[o], outs[i])) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": two outputs overlap");
  }
  const int f32 = logits_dtype == LLMOC_DTYPE_F32, splits = beam_splits(d->batch, d->beams, d->vocab, f32);
  const size_t need = beam_bytes(d, rows * splits);
  if (!workspace || workspace_bytes < need)
    return refuse(LLMOC_ERR_WORKSPACE, std::string(who) + ": workspace too small");
  if (!aligned(workspace, 8)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the workspace is not aligned to 8");
  const Rows wr{workspace, (long long)need, (long long)need, 1};
  for (const Rows& r : in)
    if (overlap(wr, r)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the workspace overlaps an input");
  for (const Rows& r : outs)
    if (overlap(wr, r)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": the workspace overlaps an output");
  OnDevice od(device);
  if (!od.ok) return no_device(who, device);
  BeamArgs a{};
  a.logits = logits;
  a.ld = ld;
  a.f32 = f32;
  a.scores = scores;
  a.fin = finished;
  a.batch = d->batch;
  a.beams = d->beams;
  a.vocab = d->vocab;
  a.n_out = d->n_out;
  a.eos = d->eos_token;
  a.parent = parent;
  a.token = token;
  a.out = out_scores;
  a.fin_out = finished_out;
  a.splits = splits;
  a.vec = vec_rows(logits, ld * (long long)es);
  const size_t lists = (size_t)rows * a.splits;
  a.cand = (float2*)workspace;
  a.stat = (float2*)((char*)workspace + up256(lists * d->n_out * 8));
  return launched(launch_beam_select(a, (cudaStream_t)stream), who, 2);
}

llmoc_status llmoc_beam_reorder(const llmoc_reorder_tensor* tensors, int n_tensors, const int32_t* parent, int batch,
                                int beams, int n_out, int device, void* stream) {
  const char* who = "llmoc_beam_reorder";
  if (n_tensors < 0 || batch < 0 || beams <= 0 || n_out <= 0 || (n_tensors > 0 && !tensors))
    return refuse(LLMOC_ERR_INVALID, std::string(who) + ": bad arguments");
  if (n_out > kReorderMaxOut || (long long)batch * (beams > n_out ? beams : n_out) > (1 << 24))
    return refuse(LLMOC_ERR_UNSUPPORTED, std::string(who) + ": more than 64 rows per sequence, or too large a batch");
  if (n_tensors == 0 || batch == 0) return LLMOC_OK;
  if (!parent || !aligned(parent, 4)) return refuse(LLMOC_ERR_INVALID, std::string(who) + ": null or unaligned parent");
  // what a tensor's rows span, and whether their segments are disjoint
  auto span = [](const llmoc_reorder_tensor& t, long long stride, long long rows, bool* ok) {
    const long long extent = (t.n_seg - 1) * (t.n_seg > 1 ? t.seg_stride : 0) + t.seg_bytes;
    const bool inner = t.n_seg == 1 || t.seg_stride >= t.seg_bytes;  // a row's segments do not meet
    const bool rows_apart = rows == 1 || (inner && stride >= extent);
    const bool seg_apart = stride >= t.seg_bytes && t.seg_stride >= (rows - 1) * stride + t.seg_bytes;
    *ok = stride >= 0 && ((inner && rows_apart) || seg_apart);
    return (rows - 1) * stride + extent;
  };
  for (int i = 0; i < n_tensors; ++i) {
    const llmoc_reorder_tensor& t = tensors[i];
    if (!t.src || !t.dst || t.n_seg <= 0 || t.seg_bytes < 0 || (t.n_seg > 1 && t.seg_stride < 0))
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": tensor " + std::to_string(i) + ": bad geometry");
    bool s_ok, d_ok;
    span(t, t.src_stride, (long long)batch * beams, &s_ok);
    span(t, t.dst_stride, (long long)batch * n_out, &d_ok);
    if (!s_ok || !d_ok)
      return refuse(LLMOC_ERR_INVALID, std::string(who) + ": tensor " + std::to_string(i) + ": rows overlap");
  }
  // a destination overlaps nothing but, in place, its own source: the ranges
  // in order of their starts, each against the furthest end before it
  struct Range {
    const char *lo, *hi;
    int tensor;
    bool dst;
  };
  Range few[2 * kReorderBatch + 1];
  Range* rg = n_tensors <= kReorderBatch ? few : new (std::nothrow) Range[2 * (size_t)n_tensors + 1];
  if (!rg) return refuse(LLMOC_ERR_NO_MEMORY, std::string(who) + ": out of memory");
  size_t nr = 0;
  rg[nr++] = Range{(const char*)parent, (const char*)(parent + (size_t)batch * n_out), -1, false};
  for (int i = 0; i < n_tensors; ++i) {
    const llmoc_reorder_tensor& t = tensors[i];
    bool ok;
    const long long ds = span(t, t.dst_stride, (long long)batch * n_out, &ok);
    const bool in_place = t.src == t.dst && t.src_stride == t.dst_stride && n_out == beams;
    if (t.seg_bytes == 0) continue;
    rg[nr++] = Range{(const char*)t.dst, (const char*)t.dst + ds, i, true};
    if (!in_place) {
      const long long ss = span(t, t.src_stride, (long long)batch * beams, &ok);
      rg[nr++] = Range{(const char*)t.src, (const char*)t.src + ss, i, false};
    }
  }
  std::sort(rg, rg + nr, [](const Range& a, const Range& b) { return a.lo < b.lo; });
  const char *any_end = nullptr, *dst_end = nullptr;
  const Range* bad = nullptr;
  for (size_t i = 0; i < nr && !bad; ++i) {
    if ((rg[i].dst ? any_end : dst_end) > rg[i].lo) bad = rg + i;
    any_end = std::max(any_end, rg[i].hi);
    if (rg[i].dst) dst_end = std::max(dst_end, rg[i].hi);
  }
  const int which = bad ? bad->tensor : 0;
  if (rg != few) delete[] rg;
  if (bad)
    return refuse(LLMOC_ERR_INVALID,
                  std::string(who) + ": a destination overlaps a source, another destination or parent (" +
                      (which < 0 ? std::string("parent") : "tensor " + std::to_string(which)) + ")");
  OnDevice od(device);
  if (!od.ok) return no_device(who, device);
  for (int i0 = 0; i0 < n_tensors; i0 += kReorderBatch) {
    ReorderArgs a{};
    a.n = n_tensors - i0 < kReorderBatch ? n_tensors - i0 : kReorderBatch;
    a.parent = parent;
    a.batch = batch;
    a.beams = beams;
    a.n_out = n_out;
    for (int i = 0; i < a.n; ++i) {
      const llmoc_reorder_tensor& t = tensors[i0 + i];
      ReorderTensor& r = a.t[i];
      r.src = (const char*)t.src;
      r.dst = (char*)t.dst;
      r.src_stride = t.src_stride;
      r.dst_stride = t.dst_stride;
      r.seg_stride = t.n_seg > 1 ? t.seg_stride : 0;
      r.seg_bytes = t.seg_bytes;
      r.n_seg = t.n_seg;
      // the widest access that every row and segment start allows
      const uintptr_t at = (uintptr_t)t.src | (uintptr_t)t.dst | (uintptr_t)t.src_stride | (uintptr_t)t.dst_stride |
                           (uintptr_t)r.seg_stride;
      r.width = 16;
      while (r.width > 1 && (at & (r.width - 1))) r.width >>= 1;
    }
    const cudaError_t e = launch_reorder(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return launched(e, who, 0);
    note_launches(1);
  }
  return LLMOC_OK;
}

}  // extern "C"
