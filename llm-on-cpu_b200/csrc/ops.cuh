// ops.cuh — argument structs and launchers of the operators around the MoE
// layer: dense INT4 products (linear.cu), residual norms (norm.cu), beam
// selection and state reordering (beam.cu).  Host side: ops_runtime.cu.
#pragma once
#include <cstddef>
#include <cstdint>
#include <string>

#include "common.cuh"

namespace llmoc {

// ---- linear.cu
// Bytes of a 256-wide block of a tile's stream: 2048 of words, then 32 for each
// group of fl * 32 (twice with zeros).
__host__ __device__ constexpr int lin_block_bytes(int fl, bool gptq) { return 2048 + 8 / fl * 32 * (gptq ? 2 : 1); }
struct LinArgs {
  const char* q;  // the packed stream
  int M, K;
  int nb;         // blocks of 256 k per tile
  int mt;         // 16-row tiles
  int zp;
  const __nv_bfloat16* X;
  long long ldx;
  int T;
  const __nv_bfloat16* R;  // [T][M] added before the rounding, or null
  long long ldr;
  void* Y;
  long long ldy;
  int y_f32;
  int x_vec;  // X rows readable by 16-byte loads
  int y_vec;  // two neighbours of Y, the first in an even column, writable at once
  int* err;   // bit 0: a bounded wait gave up
};
struct LinPack {
  const uint8_t* q;   // QLWC [M][K / 2]
  const uint16_t* s;  // [M][ng] fp16
  const uint16_t* z;  // or null
  int M, K, gs, ng, nb, fl, gptq;
  uint32_t* out;
};
cudaError_t launch_lin_pack(const LinPack& a, cudaStream_t st);
cudaError_t launch_linear(const LinArgs& a, int fl, bool awq, cudaStream_t st);
// CTAs of c-wide clusters that are resident at once on the current device, one on
// an SM (a cluster stays within a GPC, whose SMs are rarely a multiple of c)
int cluster_ctas(int c);
// linear_umma.cu: the same product for tens of tokens (tcgen05); zp < 16
cudaError_t launch_linear_umma(const LinArgs& a, int fl, bool awq, cudaStream_t st);

// ---- norm.cu
struct NormArgs {
  const void* block;
  const void* res;
  void* res_out;
  void* out;
  const void* post_w;
  const void* post_b;
  const void* pre_w;
  const void* pre_b;
  const void* gate;
  long long ld_block, ld_res, ld_res_out, ld_out, gate_row, gate_col;
  int T, H;
  int post, pre;  // LLMOC_NORM_*
  int block_f32, res_f32, out_f32, w_f32, gate_f32, gate_sigmoid;
  float w_off, eps, block_scale, res_scale;
  int vec;  // every row of every operand readable by 16-byte loads
};
constexpr int kNormMaxH = 16384;
cudaError_t launch_norm(const NormArgs& a, cudaStream_t st);

// ---- beam.cu
struct BeamArgs {
  const void* logits;  // [batch * beams][ld]
  long long ld;
  int f32;
  const float* scores;        // [batch][beams]
  const unsigned char* fin;   // [batch][beams] or null
  int batch, beams, vocab, n_out, eos;
  int* parent;
  int* token;
  float* out;
  unsigned char* fin_out;  // or null
  int splits;  // vocabulary slices per row
  int vec;                 // rows readable by 16-byte loads
  float2* cand;            // workspace [batch * beams][splits][n_out]: (logit, index bits), best first
  float2* stat;            // workspace [batch * beams][splits]: (max, sum exp(x - max))
};
constexpr int kBeamMaxOut = 128;
constexpr int kBeamMaxBeams = 128;
int beam_splits(int batch, int beams, int vocab, int f32);
long long beam_lists(int batch, int beams, int vocab, int f32);
cudaError_t launch_beam_select(const BeamArgs& a, cudaStream_t st);

struct ReorderTensor {
  const char* src;
  char* dst;
  long long src_stride, dst_stride, seg_stride;
  long long seg_bytes;
  int n_seg;
  int width;  // bytes per column access: 16, 8, 4, 2 or 1
};
constexpr int kReorderBatch = 48;  // tensors per launch
constexpr int kReorderMaxOut = 64;
struct ReorderArgs {
  ReorderTensor t[kReorderBatch];
  long long first[kReorderBatch + 1];  // first block of each tensor, then the total
  int n;
  const int* parent;
  int batch, beams, n_out;
};
cudaError_t launch_reorder(ReorderArgs& a, cudaStream_t st);

// ---- runtime.cu
void set_last_error(const std::string& msg);
void note_launches(int n);

}  // namespace llmoc
