// Host-side launch interface of the sm_100a kernels (no torch types; raw pointers).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace nsw {

enum DType : int { kBF16 = 0, kF16 = 1, kF32 = 2 };

int* device_error_flag();  // per-device error word (lazily allocated)

// ---- norms -------------------------------------------------------------------
cudaError_t rmsnorm_fwd(const void* x, const float* w, void* y, float* rstd, int64_t rows, int n,
                        float eps, int dtype, cudaStream_t s);
cudaError_t rmsnorm_bwd(const void* dy, const void* x, const float* w, const float* rstd, void* dx,
                        float* dw_partial, int partial_rows, int64_t rows, int n, int dtype,
                        cudaStream_t s, float eps = -1.f, const void* add = nullptr);

// ---- elementwise epilogues -----------------------------------------------------
// y = act(acc + bias) + residual (residual row index = row % res_period)
cudaError_t bias_act_residual(const void* acc, int acc_dtype, const float* bias, const void* residual,
                              int64_t res_period, void* y, void* preact, int64_t rows, int n,
                              int act, int dtype, cudaStream_t s);
cudaError_t gelu_bwd(const void* dy, const void* u, void* du, int64_t n, int dtype, cudaStream_t s);
// column sums of a [rows, n] matrix in fp32 (deterministic two-pass)
// out_b[:] (+)= sum over rows of part[b, :, :] (fp32, rows in order); out_b = out + b * n, except
// out_1 = out1 when given (separate destinations, e.g. two parameters' gradients); accumulate adds
// to the destination instead of overwriting it
cudaError_t sum_rows(const float* part, int64_t batches, int64_t rows, int64_t n, float* out, cudaStream_t s,
                     bool accumulate = false, float* out1 = nullptr);
cudaError_t col_sum(const void* x, float* out, float* partial, int partial_rows, int64_t rows, int n,
                    int dtype, cudaStream_t s);

// ---- patch embed / head layout ------------------------------------------------
cudaError_t im2col_patch(const void* x, int x_dtype, void* cols, int N, int C, int H, int W, int p,
                         int dtype, cudaStream_t s);
cudaError_t col2im_patch(const void* dcols, void* dx, int x_dtype, int N, int C, int H, int W, int p,
                         int dtype, cudaStream_t s);
cudaError_t unpatchify(const void* y2, void* out, int BT, int h, int w, int p, int C, int dtype,
                       cudaStream_t s);
cudaError_t patchify(const void* dout, void* dy2, int BT, int h, int w, int p, int C, int dtype,
                     cudaStream_t s);

// ---- losses ----------------------------------------------------------------------
cudaError_t weighted_sse(const void* x, int x_dtype, const void* y, int y_dtype, const float* area_w,
                         const float* ch_w, float* partial, int partial_n, float* out, int64_t lead,
                         int C, int H, int W, cudaStream_t s);
cudaError_t weighted_sse_bwd(const void* x, int x_dtype, const void* y, int y_dtype,
                             const float* area_w, const float* ch_w, const float* gscale, void* dx,
                             int64_t lead, int C, int H, int W, cudaStream_t s);
cudaError_t weighted_se_per_plane(const void* x, int x_dtype, const void* y, int y_dtype,
                                  const float* area_w, float* out, int64_t planes, int H, int W,
                                  cudaStream_t s);

// ---- optimizer -----------------------------------------------------------------
cudaError_t adamw_step(float* p, const float* g, float* m, float* v, void* shadow, int shadow_dtype,
                       const float* gscale, const int* skip, int64_t n, float lr, float b1, float b2,
                       float eps, float wd, float bc1, float bc2, bool decoupled, cudaStream_t s);
cudaError_t segment_sumsq(const float* x, const int64_t* block_lo, const int64_t* block_hi,
                          const int* block_cls, int nblocks, int ncls, float* partial, float* out,
                          cudaStream_t s);

// ---- window attention ------------------------------------------------------------
struct AttnGeom {
  int B, T, H, W;      // token grid (local)
  int nh, hd;          // local heads, head dim
  int wh, ww;          // window
  int sh, sw;          // index shift
  int mask, mask_shift, row_offset, h_global;
  float scale;
  int64_t qkv_stride;  // elements between consecutive tokens in qkv (3*nh*hd)
  int64_t out_stride;  // elements between tokens in out / dout (nh*hd)
};
cudaError_t window_attn_fwd(const void* qkv, const float* qw, const float* kw, void* out, float* lse,
                            const AttnGeom& g, int dtype, cudaStream_t s);
// tcgen05/TMEM forward (bf16, head_dim 64, T*wh*ww <= 176); same outputs as window_attn_fwd
bool window_attn_fwd_tc_supported(const AttnGeom& g, int dtype);
cudaError_t window_attn_fwd_tc(const void* qkv, const float* qw, const float* kw, void* out, float* lse,
                               const AttnGeom& g, cudaStream_t s);
// warp-specialised tcgen05 forward (same contract and support as window_attn_fwd_tc)
cudaError_t window_attn_fwd_ws(const void* qkv, const float* qw, const float* kw, void* out, float* lse,
                               const AttnGeom& g, cudaStream_t s, long long* stamps = nullptr);
// RMSNorm, one warp per row with the row in registers (n <= 2048); rmsnorm_fwd/bwd use the TMA
// version below where it applies and these otherwise
cudaError_t rmsnorm_fwd_rows(const void* x, const float* w, void* y, float* rstd, int64_t rows, int n,
                             float eps, int dtype, cudaStream_t s);
cudaError_t rmsnorm_bwd_rows(const void* dy, const void* x, const float* w, const float* rstd, void* dx,
                             float* dw_partial, int partial_rows, int64_t rows, int n, int dtype,
                             cudaStream_t s);
// RMSNorm with TMA bulk-copy row tiles (16-bit types, n % 8 == 0, n <= 4096)
bool rmsnorm_tma_supported(int64_t rows, int n, int dtype);
cudaError_t rmsnorm_fwd_tma(const void* x, const float* w, void* y, float* rstd, int64_t rows, int n, float eps,
                            int dtype, int grid, cudaStream_t s);
// eps >= 0: rstd is recomputed from x (as the forward computed it); eps < 0: read from rstd
cudaError_t rmsnorm_bwd_tma(const void* dy, const void* x, const float* w, const float* rstd, void* dx,
                            float* dw_partial, int partial_rows, int64_t rows, int n, int dtype, float eps,
                            cudaStream_t s, const void* add = nullptr);  // add: optional [rows, n] added to dx
// dqw_part / dkw_part: one row of head_dim partial sums per CTA, min(items, SM count) rows
cudaError_t window_attn_bwd_tc(const void* qkv, const float* qw, const float* kw, const void* out,
                               const void* dout, const float* lse, void* dqkv, float* dqw_part, float* dkw_part,
                               const AttnGeom& g, cudaStream_t s, long long* stamps = nullptr);
cudaError_t window_attn_bwd(const void* qkv, const float* qw, const float* kw, const void* out,
                            const void* dout, const float* lse, void* dqkv, float* dqw_part,
                            float* dkw_part, const AttnGeom& g, int dtype, cudaStream_t s);

// ---- tcgen05 GEMM ----------------------------------------------------------------
struct GemmArgs {
  const void* A;        // [M, K] row-major (K contiguous)
  const void* B;        // [N, K] row-major (K contiguous)
  void* D;              // [M, N] row-major output (ldd elements)
  int64_t M, N, K;
  int64_t lda, ldb, ldd;
  const float* bias;    // [N] or null
  const void* residual; // [*, N] (ldr) or null; row index = m % res_period
  int64_t ldr, res_period;
  void* preact;         // optional [M, N] pre-activation output (ldd)
  int act;              // 0 none, 1 gelu, 2 * gelu'(residual), 3 gelu + gelu'(u) as preact, 4 * residual
  int dtype;            // kBF16 / kF16 (A, B, D, residual, preact)
  int out_f32;          // D in fp32 instead of dtype
  float alpha;
  int accumulate;       // D += result (fp32 output only)
  // tensor-parallel all-reduce fused into the epilogue (ar_world > 1): ar_part[r] / ar_flags[r]
  // are rank r's symmetric partial buffer (ar_world slots of [M, N] in dtype, slot s receiving
  // rank s's partial) and flag words (peer pointers)
  int ar_world;
  int ar_rank;
  void* ar_part[8];
  uint32_t* ar_flags[8];
  // optional (nullptr: off): %globaltimer stamps of the fused all-reduce epilogue's phases, eight per
  // tile for the first 32 tiles of CTAs 0..3, at [(cta * 32 + i) * 8 + phase]
  long long* ar_stamps;
};
cudaError_t gemm_tcgen05(const GemmArgs& a, cudaStream_t s, int impl = 0);
int gemm_tcgen05_supported(const GemmArgs& a);

// Weight (and bias) gradient of a linear layer on the tensor cores:
//   D[m, n] (+)= sum_t dy[t, m] * x[t, n]   (fp32),   db[m] (+)= sum_t dy[t, m]   (fp32)
// dy [T, M] and x [T, N] token-major (features contiguous, leading dimensions ldy / ldx).
// D and db may be split into up to four row segments of seg_rows rows (separate buffers, e.g. the
// q / k / v weights of a fused projection); seg_rows = 0 means one segment of M rows.
struct WgradArgs {
  const void* dy;
  int64_t ldy;
  const void* x;
  int64_t ldx;
  int64_t T, M, N;
  float* D[4];
  int64_t ldd;
  int64_t seg_rows;
  int accumulate;
  float* db[4];  // db[0] null: no bias gradient
  int db_accumulate;
  int dtype;
  float* ws;   // wgrad_workspace_floats(M, N, plan) floats (none needed when that is 0)
  int splits;  // set from the plan
  int k1;      // set from the plan
};
// Work schedule: `splits` k-splits (uniform), or with k1 > 0 the balanced schedule (each tile's first
// k1 k-blocks on a pair of its own, the rest in `splits` pieces on the remaining pairs); `pairs` is
// the number of CTA pairs it was planned for.
struct WgradPlan {
  int splits, k1, pairs;
};
WgradPlan wgrad_plan(int64_t M, int64_t N, int64_t T);
int64_t wgrad_workspace_floats(int64_t M, int64_t N, const WgradPlan& plan);
int wgrad_tcgen05_supported(const WgradArgs& a);
cudaError_t wgrad_tcgen05(const WgradArgs& a, const WgradPlan& plan, cudaStream_t s);

// ---- gated feed-forward network (gated_mlp.cu) -------------------------------------------------------
// One product of the network with its epilogue.  A operands are [M, K] rows, 16-byte aligned; weights are
// read as stored.  mode:
//   kGatedUp    out0 = act(a0 b0^T + bias0) * (a0 b1^T + bias1); out1 / out2 (both or neither, ldaux): the
//               two pre-activations; b0 / b1 [N, K]
//   kGatedDown  out0 = a0 b0^T + bias0 + in0 (optional, ldin); b0 [N, K]; rows of out0 and in0 of any alignment
//   kGatedDh    d = a0 b0 with b0 [K, N]; out0 = d * in1 * act'(in0), out1 = d * act(in0) (in: g, u, ldin;
//               out0 in rows of ldout, out1 in rows of ldaux)
//   kGatedDx    out0 = a0 b0 + a1 b1 with b0, b1 [K, N]; rows of out0 of any alignment
enum GatedMode : int { kGatedUp = 0, kGatedDown = 1, kGatedDh = 2, kGatedDx = 3 };
struct GatedArgs {
  int mode, dtype, act;  // act: 0 SiLU, 1 GELU
  int64_t M, N, K;
  const void *a0, *a1;
  int64_t lda;
  const void *b0, *b1;
  int64_t ldb0, ldb1;
  const void *bias0, *bias1;  // [N] in bias_dtype, or null
  int bias_dtype;
  const void *in0, *in1;
  int64_t ldin;
  void *out0, *out1, *out2;
  int64_t ldout, ldaux;
  // kGatedDh, where gated_sum_rows(args) > 0: that many rows of 2 sums_half column sums, of out0 at [0, N), of
  // out1 at [sums_half, sums_half + N) (null: none)
  float* sums;
  int64_t sums_half;
};
int64_t gated_sum_rows(const GatedArgs& a);
// The three weight gradients, or those of them with a D, in one launch: w[i].D (+)= w[i].a^T w[i].b over T tokens; a [T, M] in rows of lda,
// b [T, N] in rows of ldb (16-byte aligned rows; w[1].b is w[0].b), D contiguous [M, N], 16-bit or (out_f32) fp32,
// added to with accumulate; ws: gated_dw_workspace floats.
struct GatedDwArgs {
  int dtype;
  int64_t T;
  struct Weight {
    const void *a, *b;
    int64_t lda, ldb, M, N;
    void* D;
    int out_f32, accumulate;
  } w[3];
  float* ws;
};
int64_t gated_dw_workspace(const GatedDwArgs& a);
cudaError_t gated_dw(const GatedDwArgs& a, cudaStream_t s);
// Column sums.  col_partial: `parts` partial rows of n sums of one or two 16-bit matrices (rows 16-byte aligned,
// ld >= n rounded up to 8).  col_finish: sums of partial rows of `stride` floats, columns [first, first + n), into
// out (null: none): fp32 (f32; added to with accumulate) or dtype.
struct ColSource {
  const void* x;
  int64_t ld, rows, n;
  int64_t parts;
  float* partial;
};
struct ColSum {
  const float* partial;
  int64_t parts, stride, first, n;
  void* out;
  int f32, accumulate;
};
constexpr int kColSums = 3;
int col_sum_parts(int64_t rows, int64_t n);
cudaError_t col_partial(const ColSource* src, int count, int dtype, cudaStream_t s);
cudaError_t col_finish(const ColSum* v, int dtype, cudaStream_t s);
// dependent: the A operand is written by the kernel before it on the stream, which this one may overlap (a
// programmatic dependent launch: it waits for that kernel before it touches anything but the weights)
cudaError_t gated_product(const GatedArgs& a, bool dependent, cudaStream_t s);
// kGatedUp (no out1 / out2) and kGatedDown for at most kGatedSkinnyTokens rows, any strides
constexpr int kGatedSkinnyTokens = 16;
cudaError_t gated_skinny(const GatedArgs& a, bool dependent, cudaStream_t s);
// 16-bit strided copies, one launch: dst[i, j] = src[i s0 + j s1] into 16-byte aligned rows of ld elements (a
// multiple of eight, the ones past cols zero)
struct PadCopy {
  const void* src;
  void* dst;
  int64_t s0, s1, ld, rows, cols;
};
constexpr int kPadCopies = 5;
cudaError_t pad_copy(const PadCopy* v, int count, cudaStream_t s);

// ---- norms with gate and skip connection (norm_gate.cu) ------------------------------------------------
// Forward: stream = skip_scale skip + gate * rms(y) * wp; normed = rms(stream) * wn (normed and wn null: only
// the stream).  Backward: dy, dskip (null: not wanted) from ds and / or dn (null: zero), and dwp, dgate (null: not wanted), dwn
// (null with wn).  Tensors are contiguous [samples, rows, n]; gate of sample i at gate + i gate_stride (null:
// ones).  part: samples * blocks * 2 * n floats.
struct NormGateArgs {
  const void *y, *skip, *ds, *dn;
  void *stream, *normed, *dy, *dskip;
  const float *wp, *gate, *wn;
  int64_t gate_stride, samples, rows;
  int n, dtype;
  float skip_scale, eps;
  float *part, *dwp, *dgate, *dwn;
};
constexpr int kNormGateMaxWidth = 16384;
constexpr int kNormGateSkipWidth = 8192;  // wider rows: dy and dskip are always written
int norm_gate_blocks(int64_t samples, int64_t rows, int n, int sms);  // of the backward, per sample
cudaError_t norm_gate_fwd(const NormGateArgs& a, int sms, cudaStream_t s);
cudaError_t norm_gate_bwd(const NormGateArgs& a, int blocks, cudaStream_t s);

// ---- gradient clipping over separate tensors (grad_clip.cu) --------------------------------------------
struct ClipTensor {
  const void* in;
  void* out;
  int64_t n;
  int dtype;
};
constexpr int kClipTensors = 512;  // tensors in one launch's parameter table
// partial: blocks floats per table of kClipTensors tensors; norm: one float
cudaError_t clip_tensors(const ClipTensor* v, int count, float max_norm, float* partial, int blocks, float* norm,
                         cudaStream_t s);

// Data-parallel reduction / sharded AdamW over peer memory (dp_fused.cu).  Every rank's buffers:
// grad / data fp32 flat buffers, shadow 16-bit (or null), flags uint32 [kDpFlagBase + world * slots]
// (flag word of (rank r, slot) at kDpFlagBase + r * slots + slot in every rank's array).
constexpr int kDpFlagBase = 16;
struct DpPeers {
  float* grad[8];
  float* data[8];
  void* shadow[8];
  uint32_t* flags[8];
  int world, rank, slots;
};
cudaError_t dp_reduce(const DpPeers& pr, int slot, uint32_t epoch, int64_t lo, int64_t hi, float scale,
                      cudaStream_t s);
cudaError_t dp_adamw(const DpPeers& pr, const int64_t* rlo, const int64_t* rhi, const int64_t* rstart, int nranges,
                     int64_t total4, float* m, float* v, int shadow_dtype, const float* gscale, const int* skip,
                     float lr, float b1, float b2, float eps, float wd, float bc1, float bc2, bool decoupled,
                     cudaStream_t s);
cudaError_t dp_barrier(const DpPeers& pr, int slot, uint32_t epoch, cudaStream_t s);

// Cyclic roll of a (B*T, H_l, W_l, C) activation sharded over an n1 x n2 (sp1 x sp2) grid of one node's
// GPUs (halo_roll.cu): band buffers and flag words in symmetric memory, one entry per group rank.
// Flag words of each rank: [kHaloEpoch] rolls completed, [kHaloPackCount] / [kHaloDoneCount] block
// counters, [kHaloReady + r] / [kHaloAck + r] the last epoch rank r published.
constexpr int kHaloEpoch = 0, kHaloPackCount = 1, kHaloDoneCount = 2, kHaloReady = 16, kHaloAck = 32;
constexpr int kHaloFlagWords = 48;
struct HaloArgs {
  const void* x;
  void* out;
  void* band[8];
  uint32_t* flags[8];
  int world, rank, n1, n2;
  int coord1[8], coord2[8];  // (sp1, sp2) shard of each group rank
  int grid_rank[8];          // group rank holding shard (i, j), at i * n2 + j
  int h_off[9], w_off[9];    // shard offsets along H (n1 + 1 entries) and W (n2 + 1)
  int bt, row_vec, sh, sw;   // B*T, 16-byte vectors per row of C elements, shifts along H and W
};
int64_t halo_band_bytes(const HaloArgs& a, int shard);
cudaError_t halo_roll(const HaloArgs& a, cudaStream_t s);

// Legendre part of the real SHT (sht.cu): table P[m, l, k] = w_k Pbar_l^m(x_k) for orders
// m0 .. m0 + m_count - 1 (packed: order index mi's rows l = m .. L-1 start at row row_off[mi]),
// and the batched contractions C[mi, l, :] = sum_k P F[mi, k, :] / dF[mi, k, :] = sum_l P dC[mi, l, :].
cudaError_t legendre_table(const double* x, const double* w, int m0, int m_count, int L, int K,
                           const int64_t* row_off, float* P, int csphase, cudaStream_t s);
cudaError_t legendre_fwd(const float* P, const int64_t* row_off, const float* F, float* C, int m0, int m_count, int L,
                         int K, int N, cudaStream_t s);
cudaError_t legendre_bwd(const float* P, const int64_t* row_off, const float* dC, float* dF, int m0, int m_count, int L,
                         int K, int N, cudaStream_t s);

}  // namespace nsw
