// C ABI between the torch binding TU (bindings.cpp) and the pure-HIP kernel
// TUs (*.hip).  `stream` is a hipStream_t passed as void*.
// Every launcher returns a hipError_t as int (0 == success).
#pragma once

#include <cstdint>

extern "C" {

// ---- l2norm.hip -----------------------------------------------------------
// x: [N, C] (bf16 if is_bf16 else fp32) -> y same dtype, inv_norm fp32 [N]
int launch_l2norm_fwd(void* stream, const void* x, void* y, float* inv_norm,
                      int64_t N, int64_t C, bool is_bf16);
int launch_l2norm_bwd(void* stream, const void* g, const void* y,
                      const float* inv_norm, void* gx, int64_t N, int64_t C,
                      bool is_bf16);

// ---- contrastive.hip ------------------------------------------------------
// q,k: [N,C] bf16; queue_kc: [K,C] bf16; out: [N,1+K] fp32
int launch_contrastive_fwd(void* stream, const void* q, const void* k,
                           const void* queue_kc, float* out, int64_t N,
                           int64_t C, int64_t K, float invT);
// g: [N,1+K] fp32; k: [N,C] bf16; queue_ck: [C,K] fp32; dq (pre-zeroed): [N,C] fp32
int launch_contrastive_bwd(void* stream, const float* g, const void* k,
                           const float* queue_ck, float* dq, int64_t N,
                           int64_t C, int64_t K, float invT);

// ---- softmax_ce.hip -------------------------------------------------------
// logits: [N, M] fp32
int launch_softmax_ce0_fwd(void* stream, const float* logits, float* loss_rows,
                           float* row_max, float* row_lse, int64_t N,
                           int64_t M);
int launch_softmax_ce0_bwd(void* stream, const float* logits,
                           const float* row_max, const float* row_lse,
                           float* dlogits, float scale, const float* gscale,
                           int64_t N, int64_t M);

// ---- queue.hip ------------------------------------------------------------
// queue: [C,K] fp32; queue_kc: [K,C] bf16 (nullable); keys: [B,C]
int launch_queue_enqueue(void* stream, float* queue, void* queue_kc,
                         const void* keys, bool keys_bf16, int64_t C,
                         int64_t K, int64_t B, int64_t ptr);
// graph-replay-safe variant: ring position read/advanced from ptr_dev
int launch_queue_enqueue_dev(void* stream, float* queue, void* queue_kc,
                             const void* keys, bool keys_bf16, int64_t C,
                             int64_t K, int64_t B, int64_t* ptr_dev);

// ---- multi_tensor.hip -----------------------------------------------------
int launch_multi_tensor_ema(void* stream, const int64_t* ptrs_dst,
                            const int64_t* ptrs_src, const int32_t* sizes,
                            int64_t nchunks, float m);
int launch_multi_tensor_sgd(void* stream, const int64_t* ptrs_p,
                            const int64_t* ptrs_g, const int64_t* ptrs_b,
                            const int32_t* sizes, int64_t nchunks, float lr,
                            float momentum, float wd);
int launch_ema_flat(void* stream, float* dst, const float* src, int64_t n,
                    float m);

// ---- adamw.hip ------------------------------------------------------------
// A table of up to ADAMW_TENSORS tensors of one dtype, passed by value in
// the kernel's arguments (which hold 4 KB).  Tensor i is at p (weights), g
// (gradients), m and v (moments, fp32 or 8-bit codes) and s (fp32 pairs of
// scales, one per 256 elements; 8-bit only).  It takes the chunks of
// ADAMW_CHUNK elements from first[i] on, of which the last has tail[i]; its
// number in the caller's list is list_base + number[i].  dtype: 0 fp32,
// 1 bf16, 2 fp16.
#define ADAMW_TENSORS 82
#define ADAMW_CHUNK 4096
struct AdamwTable {
  void* p[ADAMW_TENSORS];
  const void* g[ADAMW_TENSORS];
  void* m[ADAMW_TENSORS];
  void* v[ADAMW_TENSORS];
  void* s[ADAMW_TENSORS];
  uint32_t first[ADAMW_TENSORS];
  uint16_t tail[ADAMW_TENSORS];
  uint16_t number[ADAMW_TENSORS];
  uint32_t list_base, chunks;
  int count;
};
// the same for gradients alone
#define GRAD_TENSORS 256
struct GradTable {
  const void* g[GRAD_TENSORS];
  uint32_t first[GRAD_TENSORS];
  uint16_t tail[GRAD_TENSORS];
  uint32_t chunks;
  int count;
};
struct AdamwScalars {
  float beta1, one_minus_beta1, beta2, one_minus_beta2;
  float inv_root_bc2, eps, decay, step_size, max_norm;
};
// norm: device fp32 scalar for the clip, or null for none; once: the data go
// past the caches
int launch_adamw(void* stream, const AdamwTable* tab, const AdamwScalars* h,
                 const float* norm, int dtype, bool once);
int launch_adamw8(void* stream, const AdamwTable* tab, const AdamwScalars* h,
                  const float* norm, int dtype, bool once, uint32_t seed);
// decoded moments of the codes m, v, s into p (m) and g (v), of type dtype
int launch_adamw8_values(void* stream, const AdamwTable* tab, int dtype);
// partial[blocks]: sums of squares of the table's g
int launch_sumsq(void* stream, const GradTable* tab, int dtype,
                 double* partial, int blocks, bool once);
// out = 2-norm of the table's g, of NORM_SMALL_CHUNKS chunks at most
#define NORM_SMALL_CHUNKS 32
int launch_norm_small(void* stream, const GradTable* tab, int dtype,
                      float* out);
// out = sqrt(sum of partial[0..n))
int launch_norm_final(void* stream, const double* partial, int n, float* out);

// ---- norm_residual.hip ----------------------------------------------------
// x, r: [rows, width] of type_x; h, gate, y: of type_h (0 fp32, 1 bf16,
// 2 fp16; type_x is fp32 or type_h).  ld_*: elements from row to row of the
// inputs; outputs are contiguous.  w1, b1, scale, w2, b2: [width], null for
// none; bit j of f32: the j-th of (w1, b1, w2, b2, scale) is fp32, else
// type_h.  stats: fp32 [4, rows] (mean and 1/std after, then before), null
// where no backward follows.
enum { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
enum { NORM_GATE_NONE = 0, NORM_GATE_FULL = 1, NORM_GATE_ROW = 2 };
enum { NORM_ACT_NONE = 0, NORM_ACT_SIGMOID = 1, NORM_ACT_SILU = 2 };
#define NORM_MAX_WIDTH 16384
struct NormArgs {
  const void *x, *h, *gate, *w1, *b1, *w2, *b2, *scale;
  void *r, *y;
  float* stats;
  int64_t rows, ld_x, ld_h, ld_g;
  int width, type_x, type_h, post, pre, gate_kind, act, f32;
  float scale_value, post_eps, pre_eps;
};
// d_r, d_y: contiguous, null where an output has no gradient; d_x, d_h,
// d_gate and the vectors' (of their vector's type): null where none is
// wanted; partial[j]: fp32 [blocks, width] for column sum j (0 and 1 for d_w1,
// d_b1, d_scale; 2 for d_w2; 3 for d_b2), null where it is not needed
struct NormGrads {
  const void *d_r, *d_y;
  void *d_x, *d_h, *d_gate, *d_w1, *d_b1, *d_w2, *d_b2, *d_scale;
  float* partial[4];
};
int launch_norm_fwd(void* stream, const NormArgs* a);
int norm_bwd_blocks(const NormArgs* a);
int launch_norm_bwd(void* stream, const NormArgs* a, const NormGrads* o,
                    int blocks);
int launch_norm_columns(void* stream, const NormArgs* a, const NormGrads* o,
                        int blocks);

// ---- bn.hip ---------------------------------------------------------------
// x/y/g/res: [R, C] bf16 (NHWC flattened); stats fp32; C in {64..256 dividing
// 256, or multiples of 256 up to 2048}; part_* workspaces are [304, C] fp32.
int launch_bn_stats(void* stream, const void* x, float* part_s, float* part_q,
                    float* mean, float* rstd, float* running_mean,
                    float* running_var, int64_t R, int64_t C, float eps,
                    float momentum);
int launch_bn_apply(void* stream, const void* x, const void* res, void* y,
                    const float* mean, const float* rstd, const float* gamma,
                    const float* beta, int64_t R, int64_t C, bool relu);
int launch_bn_bwd_reduce(void* stream, const void* g, const void* y,
                         const void* x, const float* mean, const float* rstd,
                         float* part_db, float* part_dg, float* dbeta,
                         float* dgamma, int64_t R, int64_t C, bool relu);
int launch_bn_bwd_dx(void* stream, const void* g, const void* y,
                     const void* x, const float* mean, const float* rstd,
                     const float* gamma, const float* dbeta,
                     const float* dgamma, void* dx, void* dres, int64_t R,
                     int64_t C, bool relu, bool train);
// finalize mean/rstd (+ running stats) from the [P, C] slot-striped
// (sum, sumsq) partials produced by the conv-GEMM stats epilogue
int launch_bn_finalize(void* stream, const float* ssum, const float* ssq,
                       float* mean, float* rstd, float* running_mean,
                       float* running_var, int64_t R, int64_t C, int64_t P,
                       float eps, float momentum, bool zero_src);
// reduce two [P, C] slot slabs to [C] totals, re-zeroing the slabs
int launch_slot_reduce2(void* stream, float* s1, float* s2, float* o1,
                        float* o2, int64_t C, int64_t P);

// ---- augment.hip ----------------------------------------------------------
// src: [B,3,H,W] fp32; params: [M,12] fp32; out: [M,3,S,S] (bf16 or fp32,
// NCHW or NHWC per flags); tmp1/tmp2: [M,3,S,S] fp32 workspaces;
// graypart: [M, ceil(S*S / 256)] fp32
int launch_two_crop_augment(void* stream, const void* src, bool src_u8,
                            const float* params, void* out, float* tmp1,
                            float* tmp2, float* graypart, int64_t B, int64_t M,
                            int64_t H, int64_t W, int64_t S, bool out_bf16,
                            bool channels_last);

}  // extern "C"

// ---- pool.hip -------------------------------------------------------------
#ifdef __cplusplus
extern "C" {
#endif
// 3x3 stride-2 pad-1 max pool, NHWC bf16; idx: per-output uint8 tap id [0,9)
int launch_maxpool_fwd(void* stream, const void* x, void* y, void* idx,
                       int64_t N, int64_t C, int64_t H, int64_t W, int64_t Ho,
                       int64_t Wo);
int launch_maxpool_bwd(void* stream, const void* g, const void* idx, void* dx,
                       int64_t N, int64_t C, int64_t H, int64_t W, int64_t Ho,
                       int64_t Wo);
#ifdef __cplusplus
}
#endif

// ---- conv1x1.hip ----------------------------------------------------------
#ifdef __cplusplus
extern "C"
#endif
// C[M,N] = A[M,K] @ Bt[N,K]^T, bf16 in/out, fp32 accumulate (1x1-conv GEMM)
int launch_gemm_nt_bf16(void* stream, const void* A, const void* Bt, void* C,
                        int64_t M, int64_t N, int64_t K);
#ifdef __cplusplus
extern "C"
#endif
// c_add (nullable): epilogue C += c_add (requires the LDS-conforming shape)
int launch_gemm_nt_lds_bf16(void* stream, const void* A, const void* Bt,
                            void* C, int64_t M, int64_t N, int64_t K,
                            const void* c_add);
#ifdef __cplusplus
extern "C"
#endif
// a_out (nullable, needs a_scale): materialized transformed A operand [M,K]
int launch_gemm_nt_fused_bf16(void* stream, const void* A, const void* Bt,
                              void* C, int64_t M, int64_t N, int64_t K,
                              const float* a_scale, const float* a_shift,
                              bool a_relu, float* stats_sum,
                              float* stats_sumsq, void* a_out,
                              const void* c_add);
#ifdef __cplusplus
extern "C"
#endif
// 3x3 pad-1 conv (stride 1/2) as implicit MFMA GEMM (round-2 prototype).
// zero_page: [Ci + 8] bf16 — zeros, or the BN-apply neutral values.
int launch_conv3x3_fwd(void* stream, const void* x, const void* w,
                       const void* zero_page, void* out, int64_t N, int64_t H,
                       int64_t W, int64_t Ci, int64_t Co, int64_t stride,
                       const float* a_scale, const float* a_shift,
                       bool a_relu, float* stats_sum, float* stats_sumsq);
#ifdef __cplusplus
extern "C"
#endif
// strided 1x1 conv (downsample path), NHWC bf16 (round-2 prototype)
int launch_conv1x1_strided(void* stream, const void* x, const void* w,
                           void* out, int64_t N, int64_t H, int64_t W,
                           int64_t Ci, int64_t Co, int64_t stride);
#ifdef __cplusplus
extern "C"
#endif
// dgrad GEMM + fused BN-backward epilogue (round-2 prototype): C = relu-
// masked A@Bt^T, dbeta/dgamma partials accumulated (pre-zeroed, fp32).
int launch_gemm_nt_dgrad_epi(void* stream, const void* A, const void* Bt,
                             void* C, int64_t M, int64_t N, int64_t K,
                             const void* y, const void* z, const float* mean,
                             const float* rstd, float* dbeta, float* dgamma,
                             const void* c_add);

#ifdef __cplusplus
extern "C" {
#endif
// ---- weight mirrors (multi_tensor.hip) ------------------------------------
int launch_multi_cast_bf16(void* stream, const int64_t* src_ptrs,
                           const int64_t* dst_ptrs, const int32_t* sizes,
                           int64_t nchunks);
int launch_multi_transpose_bf16(void* stream, const int64_t* src_ptrs,
                                const int64_t* dst_ptrs, const int32_t* meta,
                                int64_t ntiles);
#ifdef __cplusplus
}
#endif

#ifdef __cplusplus
extern "C"
#endif
// fp8 e4m3 GEMM on the MX-scaled MFMA (per-tensor software scaling):
// C_bf16[M,N] = (A8[M,K] @ B8t[N,K]^T) * out_scale; optional bn-stats
// epilogue into [256, N] slot slabs.  M%128, N%64, K%128.
int launch_gemm_nt_fp8(void* stream, const void* A, const void* Bt, void* C,
                       int64_t M, int64_t N, int64_t K, float out_scale,
                       float* stats_sum, float* stats_sumsq);

#ifdef __cplusplus
extern "C" {
#endif
// head adaptive-avg-pool to 1x1, NHWC bf16
int launch_avgpool_fwd(void* stream, const void* x, void* y, int64_t N,
                       int64_t C, int64_t HW);
int launch_avgpool_bwd(void* stream, const void* g, void* dx, int64_t N,
                       int64_t C, int64_t HW);
#ifdef __cplusplus
}
#endif
