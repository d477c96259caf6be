// C ABI of libaeris_b200.so. Every function returns 0 on success and a negative code on a host-side argument or
// launch error. Kernels report device-side problems (bounded waits that ran out, failed bounds checks) through
// the `status` word, which the caller owns and reads after synchronising.
#pragma once
#include <stdint.h>
#ifdef __cplusplus
extern "C" {
#endif

int aeris_gemm_bf16(const void* A, const void* B, void* C, int M, int N, int K, int lda, int ldb, int ldc,
                    int a_mn, int b_mn, int epi, const void* resid, int ldr, const float* gate,
                    int rows_per_gate, void* aux, int ld_aux, int swiglu_f, int k_splits, int bn, int* status,
                    void* stream);

int aeris_gemm_bf16_2cta(const void* A, const void* B, void* C, int M, int N, int K, int lda, int ldb, int ldc,
                         int a_mn, int b_mn, int epi, const void* resid, int ldr, const float* gate,
                         int rows_per_gate, void* aux, int ld_aux, int swiglu_f, int k_splits, int* status,
                         void* stream);

// The one of the two that is the faster for the shape (see gemm2.cu). bn: tile width of the one-CTA kernel (0: from N);
// allow_2cta = 0: never the other, 2: the other wherever it takes the product. ld_gate: elements from one gate row to the
// next (a multiple of 4; N where they lie without gaps).
int aeris_gemm_auto(const void* A, const void* B, void* C, int M, int N, int K, int lda, int ldb, int ldc, int a_mn,
                    int b_mn, int epi, const void* resid, int ldr, const float* gate, int rows_per_gate, int ld_gate,
                    void* aux, int ld_aux, int swiglu_f, int k_splits, int bn, int allow_2cta, int* status, void* stream);

// 1 where aeris_gemm_auto takes the two-CTA kernel, else 0; the second for weight gradients that ask for slices
// (k_splits < 0) on a device of `sms` multiprocessors.
int aeris_gemm_takes_pairs(int M, int N, int K, int epi, int allow_2cta);
int aeris_wgrad_takes_pairs(int M, int N, int K, int k_splits, int sms);

int aeris_attn_fwd(const void* q, int ldq, int q_col0, const void* k, int ldk, int k_col0, const void* v, int ldv,
                   int v_col0, void* o, int ldo, float* lse, int n_win, int N, int H, int head_dim, float scale,
                   int* status, void* stream);

int aeris_attn_bwd(const void* qkv, int ldq, int q_col0, int k_col0, int v_col0, const void* o, const void* d_o,
                   int ldo, const float* lse, float* delta, void* dqkv, int ldg, int n_win, int N, int H,
                   int head_dim, float scale, int* status, void* stream);
// 1 where aeris_attn_bwd takes these extents on a device of `sms` multiprocessors, 0 where it returns -23.
int aeris_attn_bwd_countable(int n_win, int N, int H, int head_dim, int sms);

int aeris_gemm_scatter_heads(const void* A, const void* B, int M, int N, int K, int lda, int ldb, int b_mn,
                             const void* const* peers, int sp, int sp_rank, int n_local, int L, int sec_w, int* status,
                             void* stream);
// Variant of the attention forward kernel: poly = softmax arithmetic at head_dim 64 (-1 scalar; 0 two-wide; 2 two-wide
// with two of every eight score pairs on the polynomial exp2); p_in_tmem = probabilities kept in tensor memory as the
// A operand of P V. Returns non-zero for an unknown variant.
int aeris_attn_set_fwd_variant(int poly, int p_in_tmem);
// Checking build (-DAERIS_BOUNDS_CHECK) only: status word and source rows for the gathers launched next; returns 1 when
// the library validates gather codes, 0 when it was built without the checks.
int aeris_debug_set_gather_bounds(int* status, unsigned src_rows);
int aeris_attn_fwd_push(const void* qkv, int ld, int H_local, void* o, int ldo, float* lse, int n_win, int N,
                        int head_dim, float scale, const void* const* o_peers, int sp, int n_local, int push_ld,
                        int push_col0, int* status, void* stream);
int aeris_attn_bwd_push(const void* qkv, int ld, int H_local, const void* o, const void* d_o, int ldo, const float* lse,
                        float* delta, int n_win, int N, int head_dim, float scale, const void* const* dq_peers, int sp,
                        int n_local, int push_ld, int push_sec_w, int push_col0, int* status, void* stream);

// `w` is the bf16 norm weight, or null with the fp32 weight in `w_f32`; `h_lo` (optional) receives the bf16 rounding
// residual of `h`, so that h + h_lo carries the fp32 result (used by the fp32 output head).
int aeris_modnorm_fwd(const void* x, const void* gidx, const void* const* peer_ptrs, int n_peers, void* x_out,
                      const float* scale, const float* shift, const void* w, void* h, int rows, int D, int mode,
                      float eps, const float* w_f32, void* h_lo, void* stream);
// mod_stride: elements from one sample's scale (shift) to the next, a multiple of 4
int aeris_modnorm_fwd_batch(const void* x, const void* gidx, const void* const* peer_ptrs, int n_peers, void* x_out,
                            const float* scale, const float* shift, int mod_stride, const void* w, void* h, int batch,
                            int rows, int D, int mode, float eps, const float* w_f32, void* h_lo, void* stream);
int aeris_modnorm_bwd(const void* x, const void* dh, const void* dres, const float* scale, const float* shift,
                      const void* w, void* dx, float* dscale, float* dshift, float* dw, int rows, int D, int mode,
                      float eps, const float* w_f32, void* stream);
int aeris_modnorm_fwd_f32(const void* x, const float* scale, const float* shift, const float* w_f32, float* h, int batch,
                          int rows, int D, int mode, float eps, void* stream);
int aeris_modnorm_bwd_f32(const void* x, const float* dh, const float* scale, const float* shift, const float* w_f32,
                          void* dx, float* dscale, float* dshift, float* dw, float* sums, int sum_rows, int rows, int D,
                          int mode, float eps, void* stream);
int aeris_gather_rows(const void* gidx, const void* const* peer_ptrs, int n_peers, void* out, long long rows, int D,
                      void* stream);
int aeris_swiglu_fwd(const void* u, void* act, long long rows, int F, void* stream);
int aeris_swiglu_bwd(const void* u, const void* dact, void* du, long long rows, int F, void* stream);
int aeris_scale_rows(const void* W, const float* g, void* Wg, int R, int C, void* stream);
// In-place 2-D rotary embedding of the q and k sections of qkv [rows, 3 * heads * d] (bf16); cos / sin: [L, d / 2] fp32.
int aeris_rope_qk(void* qkv, const float* cos_t, const float* sin_t, long long rows, int L, int heads, int d, int inverse,
                  void* stream);
int aeris_gate_grad_finalize(float* G, const void* W, const float* g, float* dW, float* dg, int R, int C,
                             void* stream);
int aeris_gate_prepare(const void* W2, const float* g2, void* W2g, float* G2, int C2, const void* Wo, const float* go,
                       void* Wog, float* Go, int Co, int R, float* zero, int n_zero, void* stream);
int aeris_gate_finalize_pair(float* G2, const void* W2, const float* g2, float* dW2, float* dg2, int C2, float* Go,
                             const void* Wo, const float* go, float* dWo, float* dgo, int Co, int R, void* stream);
int aeris_sumsq(const float* x, long long n, double* out, void* stream);
int aeris_adamw(float* master, float* grad, float* m, float* v, void* wbf16, float* ema, const double* norm_sq,
                long long n, float lr, float beta1, float beta2, float eps, float weight_decay, int step,
                float grad_scale, float max_norm, float ema_beta, void* stream);

int aeris_signal_barrier(const void* const* flag_ptrs, int rank, int world, unsigned epoch, int* status,
                         double timeout_s, void* stream);
int aeris_wait_flag(const void* flag, unsigned expected, int* status, double timeout_s, void* stream);
int aeris_grad_reduce_scatter(const void* const* grad_ptrs, const void* mc_grad, int world, long long lo, long long n,
                              float scale, float* out, double* sumsq, void* stream);
int aeris_shard_adamw_allgather(float* master, const float* grad, float* m, float* v, float* ema,
                                const void* const* param_ptrs, void* mc_params, int world, long long lo, long long n,
                                const double* norm_sq, float lr, float beta1, float beta2, float eps,
                                float weight_decay, int step, float max_norm, float ema_beta, void* stream);

int aeris_gemm_allgather_a(void* A, const void* const* peers, const void* const* counter_peers, int world, int rank,
                           int rows_per_rank, unsigned call_index, const void* B, void* C, int N, int K, int ldb,
                           int ldc, int b_mn, int epi, const void* resid, int ldr, void* aux, int ld_aux, int swiglu_f,
                           int* status, void* stream);
int aeris_gemm_rs_push(const void* A, const void* B, int M, int N, int K, int lda, int ldb, int b_mn,
                       const void* const* peers, int world, int rank, int rows_per_rank, int ld_dst, int* status,
                       void* stream);
int aeris_rs_finalize(const void* slots, int world, long long rows, int D, const void* resid, const float* gate,
                      void* out, void* stream);

// Geometry of one rank's token stream and image block (see csrc/diffusion.cu).
typedef struct TokGeom {
  int B, nwy_loc, nwx_loc, ws_y, ws_x, n_local, sp_rank;
  int y0, x0, H, W;
  long long sample0;
} TokGeom;
int aeris_embed_pack(const float* x_img, const float* c_img, const float* cs, const TokGeom* g, int Cx, int Cc,
                     const float* ape_y, const float* ape_x, int ape_ch, unsigned long long seed, float sd, int noise,
                     void* out, int KP, long long row0, long long rows, void* stream);
int aeris_trigflow_loss(const float* pred, int ldp, const float* x_img, const float* cs, const TokGeom* g, int Cx,
                        unsigned long long seed, float sd, const float* w_var, const float* w_lat, float inv_rows,
                        float gscale, void* dpred, int ldd, double* loss, long long row0, long long rows, void* stream);
int aeris_sampler_update(float* x_out, const float* x_base, const float* pa, const float* pb, int ldp, float ca,
                         float cb, const TokGeom* g, int Cx, void* stream);
int aeris_noise_mix(float* x, float a, float b, unsigned long long seed, const TokGeom* g, int Cx, void* stream);
int aeris_affine_channels(float* out, const float* in, const float* a, const float* b, const float* add, long long n,
                          int C, void* stream);
int aeris_gemv_bias_act(const void* W, int flags, const void* bias, const void* x, float* y, int N, int K, int B, int act,
                        int silu_in, void* stream);
int aeris_modulation_mlp(const void* W1, int flags1, const void* b1, const void* x, float* y1, int N1, int K, const void* W2,
                         int flags2, const void* b2, float* y2, int N2, int B, void* stream);
// Gradients of aeris_gemv_bias_act without `act`; added to dW, db (may be null) and dx (may be null).
int aeris_gemv_bwd(const void* W, int flags, const void* x, const float* dy, float* dW, float* db, float* dx, int N, int K,
                   int B, int silu_in, void* stream);
int aeris_modulation_mlp_bwd(const void* W1, int flags1, const void* x, float* dW1, float* db1, float* dx, int N1, int K,
                             const void* W2, int flags2, const float* y1, const float* dy, float* dW2, float* db2,
                             float* dy1, int N2, int B, void* stream);
int aeris_noise_embedding(const float* t, void* out, int out_bf16, int B, int dim, double max_period, void* stream);
// The same of 1 to 64 levels that the host knows (no copy: they travel as kernel arguments).
int aeris_noise_embedding_of(const float* levels, void* out, int out_bf16, int n, int dim, double max_period, void* stream);
int aeris_pack_embed_weights(const float* W, const float* b, void* out, int D, int Cin, int KP, void* stream);
int aeris_fold_embed_grad(const float* G, float* dW, float* db, int D, int Cin, int KP, void* stream);
int aeris_pack_head_weights(const float* W, void* out, int C, int rows, int D, void* stream);
// Slices that k_splits <= 0 stands for: `tiles` output tiles over `units` CTAs or CTA pairs (see gemm.cu).
int aeris_choose_k_splits(int tiles, int kb_total, int units, int most, int want);
int aeris_gemm_split(const void* y, const void* w, float* C, int M, int D, int lo_row, int ldc, int* status, void* stream);

// One transformer block on one GPU (csrc/block.cu; mirrored in models/block.py). Every matrix is row-major without gaps.
typedef struct AerisBlock {
  int D, F, heads, head_dim, L, mode;
  int n_win, batch;                 // windows of one sample, samples
  int step, merged;                 // windows per chunk; merged: all samples are one chunk (forward)
  int slice_windows;                // weight gradients: slices of a quarter of that many windows' rows at most, if free
  int kept, two_cta, n_peers;       // kept: the internals are full-size buffers, not workspaces of one chunk
  float eps, scale;
  long long mod_vec, mod_sample;    // element strides of `mod`: between the six vectors, between samples
  const float* mod;                 // shift1, scale1, gate1, shift2, scale2, gate2
  const void *wn1, *wqkv, *wo, *wn2, *w1, *w2;
  const float *rope_cos, *rope_sin; // null: no rotary embedding
  void *x, *y;                      // block input (with `table`: receives the gathered rows) and output
  const unsigned* table;            // null, or gather codes of the rows of x
  const void* const* peers;
  void *h1, *qkv, *o, *lse, *x1, *h2, *act, *u;
  int* status;
  void* stream;
} AerisBlock;
typedef struct AerisBlockGrad {
  const void* dy;
  void *dx, *du, *dh, *dx1, *d_o, *dqkv, *w2g, *wog;
  float *delta, *G2, *Go, *dmod;    // dmod: [batch, 6 D], overwritten
  float *n1, *to_qkv, *wo, *n2, *w1, *w2;   // weight gradients, added to
} AerisBlockGrad;
// Both return the number of kernels launched, or a negative code: -1 where `step` is not positive, else that of the launch
// that failed less 1000 times its place.
int aeris_block_forward(const AerisBlock* b);
int aeris_block_backward(const AerisBlock* b, const AerisBlockGrad* g);
// aeris_block_forward of `n` records in a row, each with `mod + mod_offset` and on `stream`; same result codes.
int aeris_blocks_forward(const AerisBlock* blocks, int n, long long mod_offset, void* stream);


// Norms of queries and keys by head with the position rotation (csrc/qk_norm.cu; mirrored in ops/qk_norm.py). Strides in
// elements; a head's channels lie side by side.
typedef struct AerisHeads {
  const void* ptr;
  long long row, head;
} AerisHeads;
typedef struct AerisQkNorm {
  AerisHeads q, k, dq, dk, q_out, k_out;  // q_out, k_out: results (backward: gradients of q, k); may be the inputs themselves
  const void *wq, *wk;              // [d], bf16 or fp32
  const float *cos, *sin;           // [L, rot / 2], or null with rot = 0
  const void* pos;                  // table row of every row (int32 or int64), null: row mod L. Outside [0, L): recorded in
                                    // the status word, the row's results are not written
  float *dwq, *dwk, *sums;          // backward: [d] each; scratch [sum_rows, d]
  int* status;
  long long rows;
  int L, heads, kv_heads, d, rot, f32, w_bf16, pos64, add_dw, sum_rows;   // add_dw: dwq, dwk are added to
  float eps;
} AerisQkNorm;
int aeris_qk_norm_fwd(const AerisQkNorm* a, void* stream);
int aeris_qk_norm_bwd(const AerisQkNorm* a, void* stream);      // returns the number of kernels launched, or a negative code

// Orthogonalisation of matrices (csrc/orthogonalise.cu; mirrored in ops/orthogonalise.py): a batch of up to ORTHO_GROUPS groups
// whose matrices have one shorter side and at most two different longer ones. Matrix i of a group has rows x cols elements
// with row pitch ld and lies at element offsets[i] (device memory, int64, ascending, no two overlapping, inside [0, numel):
// else the status word is set and the matrix left out) or, with offsets null, at i * stride.
#define ORTHO_GROUPS 4
typedef struct AerisOrthoGroup {
  const void* offsets;
  long long stride, out_stride;     // out_stride, ld_out: where the results of `out` lie
  int rows, cols, ld, ld_out, count, behind;    // behind: offsets[-1] is the matrix before the first one
  float rate;                       // master * decay - rate * result
} AerisOrthoGroup;
typedef struct AerisOrtho {
  AerisOrthoGroup group[ORTHO_GROUPS];
  const void* x;                    // a tensor, fp32 or bf16, and its bf16 results
  void* out;
  float *grad, *momentum, *master, *ema;        // or flat buffers of an optimizer (x and out null); ema may be null
  void* weights;                    // bf16, may be null
  const double* norm_sq;            // as aeris_adamw
  void* work;                       // workspace from a 1024-byte boundary on
  int* status;
  double eps;
  long long numel, work_bytes;
  int groups, steps, bf16, nesterov, zero_grad; // 1 to 20 steps
  float beta, grad_scale, max_norm, decay, ema_beta;
} AerisOrtho;
// How a batch goes on this device, by its groups and steps, or a negative code: everything in one launch, all steps on the Gram
// matrix, or launch by launch with these, where "pairs" are products by CTA pairs.
enum {
  ORTHO_ROUTE_ONE_LAUNCH = 1, ORTHO_ROUTE_GRAM_ALONE = 2, ORTHO_ROUTE_TWO_STEPS = 4, ORTHO_ROUTE_GRAM_PARTS = 8,
  ORTHO_ROUTE_GRAM_PAIRS = 16, ORTHO_ROUTE_FACTOR_PAIRS = 32, ORTHO_ROUTE_UPDATE_PAIRS = 64
};
int aeris_ortho_route(const AerisOrtho* a);
long long aeris_ortho_work_bytes(const AerisOrtho* a);          // of its groups and steps, or a negative code
int aeris_orthogonalise(const AerisOrtho* a, void* stream);     // the number of kernels launched, or a negative code

// Layer norm (csrc/layer_norm.cu; mirrored in ops/layer_norm.py). Pitches in elements; columns lie side by side. Forward: y and
// stats (mean, 1 / sqrt(var + eps)) of x. Backward: y receives the gradient of x, dw and db the column sums, each where it is
// given. y may be x or dy itself.
typedef struct AerisLayerNorm {
  const void *x, *dy;
  void* y;
  const void *w, *b;                // [cols], bf16 or fp32 both; null: ones, zeros
  float *stats;                     // [rows, 2], from an 8-byte boundary on
  float *dw, *db, *work;            // [cols] each, null: not wanted; work: [slices, 2, cols], null where slices are one at most
  int* status;
  long long rows, ld_x, ld_dy, ld_y;
  int cols, f32, w_f32, add, slices;            // f32: type of x, dy, y; add: both of dw, db that are given are added to
  float eps;
} AerisLayerNorm;
// Both return the number of kernels launched, or a negative code.
int aeris_layer_norm_fwd(const AerisLayerNorm* a, void* stream);
int aeris_layer_norm_bwd(const AerisLayerNorm* a, void* stream);

// Linear layer (csrc/linear.cu; mirrored in ops/linear.py): y = resid + act(x w^T + bias) with x [rows, inner], w [cols, inner],
// bf16. Pitches in elements; rows may start anywhere.
enum { LIN_ACT_NONE = 0, LIN_ACT_RELU = 1, LIN_ACT_SILU = 2, LIN_ACT_GELU = 3, LIN_ACT_GELU_TANH = 4 };
typedef struct AerisLinear {
  const void *x, *w, *bias;         // bias [cols], fp32 or bf16, or null
  const void* resid;                // [rows, cols] or null
  void *y, *z;                      // z: null, or receives x w^T + bias
  void* work;                       // aeris_linear_fwd_bytes (may be none), from a 256-byte boundary on
  int* status;
  long long ld_x, ld_w, ld_resid, ld_y, ld_z, work_bytes;
  int rows, inner, cols, act, bias_bf16;
} AerisLinear;
// dz = dy act'(z), db = its column sums, dx = dz w, dw = dz^T x, each where its result is given. dw: bf16, or fp32 that is added to
// (dw_f32); db: fp32, added to with `add_db`.
typedef struct AerisLinearGrad {
  const void *dy, *x, *w, *z;       // z: null where act is LIN_ACT_NONE
  void *dx, *dw;
  float* db;
  void* work;                       // aeris_linear_bwd_bytes, from a 256-byte boundary on
  int* status;
  long long ld_dy, ld_x, ld_w, ld_z, ld_dx, ld_dw, work_bytes;
  int rows, inner, cols, act, dw_f32, add_db;
} AerisLinearGrad;
// Bytes of the workspace: copies of operands whose rows do not start on 16-byte boundaries (pad_*), dz (own_dz: with an activation,
// or for a dy of such rows), sums of slices of the rows.
long long aeris_linear_fwd_bytes(int rows, int inner, int cols, int pad_x, int pad_w);
long long aeris_linear_bwd_bytes(int rows, int inner, int cols, int own_dz, int pad_x, int pad_w, int dx, int dw, int db, int dw_f32);
// Both return the number of kernels launched, or a negative code.
int aeris_linear_fwd(const AerisLinear* a, void* stream);
int aeris_linear_bwd(const AerisLinearGrad* a, void* stream);

// Window attention with a learned bias by relative position (csrc/position_bias.cu; mirrored in ops/position_bias.py). Windows of
// high x wide tokens in rows; the relative position of query i and key j is (y_i - y_j + high - 1) (2 wide - 1) + x_i - x_j + wide - 1,
// its bucket buckets[that] (null: itself), its bias table[bucket, head]. Entries of -1e30 and less hide the pairs of their bucket.
typedef struct AerisBiasedAttn {
  const void* qkv;                  // [n_win * high * wide, 3 * heads * head_dim] bf16, (q|k|v, head, channel)
  void* o;                          // [n_win * high * wide, heads * head_dim]
  float* lse;                       // [n_win, heads, high * wide], log2; +infinity where a query sees nothing
  const void *table, *buckets;      // [table_rows, heads] fp32 or bf16; int32 or int64, outside [0, table_rows): recorded in the
                                    // status word, the pairs hidden
  const void* d_o;                  // backward: pitch of o
  void* dqkv;
  float* dtable;                    // [table_rows, heads], added to with `add`; null: not wanted
  void* work;                       // aeris_biased_attn_work_bytes (may be none), from a 256-byte boundary on
  int* status;
  long long ld_qkv, ld_o, ld_dqkv, work_bytes;
  int n_win, high, wide, heads, head_dim, table_rows, table_bf16, buckets64, add;
  float scale;
} AerisBiasedAttn;
long long aeris_biased_attn_work_bytes(int n_win, int high, int wide, int heads, int head_dim, int backward, int with_table);
// Both return the number of kernels launched, or a negative code.
int aeris_biased_attn_fwd(const AerisBiasedAttn* a, void* stream);
int aeris_biased_attn_bwd(const AerisBiasedAttn* a, void* stream);

#ifdef __cplusplus
}
#endif
