/*
 * h3b.h -- C ABI of libh3b.so, the B200-native (sm_100a) W4A8 ConvRot quantised linear.
 *
 * Every pointer argument is a device pointer unless the name ends in `_host`.  The caller owns every buffer, including
 * outputs and scratch ("workspace"): no entry point allocates device memory.  Work is enqueued on `stream` (a
 * cudaStream_t; NULL means the legacy default stream) and the call returns without synchronising.  Weight tensors may be
 * views into a larger byte buffer (256-byte aligned rows are enough).
 *
 * Return value: H3B_OK (0) or a positive H3B_ERR_* code; h3b_last_error() then returns a message (thread-local, valid
 * until the next call on the same thread).  H3B_ERR_ARG means the arguments are invalid (the Python layer raises
 * ValueError); every other code is a device or build failure (RuntimeError).
 *
 * Numerics (all entry points): identical to the reference's "ck" profile of h3turbo/h3/qlinear.py.  The int4->int8 decode,
 * the int32 accumulation and every epilogue rounding are bit-exact; the only float step that is not the reference's
 * correctly rounded fp64 computation is the ConvRot rotation, done as an fp32 fast Walsh-Hadamard transform.
 *
 * Reference interfaces named below are file:line in the reference project (Alexpoopy1/MiniMax-H3-Turbo).
 */
#ifndef H3B_H
#define H3B_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define H3B_ABI_VERSION 1

enum h3b_status {
  H3B_OK = 0,
  H3B_ERR_ARG = 1,          /* invalid argument (shape, dtype, size, alignment) */
  H3B_ERR_CUDA = 2,         /* a CUDA runtime call failed */
  H3B_ERR_UNSUPPORTED = 3,  /* valid for the reference, not supported by this build (e.g. convrot 1024) */
  H3B_ERR_DEVICE = 4        /* a kernel reported a failure (a bounded wait timed out); see h3b_device_error */
};

enum h3b_dtype {
  H3B_BF16 = 0,
  H3B_FP16 = 1,
  H3B_FP32 = 2,
  H3B_FP8_E4M3 = 3, /* float8_e4m3fn group scales (raw bytes) */
  H3B_INT32 = 4,    /* int32 accumulator output (parity dump); int32 positions */
  H3B_INT64 = 5     /* int64 positions */
};

enum h3b_quant_mode {
  H3B_QMODE_CK = 0,    /* absmax of the unrounded rotation; epilogue (acc * xs) * s_ch   (qlinear.py:278-283, :400-401) */
  H3B_QMODE_EAGER = 1  /* absmax of the dtype-rounded rotation; epilogue acc * (xs * s_ch) (qlinear.py:284-287, :402-403) */
};

/* ABI version (H3B_ABI_VERSION) and the last error message of this thread. */
int h3b_version(void);
const char* h3b_last_error(void);

/* Rotate + per-token int8 quantisation of activations (kernel KA).
 * Replaces quantize_activation / _quantize_rows (qlinear.py:267-303), the activation half of comfy_kitchen's fused
 * w4a8_int8_linear reached through _run_ck (qlinear.py:427-429).
 *   x      [M, ldx] of x_dtype (bf16/fp16/fp32); the row holds K features, or [gate | up] (2K) when swiglu != 0
 *          (input_act="swiglu", qlinear.py:376-379: silu(gate) * up in x_dtype, applied before the rotation).
 *   convrot 4, 16, 64 or 256 (the ConvRot block; K % convrot == 0).
 *   q      [M, ldq] int8 codes out; xs [M] fp32 per-row scales out. */
int h3b_rotq(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int convrot, int swiglu, int quant_mode,
             int8_t* q, int64_t ldq, float* xs, void* stream);

/* Block rotation only: y = per-convrot-block x @ H in y_dtype (one rounding of the fp32 transform).
 * Replaces rotate (qlinear.py:118-132). */
int h3b_rotate(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int convrot, void* y, int y_dtype,
               int64_t ldy, void* stream);

/* Per-head RMSNorm + split-half rotary embedding of q and k, in place (both, or one of them with the other NULL).
 * Replaces comfy_kitchen's rms_rope_split_half_ (called at layout.py:343) with the bit-exact semantics of the
 * reference's "torch" form of that kernel, norm_rope_ (layout.py:329-356) with rms_norm_fused_order (layout.py:309-326).
 *   q, k      [S, heads, head_dim] of x_dtype (bf16 or fp16), heads contiguous, token strides ldq / ldk (elements);
 *             head_dim 32, 64, 128 or 256
 *   wq, wk    [head_dim] of w_dtype;  eps as the fp32 value of the model's qk_norm_eps
 *   cos, sin  [S, half] of t_dtype, rows ldt elements apart; channel j < half pairs with j + half; 2 * half <= head_dim */
int h3b_qk_norm_rope(void* q, int64_t ldq, void* k, int64_t ldk, int x_dtype, int64_t S, int heads, int head_dim,
                     const void* wq, const void* wk, int w_dtype, float eps, const void* cos_t, const void* sin_t,
                     int64_t ldt, int t_dtype, int half, void* stream);

/* RMSNorm + AdaLN modulation of the residual stream: h = scale_shift(rms(x)).  Replaces _rms followed by _scale_shift_
 * (model.py:64-66, 106-109): n = dt((x * rsqrt(mean(x^2) + eps)) * w), then for a token with modulation row `row`
 * h = dt(dt(n * dt(1 + dt(scale[row]))) + dt(shift[row])); tokens without a row keep n.  The row sum's order is this
 * kernel's own (torch's F.rms_norm reduces in another order: rare one-ulp differences of n).
 *   x, h          [M, hidden] of x_dtype (bf16 or fp16), rows ldx / ldh elements apart; hidden a multiple of 8
 *   w             [hidden] of w_dtype;  shift, scale: [n_rows, hidden] of m_dtype, rows ldm elements apart
 *   segments      HOST table of n_segments <= H3B_MAX_SEGMENTS x (first token, end token, row), int32
 *   token_rows    optional DEVICE int32 [M] row per token (negative: none, else < n_rows, which the caller guarantees);
 *                 used instead of the segments when given
 *   every device pointer 16-byte aligned */
#define H3B_MAX_SEGMENTS 16
int h3b_rms_modulate(const void* x, int x_dtype, int64_t ldx, int64_t M, int hidden, const void* w, int w_dtype,
                     float eps, const void* shift, const void* scale, int64_t ldm, int64_t n_rows, int m_dtype,
                     const int32_t* segments, int n_segments, const int32_t* token_rows, void* h, int64_t ldh,
                     void* stream);

/* RMSNorm + AdaLN modulation fused into the rotate+quantise kernel: the codes and scales of h = _scale_shift_(_rms(x))
 * (model.py:64-66, 106-109, 239-241) without writing h; the activation side of the qkv and fc1 linears of a block.
 * Bit-identical to h3b_rms_modulate (bf16) followed by h3b_rotq on its output.  Every tensor bf16:
 *   x          [M, K], rows ldx elements apart; K a multiple of 256, at most 6144; convrot 256
 *   w          [K] norm weight (the reference rounds it to x's dtype first)
 *   shift      [n_rows, K] dt(shift);  scale1: [n_rows, K] dt(1 + dt(scale)), the factor _scale_shift_ multiplies by;
 *              rows ldm elements apart
 *   segments / token_rows as h3b_rms_modulate;  q [M, ldq] int8 codes, xs [M] fp32 scales as h3b_rotq
 *   every device pointer 16-byte aligned */
int h3b_rotq_rms_modulate(const void* x, int64_t M, int64_t K, int64_t ldx, const void* w, float eps, const void* shift,
                          const void* scale1, int64_t ldm, int64_t n_rows, const int32_t* segments, int n_segments,
                          const int32_t* token_rows, int convrot, int quant_mode, int8_t* q, int64_t ldq, float* xs,
                          void* stream);

/* Gated residual update, in place: x = dt(x + other * dt(gate[row])) for tokens with a modulation row, others
 * unchanged.  Replaces _gate_ (model.py:111-115; torch's addcmul_, bit-identical).  Arguments as h3b_rms_modulate;
 * other: [M, hidden] of x_dtype, rows ldo elements apart. */
int h3b_gate_residual(void* x, int x_dtype, int64_t ldx, const void* other, int64_t ldo, int64_t M, int hidden,
                      const void* gate, int64_t ldm, int64_t n_rows, int m_dtype, const int32_t* segments, int n_segments,
                      const int32_t* token_rows, void* stream);

/* Merge softmax attention computed over disjoint key sets (no reference counterpart: the ring key/value exchange of
 * the token-sharded DiT block, whose single-GPU form is one attention call, model.py:196-228).  For every head h and
 * query q: L' = log(exp(L) + exp(l)), A = A exp(L - L') + fp32(o) exp(l - L'), L = L'.
 *   acc    fp32 [heads, queries, head_dim] running output;  acc_lse fp32 [heads, queries] running log-sum-exp
 *   o      attention output over the next key set, element (h, q, d) at o + h*o_head_stride + q*o_query_stride + d;
 *          o_dtype must be H3B_BF16 (anything else is refused with H3B_ERR_ARG)
 *   lse    fp32 [heads, queries] its log-sum-exp (natural log);  first != 0: (acc, acc_lse) = (o, lse)
 *          a query with no keys on either side (both log-sum-exps -inf) gets a zero output
 *   out    optional bf16 [queries, heads * head_dim] (row stride ldo): the merged result, written instead of acc */
int h3b_attn_merge(float* acc, float* acc_lse, const void* o, int64_t o_head_stride, int64_t o_query_stride, int o_dtype,
                   const float* lse, int64_t heads, int64_t queries, int head_dim, int first, void* out, int64_t ldo,
                   void* stream);

/* Rotary embedding of q and k from positions on several axes (time, height, width), out of place (no reference
 * counterpart as one operator: rope_angles and the rotation of norm_rope_, layout.py:265-273, 348-355, without the norm
 * and without cos / sin tables).
 *   theta[b, s, j] = pos[b, s, axis(j)] * inv_freq[j],  j < F = sum(sections), axis(j) the section that holds j
 *   pair j: channels (j, j + F) H3B_PAIR_HALF, (2 j, 2 j + 1) H3B_PAIR_ADJACENT; channels >= 2 F are copied
 *   (a, b) -> (a cos - b sin, a sin + b cos) in fp32, one rounding;  inverse != 0: by -theta (the gradient's direction)
 *   q, k       one of them may be null; S tokens (0 is valid) of `heads` heads, strides in elements, channels contiguous;
 *              any stride (16-byte aligned rows are faster); pointers aligned to their elements; y must not overlap x or itself
 *   pos        [B, S, n_axes] of pos_dtype (fp32, int32, int64), axes contiguous, strides in elements (0: shared)
 *              (angles are exact to fp32 up to |theta| = 2^28 and to 4 * 2^-53 |theta| beyond)
 *   inv_freq   DEVICE fp32 [F];  sections: HOST int32 [n_axes], n_axes <= H3B_MAX_AXES, 2 F <= head_dim <= 1024 */
#define H3B_MAX_AXES 8
enum h3b_rope_pairing { H3B_PAIR_HALF = 0, H3B_PAIR_ADJACENT = 1 };
typedef struct h3b_rope_operand {
  const void* x;
  void* y;
  const void* pos;
  int64_t S, x_stride_b, x_stride_s, x_stride_h, y_stride_b, y_stride_s, y_stride_h, pos_stride_b, pos_stride_s;
  int64_t heads;
} h3b_rope_operand;
int h3b_rope_axes(const h3b_rope_operand* q, const h3b_rope_operand* k, int x_dtype, int64_t B, int head_dim,
                  const float* inv_freq, const int32_t* sections, int n_axes, int pos_dtype, int pairing, int inverse,
                  void* stream);

/* Cross attention: softmax attention of q over another stream's k and v (no reference counterpart: the reference's
 * attention is one stream's own, model.py:196-228).  s_ij = scale q_i . k_j + bias_j,  o_i = sum_j softmax_j(s_ij) v_j.
 *   q, o       [B, Sq, Hq, head_dim];  k, v: [B, Sk, Hkv, head_dim] of dtype (bf16 or fp16); Hq a multiple of Hkv (query
 *              head h reads key head h / (Hq / Hkv)); strides in elements, multiples of 8 and at least 8 (0, a tensor shared
 *              along an axis, is refused), those of o at least head_dim; those of extents of one are not looked at; channels
 *              contiguous, every tensor 16-byte aligned; o must not overlap k or v; head_dim a multiple of 8, at most 128;
 *              scale > 0
 *   kv_lens    optional DEVICE int32 [B]: only keys j < kv_lens[b] take part
 *   mask       optional DEVICE key mask, rows ldm elements apart (0: shared): H3B_MASK_BOOL uint8 [B, Sk], 0 leaves the
 *              key out; H3B_MASK_BIAS fp32 [B, Sk] added to the scaled scores, -inf leaves the key out
 *   lse        optional fp32 [B, Hq, Sq]: natural log of sum_j exp(s_ij - t), t = 0, or with H3B_MASK_BIAS the largest bias in
 *              use of the batch entry (a mask of large negative values keeps the scores' digits so, here and in the gradients,
 *              which take this lse).  To merge results over disjoint key sets by their log-sum-exps, add t
 *   kv_lens, an additive mask and lse are 4-byte aligned
 * A query without keys (Sk = 0, kv_lens 0, all masked) gets o = 0 and lse = -inf.  What keys that are left out hold (NaN
 * and infinities too) never reaches a result.  Products take operands of dtype and add up in fp32; softmax and sums are
 * fp32; the probabilities are rounded to dtype for the second product.
 * workspace >= h3b_cross_attention_workspace_bytes(..., backward = 0), 256-byte aligned (may be null when that is 0). */
enum h3b_mask_kind { H3B_MASK_NONE = 0, H3B_MASK_BOOL = 1, H3B_MASK_BIAS = 2 };
typedef struct h3b_attn_tensor {
  void* ptr;
  int64_t stride_b, stride_s, stride_h;
} h3b_attn_tensor;
/* 0 where none is needed, and for sizes that the calls refuse (h3b_last_error says why). */
size_t h3b_cross_attention_workspace_bytes(int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int head_dim, int mask_kind,
                                           int backward);
int h3b_cross_attention(const h3b_attn_tensor* q, const h3b_attn_tensor* k, const h3b_attn_tensor* v,
                        const h3b_attn_tensor* o, int dtype, int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv,
                        int head_dim, float scale, const int32_t* kv_lens, const void* mask, int mask_kind, int64_t ldm,
                        float* lse, void* workspace, size_t ws_bytes, void* stream);

/* Gradients of h3b_cross_attention's o with respect to q, k and v; o and lse are the forward's, the other arguments the
 * same.  grad_o, dq: as q; dk, dv: as k.  Shared heads add up; keys that are left out get zero gradients.  Every sum has a
 * fixed order (no atomics): the same call gives the same bits.  The mask has no gradient.
 * P and its gradient are rounded to dtype for the second products, in fp16 after scaling by powers of two into its range, so
 * that gradients of any size keep 11 bits.
 * workspace >= h3b_cross_attention_workspace_bytes(..., backward = 1). */
int h3b_cross_attention_backward(const h3b_attn_tensor* grad_o, const h3b_attn_tensor* q, const h3b_attn_tensor* k,
                                 const h3b_attn_tensor* v, const h3b_attn_tensor* o, const float* lse,
                                 const h3b_attn_tensor* dq, const h3b_attn_tensor* dk, const h3b_attn_tensor* dv, int dtype,
                                 int64_t B, int64_t Sq, int64_t Sk, int Hq, int Hkv, int head_dim, float scale,
                                 const int32_t* kv_lens, const void* mask, int mask_kind, int64_t ldm, void* workspace,
                                 size_t ws_bytes, void* stream);

/* ---- the residual's addition with its root-mean-square norm and 8-bit output (no reference counterpart as one operator: _gate_,
 * _rms, _scale_shift_ and the activation half of the W4A8 linear, model.py:64-66, 106-115, 239-241, qlinear.py:267-303, whose
 * intermediate roundings this one leaves out):
 *   t = dt(x + gate y);  r = rsqrt(mean t^2 + eps);  h = t r w (1 + scale) + shift in fp32, rounded once where it is written
 *   z = h rotated by blocks of 256 as the W4A8 linears take it;  scales = max|z| / 127;  codes = rint(z / scales)
 *   x, y, t, h   [M, K] rows of dtype (bf16 or fp16), K a multiple of 8 (of 256 with codes), at most H3B_MAX_RESIDUAL; t may be x
 *                or y, h may not be any of them
 *   w            [K] of w_dtype;  gate, shift, scale: [n_rows, K] of m_dtype, rows ldm apart, each row of a token's segment.
 *                gate NULL: 1 for every row; shift and scale NULL (together): none
 *   segments / token_rows as h3b_rms_modulate (numbers outside 0 .. n_rows - 1: none): a row outside every segment keeps t = x
 *                (where there is a gate) and h = t r w
 *   h, codes (with scales [M]) and rstd [M] (the gradients take it) may each be NULL: not written
 *   A row whose h has a NaN or an infinity gets codes 0 and a scale that is NaN or infinite; a row of zeros scale 0. */
#define H3B_MAX_RESIDUAL 16384
size_t h3b_residual_norm_workspace_bytes(int64_t M, int64_t K, int backward);
int h3b_residual_norm(const void* x, int64_t ldx, const void* y, int64_t ldy, int dtype, int64_t M, int64_t K, const void* w,
                      int w_dtype, float eps, const void* gate, const void* shift, const void* scale, int64_t ldm,
                      int64_t n_rows, int m_dtype, const int32_t* segments, int n_segments, const int32_t* token_rows, void* t,
                      int64_t ldt, void* h, int64_t ldh, int8_t* codes, int64_t ldc, float* scales, float* rstd,
                      void* workspace, size_t ws_bytes, void* stream);
/* Gradients with respect to x, y and w from those of t (grad_t, NULL: none) and h; t and rstd as h3b_residual_norm wrote them, the
 * other arguments the same.  dx is written; dy only with a gate (without one it is dx), NULL: not asked for; dw [K] of w_dtype or
 * NULL.  gate, shift and scale have no gradient here.  dx may be grad_t or grad_h.  Every sum has a fixed order. */
int h3b_residual_norm_backward(const void* grad_t, int64_t lddt, const void* grad_h, int64_t lddh, const void* t, int64_t ldt,
                               const float* rstd, int dtype, int64_t M, int64_t K, const void* w, int w_dtype, const void* gate,
                               const void* scale, int64_t ldm, int64_t n_rows, int m_dtype, const int32_t* segments,
                               int n_segments, const int32_t* token_rows, void* dx, int64_t lddx, void* dy, int64_t lddy,
                               void* dw, void* workspace, size_t ws_bytes, void* stream);

/* ---- low-rank adapters of many requests beside a shared projection (no reference counterpart):
 *     out_i = base_i + s_g (x_i A_g^T) B_g^T,   g the adapter of row i; a row without one keeps base_i.
 * A plan says which rows an adapter has; it is made once for a batch and serves every projection of every layer.
 *   rows [M] adapter of each row; numbers outside 0 .. adapters - 1: none.  Any order.
 *   plan  h3b_adapter_plan_ints(M, adapters) numbers (device memory, 16-byte aligned), written by h3b_adapter_plan; only plans
 *         that it wrote for the same M and adapters may be passed on. */
#define H3B_MAX_RANK 128
#define H3B_MAX_ADAPTERS 65535
int64_t h3b_adapter_plan_ints(int64_t M, int64_t adapters);
int h3b_adapter_plan(const int32_t* rows, int64_t M, int64_t adapters, int32_t* plan, int64_t plan_ints, void* stream);

/* x [M, ldx], base and out [M, ld]: bf16 or fp16 rows of K and N channels (multiples of 8; 16-byte aligned rows); a [adapters,
 * rank, K] and b [adapters, N, rank] of the same type, contiguous; scales [adapters] fp32 or NULL (1); base NULL: zeros; out may be
 * base (rows without an adapter are then left as they are), and otherwise overlaps nothing.  Sums are held in fp32; s x A^T
 * is rounded once for the second product and for the gradient of b (s grad_out B likewise for those of x and a): to bf16's 8 digits
 * beside bf16 operands, to fp16's 11 digits over fp32's range (tf32) beside fp16 ones and in the second product of few rows.
 *   hidden     h3b_low_rank_hidden_bytes(M, rank) (256-byte aligned) for the gradients, or NULL
 *   workspace  h3b_low_rank_workspace_bytes(..., backward = 0), 256-byte aligned; the size queries give 0 for refused sizes. */
size_t h3b_low_rank_hidden_bytes(int64_t M, int rank);
size_t h3b_low_rank_workspace_bytes(int64_t M, int64_t K, int64_t N, int rank, int64_t adapters, int backward);
int h3b_low_rank(const void* x, int64_t ldx, const void* a, const void* b, const void* base, int64_t ldbase, void* out,
                 int64_t ldo, int dtype, int64_t M, int64_t K, int64_t N, int rank, int64_t adapters, const float* scales,
                 const int32_t* plan, void* hidden, void* workspace, size_t ws_bytes, void* stream);
/* Gradients with respect to x, a and b (each may be NULL: not asked for); that of base is grad_out itself.  hidden as
 * h3b_low_rank left it for the same arguments.  dx, da and db overlap no input and not one another.  Adapters without rows and rows
 * without an adapter get zeros.  Every sum has a fixed order: the same call gives the same bits. */
int h3b_low_rank_backward(const void* grad_out, int64_t ldgo, const void* x, int64_t ldx, const void* a, const void* b,
                          const void* hidden, void* dx, int64_t lddx, void* da, void* db, int dtype, int64_t M, int64_t K,
                          int64_t N, int rank, int64_t adapters, const float* scales, const int32_t* plan, void* workspace,
                          size_t ws_bytes, void* stream);

/* int4 codebook indices + group scales -> the exact int8 grid [N, K] (row stride ldg bytes).
 * Replaces decode_int8_grid / _decode_rows / _pair_lut (qlinear.py:157-204).
 *   q4     [N, ldq4 bytes] packed nibbles, low nibble first (types.py:14-16)
 *   s_rel  [N, lds elements] of s_dtype (fp8 e4m3 bytes, fp16, bf16 or fp32), K / group per row
 *   codebook fp32 [16]; group >= 4 dividing 16 or a multiple of 16 (qlinear.py:146). */
int h3b_decode_grid(const void* q4, int64_t N, int64_t K, int64_t ldq4, const void* s_rel, int s_dtype, int64_t lds,
                    const float* codebook, int group, int8_t* grid, int64_t ldg, void* stream);

/* Exact int32 a[M, K] @ b[N, K]^T for int8 operands on the tcgen05 tensor cores (parity of the integer accumulator).
 * Replaces _int8_mm (qlinear.py:236-254).  lda/ldb in bytes (multiples of 16), ldc in elements. */
int h3b_int8_gemm_s32(const int8_t* a, int64_t lda, int64_t M, const int8_t* b, int64_t ldb, int64_t N, int64_t K,
                      int32_t* c, int64_t ldc, void* stream);

/* Scratch bytes h3b_w4a8_gemm / h3b_w4a8_linear need for these sizes (0 is a valid answer). */
size_t h3b_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K);
size_t h3b_linear_workspace_bytes(int64_t M, int64_t N, int64_t K);

/* W4A8 GEMM + epilogue on already-quantised activation codes (kernel KB).
 * Replaces the int8 GEMM and epilogue of _TorchRunner._a8 (qlinear.py:396-405):
 *   out = out_dtype( (fp32(acc) * xs[m]) * s_ch[n] )            quant_mode CK
 *   out = out_dtype(  fp32(acc) * (xs[m] * s_ch[n]) )           quant_mode EAGER
 *   out = out_dtype( fp32(out) + fp32(bias[n]) )                 when bias != NULL (bias already of out_dtype)
 * out_dtype H3B_INT32 stores the raw accumulator instead (xs, s_ch, bias ignored).
 *   qa [M, lda bytes] int8 codes, xs [M] fp32; weight as in h3b_decode_grid; out [M, ldo elements]. */
int h3b_w4a8_gemm(const int8_t* qa, int64_t lda, const float* xs, int64_t M, const void* q4, int64_t ldq4,
                  const void* s_rel, int s_dtype, int64_t lds, const float* s_ch, const float* codebook, int group,
                  const void* bias, void* out, int out_dtype, int64_t ldo, int64_t N, int64_t K, int quant_mode,
                  void* workspace, size_t ws_bytes, void* stream);

/* GEMM + epilogue on an already-decoded int8 weight grid [N, ldg bytes] (same epilogue contract as h3b_w4a8_gemm).
 * For callers that keep decoded grids resident (weights that never stream); no workspace.  Same reference lines as
 * h3b_w4a8_gemm (qlinear.py:396-405) with the decode (qlinear.py:194-204) hoisted out. */
/* 1 when h3b_w4a8_gemm (and so h3b_w4a8_linear) decodes the int4 weight inside the GEMM's producer warps for this
 * problem (few M tiles; fp8 e4m3 scales with group 16 or fp16/bf16/fp32 scales with group 128; 16-byte aligned packed
 * rows), 0 when it runs a separate decode pass into the workspace first.  No reference counterpart (introspection). */
int h3b_w4a8_gemm_decodes_in_kernel(int64_t M, int64_t N, int64_t K, const void* q4, int64_t ldq4, int s_dtype,
                                    int group);

int h3b_int8_gemm_epilogue(const int8_t* qa, int64_t lda, const float* xs, int64_t M, const int8_t* grid, int64_t ldg,
                           const float* s_ch, const void* bias, void* out, int out_dtype, int64_t ldo, int64_t N,
                           int64_t K, int quant_mode, void* stream);

/* The whole W4A8 linear: (swiglu) -> rotate+quantise -> GEMM -> epilogue.  The seam the reference hands to
 * comfy_kitchen: _run_ck -> w4a8_int8_linear(x2, w.q, s_rel, w.s_ch, codebook, bias, group_size, convrot_groupsize,
 * out_dtype) (qlinear.py:427-429, result contract :446-451).  workspace >= h3b_linear_workspace_bytes(M, N, K). */
int h3b_w4a8_linear(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, int swiglu, const void* q4,
                    int64_t ldq4, const void* s_rel, int s_dtype, int64_t lds, const float* s_ch, const float* codebook,
                    int group, int convrot, const void* bias, void* out, int out_dtype, int64_t ldo, int64_t N,
                    int quant_mode, void* workspace, size_t ws_bytes, void* stream);

/* Allocation-free W4A8 GEMM + epilogue: h3b_w4a8_gemm without the workspace argument.  No counterpart in the
 * reference.  For callers that cannot allocate device memory: code running inside a host framework or plugin that
 * gives it no device allocator, a C/FFI caller with no CUDA memory pool of its own, or a latency-critical loop that must
 * not call cudaMalloc (it can synchronise the whole device).  The decoded weight rows live in one file-scope device
 * array of H3B_NOALLOC_SCRATCH_BYTES that every GPU using the library holds until the process exits; the weight is
 * decoded and multiplied in slabs of rows that fit in it, so any N works, and K may be at most
 * H3B_NOALLOC_SCRATCH_BYTES / 32 (larger K is rejected with H3B_ERR_ARG).  Every call looks up the array's device
 * address in the current device's context (cudaGetSymbolAddress; the first call on a device loads the module there, so
 * make that first call before any stream capture).  All calls share the one
 * array: calls that may overlap on the GPU (different streams, or different host threads) race on it and must be
 * serialised by the caller.  Nothing in it needs to start at zero (each slab is fully rewritten before it is read). */
#define H3B_NOALLOC_SCRATCH_BYTES (16u << 20)
int h3b_w4a8_gemm_noalloc(const int8_t* qa, int64_t lda, const float* xs, int64_t M, const void* q4, int64_t ldq4,
                          const void* s_rel, int s_dtype, int64_t lds, const float* s_ch, const float* codebook, int group,
                          const void* bias, void* out, int out_dtype, int64_t ldo, int64_t N, int64_t K, int quant_mode,
                          void* stream);

/* ---- block streamer: the copy path of StreamingProvider (stream.py:115-623; copies and slot events :333-362,
 * acquire/release ordering :376-437).  An engine owns a copy stream, per-slot `ready`/`done` events and page-locked host
 * staging buffers; the caller owns the device slots.  Slot s's copy waits on the device for done[s] (recorded by
 * release on the compute stream), and acquire makes the compute stream wait for ready[s].  Host waits are bounded. */
typedef struct h3b_streamer h3b_streamer;
enum h3b_copy_mode {
  H3B_COPY_DIRECT = 0,   /* source is page-locked (registered or pinned): one async copy */
  H3B_COPY_STAGED = 1,   /* pageable source: multi-threaded memcpy into a staging buffer, then an async copy */
  H3B_COPY_PAGEABLE = 2  /* pageable source copied by the driver (returns once the source has been read) */
};
int h3b_streamer_create(int device, int n_slots, int n_staging, size_t staging_bytes, int memcpy_threads,
                        h3b_streamer** out);
int h3b_streamer_destroy(h3b_streamer* s);
int h3b_streamer_copy(h3b_streamer* s, int slot, void* dst, const void* src_host, size_t bytes, int mode);
/* A caller-driven copy (a custom transfer) on the engine's copy stream: begin (the stream waits for done[slot]),
 * enqueue the copy on h3b_streamer_stream(s), end (ready[slot] recorded). */
int h3b_streamer_begin(h3b_streamer* s, int slot);
int h3b_streamer_end(h3b_streamer* s, int slot, size_t bytes);
void* h3b_streamer_stream(h3b_streamer* s);
int h3b_streamer_acquire(h3b_streamer* s, int slot, void* stream);
int h3b_streamer_release(h3b_streamer* s, int slot, void* stream);
int h3b_streamer_wait(h3b_streamer* s, int slot, double timeout_s);
int h3b_streamer_stats(h3b_streamer* s, uint64_t* copies, uint64_t* bytes, double* busy_s);
/* Page-lock / unlock a host range in place (read_only != 0 for a read-only file mapping: cudaHostRegisterReadOnly).
 * Replaces the reference's torch.cuda.cudart().cudaHostRegister calls (stream.py:208-217, :232-238). */
int h3b_host_register(void* ptr, size_t bytes, int read_only);
int h3b_host_unregister(void* ptr);

/* Self-test of the bounded-wait failure path (no reference counterpart): one thread waits on an mbarrier that nothing
 * arrives on, gives up after limit_s (0 < limit_s <= 10) of GPU time, raises bit 0 of the device flag and writes 1 to
 * *gave_up_device (device memory).  The context stays usable; read and clear the flag with h3b_device_error(1). */
int h3b_selftest_wait_timeout(double limit_s, int* gave_up_device, void* stream);

/* Device-side failure flag of the current device: a kernel whose bounded wait ran out sets it (and returns instead of
 * hanging).  Returns the flag and, when clear != 0, resets it.  Synchronises the device. */
int h3b_device_error(int clear);

#ifdef __cplusplus
}
#endif

#endif /* H3B_H */
