/*
 * anima_attn.h — C ABI of the MI355X (gfx950) DiT attention path.
 *
 * One shared library, libanima_attn.so, holds every kernel of the path:
 * the QK-RMSNorm + 3D-RoPE prologue, per-head RMSNorm of cross-attention
 * queries, the non-causal flash-attention forward (self, and key-length
 * masked cross-attention with an optional fused padding correction), the
 * flash-attention backward, and the padding-correction kernels on their own;
 * around them the block's norms, int8 products and 8-bit copies, rotary
 * positions on their own and the attention over selected blocks.
 *
 * Conventions shared by every entry point:
 *   - Tensors are device pointers. Attention tensors are [B, S, H, hd]
 *     ("BSHD") with the head-dim stride fixed to 1 and the other three
 *     strides passed in elements (int64). Prologue tensors are contiguous.
 *   - `stream` is a hipStream_t passed as void* (NULL = the null stream).
 *     Every call is asynchronous on that stream; no call synchronises the
 *     host and none allocates or frees device memory: outputs and
 *     workspaces are allocated by the caller.
 *   - Return codes: AA_OK (0); AA_EINVAL (-1) for a bad argument (null
 *     pointer, inconsistent shape, misaligned pointer or stride);
 *     AA_EUNSUPPORTED (-2) for a shape or dtype the kernels do not
 *     implement; AA_EHIP (-3) when a HIP launch reports an error.
 *     aa_last_error() returns the calling thread's last message.
 *   - Only dtype AA_DTYPE_BF16 is implemented for activations (aa_rotary also
 *     takes FP16 and FP32); weights, rotary tables, LSE and padding logs are
 *     float32; key lengths and block lists int32.
 *   - hd (head_dim) must be 128; aa_attn_fwd (and its workspace and no-alloc
 *     forms) also takes 384, the VAE decoder's single-head attention, and
 *     aa_rotary multiples of 8 up to 512.
 *
 * The reference (anima-flat) has no C FFI of its own: its path is Python
 * calling FlashAttention-4 (CuTe DSL) and Triton kernels. Each entry point
 * below names the reference function (file:line under src/) whose work it
 * replaces; the Python host layer in anima-flat_amd/ keeps those functions'
 * signatures and calls these entry points through ctypes.
 */
#ifndef ANIMA_ATTN_H
#define ANIMA_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define AA_ABI_VERSION 3

enum {
  AA_OK = 0,
  AA_EINVAL = -1,
  AA_EUNSUPPORTED = -2,
  AA_EHIP = -3,
};

enum {
  AA_DTYPE_BF16 = 0,
  AA_DTYPE_FP16 = 1, /* aa_rotary only */
  AA_DTYPE_FP32 = 2, /* aa_rotary, and modulation rows of aa_adaln_fwd / _bwd, only */
};

/* ABI version of the loaded library (AA_ABI_VERSION when built from this header). */
int aa_abi_version(void);

/* Last error message of the calling thread ("" if none). Valid until the next call. */
const char* aa_last_error(void);

/* ------------------------------------------------------------------------ */
/* Prologue                                                                  */
/* ------------------------------------------------------------------------ */

/*
 * Per-head RMSNorm of the q and k sections of a fused QKV projection output,
 * rounded to the activation dtype, then rotate-half RoPE; optional V copy.
 *   qkv [B, S, 3*H*hd] contiguous; q, k [B, S, H, hd] contiguous outputs;
 *   v   [B, S, H, hd] output or NULL (NULL: V is not copied);
 *   q_weight, k_weight [hd] float32; cos, sin [S, hd/2] float32;
 *   position of token (b, s) is s.
 * Replaces: src/kernels/rope.py:175-193 (_qkv_norm_rope, v == NULL) and
 *           src/kernels/rope.py:504-523 (_qkv_norm_rope_v, v != NULL),
 *           kernel src/kernels/rope.py:61-143.
 */
int aa_qkv_norm_rope_fwd(const void* qkv, void* q, void* k, void* v,
                         const float* q_weight, const float* k_weight,
                         const float* cos, const float* sin,
                         int64_t B, int64_t S, int64_t H, int64_t hd,
                         float eps, int dtype, void* stream);

/*
 * QKV projection fused with the prologue: q, k, v = aa_qkv_norm_rope_fwd of
 * qkv = hid @ weight^T (bf16), without qkv ever reaching memory.
 *   hid [B*S rows, H*hd], row r at hid + r * hid_row_stride elements
 *   (hid_row_stride >= H*hd, a multiple of 8, at most 2^27); weight [3*H*hd, H*hd]
 *   contiguous (nn.Linear layout, no bias); q, k, v [B, S, H, hd] contiguous
 *   outputs (v is the projection's V section as it is); q_weight, k_weight,
 *   cos, sin as for aa_qkv_norm_rope_fwd. H <= 64.
 * Replaces: src/model.py:308-316 (b.qkv(hid), model.py:134, followed by
 *           qkv_norm_rope, src/kernels/rope.py:616-645) on the inference path.
 */
int aa_qkv_proj_norm_rope(const void* hid, int64_t hid_row_stride, const void* weight,
                          void* q, void* k, void* v,
                          const float* q_weight, const float* k_weight,
                          const float* cos, const float* sin,
                          int64_t B, int64_t S, int64_t H, int64_t hd,
                          float eps, int dtype, void* stream);

/*
 * A projection fused with per-head RMSNorm: y = aa_head_norm_fwd of
 * x @ weight^T (bf16), the projection never reaching memory.
 *   x [B*S rows, K], row r at x + r * x_row_stride elements (x_row_stride >= K,
 *   a multiple of 8, at most 2^27; K a multiple of 32); weight [H*hd, K] contiguous (nn.Linear
 *   layout, no bias); y [B, S, H, hd] contiguous; norm_weight [hd] float32.
 * Replaces: src/model.py:324 (b.xq(hid), model.py:138, followed by head_norm,
 *           src/kernels/rope.py:648-652) on the inference path.
 */
int aa_proj_head_norm(const void* x, int64_t x_row_stride, const void* weight, int64_t K,
                      void* y, const float* norm_weight,
                      int64_t B, int64_t S, int64_t H, int64_t hd,
                      float eps, int dtype, void* stream);

/*
 * The context's keys and values with the key-side RMSNorm fused:
 * kv = ctx @ weight^T (bf16, [B, S, 2, H, hd]), k = RMSNorm(kv[:, :, 0]) with
 * k_weight, v = kv[:, :, 1], kv never reaching memory.
 *   ctx [B*S rows, K] as x above; weight [2*H*hd, K] contiguous; k, v
 *   [B, S, H, hd] contiguous; k_weight [hd] float32 (pass the bf16 weight
 *   widened, as F.rms_norm applies it in the activation dtype).
 * Replaces: src/model.py:256-258 (b.xkv(ctx), model.py:139, .view().unbind(),
 *           F.rms_norm of k) in encode_context, inference path.
 */
int aa_kv_proj_norm(const void* ctx, int64_t ctx_row_stride, const void* weight, int64_t K,
                    void* k, void* v, const float* k_weight,
                    int64_t B, int64_t S, int64_t H, int64_t hd,
                    float eps, int dtype, void* stream);

/*
 * Per-head RMSNorm: x [B, S, H*hd] contiguous -> y [B, S, H, hd] contiguous.
 * Replaces: src/kernels/rope.py:203-212 (_head_norm), kernel rope.py:146-172.
 */
int aa_head_norm_fwd(const void* x, void* y, const float* weight,
                     int64_t B, int64_t S, int64_t H, int64_t hd,
                     float eps, int dtype, void* stream);

/* Bytes of workspace aa_qkv_norm_rope_bwd needs (weight-grad partials: one
 * 2*hd float record per 8 tokens). */
size_t aa_qkv_norm_rope_bwd_workspace(int64_t B, int64_t S, int64_t H, int64_t hd);

/*
 * Backward of aa_qkv_norm_rope_fwd (with V copied):
 *   dq, dk, dv [B, S, H, hd] contiguous -> dqkv [B, S, 3*H*hd],
 *   dq_weight, dk_weight [hd] float32 (sums over every token and head).
 * The weight-gradient reduction runs in a fixed order (deterministic).
 * Replaces: src/kernels/rope.py:540-577 (_qkv_norm_rope_bwd),
 *           kernel rope.py:277-383, helper rope.py:223-274.
 */
int aa_qkv_norm_rope_bwd(const void* qkv, const void* dq, const void* dk,
                         const void* dv, void* dqkv,
                         const float* q_weight, const float* k_weight,
                         const float* cos, const float* sin,
                         float* dq_weight, float* dk_weight,
                         void* workspace, size_t workspace_bytes,
                         int64_t B, int64_t S, int64_t H, int64_t hd,
                         float eps, int dtype, void* stream);

/* Bytes of workspace aa_head_norm_bwd needs (as above with hd floats). */
size_t aa_head_norm_bwd_workspace(int64_t B, int64_t S, int64_t H, int64_t hd);

/*
 * Backward of aa_head_norm_fwd: x, dy [B, S, H*hd] -> dx [B, S, H*hd],
 * dweight [hd] float32.
 * Replaces: src/kernels/rope.py:443-471 (_head_norm_bwd), kernel rope.py:386-436.
 */
int aa_head_norm_bwd(const void* x, const void* dy, void* dx,
                     const float* weight, float* dweight,
                     void* workspace, size_t workspace_bytes,
                     int64_t B, int64_t S, int64_t H, int64_t hd,
                     float eps, int dtype, void* stream);

/* ------------------------------------------------------------------------ */
/* Flash attention                                                           */
/* ------------------------------------------------------------------------ */

typedef struct aa_attn_fwd_args {
  const void* q;        /* [B, Sq, H, hd] */
  const void* k;        /* [B, Sk, H, hd]; may be NULL when Sk == 0 */
  const void* v;        /* [B, Sk, H, hd]; may be NULL when Sk == 0 */
  void* out;            /* [B, Sq, H, hd]; Sk == 0 gives out = 0 and lse = -inf */
  float* lse;           /* [B, H, Sq] contiguous natural-log LSE, or NULL */
  const int32_t* seqused_k; /* [B] keys attended per batch item, or NULL (all Sk) */
  const float* ln_pad;  /* [B] log(#padding keys) for the fused padding
                           correction out *= 1/(1+exp(ln_pad-lse)), or NULL */
  int64_t q_stride[3];  /* batch, seq, head strides in elements */
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t out_stride[3];
  int64_t B, Sq, Sk, H, hd;
  float softmax_scale;  /* usually 1/sqrt(hd) */
  int dtype;
  void* workspace;      /* device scratch of aa_attn_fwd_workspace() bytes (may be 0) */
  size_t workspace_bytes;
} aa_attn_fwd_args;

/* Bytes of device workspace aa_attn_fwd needs on the current device: partial
 * results (bf16 normalised O and fp32 LSE, at both head dims) when the work items (256
 * queries of one (batch, head); 128 at hd 384) of a partial last round of
 * workgroups (at hd 384: of too few work items to fill the device) are split
 * over key ranges, else 0. */
size_t aa_attn_fwd_workspace(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t hd);

/*
 * out = softmax(q k^T * softmax_scale) v, non-causal, per (batch, head);
 * keys j >= seqused_k[b] are excluded when seqused_k != NULL; lse is the
 * natural-log row log-sum-exp of the scaled scores over the attended keys.
 * One kernel launch, plus a combine pass when aa_attn_fwd_workspace() > 0.
 * From about two rounds of 64-tile work items on (e.g. B=2 at 4096 keys),
 * the hd-128 forward keeps each row's first key tile max and follows its
 * launch with a fix-up launch that re-runs, with a running max, the work
 * items whose scores left that exponent range (AA_FWD_FIRST_TILE_MAX=0|1
 * forces the form). Every launch goes to `stream`; none allocates.
 * Replaces: src/attention.py:43-53 (anima_flat::fa_fwd),
 *           src/attention.py:63-66 (anima_flat::fa_fwd_nolse),
 *           src/attention.py:74-81 (anima_flat::fa_fwd_k), and with
 *           ln_pad != NULL also the ctx_scale pass of
 *           src/attention.py:156-180 (cross_attention_trimmed).
 * With hd == 384 (one kernel for that width, plus a combine pass when its keys
 * are split): replaces the VAE's mid-block attention, src/vae.py:239
 * (ffpa_attn_func / SDPA on [B, 1, S, 384], vae.py:10-13, 230-241).
 */
int aa_attn_fwd(const aa_attn_fwd_args* args, void* stream);

/*
 * aa_attn_fwd without a caller workspace and without any allocation: the
 * split partials go to a fixed device array of 25,296,896 bytes that the
 * library holds on each device it runs on until the process ends (every
 * forward, head_dim 128 or 384, on a 256-CU device fits; a plan that needs
 * more returns AA_EUNSUPPORTED). args->workspace / workspace_bytes are ignored. Calls on
 * one device share that array: calls that overlap on one device (two streams
 * at once) race and must be serialised by the caller. Same results as
 * aa_attn_fwd (same kernels). No counterpart in the reference: for callers
 * that cannot allocate device memory (code under HIP graph capture, serving
 * loops, harnesses that forbid hipMalloc).
 */
int aa_attn_fwd_noalloc(const aa_attn_fwd_args* args, void* stream);

typedef struct aa_attn_bwd_args {
  const void* dout;     /* [B, Sq, H, hd] */
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const float* lse;     /* [B, H, Sq] contiguous, from aa_attn_fwd */
  void* dq;             /* [B, Sq, H, hd] */
  void* dk;             /* [B, Sk, H, hd] */
  void* dv;             /* [B, Sk, H, hd] */
  int64_t dout_stride[3];
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t out_stride[3];
  int64_t dq_stride[3];
  int64_t dk_stride[3];
  int64_t dv_stride[3];
  int64_t B, Sq, Sk, H, hd;
  float softmax_scale;
  int dtype;
} aa_attn_bwd_args;

/* Bytes of workspace aa_attn_bwd needs, 16-byte aligned: 1 KB of softmax
 * statistics per 64 queries, for every (batch, head); 0 if Sq == 0. */
size_t aa_attn_bwd_workspace(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t hd);

/*
 * dq, dk, dv of aa_attn_fwd (no key mask), softmax recomputed from lse.
 * Deterministic: no atomics, every sum runs in a fixed order.
 * Replaces: src/attention.py:91-103 (anima_flat::fa_bwd), reached through
 *           the autograd registration at src/attention.py:111-123.
 */
int aa_attn_bwd(const aa_attn_bwd_args* args, void* workspace,
                size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------ */
/* Padding correction of trimmed cross-attention                             */
/* ------------------------------------------------------------------------ */

/*
 * y = out * 1/(1 + exp(ln_pad[b] - lse[b, h, s])); out, y [B, S, H, hd]
 * contiguous, lse [B, H, S], ln_pad [B].
 * Replaces: src/kernels/ctx_scale.py:39-55 (kernel ctx_scale.py:8-36).
 */
int aa_ctx_scale_fwd(const void* out, const float* lse, const float* ln_pad,
                     void* y, int64_t B, int64_t S, int64_t H, int64_t hd,
                     int dtype, void* stream);

/*
 * dout = dy * g, dlse[b,h,s] = sum_d(dy * out) * g * (1 - g) with
 * g = 1/(1 + exp(ln_pad[b] - lse[b,h,s])).
 * Replaces: src/kernels/ctx_scale.py:98-117 (kernel ctx_scale.py:63-95).
 */
int aa_ctx_scale_bwd(const void* out, const float* lse, const float* ln_pad,
                     const void* dy, void* dout, float* dlse,
                     int64_t B, int64_t S, int64_t H, int64_t hd,
                     int dtype, void* stream);

/* ------------------------------------------------------------------------ */
/* Text-context length bookkeeping                                           */
/* ------------------------------------------------------------------------ */

/* Bytes of workspace aa_context_lengths needs (one int32 per 32 rows per item). */
size_t aa_context_lengths_workspace(int64_t B, int64_t S);

/*
 * Lengths of a zero-padded text context ctx [B, S, C] (element strides
 * stride_b, stride_s; last dim contiguous; elem_bytes 2 for bf16/fp16 or 4
 * for fp32): seqused[b] = 1-based index of the last row with a non-zero
 * element, at least 1 (int32 [B]); ln_pad[b] = log(S - seqused[b]) (float
 * [B], -inf when nothing is padded). Computed on the device with no host
 * read: K/V projected from the untrimmed context can go straight to
 * aa_attn_fwd with seqused_k / ln_pad, which reads only the first seqused[b]
 * keys, so the reference's trim to roundup8(max length) rows (and its
 * device-to-host read) is not needed. Rows must be 16-byte aligned and
 * C * elem_bytes a multiple of 16.
 * Replaces: src/model.py:248-253 (the length, seqused and ln_pad lines of
 *           encode_context's trim; the ctx[:, :keep] slice is dropped).
 */
int aa_context_lengths(const void* ctx, int64_t B, int64_t S, int64_t C,
                       int64_t stride_b, int64_t stride_s, int elem_bytes,
                       int32_t* seqused, float* ln_pad,
                       void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------ */
/* FP8 row quantisation (consumer of the attention output)                   */
/* ------------------------------------------------------------------------ */

/*
 * Per-row FP8 quantisation: for each of `rows` rows of x [rows, K] bf16
 * (contiguous), y = x or GELU(x) (gelu != 0; Abramowitz-Stegun 7.1.26 erf),
 * s[row] = max(max|y|, 1e-12) / 448 (float), q = e4m3fn(clamp(y / s, +-448))
 * rounded to nearest even (uint8 [rows, K], OCP E4M3 "fn" bytes).
 * K a multiple of 8 and at most 8192; x 16-byte and q 8-byte aligned.
 * Replaces: src/kernels/fp8.py:295-328 (rowquant, op anima_flat::rowquant),
 *           kernel fp8.py:275-292.
 */
int aa_rowquant(const void* x, int64_t rows, int64_t K, int gelu,
                void* q, float* s, int dtype, void* stream);

/* ------------------------------------------------------------------------ */
/* Norms, gate and residual around the sublayers                             */
/* ------------------------------------------------------------------------ */

typedef struct aa_adaln_args {
  const void* x;        /* [B, S, D] residual stream */
  const void* y;        /* [B, S, D] the sublayer's output, or NULL: no residual add */
  const void* gate;     /* rows of D (mod_dtype), batch item b's at b * gate_stride; unused without y */
  const void* scale;
  const void* shift;
  int64_t gate_stride;  /* elements; 0: one row for all batch items */
  int64_t scale_stride;
  int64_t shift_stride;
  const float* weight;  /* [D] RMSNorm weight of a norm on y, or NULL: y as it is */
  void* r;              /* [B, S, D] x + branch_scale * gate * norm(y); unused without y */
  void* h;              /* [B, S, D] modulated norm of r, or NULL when q is set */
  void* q;              /* [B, S, D] int8 codes of h in place of h, or NULL */
  float* q_scale;       /* [B * S] scales of q */
  float* stats;         /* [B * S, 4] for aa_adaln_bwd, or NULL */
  int64_t B, S, D;
  float eps;
  float branch_scale;
  int dtype;            /* of x, y, r, h */
  int mod_dtype;        /* of gate, scale, shift: AA_DTYPE_BF16 or AA_DTYPE_FP32 */
} aa_adaln_args;

/*
 * n = y, or y * rsqrt(mean(y^2) + eps) * weight; r = x + branch_scale * gate * n
 * (r = x without y); h = (r - mean(r)) * rsqrt(var(r) + eps) * (1 + scale) + shift,
 * per token over D channels, all in fp32; r and h are rounded to bf16 once each
 * (h is that of the fp32 r). With q: s = max(max|h|, 1e-12) / 127 and q as
 * aa_rowquant_int8 makes them, of the fp32 h; a token with a value that is not
 * finite has the scale NaN.
 * x, y, r, h, q contiguous; D a multiple of 8, at most 8192; 16-byte aligned
 * pointers and modulation rows.
 * Stands for the work of src/kernels/adaln.py:298-314 (residual_adaln, adaln;
 * kernel adaln.py:10-46) and, with q, of src/kernels/fp8.py:56-97 in int8.
 */
int aa_adaln_fwd(const aa_adaln_args* args, void* stream);

typedef struct aa_adaln_bwd_args {
  const void* dr;       /* [B, S, D] gradient of r (of h's input x without y), or NULL: zero */
  const void* dh;       /* [B, S, D] gradient of h, or NULL: zero */
  const void* x;        /* x, y, gate, scale, weight, strides: as in the forward */
  const void* y;
  const void* gate;
  const void* scale;
  int64_t gate_stride;
  int64_t scale_stride;
  const float* weight;
  const float* stats;   /* from aa_adaln_fwd */
  void* dx;             /* [B, S, D] */
  void* dy;             /* [B, S, D]; unused without y */
  void* dgate;          /* [gate_rows, D] in mod_dtype, or NULL: not computed */
  void* dscale;
  void* dshift;
  float* dweight;       /* [D], or NULL */
  int64_t gate_rows;    /* B, or 1: the sum over all batch items */
  int64_t scale_rows;
  int64_t shift_rows;
  int64_t B, S, D;
  float branch_scale;
  int dtype;
  int mod_dtype;
} aa_adaln_bwd_args;

/* Bytes of workspace aa_adaln_bwd needs on the current device, 16-byte aligned:
 * partial sums of the modulation's and the weight's gradients; 0 when none of
 * them is asked for (sums == 0). */
size_t aa_adaln_bwd_workspace(int64_t B, int64_t S, int64_t D, int sums);

/*
 * Gradients of aa_adaln_fwd (not of its int8 form), every sum in a fixed order.
 * Stands for the work of the backward in src/kernels/adaln.py (kernel :111-172).
 */
int aa_adaln_bwd(const aa_adaln_bwd_args* args, void* workspace, size_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------ */
/* Int8 products                                                             */
/* ------------------------------------------------------------------------ */

/*
 * Per-row int8 quantisation of x [rows, K] bf16 (contiguous): y = x or GELU(x)
 * (gelu != 0; erf form, to 3e-5 relative or 2e-18), s[row] = max(max|y|, 1e-12)
 * / 127 (float), q = round-to-nearest-even(127 y / max(max|y|, 1e-12)) (int8
 * [rows, K]): without GELU as in exact arithmetic, after it but for quotients as
 * near a tie as GELU's error. A row with a value that is not finite has the
 * scale NaN and codes 0. K a multiple of 8 and at most 8192; x 16-byte and q 8-byte
 * aligned.
 */
int aa_rowquant_int8(const void* x, int64_t rows, int64_t K, int gelu,
                     void* q, float* s, int dtype, void* stream);

/*
 * y[m, n] = s[m] * weight_scale[n] * sum_k q[m, k] weight[n, k], the sum exact
 * in int32; q [M, K], weight [N, K] int8, y [M, N] of `dtype` (bf16), all
 * contiguous and 16-byte aligned; s [M], weight_scale [N] float.
 * K a multiple of 16 and at most 65536; N a multiple of 8.
 * Stands for the work of src/kernels/fp8.py:234-257 (fp8_linear) in int8.
 */
int aa_int8_linear(const void* q, const float* s, const void* weight, const float* weight_scale,
                   void* y, int64_t M, int64_t N, int64_t K, int dtype, void* stream);

/* ------------------------------------------------------------------------ */
/* Activations kept in 8 bits for the backward pass                          */
/* ------------------------------------------------------------------------ */

/*
 * The 8-bit checkpoint of rows x [rows, K] bf16: per row, groups of 32 channels
 * (G = ceil(K / 32), the last one may be shorter) share a step, a power of two
 * 2^(e - 127) with 2^6 <= max|x| / step < 2^7 (e >= 1): code = round-to-nearest-
 * even(x / step) clamped to +-127. codes: int8 [rows, 32 G], zero past K;
 * exps: uint8 biased exponents e, 255 for a group with a value that is not
 * finite (it reads back as NaN).
 *
 * aa_gelu8_fwd: y = GELU(x) (erf form), and the checkpoint, exps [rows, G];
 * codes NULL: y only. aa_gelu8_bwd: dx = dy * GELU'(code * step).
 * x, y, dy, dx [rows, K] contiguous, codes: 16-byte aligned; K a multiple of 8,
 * at most 65536.
 */
int aa_gelu8_fwd(const void* x, void* y, void* codes, void* exps, int64_t rows, int64_t K,
                 int dtype, void* stream);
int aa_gelu8_bwd(const void* dy, const void* codes, const void* exps, void* dx, int64_t rows,
                 int64_t K, int dtype, void* stream);

/*
 * t = x a^T (x [M, K], a [R, K], t [M, R], bf16, contiguous), and x's checkpoint
 * with exps [G, Mp], Mp = M rounded up to a multiple of 16; codes NULL: t only.
 * R a multiple of 8, at most 64; K a multiple of 8, at most 65536; all pointers
 * 16-byte aligned.
 */
int aa_lora8_fwd(const void* x, const void* a, void* t, void* codes, void* exps,
                 void* workspace, size_t workspace_bytes, int64_t M, int64_t K, int64_t R,
                 int dtype, void* stream);

/* Bytes of workspace aa_lora8_fwd and aa_lora8_bwd (for da) need on the current
 * device, 16-byte aligned: fp32 partial sums of ranges of channels and rows. */
size_t aa_lora8_fwd_workspace(int64_t M, int64_t K, int64_t R);
size_t aa_lora8_bwd_workspace(int64_t M, int64_t K, int64_t R);

/*
 * dx = dt a [M, K] and da = dt^T (codes * step) [R, K] (bf16; either may be
 * NULL: not computed), every sum in a fixed order.
 */
int aa_lora8_bwd(const void* dt, const void* a, const void* codes, const void* exps, void* dx,
                 void* da, void* workspace, size_t workspace_bytes, int64_t M, int64_t K,
                 int64_t R, int dtype, void* stream);

/* ------------------------------------------------------------------------ */
/* Rotary positions                                                          */
/* ------------------------------------------------------------------------ */

enum { AA_POSITION_INT32 = 0, AA_POSITION_INT64 = 1, AA_POSITION_FP32 = 2, AA_POSITION_FP64 = 3 };
enum { AA_SCALING_NTK = 0, AA_SCALING_LINEAR = 1, AA_SCALING_YARN = 2 };

typedef struct aa_rotary_tables_args {
  const void* positions; /* [rows, axes] of position_type */
  float* cos;            /* [rows, pairs], pairs = sum(dims) / 2 */
  float* sin;
  int64_t rows, axes;    /* 1 to 4 axes */
  int64_t dims[4];       /* values of a head that turn with each axis: even, 2 to 512 together */
  double theta[4];       /* base of each axis' frequencies */
  double scale[4];       /* >= 1: how much longer the axis is than in training */
  double original;       /* AA_SCALING_YARN: the trained length */
  int scaling;
  int position_type;
} aa_rotary_tables_args;

/*
 * cos and sin of positions[t, axis(i)] * f_i, the angle in 64 bits; f_i =
 * theta^(-2 i / d) for pair i of an axis of d dims, and for a scale s:
 *   AA_SCALING_NTK     theta s^(d / (d - 2)) in theta's place (d > 2);
 *   AA_SCALING_LINEAR  f_i / s;
 *   AA_SCALING_YARN    f_i (g + (1 - g) / s), g = (original f_i / (2 pi) - 1) / 31
 *                      clamped to 0 .. 1 (linear in the number of turns, not in i),
 *                      and both tables times 0.1 ln(max s) + 1.
 * The angle is exact to 2^-52 of itself: positions up to 10^8 are told apart.
 * Generalises src/model.py:51-84 (rope_tables), whose tables at 1 x 1 to h x w
 * are AA_SCALING_NTK's of axes (t, y, x).
 */
int aa_rotary_tables(const aa_rotary_tables_args* args, void* stream);

typedef struct aa_rotary_args {
  const void* q;           /* [B, S, H, hd] */
  const void* k;           /* [B, S, Hk, hd]; unused when Hk == 0 */
  void* q_out;             /* [B, S, H, hd], no memory shared with the inputs */
  void* k_out;
  const float* cos;        /* [S, part / 2] contiguous, batch item b's at b * table_stride */
  const float* sin;
  int64_t q_stride[3];     /* batch, token, head strides in elements, head-dim stride 1 */
  int64_t k_stride[3];
  int64_t q_out_stride[3];
  int64_t k_out_stride[3];
  int64_t table_stride;    /* 0: one table for all batch items; else S * part / 2 or more */
  int64_t B, S, H, Hk, hd;
  int64_t part;            /* values of a head that are turned; the others are copied */
  int interleaved;         /* pairs (2 i, 2 i + 1), not (i, i + part / 2) */
  int inverse;             /* by minus the angles: the backward */
  int dtype;               /* AA_DTYPE_BF16, AA_DTYPE_FP16 or AA_DTYPE_FP32 */
} aa_rotary_args;

/*
 * (a, b) -> (a cos - b sin, b cos + a sin) for every pair of the first `part`
 * values of every head, in fp32, rounded once. hd a multiple of 8, at most 512;
 * pointers 16-byte aligned, strides multiples of 16 bytes.
 * Stands beside src/kernels/rope.py:61-143, whose turn is fused with its norm.
 */
int aa_rotary(const aa_rotary_args* args, void* stream);

/* ------------------------------------------------------------------------ */
/* Attention over selected blocks                                            */
/* ------------------------------------------------------------------------ */

/*
 * Blocks: 64 consecutive queries, 64 consecutive keys, the last of either may be
 * shorter. A list of key blocks for each block of queries: int32 [B, H, nq,
 * count] contiguous, nq = ceil(Sq / 64). Entries below 0 or past the last block
 * with a key are no blocks; a block that is named twice counts once; a list
 * without blocks gives out = 0 and lse = -inf. q has H heads, k and v Hk: head h
 * of q reads head h / (H / Hk).
 */
typedef struct aa_block_select_args {
  const void* q;            /* [B, Sq, H, hd] */
  const void* k;            /* [B, Sk, Hk, hd]; may be NULL when Sk == 0 */
  const int32_t* seqused_k; /* [B] keys that count, or NULL (all Sk) */
  int32_t* blocks;          /* [B, H, nq, count] */
  int64_t q_stride[3];      /* batch, seq, head strides in elements */
  int64_t k_stride[3];
  int64_t B, Sq, Sk, H, Hk, hd;
  int64_t count;            /* 1 to 4096 */
  int dtype;
} aa_block_select_args;

/* Bytes of workspace aa_block_select needs: the blocks' means, in 64 bits. */
size_t aa_block_select_workspace(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk);

/*
 * For each block of queries the `count` key blocks with the largest product of
 * mean query and mean key (both over the rows there are), ties to the lower
 * index, NaN before everything; in ascending order, -1 behind them where fewer
 * blocks hold a key. Means and products are fp64. Sk at most 262144.
 * No counterpart in the reference.
 */
int aa_block_select(const aa_block_select_args* args, void* workspace, size_t workspace_bytes, void* stream);

typedef struct aa_sparse_fwd_args {
  const void* q;            /* [B, Sq, H, hd] */
  const void* k;            /* [B, Sk, Hk, hd]; k, v may be NULL when Sk == 0 */
  const void* v;
  void* out;                /* [B, Sq, H, hd] */
  float* lse;               /* [B, H, Sq] contiguous, or NULL */
  const int32_t* seqused_k; /* [B], or NULL */
  const int32_t* blocks;    /* [B, H, nq, count] */
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t out_stride[3];
  int64_t B, Sq, Sk, H, Hk, hd;
  int64_t count;
  float softmax_scale;
  int dtype;
} aa_sparse_fwd_args;

/* Bytes of workspace aa_sparse_fwd needs on the current device, 16-byte aligned:
 * fp32 partial results where there are fewer blocks of queries than SIMDs and
 * the lists are split, else 0. */
size_t aa_sparse_fwd_workspace(int64_t B, int64_t Sq, int64_t H, int64_t count);

/*
 * out = softmax(q k^T * softmax_scale) v over the keys of the listed blocks below
 * seqused_k, lse its natural-log row log-sum-exp. One launch, plus a combine pass
 * when aa_sparse_fwd_workspace() > 0. Rows of k and v at or past seqused_k are
 * not read. B H nq at most 0x1fffff0; with lse also what aa_sparse_bwd takes. Stands beside src/attention.py:43-81, which attends every key.
 */
int aa_sparse_fwd(const aa_sparse_fwd_args* args, void* workspace, size_t workspace_bytes, void* stream);

typedef struct aa_sparse_bwd_args {
  const void* dout;         /* [B, Sq, H, hd] */
  const void* q;            /* as in the forward */
  const void* k;
  const void* v;
  const void* out;          /* from aa_sparse_fwd */
  const float* lse;         /* [B, H, Sq] contiguous, from aa_sparse_fwd */
  const int32_t* seqused_k;
  const int32_t* blocks;
  void* dq;                 /* [B, Sq, H, hd] */
  void* dk;                 /* [B, Sk, Hk, hd]: 0 where no list names a key's block */
  void* dv;
  int64_t dout_stride[3];
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t out_stride[3];
  int64_t dq_stride[3];
  int64_t dk_stride[3];
  int64_t dv_stride[3];
  int64_t B, Sq, Sk, H, Hk, hd;
  int64_t count;
  float softmax_scale;
  int dtype;
} aa_sparse_bwd_args;

/* Bytes of workspace aa_sparse_bwd needs on the current device, 16-byte aligned:
 * 1 KB of softmax statistics per block of queries, the lists turned round, the
 * mean key of each block and, where few blocks are split over more of the device,
 * fp32 partial sums. */
size_t aa_sparse_bwd_workspace(int64_t B, int64_t Sq, int64_t Sk, int64_t H, int64_t Hk, int64_t count);

/*
 * dq, dk, dv of aa_sparse_fwd, softmax recomputed from lse; dk and dv are sums
 * over the heads of q that share a head of k. Deterministic: no atomics on
 * floats, every sum in a fixed order. With Sq == 0 or Sk == 0 nothing is written.
 * Sequence strides of dout, q, k and v are 0 to 2^24 - 1 (in the forward those of
 * k and v). With nk = ceil(Sk / 64): B H nq and B Hk nk at most 0x1fffff0, B H ceil(nq / 64) +
 * B Hk nk / 4 and B Hk nk below 2^24.
 */
int aa_sparse_bwd(const aa_sparse_bwd_args* args, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* ANIMA_ATTN_H */
