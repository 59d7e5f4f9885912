/*
 * loopback_model.h -- C ABI of libloopback_model.so: MI355X (gfx950) kernels of a language model's training step that stand
 * beside those of loopback_lm.h: layer norm with the residual's add and the distillation loss from a teacher's highest
 * logits, each forward and backward in passes over their rows, and differential attention on the matrix cores.
 *
 * Conventions: device pointers; dtype is LDR_F32, LDR_BF16 or LDR_F16 (loopback_read.h); every statistic and sum is fp32,
 * results are rounded once from fp32; stream is a hipStream_t; nothing synchronizes with the host or allocates. The return
 * value is 0, a negative code (rejected before any launch: -1 argument, -2 shape, -3 alignment, -4 dtype) or a positive
 * hipError_t. Sums have a fixed order: the same call gives the same bits.
 */
#ifndef LOOPBACK_MODEL_H
#define LOOPBACK_MODEL_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LMO_ABI_VERSION 1
int lmo_abi_version(void);

/* ---- layer norm ---------------------------------------------------------------------------------------------------
 * Contiguous rows of d elements at element alignment (16-byte aligned rows of a multiple of 8 take the wider loads).
 * h = round(x + add) into h_out, or x where add is NULL (h_out is not used); m = mean(h), r = rsqrt(mean((h - m)^2) + eps),
 * y = round((h - m) r w + b). w and b [d] may each be NULL (1 and 0). stats [rows, 2] receives m and r for the backward
 * (NULL: not wanted). d up to LMO_NORM_MAX_WIDTH, rows below 2^31. */
#define LMO_NORM_MAX_WIDTH 16384
int lmo_layer_norm_fwd(const void* x, const void* add, const void* w, const void* b, void* h_out, void* y, float* stats,
                       int64_t rows, int64_t d, float eps, int dtype, void* stream);

/* Floats of lmo_layer_norm_bwd's scratch. */
int64_t lmo_layer_norm_scratch(int64_t rows, int64_t d);

/* dx = round(r (t - mean(t) - hat mean(t hat)) + dres), t = dy w, hat = (h - m) r (dres, another gradient of h, may be
 * NULL); dw = round(sum of dy hat), db = round(sum of dy) over the rows. Each result may be NULL (not wanted). scratch is
 * needed for dw and db. */
int lmo_layer_norm_bwd(const void* dy, const void* h, const void* w, const float* stats, const void* dres, void* dx,
                       void* dw, void* db, float* scratch, int64_t rows, int64_t d, int dtype, void* stream);

/* ---- distillation from a teacher's highest logits -----------------------------------------------------------------
 * logits x [rows, vocab] at element alignment; ids [rows, k] (int32, or int64 where wide_ids) the classes of the teacher's
 * logits top [rows, k] (top_dtype), an id below 0 names nothing and its logit is not read into anything; tau the
 * temperature; teacher_lse [rows] fp32, the log of the teacher's sum of exp(z / tau) over every class, or NULL (its k are
 * then all it has); labels [rows] int64, or NULL, -100 for a row without one; hard in [0, 1].
 *
 * A row counts where it names a class. p_i = exp(top_i / tau - teacher_lse), or its softmax over the row's k; P the sum of
 * the p and rest = max(0, 1 - P) with a teacher_lse and a class that is not named, else 0; q = softmax(x / tau); q_rest the sum of q over the classes
 * that are not named. kl = sum p_i (log p_i - log q[id_i]) + rest (log rest - log q_rest), terms of p 0 left out.
 *   loss = (1 - hard) tau^2 mean(kl over the rows that count) + hard mean(-log softmax(x)[label] over those with a label)
 * a mean over no rows is 0. An id of vocab or more and a label outside [0, vocab) other than -100 make the loss NaN. An id
 * named twice has the sum of its p.
 *
 * saved [rows, LMO_DISTILL_SAVED] and coef [2] receive what the backward needs. loss: one fp32. k up to
 * LMO_DISTILL_MAX_TOP, vocab below 2^31, and with a teacher_lse up to LMO_DISTILL_MAX_TAIL; rows below 2^31. */
#define LMO_DISTILL_SAVED 12
#define LMO_DISTILL_MAX_TOP 1024
#define LMO_DISTILL_MAX_TAIL 524288
int lmo_distill_fwd(const void* logits, const void* top, int top_dtype, const void* ids, int wide_ids,
                    const float* teacher_lse, const int64_t* labels, float tau, float hard, float* saved, float* coef,
                    float* loss, int64_t rows, int64_t vocab, int64_t k, int dtype, void* stream);

/* dlogits = round(dloss times the loss's gradient); tail: the forward had a teacher_lse; rows that neither count nor have a label are zeros. */
int lmo_distill_bwd(const void* logits, const void* top, int top_dtype, const void* ids, int wide_ids,
                    const int64_t* labels, float tau, const float* saved, const float* coef, const float* dloss,
                    void* dlogits, int64_t rows, int64_t vocab, int64_t k, int tail, int dtype, void* stream);

/* ---- differential attention -----------------------------------------------------------------------------------------
 * y[b, i, h] = (P1 - lam P2) v, Pm = softmax over the keys j that the query sees of scale q[b, i, 2 h + m - 1] k[b, j, 2 h' + m - 1],
 * h' = h hk / H: groups of H / hk heads share a pair of keys and its values. q [b, tq, 2 H, dh], k [b, tk, 2 hk, dh], v [b, tk,
 * hk, dv], bf16 or fp16, by strides in elements, multiples of 8, the last dimension's 1 and bases 16-byte aligned; dh a multiple
 * of 8 up to 128, dv up to 256. Query i sees the keys j < lengths[b] (NULL: tk) and, causal, j <= starts[b] + i (NULL: tk - tq);
 * one that sees none has zeros and no gradient. Keys and values at and past lengths[b] are not read into anything; lengths are
 * taken as within 0 .. tk. lam by strides too (0 where it is shared), fp32 where lam32, else the rows' type. */
typedef struct { const void* p; int64_t b, t, h; } lmo_strides;
typedef struct { int64_t b, tq, tk, h, hk, dh, dv; int causal; float scale; } lmo_diff_shape;

/* Floats of lmo_diff_attn_fwd's scratch; record: with second and lse. */
int64_t lmo_diff_attn_scratch(const lmo_diff_shape* shape, int record);

/* out [b, tq, H, dv] contiguous. For a backward, both or neither: second [b, tq, H, dv], P2 v, and lse [2, b, H, tq], the base-2
 * logarithms of the sums of exp(scores) (infinite for a query that sees no key). */
int lmo_diff_attn_fwd(const lmo_strides* q, const lmo_strides* k, const lmo_strides* v, const lmo_strides* lam, int lam32,
                      const int32_t* lengths, const int32_t* starts, void* out, void* second, float* lse, float* scratch,
                      const lmo_diff_shape* shape, int dtype, void* stream);

/* What dlam has: one value, one per head [H], or one per query and head [b, tq, H]; of lam's type. */
#define LMO_LAM_LAYER 0
#define LMO_LAM_HEAD 1
#define LMO_LAM_TOKEN 2

/* Floats of lmo_diff_attn_bwd's scratch. */
int64_t lmo_diff_attn_bwd_scratch(const lmo_diff_shape* shape, int lam_kind);

/* The gradients, contiguous, of the forward's shapes: dq, and, where wanted (dk and dv both or neither), dk, dv and dlam. dy is
 * contiguous, its rows H dv of up to 2^26 elements where there are several. Rows of dk and dv that no query sees are zeros. */
int lmo_diff_attn_bwd(const lmo_strides* q, const lmo_strides* k, const lmo_strides* v, const lmo_strides* lam, int lam32,
                      const int32_t* lengths, const int32_t* starts, const void* out, const void* second, const float* lse,
                      const void* dy, void* dq, void* dk, void* dv, void* dlam, int lam_kind, float* scratch,
                      const lmo_diff_shape* shape, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif
