/*
 * loopback_block.h -- C ABI of libloopback_block.so: MI355X (gfx950) kernels of a transformer block's training step that
 * stand beside those of loopback_lm.h: the join of a block's output with the residual stream (a norm after the block, a
 * gate, a residual scale, dropout, the add, the next norm) and dropout alone, each forward and backward in one pass over
 * its rows, and the gated feed-forward block on the matrix cores.
 *
 * Conventions: device pointers to contiguous row-major tensors at element alignment (16-byte aligned rows of a multiple
 * of 8 elements take the wider loads); dtype is LDR_F32, LDR_BF16 or LDR_F16 (loopback_read.h); every statistic and sum
 * is fp32, results are rounded once from fp32; stream is a hipStream_t; nothing synchronizes with the host or allocates.
 * The return value is 0, a negative code (rejected before any launch: -1 argument, -2 shape, -3 alignment, -4 dtype) or
 * a positive hipError_t. Sums have a fixed order: the same call gives the same bits.
 */
#ifndef LOOPBACK_BLOCK_H
#define LOOPBACK_BLOCK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LBK_ABI_VERSION 3   /* 2: lbk_join_bwd takes x in h's place; 3: lbk_product_tiling */
int lbk_abi_version(void);

/* ---- dropout ----------------------------------------------------------------------------------------------------
 * The mask of a (rows, d) tensor is never stored: element (r, c) is kept where its 16 bits are at or above `drop` (0 to
 * 65536, the probability's 65536ths), and a kept value is multiplied by 65536 / (65536 - drop). The bits are the half
 * c mod 2 of word (c mod 8) / 2 of Philox-4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011)
 * with the 64-bit key rng[0] and the counter (c / 8, r, site, rng[1] mod 2^32). rng: two int64 on the device, read when
 * the kernel runs (a captured graph draws a new mask when they have changed). A dropped NaN or infinity is 0. */
int lbk_dropout(const void* x, const int64_t* rng, uint32_t site, int drop, void* out, int64_t rows, int64_t d, int dtype,
                void* stream);

/* ---- block join --------------------------------------------------------------------------------------------------
 * z = y; post: z = y r1 post, r1 = rsqrt(mean(y^2) + eps); gate: z = z gate[row / gate_rows]; z = scale z; drop: as above;
 * h = round(x + z); pre: n = round((x + z) r2 pre), r2 = rsqrt(mean((x + z)^2) + eps). post, gate, pre may be NULL. gate
 * has ceil(rows / gate_rows) rows of d; rng is read where drop > 0. r_post and r_pre [rows] receive r1 and r2 for the
 * backward (NULL: not wanted). d up to LBK_JOIN_MAX_WIDTH, rows below 2^31. */
#define LBK_JOIN_MAX_WIDTH 8192
int lbk_join_fwd(const void* x, const void* y, const void* post, const void* gate, int64_t gate_rows, const void* pre,
                 const int64_t* rng, uint32_t site, int drop, float scale, float eps, void* h, void* n, float* r_post,
                 float* r_pre, int64_t rows, int64_t d, int dtype, void* stream);

/* Floats of lbk_join_bwd's scratch. */
int64_t lbk_join_scratch(int64_t rows, int64_t d, int64_t gate_rows);

/* The gradients for dh and dn (either may be NULL, not both; dn needs pre): dx = dh + the norm's share, dy through the
 * dropout, scale, gate and norm, and the sums dpost, dgate (gate's shape), dpre, rounded once. Each result may be NULL
 * (not wanted). x and y are the forward's inputs: the norm's gradient is formed at x + z before its rounding. */
int lbk_join_bwd(const void* dh, const void* dn, const void* x, const void* y, const void* post, const void* gate,
                 int64_t gate_rows, const void* pre, const float* r_post, const float* r_pre, const int64_t* rng,
                 uint32_t site, int drop, float scale, void* dx, void* dy, void* dpost, void* dgate, void* dpre,
                 float* scratch, int64_t rows, int64_t d, int dtype, void* stream);

/* ---- gated feed-forward block, bf16 and fp16 ---------------------------------------------------------------------
 * y = (a(x Wg^T) * (x Wu^T)) Wd^T for x [t, d], w = [Wg; Wu] [2 n, d], Wd [d_out, n]; activation 0: a(g) = g sigmoid(g)
 * (silu), 1: gelu in its tanh form. Sizes below 2^31. Every matrix has its rows ld elements apart (up to 2^22). Operands are
 * 16-byte aligned with ld a multiple of 8, all ld elements of a row readable -- lbk_pad_rows makes such a copy of one that
 * is not -- or, for up to LBK_FEW_TOKENS tokens of lbk_linear_fwd, and of lbk_ffn_gate_up without `saved`, of any alignment.
 * Results may have any. */
#define LBK_FEW_TOKENS 32

/* out [rows, ld] = x [rows, cols], contiguous, with zeros past the columns. */
int lbk_pad_rows(const void* x, int64_t rows, int64_t cols, int64_t ld, void* out, int dtype, void* stream);

/* Bytes of `saved`, what the backward needs of the two projections: (u a'(g), a(g)) per (token, column) in the kernels' own
 * order, 24 bits each (six bytes per token and column, of blocks of 32 x 32). 16-byte aligned. */
int64_t lbk_ffn_saved_bytes(int64_t t, int64_t n);

/* act [t, n] = round(a(x Wg^T) * (x Wu^T)): both projections, the activation and the product in one kernel. saved: NULL
 * where no backward follows. */
int lbk_ffn_gate_up(const void* x, int64_t ldx, const void* w, int64_t ldw, void* act, int64_t ld_act, void* saved, int64_t t,
                    int64_t d, int64_t n, int activation, int dtype, void* stream);

/* dgate_up [t, 2 n]: the gradients of the two projections for dy [t, d] (the block's output), the product dy Wd and the
 * activation's gradient in one kernel. w_down [d, n]. */
int lbk_ffn_dgate_up(const void* dy, int64_t ld_dy, const void* w_down, int64_t ldw, const void* saved, void* dgate_up,
                     int64_t ld_dgu, int64_t t, int64_t n, int64_t d, int dtype, void* stream);

/* The block's plain products: y [t, n] = x [t, k] w [n, k]^T; dx [t, k] = dy [t, n] w [n, k]; dw [n, k] = dy^T x (contiguous).
 * The summed dimension is split where that fills the GPU; scratch has lbk_linear_scratch(columns and rows of the result,
 * summed dimension) floats (NULL where that is 0), 16-byte aligned. */
int64_t lbk_linear_scratch(int64_t columns, int64_t rows, int64_t summed);

/* Which tiles the product of a result of `columns` x `rows` takes on the tiled kernels: 0 is 128 x 128, 1 is 256 x 256 and
 * 2 is 192 x 256 (columns x rows), and into *splits in how many the summed dimension is split. product: 0 the plain ones, 1 the
 * gate and up projection (columns 2 n, rows t, summed d), 2 the gradients of the two (columns n, rows t, summed d). */
int lbk_product_tiling(int product, int64_t columns, int64_t rows, int64_t summed, int* splits);
int lbk_linear_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, void* y, int64_t ldy, float* scratch, int64_t t,
                   int64_t k, int64_t n, int dtype, void* stream);
int lbk_linear_dx(const void* dy, int64_t ld_dy, const void* w, int64_t ldw, void* dx, int64_t ld_dx, float* scratch, int64_t t,
                  int64_t n, int64_t k, int dtype, void* stream);
int lbk_linear_dw(const void* dy, int64_t ld_dy, const void* x, int64_t ldx, float* scratch, void* dw, int64_t t, int64_t n,
                  int64_t k, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LOOPBACK_BLOCK_H */
