/*
 * Operators of a transformer block around its attention on gfx950: the residual stream's gated norm (forward and
 * backward), rotary positions, and linears with 4-bit weights. Conventions of lbw_attn.h: device pointers owned by
 * the caller, int64 sizes and strides in elements, a hipStream_t as void*, an int status; nothing is allocated and
 * nothing synchronises, so every call can be captured in a HIP graph. Arguments are checked before anything is
 * launched.
 */
#ifndef LBW_BLOCK_H
#define LBW_BLOCK_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element formats (LBW_DTYPE_BF16 and LBW_DTYPE_FP16 of lbw_attn.h, and fp32). */
#define LBW_DTYPE_FP32 2

/* Norm kinds. */
#define LBW_NORM_NONE 0
#define LBW_NORM_LAYER 1   /* (x - mean) * rsqrt(var + eps) */
#define LBW_NORM_RMS 2     /* x * rsqrt(mean(x^2) + eps) */

#define LBW_NORM_MAX_WIDTH 12288

/*
 * What stands between two sub-layers of a block, in one pass over the rows:
 *   p = post(y) * post_weight            the branch's own norm (post_norm; LBW_NORM_NONE: p = y)
 *   s = residual_scale * x + branch_scale * gate * p
 *   h = (norm(s) * weight + bias) * (1 + scale) + shift
 * with every step in fp32 and one rounding each to s_out and h_out (the norm reads s before it is rounded). Replaces
 * the gated residual addition, the norms and their modulation around the sub-layers of the DiT's block
 * (lingbot/models/lingbot_world/transformer.py:281-360). x, y [batch][len][width] of `dtype` (strides *_s_batch,
 * *_s_tok; channels contiguous); y may be null (then s = residual_scale * x). gate, shift, scale: null, or vectors of
 * `vec_dtype` (`dtype` or fp32) with strides *_s_batch, *_s_group: token t of batch entry b takes row (b, t /
 * group_len); stride 0 for a vector that all share. weight, bias, post_weight: null or [width] of vec_dtype. s_out,
 * h_out: packed [batch][len][width] of `dtype`; either may be null, h_out has to be where norm is LBW_NORM_NONE.
 * batch * len <= 2^30.
 */
int lbw_gated_norm(const void* x, const void* y, int dtype, int vec_dtype, int64_t batch, int64_t len, int64_t width,
                   int64_t x_s_batch, int64_t x_s_tok, int64_t y_s_batch, int64_t y_s_tok,
                   const void* gate, int64_t gate_s_batch, int64_t gate_s_group,
                   const void* shift, int64_t shift_s_batch, int64_t shift_s_group,
                   const void* scale, int64_t scale_s_batch, int64_t scale_s_group, int64_t group_len,
                   const void* weight, const void* bias, const void* post_weight, int norm, int post_norm, float eps,
                   float residual_scale, float branch_scale, void* s_out, void* h_out, void* stream);

/*
 * Gradients of lbw_gated_norm: ds, dh (packed, of `dtype`; either may be null) are those of s_out and h_out; the
 * other inputs as there. Any of the outputs may be null: dx, dy packed [batch][len][width] of `dtype`; dgate, dshift,
 * dscale packed [batch][groups][width] of vec_dtype where `rowwise` says that the vector has rows of its own (1:
 * gate, 2: shift, 4: scale), else [width]; dweight, dbias, dpost_weight [width] of vec_dtype. groups: rows of the
 * modulation vectors an entry of the batch has (1 where all share them); those past the last token get zeros. The
 * sums over rows are formed in fp32 in a fixed order. `workspace` holds lbw_gated_norm_bwd_workspace_bytes() bytes,
 * 16-byte aligned (only read and written where a vector's gradient is asked for); calls that share a workspace must
 * not overlap.
 */
int lbw_gated_norm_bwd(const void* ds, const void* dh, const void* x, const void* y, int dtype, int vec_dtype,
                       int64_t batch, int64_t len, int64_t width,
                       int64_t x_s_batch, int64_t x_s_tok, int64_t y_s_batch, int64_t y_s_tok,
                       const void* gate, int64_t gate_s_batch, int64_t gate_s_group,
                       const void* scale, int64_t scale_s_batch, int64_t scale_s_group, int rowwise,
                       int64_t groups, int64_t group_len, const void* weight, const void* bias,
                       const void* post_weight, int norm, int post_norm, float eps, float residual_scale,
                       float branch_scale, void* dx, void* dy, void* dgate, void* dshift, void* dscale, void* dweight,
                       void* dbias, void* dpost_weight, void* workspace, void* stream);

/* Bytes of scratch lbw_gated_norm_bwd needs for its sums over rows. */
int64_t lbw_gated_norm_bwd_workspace_bytes(int64_t batch, int64_t len, int64_t width, int64_t groups,
                                           int64_t group_len);

#define LBW_ROTARY_MAX_DIM 512

/*
 * Rotary positions: the first 2 * pairs channels of every head of q [batch][len][q_heads][dim] and k
 * [batch][len][k_heads][dim] (`dtype`; strides *_s_batch, *_s_tok, *_s_head; channels contiguous) are rotated,
 *   (a, b) -> factor * (a cos w - b sin w, b cos w + a sin w),   w = position[axis of the pair] * freq[pair],
 * the others copied. interleaved: pair i is channels (2 i, 2 i + 1), else (i, pairs + i). inverse: w negated (the
 * gradient's rotation). The angle is formed in 64 bits and reduced to a turn before the sine and cosine are taken in
 * fp32, so far positions keep theirs; one rounding to `dtype`. freq: float64 [pairs], radians a position. axis: int32
 * [pairs] with values in 0 .. axes - 1, or null (all 0); a pair of another axis comes out as NaN. positions: int64
 * (pos_is_i64) or int32 with strides p_s_batch, p_s_tok, p_s_axis, or null: token t of every entry is at pos_start + t
 * on every axis. q_out, k_out as q, k (strides qo_*, ko_*); a call in place passes the same pointer and strides twice,
 * any other overlap is an error of the caller. k may be null with k_heads 0. dim even is not required; 2 * pairs <= dim
 * <= LBW_ROTARY_MAX_DIM, batch * len <= 2^30, 4096 heads at most.
 */
int lbw_rotary(const void* q, const void* k, int dtype, int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads,
               int64_t dim, int64_t pairs, int64_t q_s_batch, int64_t q_s_tok, int64_t q_s_head, int64_t k_s_batch,
               int64_t k_s_tok, int64_t k_s_head, const void* positions, int pos_is_i64, int64_t p_s_batch,
               int64_t p_s_tok, int64_t p_s_axis, int64_t pos_start, const double* freq, const int32_t* axis,
               int64_t axes, int interleaved, int inverse, float factor, void* q_out, void* k_out,
               int64_t qo_s_batch, int64_t qo_s_tok, int64_t qo_s_head, int64_t ko_s_batch, int64_t ko_s_tok,
               int64_t ko_s_head, void* stream);

/* Code formats of the 4-bit weights. */
#define LBW_W4_INT4 0   /* value code - zero, a zero for each group (8 without zeros) */
#define LBW_W4_FP4 1    /* e2m1: sign, two exponent bits, one mantissa bit: +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} */

/*
 * 4-bit weights of a linear [n][k], in tiles of 16 rows x 128 columns (n, k rounded up; nt = ceil(n / 16), kt =
 * ceil(k / 128)), `group` (32, 64 or 128) columns sharing a scale:
 *   w4     uint8 [nt][kt][1024]: word j (0 .. 3) of lane 16 q + r holds the codes of row r at columns 32 j + 8 q + i,
 *          i = 0 .. 7; its nibble s holds i = s for LBW_W4_FP4 and i = 2 s (s < 4), 2 s - 7 (s >= 4) for LBW_W4_INT4
 *   scale  bf16  [nt][kt][16][128 / group]
 *   zero   uint8 [nt][kt][16][128 / group], LBW_W4_INT4 only, or null (8); lbw_quant_w4 makes 0 .. 15, any is taken
 * (All 16-byte aligned.) A weight is scale * value. Rows and columns past n and k hold scale 0 where a whole group
 * lies there, and any code.
 *
 * lbw_quant_w4 makes them from w [n][k] (bf16, or fp32 when w_is_fp32; row stride s_row): scale = amax / 6 (fp4),
 * amax / 7 (int4 without zeros) or (max(x, 0) - min(x, 0)) / 15 (with zeros), rounded to bf16, codes to the nearest
 * value of the rounded scale by arithmetic in fp32 (integers: w * (1 / scale) + zero, ties to even codes; fp4: w / scale,
 * ties to the smaller magnitude). Values are finite; a group that holds none but zeros gets scale 0.
 */
int lbw_quant_w4(const void* w, int w_is_fp32, int64_t n, int64_t k, int64_t s_row, int fmt, int64_t group,
                 uint8_t* w4, uint16_t* scale, uint8_t* zero, void* stream);

/* Beside the element format of lbw_gemm_w4: the bias is fp32. */
#define LBW_W4_BIAS_FP32 256

/*
 * out[m][n] = x w^T + bias: x [m][k] of `dtype` (bf16 or fp16; row stride x_s_row; the k that w was packed for), w
 * as above, bias [n] of `dtype` (of fp32 where dtype has LBW_W4_BIAS_FP32 added) or null, out [m][n] packed of `dtype`.
 * Codes enter the products exactly; sums and group scales are fp32, the bias is added in fp32, with one rounding at the
 * end. m <= 2^24, n <= 1048560, k <= 2^20. With LBW_W4_INT4 a row of x that holds an infinity gives NaN (the codes'
 * offset is taken off the sums), and one of bf16 values of 2^115 and more may (the offset's part leaves fp32's range).
 */
int lbw_gemm_w4(const void* x, int dtype, int64_t m, int64_t k, int64_t x_s_row, const uint8_t* w4,
                const uint16_t* scale, const uint8_t* zero, int fmt, int64_t group, int64_t n, const void* bias,
                void* out, void* stream);

#ifdef __cplusplus
}
#endif

#endif
