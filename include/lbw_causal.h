/*
 * Causal self-attention on gfx950, from the projections to a cache held in 4 bits: norms of q and k by head with the
 * rotation, attention over packed sequences (forward and backward), and pages of e2m1 codes with the attention that reads
 * them. Conventions of lbw_attn.h and lbw_block.h: device pointers owned by the caller, int64 sizes and strides in
 * elements, a hipStream_t as void*, an int status; nothing is allocated and nothing synchronises, so every call can be
 * captured in a HIP graph. Arguments are checked before anything is launched; what lies in device memory (starts, lengths,
 * pages) cannot be checked then, and the kernels hold it inside the buffers.
 */
#ifndef LBW_CAUSAL_H
#define LBW_CAUSAL_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Every head of q [batch][len][q_heads][dim] and k [batch][len][k_heads][dim] (`dtype`; strides *_s_batch, *_s_tok,
 * *_s_head; channels contiguous) divided by the root of its mean square (plus eps), multiplied by q_weight / k_weight
 * ([dim] of vec_dtype, `dtype` or fp32, 16-byte aligned, or null: 1), and its first 2 * pairs channels turned as lbw_rotary turns them.
 * fp32 from the load to the one rounding. Outputs with strides qo_*, ko_*, apart from the inputs. k may be null with
 * k_heads 0. Limits of lbw_rotary.
 */
int lbw_norm_rotary(const void* q, const void* k, int dtype, int vec_dtype, int64_t batch, int64_t len, int64_t q_heads,
                    int64_t k_heads, int64_t dim, int64_t pairs, int64_t q_s_batch, int64_t q_s_tok, int64_t q_s_head,
                    int64_t k_s_batch, int64_t k_s_tok, int64_t k_s_head, const void* q_weight, const void* k_weight,
                    float eps, const void* positions, int pos_is_i64, int64_t p_s_batch, int64_t p_s_tok,
                    int64_t p_s_axis, int64_t pos_start, const double* freq, const int32_t* axis, int64_t axes,
                    int interleaved, float factor, void* q_out, void* k_out, int64_t qo_s_batch, int64_t qo_s_tok,
                    int64_t qo_s_head, int64_t ko_s_batch, int64_t ko_s_tok, int64_t ko_s_head, void* stream);

/*
 * Gradients of lbw_norm_rotary from those of its outputs, dq and dk (strides dq_*, dk_*; either null: zero): dq_in and
 * dk_in of `dtype` (strides qo_*, ko_*), dq_weight and dk_weight [dim] of vec_dtype (16-byte aligned); any of the four may be null. The sums
 * over tokens and heads are fp32 in a fixed order. `workspace`: lbw_norm_rotary_bwd_workspace_bytes(dim) bytes, 16-byte
 * aligned, used where a weight's gradient is asked for; calls that share it must not overlap.
 */
int lbw_norm_rotary_bwd(const void* dq, const void* dk, const void* q, const void* k, int dtype, int vec_dtype,
                        int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t pairs,
                        int64_t dq_s_batch, int64_t dq_s_tok, int64_t dq_s_head, int64_t dk_s_batch, int64_t dk_s_tok,
                        int64_t dk_s_head, int64_t q_s_batch, int64_t q_s_tok, int64_t q_s_head, int64_t k_s_batch,
                        int64_t k_s_tok, int64_t k_s_head, const void* q_weight, const void* k_weight, float eps,
                        const void* positions, int pos_is_i64, int64_t p_s_batch, int64_t p_s_tok, int64_t p_s_axis,
                        int64_t pos_start, const double* freq, const int32_t* axis, int64_t axes, int interleaved,
                        float factor, void* dq_in, void* dk_in, int64_t qo_s_batch, int64_t qo_s_tok,
                        int64_t qo_s_head, int64_t ko_s_batch, int64_t ko_s_tok, int64_t ko_s_head, void* dq_weight,
                        void* dk_weight, void* workspace, void* stream);
int64_t lbw_norm_rotary_bwd_workspace_bytes(int64_t dim);

/*
 * Attention over packed sequences: rows starts[s] .. starts[s + 1] of q [q_rows][q_heads][dim] are the queries of sequence
 * s, rows k_starts[s] .. k_starts[s + 1] of k and v [k_rows][k_heads][dim] its keys (int32, seqs + 1 each, not falling).
 * Head h of q reads head h / (q_heads / k_heads) of k and v. causal: the last query sees every key, each one before it one
 * less; a query that sees none gives 0, and so do the rows of no sequence. `dtype` bf16 or fp16, dim 64 or 128, strides
 * *_s_tok, *_s_head (multiples of 8, rows 16-byte aligned). Products of that type summed in fp32, softmax in fp32, its
 * weights rounded to the type before they meet v. out packed [q_rows][q_heads][dim]; rest: null, or the same of what
 * the rounding of out took off (rows of no sequence are left as they are). lse: null, or fp32
 * [q_heads][q_rows], the base-2 logarithm of each row's sum of exponentials (+inf where a row sees nothing).
 * sm_scale positive. seqs <= 65535, rows < 2^31, at most 4096 heads, token strides of dim to 2^24 - 1.
 */
int lbw_packed_attn_fwd(const void* q, const void* k, const void* v, int dtype, int64_t seqs, int64_t q_rows,
                        int64_t k_rows, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t q_s_tok,
                        int64_t q_s_head, int64_t k_s_tok, int64_t k_s_head, int64_t v_s_tok, int64_t v_s_head,
                        const int32_t* starts, const int32_t* k_starts, int causal, float sm_scale, void* out,
                        void* rest, float* lse, void* stream);

/*
 * Gradients of lbw_packed_attn_fwd: d_out (strides do_*) that of out; out, rest and lse as the forward left them. dq, dk, dv
 * packed like q, k, v would be; null where not wanted (dk and dv together). Rows of no sequence get zeros. Sums over heads
 * and rows have a fixed order. `workspace`: lbw_packed_attn_bwd_workspace_bytes(...) bytes, 16-byte aligned; calls that
 * share it must not overlap.
 */
int lbw_packed_attn_bwd(const void* d_out, const void* out, const void* rest, const float* lse, const void* q,
                        const void* k, const void* v, int dtype, int64_t seqs, int64_t q_rows, int64_t k_rows, int64_t q_heads,
                        int64_t k_heads, int64_t dim, int64_t do_s_tok, int64_t do_s_head, int64_t q_s_tok,
                        int64_t q_s_head, int64_t k_s_tok, int64_t k_s_head, int64_t v_s_tok, int64_t v_s_head,
                        const int32_t* starts, const int32_t* k_starts, int causal, float sm_scale, void* dq, void* dk,
                        void* dv, void* workspace, void* stream);
int64_t lbw_packed_attn_bwd_workspace_bytes(int64_t q_rows, int64_t k_rows, int64_t q_heads, int64_t k_heads);

#define LBW_KV4_PAGE 64   /* tokens of a page */

/*
 * Pages of a cache in 4 bits: for each page and head, of 64 tokens (32 channels of a token share a scale):
 *   k4  [page][head][64][dim / 2]: a token's codes in four parts, part p holding channels 32 j + 8 p .. + 8 of every j in
 *       order; two codes a byte, the lower channel in the low bits
 *   ks  [page][head][64][dim / 32]
 *   v4  [page][head][64 * dim / 2]: byte [half h][dim / 64: w][part p][n 0 .. 15][b 0 .. 1][e 0 .. 7] holds the codes of token
 *       32 h + 16 (e / 4) + 4 p + e % 4 at channels 64 w + 32 b + n (low bits) and 16 further
 *   vs  [page][head][64 * dim / 32]: byte [half h][part p][group dim / 32][e 0 .. 7], the scale of that token and group
 * Codes are e2m1 (LBW_W4_FP4), scales E8M0: a value is code * 2^(scale - 127); scale 255: the group held a value that is
 * not finite, and stands for NaN. A scale is the least power of two, 2^-125 or more, at which no magnitude is over 6;
 * codes are the nearest, ties to the even one; magnitudes over 3 * 2^126 count as that.
 *
 * The tokens of a call: rows starts[s] .. starts[s + 1] (int32, seqs + 1, not falling; null: one row for each sequence) are the
 * newest of the lens[s] (int32) tokens of sequence s, the last row its last token. Token t of sequence s lies in page
 * table[s][t / 64] (int32, row stride t_s_seq, `width` pages a row). Tokens past a row of the table, in pages that are not
 * 0 .. pages - 1 or before the first are not written, read as 0, and not attended.
 */

/* k, v [rows][heads][dim] of `dtype` (bf16 or fp16) into the pages. No page may be in the table twice for tokens of the call. */
int lbw_kv4_write(const void* k, const void* v, int dtype, int64_t seqs, int64_t rows, int64_t heads, int64_t dim,
                  int64_t k_s_tok, int64_t k_s_head, int64_t v_s_tok, int64_t v_s_head, const int32_t* starts,
                  const int32_t* lens, const int32_t* table, int64_t t_s_seq, int64_t width, int64_t pages,
                  uint8_t* k4, uint8_t* ks, uint8_t* v4, uint8_t* vs, void* stream);

/* The values of the call's tokens, bf16 [rows][heads][dim] (exact; rows of no sequence 0). */
int lbw_kv4_read(int64_t seqs, int64_t rows, int64_t heads, int64_t dim, const int32_t* starts, const int32_t* lens,
                 const int32_t* table, int64_t t_s_seq, int64_t width, int64_t pages, const uint8_t* k4,
                 const uint8_t* ks, const uint8_t* v4, const uint8_t* vs, void* k, void* v, void* stream);

/*
 * Attention of q [rows][q_heads][dim] (bf16 or fp16) over the pages: row r of sequence s sees the tokens up to its own, those
 * of them that are in the table where a length passes it.
 * Head h of q reads head h / (q_heads / heads). out packed, of q's type; a row that sees nothing, or of no sequence, is 0.
 * The values of the cache enter the products exactly, sums and softmax are fp32, its weights are rounded to bf16 for bf16
 * q and to twice that length for fp16. `workspace`: lbw_kv4_attn_workspace_bytes(...) bytes, 16-byte aligned; calls that
 * share it must not overlap.
 */
int lbw_kv4_attn(const void* q, int dtype, int64_t seqs, int64_t rows, int64_t q_heads, int64_t heads, int64_t dim,
                 int64_t q_s_tok, int64_t q_s_head, const int32_t* starts, const int32_t* lens, const int32_t* table,
                 int64_t t_s_seq, int64_t width, int64_t pages, const uint8_t* k4, const uint8_t* ks, const uint8_t* v4,
                 const uint8_t* vs, float sm_scale, void* out, void* workspace, void* stream);
/* (single: starts is null) */
int64_t lbw_kv4_attn_workspace_bytes(int64_t seqs, int64_t rows, int64_t q_heads, int64_t heads, int64_t dim,
                                     int64_t width, int single);

#ifdef __cplusplus
}
#endif

#endif
