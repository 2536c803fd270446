/*
 * exl3_layer.h — C-ABI of the MI355X (gfx950) kernels of the layer pipeline
 * around the trellis encoder (alpha2beta/EXL3_Intel_Arc_quantizer's
 * exl3_quant/hadamard.py, regularize.py and ldlq.py, which do this work with
 * torch tensor operations). Same conventions as exl3_encoder.h: device
 * buffers owned by the caller, nothing allocated, work enqueued on `stream`
 * (a hipStream_t, NULL = the null stream), 0 on success and a message in
 * exl3_last_error() otherwise. Matrices are float32, row-major, contiguous.
 * The last section holds the operators of a served model's 4-bit attention
 * cache.
 */
#ifndef EXL3_LAYER_H
#define EXL3_LAYER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Replaces preapply_had_l / preapply_had_r (hadamard.py:73-96) and their
 * in-place forms (hadamard.py:99-126): the orthonormal Sylvester matrix of
 * order 128, H[i][j] = (-1)^popcount(i & j) / sqrt(128), applied blockwise.
 * side = 0: out = H @ in on every 128-row block (rows % 128 == 0);
 * side = 1: out = in @ H on every 128-column block (cols % 128 == 0).
 * Computed as a fast Walsh-Hadamard transform in fp32; in == out is allowed. */
int exl3_hadamard128(const float* in, float* out, int64_t rows, int64_t cols, int side,
                     void* stream);

/* Division by a scale vector and the blockwise Hadamard transform in one pass
 * over HBM, the arithmetic of a division (correctly rounded fp32) followed by
 * exl3_hadamard128: the single steps that exl3_rotate and exl3_row_energy
 * join (regularize.py:171-181), for a caller that wants them apart.
 * side = 1: out = (in / divisor[col]) @ H, divisor of `cols` floats (the
 *           fold of sv before H_r); slice_sumsq, if not NULL, receives the
 *           sum of squares of every 32-element slice of every output row,
 *           slice_sumsq[row * (cols / 32) + slice] (the first pass of the
 *           row RMS that regularize takes next).
 * side = 0: out = H @ (in / divisor[row]), divisor of `rows` floats (the
 *           fold of su before H_l); slice_sumsq must be NULL.
 * divisor may be NULL (no division); in == out is allowed. */
int exl3_hadamard128_scaled(const float* in, float* out, int64_t rows, int64_t cols, int side,
                            const float* divisor, float* slice_sumsq, void* stream);

/* The two matrix passes of regularize (regularize.py:159-181) for a matrix of
 * multiples of 128, each one read of `in`: sums[row * (cols / 128) + segment] =
 * the sum of squares of every 128-element segment of the rows of (in / sv) H,
 * and out = H (((in / sv) H) / su). H is orthonormal, so the sums are taken
 * without it; out has the values of exl3_hadamard128_scaled side 1 (divisor
 * sv) and then side 0 (divisor su). sv holds `cols` floats, su `rows`; out
 * does not overlap in. */
int exl3_row_energy(const float* in, const float* sv, float* sums, int64_t rows, int64_t cols,
                    void* stream);
int exl3_rotate(const float* in, const float* sv, const float* su, float* out, int64_t rows,
                int64_t cols, void* stream);

/* Replaces weight_from_quantized (hadamard.py:129-140): out = (H (in) * su)
 * H * sv with the blockwise transforms of exl3_hadamard128, su of `rows`
 * floats (one per row), sv of `cols` floats, in one pass over HBM; the same
 * fp32 operations as the separate transforms and scalings. rows and cols are
 * multiples of 128; out and sv are 8-byte aligned; out does not overlap in. */
int exl3_unrotate(const float* in, const float* su, const float* sv, float* out, int64_t rows,
                  int64_t cols, void* stream);

/* Replaces decode_weight_from_storage (serialization.py:223-266): the weight
 * of a stored projection, exl3_unrotate of the codebook values of its packed
 * tiles (uint16 [rows / 16][cols / 16][16 K], the words exl3_pack_trellis
 * writes, 4-byte aligned) with codebook cb, in one pass. */
int exl3_decode_weight(const uint16_t* packed, const float* su, const float* sv, float* out,
                       int64_t rows, int64_t cols, int K, int cb, void* stream);

/* Second pass of block_rms (regularize.py:41-56) over slice sums made
 * elsewhere: out[o] = sqrt(S_o / n), S_o the sum of slice_sumsq[o * slices
 * + s] over s = 0 .. slices - 1 taken in slice order. */
int exl3_block_rms_from_slices(const float* slice_sumsq, float* out, int64_t outputs, int64_t n,
                               int64_t slices, void* stream);

/* The input-channel step of regularize (regularize.py:171-181): scales[r] as
 * exl3_block_rms_from_slices, 0.1 where that is below 1e-30, and su_out[r] =
 * su[r] * scales[r] / -1.24371088 + 1e-10. */
int exl3_input_scales(const float* slice_sumsq, const float* su, float* scales, float* su_out,
                      int64_t rows, int64_t n, int64_t slices, void* stream);

/* The output-channel step of regularize (regularize.py:102-168) for a
 * rows x cols matrix x: scales = its column RMS (32-row slices, as
 * exl3_block_rms) divided by their mean unless that is below 1e-30 (no
 * energy); where the scales apply, columns whose scale is below 1e-30 get
 * 0.1 and divisor[c] = sv[c] * scales[c] + 1e-10, elsewhere divisor = sv;
 * sv_out = divisor with 0 for those columns. decide: 0 the scales do not
 * apply, 1 they do, 2 they do if the skew is below 0.15; forced != 0: they
 * also apply to a matrix without energy. With diag (diag_len values,
 * diag_stride apart; may be NULL) the skew is the share of sum(sqrt(diag))
 * that its largest diag_len / 50 values hold and is written to flags[1];
 * without it flags[1] is read when decide = 2. flags (device doubles):
 * {has energy, skew, applied}. workspace: exl3_block_rms_workspace(rows,
 * cols, 0, 32) floats. */
int exl3_output_scales(const float* x, int64_t rows, int64_t cols, const float* diag,
                       int64_t diag_stride, int64_t diag_len, const float* sv, int decide,
                       int forced, float* workspace, int64_t workspace_elems, float* scales,
                       float* divisor, float* sv_out, double* flags, void* stream);

/* The sum of hessian_from_activations (calibration.py:337-357): h = scale *
 * X^T X for X of `tokens` rows (row stride ldx elements) and d columns, bf16
 * (bf16 != 0) or fp16, products and sums in float32, h float32 d x d
 * contiguous and exactly symmetric. d and ldx are multiples of 8, x is
 * 16-byte aligned. No float32 sum runs over more than chunk_tokens tokens
 * (>= 1; taken down to a multiple of 64, or 64): the chunks' sums are added
 * in float32, in token order. exl3_gram is exl3_gram_chunked with 8192.
 * workspace: exl3_gram_workspace floats (0 where the tokens are not shared
 * out). */
int exl3_gram_chunked(const uint16_t* x, int bf16, int64_t tokens, int64_t ldx, int64_t d,
                      float scale, int64_t chunk_tokens, float* h, float* workspace,
                      int64_t workspace_elems, void* stream);
int exl3_gram(const uint16_t* x, int bf16, int64_t tokens, int64_t ldx, int64_t d, float scale,
              float* h, float* workspace, int64_t workspace_elems, void* stream);

/* Floats of workspace exl3_gram needs on the current device, or -1 for a
 * shape it does not take. */
int64_t exl3_gram_workspace(int64_t tokens, int64_t d);

/* The damping of hessian_from_activations (calibration.py:359-385) on the
 * diagonal of h (row stride ld): adds max(1e-8, lambda * mean(diagonal)),
 * then replaces values below floor_value in magnitude by it. mean (device)
 * receives the mean. */
int exl3_damp_diagonal(float* h, int64_t d, int64_t ld, double lambda, float floor_value,
                       float* mean, void* stream);

/* Replaces block_rms (regularize.py:41-56): out = sqrt(S / n), S the sum of
 * squares along `dim` (0: over rows, one output per column; 1: over
 * columns, one per row) taken in slices of `blocksize` whose sums are
 * accumulated in slice order. workspace: device floats, at least
 * exl3_block_rms_workspace(rows, cols, dim, blocksize) of them (the slice
 * sums). */
int exl3_block_rms(const float* x, float* out, int64_t rows, int64_t cols, int dim, int blocksize,
                   float* workspace, int64_t workspace_elems, void* stream);

/* Floats of workspace exl3_block_rms needs (outputs x slices), or -1 for
 * invalid arguments. */
int64_t exl3_block_rms_workspace(int64_t rows, int64_t cols, int dim, int blocksize);

/* The diagonal-block step of a blocked Cholesky factorisation, which
 * replaces torch.linalg.cholesky_ex in block_ldl (ldlq.py:76-142): factors
 * the nb x nb block at `a` (leading dimension lda, lower triangle read,
 * nb <= exl3_cholesky_block_order()) in place into L (zeros above the
 * diagonal). A non-positive or NaN pivot k sets *info (device int32) to
 * offset + k + 1 unless it is already non-zero. */
int exl3_cholesky_diag_block(float* a, int64_t lda, int nb, int64_t offset, int32_t* info,
                             void* stream);

/* Replaces torch.linalg.cholesky_ex in block_ldl (ldlq.py:76-142): factors
 * the n x n matrix at `a` (contiguous, lower triangle read) in place into L;
 * the entries above the diagonal outside the diagonal blocks of order 128
 * are not touched, those inside become 0. inverses receives the inverses of
 * L's 16 x 16 diagonal tiles, [ceil(n / 16)][16][16] (a last tile that n
 * cuts is completed by an identity). A non-positive or NaN pivot k sets
 * *info (device int32) to k + 1 unless it is already non-zero. Two launches
 * per 128 columns, no host synchronisation. */
int exl3_cholesky(float* a, int64_t n, float* inverses, int32_t* info, void* stream);

/* Floats of `inverses` exl3_cholesky needs, or -1 for n < 1. */
int64_t exl3_cholesky_inverse_elems(int64_t n);

/* The fold of block_ldl (ldlq.py:120-142) for 16-wide blocks: out's block
 * column b = l's block column b times inverses[b] below the diagonal tile,
 * an identity in it, zeros above. n is a multiple of 16, l lower
 * triangular; out does not overlap l. */
int exl3_block_fold(const float* l, const float* inverses, float* out, int64_t n, void* stream);

/* Largest block order exl3_cholesky_diag_block accepts (128). */
int exl3_cholesky_block_order(void);

/* One 16-row block of an LDLQ traversal inside an encoder call: device
 * addresses (as integers) of the block's first row in W, in its
 * compensation rows, in Wq and in E = W - Wq (all float, row stride n), of
 * its (n / 16, 256) int16 states, and the block's first tile in the call's
 * batch. A call's blocks are listed in batch order, back to back
 * (tile0 of block b + 1 = tile0 + n / 16 of block b). The table itself is
 * read by the kernels, so it lives in device memory. */
typedef struct exl3_ldlq_block {
  int64_t w;
  int64_t comp;
  int64_t wq;
  int64_t err;
  int64_t states;
  int64_t n;
  int64_t tile0;
  int64_t reserved;
} exl3_ldlq_block;

/* Replaces the tile formation of one LDLQ step (ldlq.py:276-287) for every
 * block of an encoder call: x[tile0 + t][p] = W[r][16 t + c] + comp[r][16 t + c]
 * with (r, c) the row and column of tensor_core_perm(p) in a 16 x 16 tile.
 * x is f32 [tiles][256]; tiles = the sum of the blocks' n / 16. */
int exl3_ldlq_gather(const exl3_ldlq_block* blocks, int nblocks, int64_t tiles, float* x,
                     void* stream);

/* Replaces the write-back of one LDLQ step (ldlq.py:289-300) for every
 * block of an encoder call, from the encoder's tensor-core-order outputs
 * recon (f32 [tiles][256]) and idx (int16 [tiles][256]): Wq[r][16 t + c] =
 * recon, E[r][16 t + c] = W - recon at the same position, and the block's
 * states[t][p] = idx[tile0 + t][p]. */
int exl3_ldlq_scatter(const exl3_ldlq_block* blocks, int nblocks, int64_t tiles,
                      const float* recon, const int16_t* idx, void* stream);

/* ---- Products with weights as they are stored (no counterpart in the
 * reference). ---- */

/* Bytes of workspace that exl3_linear needs for `rows` rows and a (k, n) weight,
 * or -1 where it takes no such sizes. */
int64_t exl3_linear_workspace(int64_t rows, int64_t k, int64_t n, int type);

/* out (rows, n) = x W, W the (k, n) weight that exl3_decode_weight decodes from
 * `words` (k / 16 x n / 16 tiles of 16 K) with input scales su and output
 * scales sv: y = ((x su) H W_tiles) H sv. Rows of x are `stride` elements apart,
 * type 1 float16 or 2 bfloat16, as is out. half_scales: bit 0 if su, bit 1 if sv
 * is float16, else float32. Rows are transformed in float32 and count with 22
 * bits (11 where there are more than 64 of bfloat16), sums are float32. Rows with a
 * value that is not finite are NaN. k and n are multiples of 128; all memory is
 * 16-byte aligned. */
int exl3_linear(const void* x, int64_t stride, int64_t rows, int type, const uint16_t* words,
                const void* su, const void* sv, int half_scales, int64_t k, int64_t n, int K,
                int cb, void* out, void* workspace, int64_t workspace_bytes, void* stream);

/* ---- The 4-bit attention cache of a served model (no counterpart in the
 * reference). Element types: 0 float32, 1 float16, 2 bfloat16. Rows are
 * (tokens, heads, head_dim) tensors whose last axis is contiguous, given by
 * their first element and the strides of tokens and heads in elements.
 *
 * A cache is num_pages x kv_heads x (page_size / 32) tiles of 36 head_dim
 * bytes: page_size 32, 64, 128 or 256 tokens, head_dim 64, 128 or 256. A group
 * of 32 values x is held as y = H x / 8 (H the Sylvester matrix of order 32,
 * entries +-1), s = float16(bfloat16(max|y| / 7)), at most 9344, and codes
 * clamp(rint(y / s), -7, 7) + 8 in 4 bits; it stands for H ((code - 8) s) / 4.
 * A group with an infinity or a NaN is held as NaN. A tile of 32 tokens of one
 * kv head:
 *   16 head_dim bytes  key codes: dwords [token][j 0..3][group] of dims
 *                      32 group + 8 j .. + 7, dim 2 u in nibble u and
 *                      dim 2 u + 1 in nibble u + 4
 *   16 head_dim bytes  value codes: dwords [token / 8][r][token % 8] of dims
 *                      8 r .. 8 r + 7 in nibble order
 *    2 head_dim bytes  key scales: float16 [token][group]
 *    2 head_dim bytes  value scales: float16 [token / 8][group][token % 8]
 * The slot of a token is page * page_size + its position in the page. ---- */

/* Rotary positions of queries and keys in one launch: of every head's values
 * the pairs (i, i + pairs) (layout 0) or (2 i, 2 i + 1) (layout 1), i < pairs,
 *   y1 = magnitude (x1 cos a - x2 sin a), y2 = magnitude (x2 cos a + x1 sin a),
 * a = position * frequencies[i] (`inverse`: -a, which gives the gradient);
 * the other head_dim - 2 pairs values are copied. positions: int32, or int64
 * if wide_positions. Angles are taken in 64 bits, sums in 32. Outputs may be
 * the inputs, with their strides, and share no memory otherwise. q_heads or
 * k_heads may be 0, its pointers NULL. */
int exl3_rotary(const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t qo_token,
                int64_t qo_head, int q_heads, const void* k, int64_t k_token, int64_t k_head,
                void* k_out, int64_t ko_token, int64_t ko_head, int k_heads, int64_t tokens,
                int head_dim, int type, const void* positions, int wide_positions,
                const double* frequencies, int pairs, int layout, float magnitude, int inverse,
                void* stream);

/* exl3_rotary with positions of several axes (time, height and width):
 * positions is (num_axes, tokens), and pair i turns by positions[axes[i]]; a
 * pair whose axis is not one of them turns by 0. axes NULL: as exl3_rotary. */
int exl3_rotary_axes(const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t qo_token,
                     int64_t qo_head, int q_heads, const void* k, int64_t k_token, int64_t k_head,
                     void* k_out, int64_t ko_token, int64_t ko_head, int k_heads, int64_t tokens,
                     int head_dim, int type, const void* positions, int wide_positions,
                     const int32_t* axes, int num_axes, const double* frequencies, int pairs,
                     int layout, float magnitude, int inverse, void* stream);

/* The tables of one serving step from the requests' lengths (cached: tokens
 * held, fresh: new ones; negative counts as 0; at most 4096 requests). A
 * request holds ceil(cached / page_size) pages in its row of `tables`
 * (requests x width) and takes those its new tokens need from free_pages,
 * from *taken on; the new entries are written into the row, -1 once the
 * free_count entries are used up. Writes, for token t of max_tokens in request
 * order, slots[t] and positions[t] (its place in the request); -1 and 0 past
 * the last, slot -1 where no page is; starts [requests + 1], the prefix sums
 * of fresh; lengths [requests] = cached + fresh; taken_out = *taken plus the
 * pages used; status: 1 tokens without a page (the free ones ran out, in this
 * step or in the one that should have given a page held in part), 2 a request
 * outgrew its row, 4 more tokens than max_tokens, added up. */
int exl3_plan_step(const int32_t* cached, const int32_t* fresh, int requests, int32_t* tables,
                   int width, const int32_t* free_pages, int free_count, const int32_t* taken,
                   int page_size, int64_t max_tokens, int64_t* slots, int32_t* positions,
                   int32_t* starts, int32_t* lengths, int32_t* taken_out, int32_t* status,
                   void* stream);

/* Writes token t's keys and values to slots[t]; slots outside the cache are
 * skipped, and no slot may be given twice. With pairs > 0 (a multiple of 8)
 * the keys, and q_heads queries beside them into q_out (contiguous), first
 * turn by their positions as in exl3_rotary; keys stay in 32 bits between.
 * Rows are 16-byte aligned. */
int exl3_cache_append(const void* q, int64_t q_token, int64_t q_head, void* q_out, int q_heads,
                      const void* k, int64_t k_token, int64_t k_head, const void* v,
                      int64_t v_token, int64_t v_head, int64_t tokens, int type,
                      const int64_t* slots, const void* positions, int wide_positions,
                      const double* frequencies, int pairs, int layout, float magnitude,
                      void* pages, int64_t num_pages, int page_size, int kv_heads, int head_dim,
                      void* stream);

/* exl3_cache_append with positions of several axes, as in exl3_rotary_axes. */
int exl3_cache_append_axes(const void* q, int64_t q_token, int64_t q_head, void* q_out, int q_heads,
                           const void* k, int64_t k_token, int64_t k_head, const void* v,
                           int64_t v_token, int64_t v_head, int64_t tokens, int type,
                           const int64_t* slots, const void* positions, int wide_positions,
                           const int32_t* axes, int num_axes, const double* frequencies, int pairs,
                           int layout, float magnitude, void* pages, int64_t num_pages,
                           int page_size, int kv_heads, int head_dim, void* stream);

/* The keys and values that the entries at `slots` stand for, contiguous
 * (tokens, kv_heads, head_dim); zeros for slots outside the cache. */
int exl3_cache_read(const void* pages, int64_t num_pages, int page_size, int kv_heads, int head_dim,
                    const int64_t* slots, int64_t tokens, int type, void* k, void* v, void* stream);

/* Bytes of workspace that exl3_cache_attention needs with these arguments, or
 * -1. */
int64_t exl3_cache_attention_workspace(int64_t tokens, int q_heads, int kv_heads, int head_dim,
                                       int requests, int64_t max_new);

/* Attention of new tokens over the cache. Request r's queries are rows
 * starts[r] .. starts[r + 1] - 1 of q (float16 or bfloat16), its last of
 * lengths[r] positions; each attends its own position and the window - 1
 * before it: out = sum softmax(scale q . k) v, (tokens, q_heads, head_dim)
 * contiguous. Query head h reads kv head h / (q_heads / kv_heads). Rows that
 * attend nothing and rows of no request are 0; positions whose table entry
 * names no page of the cache are not attended. max_new, the most new tokens of
 * a request, or a bound, only chooses kernels: results depend on it in rounding
 * at most. Queries count with 22 bits, scores, maxima and sums are float32;
 * weights count with 22 bits for requests of up to 16 rows to a kv head (their
 * tokens times q_heads / kv_heads; 32 rows of head_dim 256), with 11 beyond. */
int exl3_cache_attention(const void* q, int64_t q_token, int64_t q_head, void* out, int64_t tokens,
                         int q_heads, int type, const void* pages, int64_t num_pages, int page_size,
                         int kv_heads, int head_dim, const int32_t* tables, int width,
                         const int32_t* starts, const int32_t* lengths, int requests, float scale,
                         int64_t window, int64_t max_new, void* workspace, int64_t workspace_bytes,
                         void* stream);

/* exl3_cache_attention with trees of drafted tokens. masks is (tokens, words) of
 * 64 bits (1 to 16 words). Of a request with n <= 64 words new tokens, which are
 * the last n of its lengths[r] positions, row i attends the positions before them
 * and new token j where bit j of its mask is set, of this sequence the last
 * `window` places; a mask may leave a row empty, which is 0 then. Requests with
 * more new tokens attend as in exl3_cache_attention. masks NULL:
 * exl3_cache_attention, with its workspace. */
int64_t exl3_cache_attention_trees_workspace(int64_t tokens, int q_heads, int kv_heads, int head_dim,
                                             int requests, int64_t max_new);
int exl3_cache_attention_trees(const void* q, int64_t q_token, int64_t q_head, void* out,
                               int64_t tokens, int q_heads, int type, const void* pages,
                               int64_t num_pages, int page_size, int kv_heads, int head_dim,
                               const int32_t* tables, int width, const int32_t* starts,
                               const int32_t* lengths, int requests, const int64_t* masks, int words,
                               float scale, int64_t window, int64_t max_new, void* workspace,
                               int64_t workspace_bytes, void* stream);

/* Masks and positions of trees of drafted tokens. Request r's are tokens
 * starts[r] .. starts[r + 1] - 1 of max_tokens, the last of lengths[r]
 * positions; parents[t] is the place among them (0 the first) of the token that t
 * follows, which is before t, or -1 (as is any other number) for the tokens
 * cached before. A token's mask, `words` (1 to 16) of 64 bits, names its ancestors
 * and itself, its position is that of the first new token plus its ancestors'
 * number. Requests of more than 64 words tokens are no trees: masks 0, positions
 * counting up. Tokens of no request: 0. */
int exl3_plan_tree(const int32_t* parents, const int32_t* starts, const int32_t* lengths,
                   int requests, int64_t max_tokens, int words, int64_t* masks, int32_t* positions,
                   void* stream);

/* The drafted tokens that the model would have chosen itself, of trees that
 * exl3_plan_tree planned with masks of `words` words. choices[t] is its
 * choice after token t; both are int64 if `wide`, else int32. A request keeps its
 * first certain[r] tokens (at least its first; certain NULL: that one), and then
 * from the last of them down, as long as there is one, the first token past them
 * whose parent is the last kept and which is the choice after it. places[t] is a
 * token's place among those kept, -1 if it is not (or of no request); kept[r] the
 * request's tokens cached before plus those kept, next[r] the choice after the
 * last kept, -1 where there are no new tokens. Of requests of more than 64 words
 * tokens, which are no trees, a token's parent is the one before it. */
int exl3_accept_trees(const void* tokens, const void* choices, int wide, const int32_t* parents,
                      const int32_t* starts, const int32_t* lengths, const int32_t* certain,
                      int requests, int64_t max_tokens, int words, int32_t* places, int32_t* kept,
                      void* next, void* stream);

/* exl3_accept_trees with the most words, 16. */
int exl3_accept_drafts(const void* tokens, const void* choices, int wide, const int32_t* parents,
                       const int32_t* starts, const int32_t* lengths, const int32_t* certain,
                       int requests, int64_t max_tokens, int32_t* places, int32_t* kept, void* next,
                       void* stream);

/* Moves the entry of every token t with 0 <= places[t] < its place in its request
 * to the slot of the request's token of that place, keys and values of all heads.
 * places grow along a request's kept tokens, as exl3_accept_drafts gives them, and
 * no two slots are alike. Moves from or to a slot outside the cache are skipped. */
int exl3_cache_keep(void* pages, int64_t num_pages, int page_size, int kv_heads, int head_dim,
                    const int64_t* slots, const int32_t* starts, const int32_t* places, int requests,
                    int64_t max_tokens, void* stream);

/* Gives back the pages of requests that held before[r] tokens and keep after[r]
 * of them (none: all its pages): entries ceil(after / page_size) to ceil(before /
 * page_size) of its row become -1, and their pages (where there are any) the last
 * of free_pages before *taken, in order; *taken_out = *taken less their number, 0
 * at least. Pages that have no place there, the first ones where more come back than
 * were taken, stay in their rows. */
int exl3_release_pages(const int32_t* before, const int32_t* after, int requests, int32_t* tables,
                       int width, int page_size, int32_t* free_pages, int free_count,
                       const int32_t* taken, int32_t* taken_out, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* EXL3_LAYER_H */
