/*
 * tpx_b200 — C ABI for sequences of different lengths laid end to end, without padding, and a cache that holds keys and
 * values in 4 bits. Conventions are those of tpx_b200.h; activations are bf16.
 *
 * Tokens. A call has T token rows. cu_seqlens [B + 1] (device, int32, not decreasing) cuts them into sequences: sequence b has
 * the rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1, none at all is allowed. Rows in front of the first and behind the last
 * sequence belong to none: outputs have theirs left as they were. cu_seqlens == NULL: row b is the one token of sequence b, T == B.
 *
 * The cache of one layer is `pages` pages [kv_heads][36 H] bytes; a page holds 32 tokens of one sequence, table[b][i] (int32,
 * rows of table_cols) names the page of the tokens 32 i .. 32 i + 31 of sequence b. An entry outside [0, pages) is no page:
 * what is written there is dropped, keys there are seen by nobody. lengths[b] tokens are cached before the call (below 0 counts as 0); the
 * call's token i of sequence b has the place lengths[b] + i. Places from 32 table_cols on are none either. Nothing here advances lengths.
 *
 * 64 consecutive values of a key or value row (the bf16 values) share a minimum and a scale, both bf16:
 *   scale = bf16((max - min) / 15), code = min(15, round((x - min) / scale)) (0 where scale is 0), value = min + code * scale.
 * Rows of 64 with an infinity or a NaN have NaN for both. One head of a page is
 *   K codes   [32 tokens][4][H / 32] 32-bit words: word (t, i) holds values 32 i + 8 t + 0..7, lowest nibble first
 *   K params  [32 tokens][H / 64] pairs (scale, min)
 *   V codes   [4 groups of 8 tokens][8][4][2][H / 64] words: word (g, t, u, h) holds values 64 h + 8 g + 0..7 of token t + 4 u of its group
 *   V params  as K params
 * in that order: a lane of the attention kernel finds the operands of its matrix instructions in 16-byte pieces.
 */
#ifndef TPX_PACKED_H
#define TPX_PACKED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  uint8_t* pool; /* 16-byte aligned */
  const int32_t *table, *lengths;
  int64_t pages, table_cols, B, kv_heads, H;
} TpxInt4Cache;

/* One pass over the heads behind a q/k/v linear: RMS norm of every query and key head (norm weights [H], bf16 or fp32; NULL: no
 * norm; the mean of squares in fp32, which heads with values from 2^60 on may pass), then the rotation of its first rot values in pairs (i, i + rot / 2) by the token's row of the table ep [2][max_pos][ld_ep]
 * fp32 (cosines, sines; NULL: none; positions outside [0, max_pos) leave the head as it is); q and k are rounded once, to bf16, and written to
 * q_out [T][Nq][H] and k_out [T][Nkv][H] (NULL: not written). With a cache the keys (as rounded) and the values v go to their places in it. pos NULL: a
 * token's position is its place in the cache (0 without one). H: a multiple of 16 up to 256, with a cache 64 or 128; rot a multiple of 16. Rows
 * of q, k and v are ld* elements apart, heads lie side by side; all of them 16-byte aligned. q may be NULL with Nq == 0. */
typedef struct {
  const uint16_t *q, *k, *v;
  const void *q_norm, *k_norm;
  const float* ep;
  const int64_t* pos;
  const int32_t* cu_seqlens;
  uint16_t *q_out, *k_out;
  const TpxInt4Cache* cache; /* host pointer, NULL: none */
  int64_t T, Nq, Nkv, H, ldq, ldk, ldv, rot, max_pos, ld_ep;
  float eps;
  int norm_is_f32;
} TpxHeadPrep;
int tpx_head_prep(const TpxHeadPrep* a, void* stream);

/* The values that the cache holds in the places of T tokens, as bf16: k_out, v_out [T][kv_heads][H], zeros where there is no page. */
int tpx_int4_read(const TpxInt4Cache* cache, const int32_t* cu_seqlens, int64_t T, uint16_t* k_out, uint16_t* v_out, void* stream);

/* Attention over the cache: softmax(q k^T * scale) v for the T query rows q [T][Nq][H] (ldq elements apart) over the tokens of
 * their sequence in the cache, the call's own included: token i of sequence b sees the places 0 .. lengths[b] + i (causal) or all
 * of lengths[b] + n. A row that sees nothing becomes zero. Weights that differ from their row's largest by 2^126 or more are 0, weights times scales
 * are rounded to 11 bits, or to 2^-31 of the largest such product of their row and group of 64 where that is more. Sums are fp32, of weights up to 2^8
 * before they are divided: values from 2^100 on may pass them (here and in tpx_packed_attention). scratch: tpx_int4_attention_scratch_bytes(...) bytes that nobody else
 * uses meanwhile, 256-byte aligned, of any content. */
typedef struct {
  const uint16_t* q;
  const TpxInt4Cache* cache;
  const int32_t* cu_seqlens;
  uint16_t* out; /* [T][Nq][H] */
  void* scratch;
  size_t scratch_bytes;
  int64_t T, Nq, ldq;
  float scale;
  int causal;
} TpxInt4Attention;
size_t tpx_int4_attention_scratch_bytes(int64_t T, int64_t B, int64_t Nq, int64_t kv_heads, int64_t H);
int tpx_int4_attention(const TpxInt4Attention* a, void* stream);
/* The same for the sequences with lengths[b] > 0 alone; rows of the others are left as they are in out. */
int tpx_int4_attention_behind(const TpxInt4Attention* a, void* stream);

/* Attention over whole prompts: softmax(q k^T * scale) v for the T rows q [T][Nq][H], k and v [T][Nkv][H] (ld* elements apart, heads
 * side by side, 16-byte aligned), each within its sequence; causal: token i of a sequence sees the keys 0 .. i. Only the rows of
 * sequences are written to out [T][Nq][H]. H 64 or 128, at most 128 query heads per key head, scale > 0. Values that a row does not see
 * never reach it, infinities and NaN included. Waits inside the kernel are bounded: tpx_packed_status reads and clears the code of one that gave up. */
typedef struct {
  const uint16_t *q, *k, *v;
  const int32_t* cu_seqlens;
  uint16_t* out;
  int64_t T, B, Nq, Nkv, H, ldq, ldk, ldv;
  float scale;
  int causal;
} TpxPackedAttention;
int tpx_packed_attention(const TpxPackedAttention* a, void* stream);
/* The same for the sequences with lengths[b] <= 0 alone (lengths [B], int32 on the device: tokens cached before the call); rows of the
 * others are left as they are in out. With tpx_int4_attention_behind on the same out every row of a call gets what it has to see. */
int tpx_packed_attention_new(const TpxPackedAttention* a, const int32_t* lengths, void* stream);
int tpx_packed_status(void* stream, unsigned* status_host);

#ifdef __cplusplus
}
#endif

#endif
