/*
 * tmhd_lowbit.h - block-scaled low-bit storage: MXFP4 projections and a K/V
 * cache held in 8 bits.  Conventions and status codes are tmhd.h's.  Every
 * scale is a power of two, 2^(byte - 127) (byte 255: NaN), and a code that these
 * entries write times its scale is a finite bf16 number exactly.
 *
 * MXFP4 matrix [rows][k], k a multiple of 32
 *   codes : uint8 [rows][k / 2], two e2m1 values a byte, the even column in the
 *           low half; e2m1 = sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6
 *   scale : one byte per 32 columns, uint8 [ceil(k / 512)][4][R][4] with R =
 *           rows rounded up to a multiple of 4: byte b of entry (s, g, row) is
 *           that of columns 512 s + 128 b + 32 g .. + 31; bytes of columns or
 *           rows that do not exist are zero.  (One 32-bit word is what a lane of
 *           the 16 x 16 x 128 MFMA needs for 512 columns.)
 *   16-byte aligned bases, row strides of the codes a multiple of 16.
 *
 * 8-bit slot ("KVSlot8": the tmhd.h slot with 8-bit values)
 *   k : [H][cap / 32][D / 16][32][16]: value (t, d) of head h at tile t / 32,
 *       d / 16, t % 32, d % 16
 *   v : [H][cap / 32][D / 32][2][32][16]: value (t, d) at tile t / 32, d / 32,
 *       (t >> 2) & 1, d % 32, (t & 3) | ((t >> 3) & 3) << 2
 *   ks, vs : scale bytes [H][cap / 64], one per 64 tokens of a head
 *   format TMHD_KV8_E4M3 (OCP e4m3) or TMHD_KV8_INT8.  cap is a multiple of 64;
 *   rows in [tokens, round_up(tokens, 64)) are zero codes.
 *   Each 16-byte chunk is what one lane of a 32-key MFMA tile consumes.
 */
#ifndef TMHD_LOWBIT_H
#define TMHD_LOWBIT_H

#include "tmhd.h"
#include "tmhd_batch.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rows of bf16 to MXFP4.  Per 32 columns: e = floor(log2(max |x|)) - 2, not
 * below -125 (the OCP microscaling rule), code = x 2^-e rounded to the nearest
 * e2m1 value, ties to the even code, saturated at 6; a block that holds an
 * infinity or NaN gets the scale byte 255 and codes 0.  Sibling of
 * tmhd_token_quant_i8; the reference has no 4-bit path.  x: 16-byte aligned,
 * row stride a multiple of 8 elements.
 */
int tmhd_mxfp4_quant(uint8_t *q, uint8_t *scale, const void *x, int32_t rows, int32_t cols, int64_t x_stride,
                     void *stream);
/* The bf16 values that an MXFP4 matrix stands for (contiguous codes and output). */
int tmhd_mxfp4_dequant(void *x, const uint8_t *q, const uint8_t *scale, int32_t rows, int32_t cols, void *stream);

/*
 * out[m][n] = bf16(sum_k a[m][k] * b[n][k] (+ bias[n])) of two MXFP4 matrices,
 * fp32 accumulation.  lda / ldb: bytes between code rows; ldo: elements
 * between output rows; bias: bf16 or NULL.  Sibling of tmhd_gemm_w8a8.
 */
int tmhd_gemm_mxfp4(void *out, const uint8_t *a, const uint8_t *b, const uint8_t *a_scale, const uint8_t *b_scale,
                    const void *bias, int32_t m, int32_t n, int32_t k, int64_t lda, int64_t ldb, int64_t ldo,
                    void *stream);

/*
 * The form that an m x n x k product takes on a device of `cus` CUs (0: the
 * current one; 32-bit offsets): 16 x 16 tiles straight from memory, or tiles of the
 * stated rows x columns (X2: two workgroups a CU), which may stand behind whole
 * rounds of 256 x 256 tiles.  -1 for sizes that no product has.  Launches
 * nothing, and needs no GPU if cus > 0.
 */
enum {
  TMHD_MXFP4_ROWS,
  TMHD_MXFP4_64X64,
  TMHD_MXFP4_128X64,
  TMHD_MXFP4_128X128,
  TMHD_MXFP4_128X128X2,
  TMHD_MXFP4_256X256
};
int tmhd_gemm_mxfp4_form(int32_t m, int32_t n, int32_t k, int32_t cus);

/*
 * tmhd_mxfp4_quant of x [m][k] (bf16, ldx elements between rows) and the product
 * with b, with the same results: in one launch for few rows, whose blocks the
 * product quantizes as it reads them, else in two with the rows' codes and
 * scales in workspace (tmhd_linear_mxfp4_workspace_bytes; 16-byte aligned, may
 * be NULL if that is 0; calls that share it must be ordered).
 */
int tmhd_linear_mxfp4(void *out, const void *x, const uint8_t *b, const uint8_t *b_scale, const void *bias, int32_t m,
                      int32_t n, int32_t k, int64_t ldx, int64_t ldb, int64_t ldo, void *workspace,
                      int64_t workspace_bytes, void *stream);
int64_t tmhd_linear_mxfp4_workspace_bytes(int32_t m, int32_t n, int32_t k);

enum { TMHD_KV8_E4M3 = 0, TMHD_KV8_INT8 = 1 };

/* Rows row0 .. of an 8-bit slot as one attention segment (pointers to the slot's
 * own arrays; row0 a multiple of 64). */
typedef struct tmhd_kv8_segment {
  const void *k;
  const void *v;
  const uint8_t *ks;
  const uint8_t *vs;
  int32_t cap;    /* tokens the slot holds, a multiple of 64 (below 2^23) */
  int32_t row0;
  int32_t tokens; /* valid tokens of the view, 0 < tokens, row0 + tokens <= cap */
  int32_t format;
} tmhd_kv8_segment;

/*
 * tmhd_kv_pack_ranges into an 8-bit slot: each range's rows go to slot rows
 * dst .. (dst a multiple of 64), rows up to the next multiple of 64 become zero.
 * Per 64 tokens of a head, K and V apart: e = the least integer, not below
 * -117, with max |x| <= Q 2^e (Q = 448 for e4m3, 127 for int8), code = x 2^-e
 * rounded to nearest even, but not up to one that stands for 2^128 (in e4m3 blocks
 * with max |x| >= 1.9375 2^127 and int8 blocks that hold the largest finite bf16, the
 * code below is the last); an infinity or NaN gives the block the scale byte 255 and
 * codes 0.  zero_to of a range is not used.
 */
int tmhd_kv8_pack_ranges(const void *k, const void *v, int64_t token_stride, int64_t head_stride,
                         const tmhd_pack_range *ranges, int32_t n_ranges, const tmhd_kv8_segment *slot, int32_t heads,
                         int32_t head_dim, void *stream);

/*
 * The values of n views (all of one head count and head_dim) in bf16, into the
 * slot format of tmhd.h: view i at slot rows dst[i] .. (multiples of 64; no two views
 * in one 64-row block), zero up to the next multiple of 64.  Exact.
 */
int tmhd_kv8_expand(const tmhd_kv8_segment *views, const int32_t *dst, int32_t n, void *k_slot, void *vt_slot,
                    int64_t k_head_stride, int64_t vt_head_stride, int32_t vt_row_stride, int32_t heads,
                    int32_t head_dim, void *stream);
/* The values of one view as token-major [tokens][heads][head_dim] bf16. */
int tmhd_kv8_token_major(const tmhd_kv8_segment *view, void *k, void *v, int32_t heads, int32_t head_dim,
                         void *stream);

/*
 * One attention call over 8-bit segments: softmax(q k^T * scale) v over the
 * values they stand for, no mask.  Weighted values are summed in fp32 and divided
 * by the weights' sum at the end, with weights up to 2^8: values above about 2^120 /
 * tokens may overflow on the way.  Q is not rounded again (scores are scaled in
 * fp32).  Codes are turned into bf16 once for up to 256 query rows; calls of many more
 * rows take less time over a slot that tmhd_kv8_expand wrote, whose kernel rounds the
 * scaled Q to bf16.  Queries and outputs as in tmhd_attn_args.
 */
typedef struct tmhd_kv8_call {
  const void *q;
  int64_t q_token_stride;
  int64_t q_head_stride;
  const int32_t *q_rows;
  int32_t q_row0;
  int32_t lq;
  void *o;
  int64_t o_token_stride;
  int64_t o_head_stride;
  const int32_t *o_rows;
  int32_t o_row0;
  int32_t n_segments; /* 1 .. TMHD_MAX_SEGMENTS */
  tmhd_kv8_segment seg[TMHD_MAX_SEGMENTS];
} tmhd_kv8_call;

/*
 * n independent calls that share heads, head_dim, scale and the format, in as
 * few launches as they fit (16 calls and 24 segments each).  workspace holds
 * the partial results of key ranges (tmhd_attn_kv8_workspace_bytes; 16-byte
 * aligned; may be NULL if that is 0); calls that share it must be ordered.
 */
int tmhd_attn_fwd_kv8(const tmhd_kv8_call *calls, int32_t n, int32_t heads, int32_t head_dim, float scale,
                      void *workspace, int64_t workspace_bytes, void *stream);
int64_t tmhd_attn_kv8_workspace_bytes(const tmhd_kv8_call *calls, int32_t n, int32_t heads, int32_t head_dim);
/* Query rows of the items (32, 128 or 256) that the first launch of these calls is cut into on a device of `cus` CUs
 * (0: the current device); -1 for calls that are refused. */
int tmhd_attn_kv8_item_rows(const tmhd_kv8_call *calls, int32_t n, int32_t heads, int32_t head_dim, int32_t cus);

#ifdef __cplusplus
}
#endif

#endif /* TMHD_LOWBIT_H */
