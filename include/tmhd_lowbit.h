/*
 * tmhd_lowbit.h - block-scaled low-bit storage: MXFP4 projections.  Conventions and status codes are tmhd.h's.  Every
 * scale is a power of two, 2^(byte - 127) (byte 255: NaN), so a stored value
 * times its scale is a bf16 number exactly.
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
 */
#ifndef TMHD_LOWBIT_H
#define TMHD_LOWBIT_H

#include "tmhd.h"

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

#ifdef __cplusplus
}
#endif

#endif /* TMHD_LOWBIT_H */
