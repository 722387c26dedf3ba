/*
 * nkmx.h — C-ABI of the MI355X (gfx950) microscaled storage operators: 4-bit floating point
 * (quantize, decode, product) and 8-bit activation checkpoints (save with the activation, load,
 * gradient of the activation, weight gradient).  They live in libnkmx.so, beside the 2-bit gradient
 * quantizer of nklq.h, and follow its conventions: plain pointers and sizes, `stream` is a
 * hipStream_t as an opaque pointer (NULL = the default stream), every call is asynchronous on it,
 * allocates no device memory, keeps no state, and may be made from several host threads at once.
 * Return value: 0, one of the NKMX_E* argument errors (< 0), or the launch's own hipError_t (> 0).
 *
 * A matrix [rows, cols] is cut along its rows into blocks of 32 neighbouring columns.  A block has
 * one power of two 2^e as its scale, kept as the byte e + 127.  Rows are padded to whole steps of
 * 128 columns with zeros, so a packed matrix has steps = ceil(cols / 128) steps a row:
 *
 *   mx4   codes  uint8 [rows, steps * 64], 2 codes a byte, the even column in the low half:
 *                bit 3 the sign, bits 2..0 = 0, .5, 1, 1.5, 2, 3, 4, 6
 *         e    = floor(log2(max |x|)) - 2; the code of x / 2^e is the nearest value, ties to the
 *                even code, 6 beyond the last
 *   act8  codes  int8 [rows, steps * 128]
 *         e    = floor(log2(max |x|)) - 6; the code is x / 2^e rounded to the nearest whole number,
 *                ties to even, limited to -127 .. 127
 *   both  scales uint8 [rows, steps * 4]; e >= -127; a block of zeros has the byte 0; a block that
 *                holds an infinity or a NaN has the byte 255 and codes 0 and decodes to NaN
 *
 * Codes start on 16-byte boundaries, scales on 4-byte ones (NKMX_EALIGN otherwise); they are
 * contiguous.  Matrices of numbers have a leading dimension in elements (ld >= cols) and need the
 * alignment of their type only.  rows, cols, ld < 2^31.  A product, weight gradient or transpose whose
 * launch would take 2^32 threads (2^27 rows of a weight, 2^30 columns of a transpose, as orders of
 * magnitude) gets NKMX_ERANGE; the passes along rows take all sizes.
 */
#ifndef NKMX_H
#define NKMX_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NKMX_VERSION 100
#define NKMX_BLOCK 32 /* columns that share a scale */
#define NKMX_STEP 128 /* columns that rows are padded to */

#define NKMX_OK 0
#define NKMX_ENULL (-1)  /* a required pointer is NULL */
#define NKMX_EALIGN (-2) /* a pointer is not aligned as described above */
#define NKMX_ERANGE (-3) /* a size, leading dimension, type or activation is out of range */
#define NKMX_EALIAS (-4) /* an output overlaps another buffer of the call (exceptions are named at the calls) */
#define NKMX_EWORK (-5)  /* the workspace is missing, too small or not on a 16-byte boundary */

/* element types */
#define NKMX_F32 0
#define NKMX_BF16 1
#define NKMX_F16 2

/* activations: none, x Phi(x) with the normal distribution function, x / (1 + e^-x) */
#define NKMX_NONE 0
#define NKMX_GELU 1
#define NKMX_SILU 2

/*
 * x [rows, cols] -> mx4.  transpose = 0: the packed matrix is x.  transpose = 1: it is the transpose,
 * [cols, rows] with blocks along x's rows (what the gradient of a product's input contracts over).
 */
int nkmx_mx4_quantize(const void* x, int type, uint64_t rows, uint64_t cols, uint64_t ldx, uint8_t* codes,
                      uint8_t* scales, int transpose, void* stream);

/* mx4 [rows, cols] -> out, rounded once to its type (exact in fp32 and bf16). */
int nkmx_mx4_dequantize(void* out, int type, uint64_t rows, uint64_t cols, uint64_t ldo, const uint8_t* codes,
                        const uint8_t* scales, void* stream);

/*
 * y[i, j] = sum over c of a[i, c] * b[j, c] (+ bias[j]): a [m, k] and b [n, k] are mx4, y and bias are of
 * `type`; bias may be NULL.  Summed in fp32, rounded once.  k = 0 gives the bias or zeros.
 */
int nkmx_mx4_matmul(void* y, int type, uint64_t m, uint64_t n, uint64_t k, uint64_t ldy, const uint8_t* a_codes,
                    const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales, const void* bias,
                    void* stream);

/*
 * The same with a = the mx4 of x [m, k] (of y's type): bit for bit nkmx_mx4_quantize followed by
 * nkmx_mx4_matmul, in one launch where there are few rows.  `workspace` (nkmx_mx4_linear_workspace
 * bytes, on a 16-byte boundary) holds a's codes where they are laid out; NULL if that is 0 bytes.
 */
int nkmx_mx4_linear(void* y, const void* x, int type, uint64_t m, uint64_t n, uint64_t k, uint64_t ldy, uint64_t ldx,
                    const uint8_t* b_codes, const uint8_t* b_scales, const void* bias, void* workspace,
                    uint64_t workspace_bytes, void* stream);
uint64_t nkmx_mx4_linear_workspace(uint64_t m, uint64_t n, uint64_t k);

/*
 * x -> act8 codes of x, and y = fn(x) of the same type unless fn is NKMX_NONE (then y is NULL).  fn is
 * taken of x itself, not of its codes, in fp32.  For fp32 they and their slopes are off by a few
 * roundings of the result (gelu, below -1.25: some 14 + 1.5 x^2 of them); for the 16-bit types gelu's
 * formula is within 7.5e-7 of the normal distribution function.  y may be x (with the same leading
 * dimension).  With an activation, codes and scales may both be NULL: y alone is written, the same bits.
 */
int nkmx_act8_save(const void* x, void* y, int type, int fn, uint64_t rows, uint64_t cols, uint64_t ldx, uint64_t ldy,
                   uint8_t* codes, uint8_t* scales, void* stream);

/* act8 [rows, cols] -> out, rounded once to its type (exact in fp32 and bf16). */
int nkmx_act8_load(void* out, int type, uint64_t rows, uint64_t cols, uint64_t ldo, const uint8_t* codes,
                   const uint8_t* scales, void* stream);

/* dx = dy * fn'(x^), x^ the value the codes stand for; dx may be dy (with the same leading dimension). */
int nkmx_act8_grad(void* dx, const void* dy, int type, int fn, uint64_t rows, uint64_t cols, uint64_t lddx,
                   uint64_t lddy, const uint8_t* codes, const uint8_t* scales, void* stream);

/*
 * dw[j, c] = (accumulate ? dw[j, c] : 0) + sum over i of dy[i, j] * x^[i, c] for dy [t, n] of `type` and x
 * [t, k] in act8; dw is fp32 [n, k].  db (fp32 [n], may be NULL) gets the sums of dy's columns the same
 * way.  Every product is exact and the sums are fp32 for all three types (an fp32 dy keeps all its bits
 * from 2^-110 up).  k = 0 gives db alone (dw, codes and scales are not read or written).  The result does
 * not depend on timing.  `workspace`: nkmx_act8_wgrad_workspace bytes on a 16-byte boundary, NULL if that
 * is 0.
 */
int nkmx_act8_wgrad(float* dw, float* db, const void* dy, int type, uint64_t t, uint64_t n, uint64_t k, uint64_t lddw,
                    uint64_t lddy, const uint8_t* codes, const uint8_t* scales, int accumulate, void* workspace,
                    uint64_t workspace_bytes, void* stream);
uint64_t nkmx_act8_wgrad_workspace(int type, uint64_t t, uint64_t n, uint64_t k);

/* Text for a return value (static storage); NKMX_VERSION the library was built from. */
const char* nkmx_strerror(int code);
int nkmx_version(void);

#ifdef __cplusplus
}
#endif
#endif /* NKMX_H */
