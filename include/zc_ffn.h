/* zc_ffn.h — C ABI of the dense feed-forward operators on B200 (sm_100a): microscaled 4-bit matrices (quantisation, products) and
 * the gated block in 16 bits with its gradient. They stand beside the expert layer of zc_moe.h: the same block without routing, for
 * the shared or dense feed-forward layers of a model. No counterpart in the reference, whose 4-bit format is affine and whose engine
 * does not train.
 *
 * Conventions (those of zc_moe.h where not stated here)
 *  - Plain C: ZC_OK or a negative code; zc_last_error() has the text. Everything is validated on the host before a launch.
 *  - No handle and no allocation: every buffer is the caller's device memory, on the current device. Codes, tiled scales and the buffers of the 16-bit block
 *    are 16-byte aligned (its rows too); the plain matrices of the microscaled calls need no more than their type's alignment, and no row stride in
 *    particular (those whose rows are 16-byte aligned are read and written in wider pieces); row-major scales need none. Calls are
 *    stream-ordered, do not block the host and may be captured into a graph (a process's first call of an entry point too: an entry point has
 *    kernels of several sizes and types, and what a capture meets first is loaded then). Calls on different streams share nothing but the status word of the device.
 *  - Row strides count elements; that of a single row has no meaning and may be anything.
 *  - What a call writes shares no memory with what it reads, or the call is refused; columns side by side in the rows of one buffer share none.
 *  - Zero tokens (rows) is a valid call: nothing is read or written, but that gradients of the weights become zero.
 *  - Results do not depend on what else runs and are the same bits on every call: no atomics, a fixed order of sums.
 *  - A wait inside a kernel is bounded (zc_ffn_wait_limit); one that runs out raises ZC_STATUS_TIMEOUT in a word of the device (zc_ffn_status).
 *    The results of that call are not meaningful then; the kernel ends what it has started and the device stays usable.
 *
 * Microscaled matrix (MX4) of [rows, cols], cols a multiple of 32: the MXFP4 format of the OCP Microscaling Formats specification v1.0.
 *  - codes: [rows, cols / 2] bytes, two e2m1 values a byte (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6),
 *    the even column in the low half;
 *  - scales: one byte s per 32 columns of a row, the factor 2^(s - 127); s = 255 makes the 32 values NaN. They are stored in tiles of
 *    128 rows x 4 scales, as the tensor cores read them: byte (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4 of tile
 *    (row / 128, block / 4); tiles of 512 bytes, row-major, ceil(rows / 128) x ceil(cols / 128) of them. Scales past the last column
 *    must not be 255 (the library writes 0); those past the last row are not used.
 */
#ifndef ZC_FFN_H
#define ZC_FFN_H

#include "zc_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of the scales of a [rows, cols] matrix: ceil(rows / 128) * ceil(cols / 128) * 512. */
int zc_mx4_scale_bytes(uint32_t rows, uint32_t cols, uint64_t* bytes);

/* x [rows, cols] (dtype; row stride ld elements) -> codes, scales. Per 32 values of a row, a = their largest magnitude:
 * scale 2^e with e = floor(log2 a) - 2 (at least -127; a = 0: -127), value -> x 2^-e rounded to the nearest e2m1 value, ties to
 * the even code, magnitudes above 6 to 6. A NaN or an infinity among the 32 makes their scale 255 and their codes 0. */
int zc_mx4_quantize(const void* x, int dtype, uint32_t rows, uint32_t cols, uint64_t ld, void* codes, void* scales, void* stream);

/* The values of a microscaled matrix in dtype, out row stride ld elements. BF16 and F32 hold every one below 2^128 exactly (those
 * above, which zc_mx4_quantize does not produce, become infinite); F16 rounds once. */
int zc_mx4_dequantize(const void* codes, const void* scales, uint32_t rows, uint32_t cols, void* out, int dtype, uint64_t ld, void* stream);

/* Row-major scales [rows, cols / 32], as checkpoints hold them, -> the tile layout. */
int zc_mx4_tile_scales(const void* row_scales, uint32_t rows, uint32_t cols, void* scales, void* stream);

/* out [tokens, rows] = x . w^T, FP32 accumulation, rounded once to out_dtype (BF16, F16 or F32; row stride out_ld elements); w is a
 * microscaled matrix [rows, cols]. x [tokens, cols] is either one too (x NULL: x_codes, x_scales are its codes and scales) or plain
 * (x not NULL, x_dtype, row stride x_ld): then it is quantised by the rule of zc_mx4_quantize on the way, and x_codes, x_scales are
 * scratch of the sizes of its codes and scales, whose contents after the call are not specified. */
int zc_mx4_linear(const void* x, int x_dtype, uint64_t x_ld, void* x_codes, void* x_scales, uint32_t tokens, uint32_t cols,
                  const void* w_codes, const void* w_scales, uint32_t rows, void* out, int out_dtype, uint64_t out_ld, void* stream);

/* h [tokens, ffn] = silu(x . gate^T) * (x . up^T): both products, the activation and the product of the two in one kernel; gate and up
 * [ffn, cols] microscaled, x and h as x and out above. The activation is evaluated on the FP32 sums. */
int zc_mx4_gated(const void* x, int x_dtype, uint64_t x_ld, void* x_codes, void* x_scales, uint32_t tokens, uint32_t cols,
                 const void* gate_codes, const void* gate_scales, const void* up_codes, const void* up_scales, uint32_t ffn,
                 void* h, int out_dtype, uint64_t out_ld, void* stream);

/* The gated block in 16 bits. x [tokens, hidden] (row stride x_ld), gate and up [ffn, hidden], all of one dtype (BF16 or F16), hidden and
 * ffn multiples of 8. h [tokens, ffn] = silu(x . gate^T) * (x . up^T), rounded once from FP32. g and u (both or neither): the two products
 * themselves, [tokens, ffn], for zc_gated_backward: in FP32 (saved_dtype ZC_F32), or rounded to dtype (saved_dtype = dtype), which halves what
 * is kept between the two calls and adds two roundings of dtype to the gradients' error. */
int zc_gated_forward(const void* x, uint64_t x_ld, const void* gate, const void* up, int dtype, uint32_t tokens, uint32_t hidden, uint32_t ffn,
                     void* h, void* g, void* u, int saved_dtype, void* stream);

/* Its gradient: dh [tokens, ffn] (row stride dh_ld) and what zc_gated_forward was given and gave.
 *   s = sigmoid(g);  dg = dh u s (1 + g (1 - s));  du = dh g s
 *   dx [tokens, hidden] = dg . gate + du . up;  dgate [ffn, hidden] = dg^T . x;  dup = du^T . x
 * dg and du [tokens, ffn] are written too (the operands of the products, rounded to dtype); dx or both of dgate and dup may be NULL
 * where they are not wanted. dx, dgate and dup are rounded once from FP32 sums. */
int zc_gated_backward(const void* dh, uint64_t dh_ld, const void* x, uint64_t x_ld, const void* gate, const void* up, const void* g, const void* u,
                      int saved_dtype, int dtype, uint32_t tokens, uint32_t hidden, uint32_t ffn, void* dg, void* du, void* dx, void* dgate, void* dup, void* stream);

/* Waits for `stream` and returns the current device's status word of these operators (then clears it). The word is that of all streams of the device: a
 * call may return, and clear, a time-out of another stream's kernels; none is cleared that no call returned. */
int zc_ffn_status(void* stream, uint32_t* status);

/* How often a wait inside the products' kernels polls before it gives up, for the calls of this process that follow (a captured call keeps what it was
 * captured with), up to 2^27: a poll takes about a microsecond at most. before (may be NULL) receives the limit so far. */
#define ZC_FFN_WAIT_POLLS 1048576u   /* the limit that holds until the first such call */
int zc_ffn_wait_limit(uint32_t polls, uint32_t* before);

#ifdef __cplusplus
}
#endif
#endif /* ZC_FFN_H */
