// fp8.h — the host side of the 8-bit products (tu_fp8_quant.hip, tu_fp8_gemm.hip): e4m3 (or e5m2) values with one
// power-of-two scale, held as its exponent byte, for each block of 128.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace siren {

enum Fp8Type : int { FP8_F32 = 0, FP8_BF16 = 1, FP8_F16 = 2 };  // types of unquantised tensors
enum Fp8Act : int { FP8_ACT_NONE = 0, FP8_ACT_SINE = 1 };

inline int64_t fp8_blocks(int64_t n) { return n / 128 + (n % 128 != 0); }  // of any n >= 0: no sum to overflow
inline int64_t fp8_padded(int64_t n) { return fp8_blocks(n) * 128; }            // bytes of a quantised row
inline int64_t fp8_scale_cols(int64_t n) { return (fp8_blocks(n) + 3) / 4 * 4; }  // scale bytes of a row: whole words

// x (rows, cols) of row stride ld, times mult (rows, cols; bf16, contiguous; nullable) ->
//   q  (rows, padded cols), s  (rows or row blocks, scale_cols(cols))       blocks along the columns
//   qt (cols, padded rows), st (cols or column blocks, scale_cols(rows))    the transpose, blocks along the rows
// either pair may be NULL. tiles: one scale per 128 x 128 instead of per 1 x 128. colsum (row blocks, cols), nullable:
// each row block's column sums of the unquantised values.
struct Fp8Quant {
    const void* x;
    int64_t ld, rows, cols;
    const void* mult;
    uint8_t *q, *s, *qt, *st;
    float* colsum;
    int type, e5m2, tiles, panels;  // panels, as in Fp8Operand: 1 of q, 2 of qt
};
void launch_fp8_quant(hipStream_t st, const Fp8Quant& a);
void launch_fp8_quant2(hipStream_t st, const Fp8Quant& a, const Fp8Quant& b);  // in one launch where their types are alike
// out[c] = sum over the row blocks of colsum (blocks, cols), in order
void launch_fp8_colsum(hipStream_t st, const float* colsum, int64_t blocks, int64_t cols, float* out);

// One operand of a product, block scales per row (shift 0) or per 128 rows (shift 7). data: rows of `padded` bytes, or in
// panels (padded / 64, rows, 64): 64 k of all rows, then the next 64.
struct Fp8Operand {
    const uint8_t* data;
    const uint8_t* scale;
    int64_t rows;
    int shift, panels;
};
// out (a.rows, b.rows) = act(a b^T + bias), sums over k; deriv (nullable, bf16): omega cos(omega z) of the sine
struct Fp8Product {
    Fp8Operand a, b;
    int64_t k;
    const float* bias;
    int act;
    float omega;
    void* out;
    int type;
    void* deriv;
    int e5m2_a;
    void* ws;
};
// y (m, n) = act(x w^T + bias) for a few rows m in one launch, x quantised on the way (w: rows, tiles)
bool fp8_few_rows(int64_t m, int64_t n, int64_t k);
void launch_fp8_few_rows(hipStream_t st, const void* x, int type, int64_t ld, int64_t m, int64_t k, const uint8_t* w,
                         const uint8_t* sw, int64_t n, const float* bias, int act, float omega, void* y, void* deriv);
int64_t fp8_product_ws_bytes(int64_t m, int64_t n, int64_t k);
void launch_fp8_product(hipStream_t st, const Fp8Product& p);

}  // namespace siren
