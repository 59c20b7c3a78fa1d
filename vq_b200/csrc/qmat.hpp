// qmat.hpp -- products of 8-bit codes with a scale for each row (tokens) and for each channel (matrix rows).
//
//   y[i][j] = (sum_k q[i][k] w[j][k]) s[i] t[j] + b[j]        q, w: int8; the sum is a whole number, exact in 32 bits
//
// for one matrix, or for one matrix per group of consecutive rows (offsets); and the gradient of that with respect to what the rows
// were quantized from.  rows.cu makes codes, product_tc.cu, product_few.cu and product_plain.cu multiply them.
#pragma once
#include <cstddef>
#include <cstdint>

namespace vqb {

class CudaDevice;

enum ValueType : int { VALUE_F32 = 0, VALUE_F16 = 1, VALUE_BF16 = 2 };
inline size_t value_bytes(int type) { return type == VALUE_F32 ? 4 : 2; }

// 128 * 128 * QMAT_MOST_WIDTH < 2^31: no sum of products of codes leaves 32 bits
constexpr size_t QMAT_MOST_WIDTH = 131071;
constexpr size_t QMAT_MOST_GROUPS = 1024; // the products keep the groups' rows and tiles in shared memory
constexpr size_t QMAT_MOST_ROWS = (size_t(1) << 30) - 1; // (rows and tiles are numbered in 32 bits)

// codes rows are 16-byte aligned: what TMA and 16-byte loads ask for
inline size_t codes_ld(size_t width) { return (width + 15) / 16 * 16; }

struct Qmat {
    size_t groups = 0, outputs = 0, inputs = 0;
    int8_t *codes = nullptr;  // groups x outputs x codes_ld(inputs), zeros behind the inputs
    float *scales = nullptr;  // groups x outputs
    int8_t *turned = nullptr; // groups x inputs x codes_ld(outputs): the codes transposed, for gradients; null without
};

// One product: `channels` rows of codes for each group times n rows.  Nothing that may still be running has written the codes and scales of channels
// (whoever makes a matrix waits for it); the rest is read once the kernels before this one have ended.
struct Product {
    const int8_t *codes = nullptr;        // groups x channels x codes_ld(width)
    const float *channel_scales = nullptr; // groups x channels; null: 1
    size_t groups = 1, channels = 0, width = 0;
    const int8_t *rows = nullptr; // n x rows_ld; of three digits, three times that, the first digits in front
    size_t rows_ld = 0, n = 0;
    int digits = 1; // 3: a row's values are 65536 d0 + 256 d1 + d2
    const float *row_scales = nullptr; // n
    const int64_t *offsets = nullptr;  // groups + 1: group g has rows offsets[g] .. offsets[g + 1] - 1; null: one group of all rows
    const float *bias = nullptr;       // groups x channels, or null
    void *y = nullptr;                 // n x y_ld values of y_type
    int y_type = VALUE_F32;
    size_t y_ld = 0;
    bool zero_rest = false;   // rows of no group become 0 (otherwise they are left as they are)
    bool rows_follow = false; // the kernel directly before wrote `rows` and `row_scales`, and had itself waited for all that was before it
};

// codes[i][k] = x[i][k] / s[i] to the nearest whole number (halves to even, of the real quotient), s[i] = max(max_k |x[i][k]| / 127, 2^-126); s is 0 for
// a row of zeros and NaN for one with an infinity or a NaN, with codes 0.  Bytes behind the row's width stay as they are.
// product_follows: the caller's next launch is launch_product or launch_product_few (which waits for these codes itself; other kernels that may start early take
// what was written for invariant).
void launch_quantize_rows(CudaDevice &dev, const void *x, int type, size_t n, size_t width, size_t ld, int8_t *codes, size_t ld_codes, float *scales, bool product_follows);
// u[i][j] = x[i][j] column_scales[g][j] of the row's group g as the whole number next to u / t, t = max(max |u| / (127 * 65536), 2^-126), in three digits (Product).  24 bits of the row's
// largest are what a sum of the u in f32 holds.  (With the 15 that two digits of 128 have, rows of one large entry and many small ones, as a softmax's gradient has, lose the small
// ones: of 128,256 outputs 5 to 15 % of the result where a channel's weights have a mean of 0.1 to 0.3 of their spread.  The third digit takes half as long again on the tensor cores:
// 4096 x 4096 x 4096 bf16 in 120 us, 81 before.)  digits: n x ld_codes of each.
void launch_digit_rows(CudaDevice &dev, const void *x, int type, size_t n, size_t width, size_t ld, const float *column_scales, size_t groups, const int64_t *offsets,
                       int8_t *digits, size_t ld_codes, float *scales);
// turned[g][k][j] = codes[g][j][k]
void launch_turn_codes(CudaDevice &dev, const int8_t *codes, size_t groups, size_t rows, size_t width, int8_t *turned);
// rows of any alignment to rows of codes_ld(width) bytes
void launch_align_codes(CudaDevice &dev, const int8_t *codes, size_t n, size_t width, size_t ld, int8_t *aligned);

void launch_product(CudaDevice &dev, const Product &p);
// Up to sixteen rows with one matrix: takes one or two as values (p.rows and p.row_scales unused) or, where x is null, codes (16-byte aligned rows).  False, having done nothing,
// when it does not take them.  The matrix may not be written by what is still running.
bool launch_product_few(CudaDevice &dev, const Product &p, const void *x, int type, size_t ld);
void launch_product_plain(CudaDevice &dev, const Product &p); // CUDA cores

} // namespace vqb
