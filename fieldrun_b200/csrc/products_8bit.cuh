// Products in 8-bit integers: how rows are stored, and what the kernels of the operators take.
//
// A row (a token's entries, or the weights of one output channel) is stored as codes with one float32 scale,
//     a = max |x|,  scale = a / 127,  code = 127 x / a rounded to an integer, half to even,
// and a product of two rows is scale_x * scale_w * sum of code_x * code_w: the sum is one of whole numbers, so it is exact and does
// not depend on the order in which it is made, on the other rows of the step or on how the work was cut.  Rows of codes are filled up
// with zeros to a multiple of 128 (a k-block of the tensor core: the 128 bytes of a swizzled row).  A row whose largest entry is below
// 2^-96 is stored as zeros with scale zero (127 / a would leave float32's range); one with an entry that is not finite gets the scale
// NaN and codes of zero, so that whatever it is multiplied with becomes NaN.
#pragma once

#include "common.cuh"

#define FRB_8BIT_KBLOCK 128            // entries of a k-block; rows of codes are multiples of it
#define FRB_8BIT_ROWS 16               // a weight's rows are filled up to multiples of it
#define FRB_8BIT_MOST_INNER 131072     // 127^2 entries of it stay below 2^31
#define FRB_8BIT_SMALLEST_ROW 1.2621774e-29f      // 2^-96

// Gates of a unit with two products in.
enum Frb8BitGate { FRB_GATE_SILU = 0, FRB_GATE_GELU_TANH = 1 };

namespace frb_products8 {

__host__ __device__ inline int up_to(int n, int step) { return (n + step - 1) / step * step; }

// Lists of tiles: rows tile_row0[t] .. of expert tile_expert[t], at most `tile_rows` of them and none beyond offsets[expert + 1].
// Null pointers: one expert whose rows are all rows.
struct Lists {
    const int* tile_expert;
    const int* tile_row0;
    const int* num_tiles;
    const int* offsets;
    int max_tiles;
    int tile_rows;
};

struct Product {
    const void* w;             // codes [experts][parts][F up to 16][K up to 128]
    const float* w_scale;      // [experts][parts][F up to 16]
    int experts, parts;        // parts 2: gate and up
    int F, K;
    const void* x;             // codes [rows][K up to 128]
    const float* x_scale;      // [rows]
    int rows;
    Lists lists;
    void* out;                 // [rows][F]
    int out_type;
    int gate;                  // parts 2: Frb8BitGate
    float limit;               // parts 2: > 0 the clamped gate
    int* status;               // 0, or the code of the wait that gave up
};

// rows_8bit.cu
int rows_codes(const void* x, int x_type, int rows, int K, const int* places, int copies, void* codes, float* scales, cudaStream_t stream);
int plan(const int* ids, int tokens, int top_k, int experts, int tile_rows, int* offsets, int* row_of_assign, int* tile_expert, int* tile_row0,
         int* num_tiles, cudaStream_t stream);
int combine(const float* y, const float* weights, const int* row_of_assign, int tokens, int top_k, int width, void* out, int out_type,
            cudaStream_t stream);
// products_8bit.cu
int product(const Product& p, cudaStream_t stream);

}  // namespace frb_products8
