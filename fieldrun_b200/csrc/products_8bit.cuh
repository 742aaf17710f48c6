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
#include "pairs.cuh"

#define FRB_8BIT_KBLOCK 128            // entries of a k-block; rows of codes are multiples of it
#define FRB_8BIT_ROWS 16               // a weight's rows are filled up to multiples of it
#define FRB_8BIT_MOST_INNER 131072     // 127^2 entries of it stay below 2^31
#define FRB_8BIT_SMALLEST_ROW 1.2621774e-29f      // 2^-96

// Gates of a unit with two products in: silu or tanh-gelu of the gate, times up; with a limit L > 0 the clamped gate.
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
    const void* x;             // codes [rows][K up to 128], or (x_scale null) rows as they are, x_stride entries apart, which the kernel rounds itself
    const float* x_scale;      // [rows]
    int x_stride, x_type;      // without x_scale
    int rows;
    bool weights_final;        // the weights were complete before the kernel before this one began
    Lists lists;
    void* out;                 // [rows], out_stride entries from one to the next
    int out_stride, out_type;
    int gate;                  // parts 2: Frb8BitGate
    float limit;               // parts 2: > 0 the clamped gate
    int* status;               // 0, or the code of the wait that gave up
};

// rows_8bit.cu; early: the kernel after this one may start before this one's wait is over (what it reads ahead is complete)
int rows_codes(const void* x, int x_type, int x_stride, int rows, int K, const int* places, int copies, void* codes, float* scales, bool early, cudaStream_t stream);
int plan(const int* ids, int tokens, int top_k, int experts, int tile_rows, int* offsets, int* row_of_assign, int* tile_expert, int* tile_row0,
         int* num_tiles, cudaStream_t stream);
int combine(const float* y, int y_stride, const float* weights, const int* row_of_assign, int tokens, int top_k, int width, void* out, int out_type,
            cudaStream_t stream);
// products_8bit.cu
bool tokens_fit(int rows, int K);
int product(const Product& p, cudaStream_t stream);

}  // namespace frb_products8

// ----------------------------------------------------------------------------- rows as codes, on the device

#ifdef __CUDACC__
namespace frb_products8 {

// Eight neighbouring entries as they are stored; those behind the row's end (`left`) are zeros.
template <typename T> struct Eight;
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void read(const float* p, int left, bool whole) {
        if (whole && left >= 8) {
            const float4 a = load4(p), b = load4(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    __device__ __forceinline__ float entry(int i) const { return v[i]; }
};
template <> struct Eight<bf16> {
    uint32_t w[4];
    __device__ __forceinline__ void read(const bf16* p, int left, bool whole) {
        if (whole && left >= 8) {
            const uint4 raw = *reinterpret_cast<const uint4*>(p);
            w[0] = raw.x; w[1] = raw.y; w[2] = raw.z; w[3] = raw.w;
            return;
        }
        const unsigned short* bits = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (2 * i < left ? (uint32_t)bits[2 * i] : 0u) | (2 * i + 1 < left ? (uint32_t)bits[2 * i + 1] << 16 : 0u);
    }
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0u; }
    __device__ __forceinline__ float entry(int i) const { return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16); }
};

// The magnitude's bits order like the magnitudes, with infinities and NaN above all numbers.
template <typename T>
__device__ __forceinline__ uint32_t top_of(const Eight<T>& v, uint32_t top) {
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v.entry(i)) & 0x7fffffffu);
    return top;
}

// What a row's largest magnitude a (its bits) gives: the factor of its entries before they are rounded, and the scale that is stored.
//
// bfloat16: with the factor rounded up every product is rounded as the quotient is.  Let x and a be integers of 8 bits, 127 x / (a 2^s) their quotient.
// If it is not a middle n + 1/2, it is at least 1 / (254 x) > 1.5e-5 of itself from one, and the factor's error (2^-23 of itself) takes it past none.
// If it is one, (2 n + 1) a 2^s = 254 x.  Either 127 divides a, so a = 254: the factor is a power of two and the product exact.  Or 127 divides
// 2 n + 1, so n = 63, and rounding up gives the even code, 64.
template <typename T>
__device__ __forceinline__ void row_factor(uint32_t top, float& factor, float& scale) {
    const float a = __uint_as_float(top);
    factor = scale = 0.f;
    if (top >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
    else if (a >= FRB_8BIT_SMALLEST_ROW) { factor = sizeof(T) == 4 ? __fdiv_rn(127.f, a) : __fdiv_ru(127.f, a); scale = __fdiv_rn(a, 127.f); }
}

#define FRB_8BIT_WHOLE 12582912.f      // 1.5 * 2^23: a number added to it is rounded to a whole one, whose lowest byte is the sum's
#define FRB_8BIT_BORDER 0.49998f       // the factor is off by 2^-23 of itself at most, a product by 127 * 2^-23 < 1.6e-5

// 127 x / a rounded half to even, for eight entries; `near`: one of them (of float32) is so near to the middle of two codes that slow_codes() has to
// decide.
template <typename T>
__device__ __forceinline__ uint2 codes_of(const Eight<T>& v, float factor, bool& near) {
    near = false;
    if (factor == 0.f) return make_uint2(0u, 0u);
    float t[8];
    const uint64_t factors = pair_of(factor, factor), whole = pair_of(FRB_8BIT_WHOLE, FRB_8BIT_WHOLE), less = pair_of(-1.f, -1.f);
    float middle = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint64_t x = pair_of(v.entry(i), v.entry(i + 1)), sums = fma_pairs(x, factors, whole);
        halves_of(sums, t[i], t[i + 1]);
        if (sizeof(T) == 4) {
            float r0, r1;
            halves_of(fma_pairs(x, factors, fma_pairs(sums, less, whole)), r0, r1);
            middle = fmaxf(middle, fmaxf(fabsf(r0), fabsf(r1)));
        }
    }
    near = sizeof(T) == 4 && middle > FRB_8BIT_BORDER;
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(t[i]);
    return make_uint2(__byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410));
}

// The code next to c (or c itself) that 127 x / a is nearest to, half to even, where it lies next to the middle of two codes.  Exact: with 127 x =
// p + e and c a = q + f, both sums of two float32, the remainder against half of a is (p - q -+ a/2) + (e - f), where both differences in the
// first bracket are of numbers within a factor of two of one another and so without rounding, and so is e - f: every term is a
// whole multiple of x's last place, e below 2^7 and f below 2^15 of them (a is less than 2^8 times x, or its code were 0).
// (p, q and their difference by name: a compiler may join a product and a subtraction into one rounding, and e and f would then count twice.)
__device__ __forceinline__ float decided_code(float x, float c, float a) {
    if (a > 1.2676506e30f) { x *= 9.5367432e-7f; a *= 9.5367432e-7f; }               // above 2^100: times 2^-20, or 127 x would be infinite
    const float p = __fmul_rn(127.f, x), e = fmaf(127.f, x, -p), q = __fmul_rn(c, a), f = fmaf(c, a, -q), d = __fsub_rn(p, q);
    const float toward = copysignf(1.f, d), over = toward * ((d - toward * (0.5f * a)) + (e - f));
    return over > 0.f || (over == 0.f && ((int)c & 1)) ? c + toward : c;
}

// The codes of eight float32 entries that stand at p, decided one after another.  (Few runs come here; the code is short, and the registers of those
// that do not come are left alone.)
template <typename T>
__device__ __forceinline__ uint2 slow_codes(const T* p, int left, float factor, float top) {
    unsigned long long codes = 0;
#pragma unroll 1
    for (int i = 0; i < 8 && i < left; ++i) {
        const float x = to_f32(p[i]);
        float t = fmaf(x, factor, FRB_8BIT_WHOLE);
        if (fabsf(fmaf(x, factor, FRB_8BIT_WHOLE - t)) > FRB_8BIT_BORDER) t = FRB_8BIT_WHOLE + decided_code(x, t - FRB_8BIT_WHOLE, top);
        codes |= (unsigned long long)(__float_as_uint(t) & 0xffu) << (8 * i);
    }
    return make_uint2((uint32_t)codes, (uint32_t)(codes >> 32));
}

}  // namespace frb_products8
#endif
