// Keys and values held in 8 bits: how a row is stored and how its codes come back.
//
// A row is one token's key or value of one head.  It is stored as 8-bit codes with one float32 scale,
//     a = max |x|,  scale = a / Q,  code = x * (Q / a) rounded to the type, half to even,
// Q = 448 for e4m3 and 127 for int8.  A row whose largest entry is below 2^-96 is stored as zeros with scale zero (Q / a would
// leave float32's range); one with an entry that is not finite gets the scale NaN and codes of zero, so that it reads back as NaN.
// Pages hold 64 tokens: codes [pages, heads, 64, entries], the row's entries side by side (keys and values alike), and scales
// [pages, heads, 64].
#pragma once

#include <cuda_fp16.h>

#include <cstring>
#include <tuple>

#include "common.cuh"

// Types of the codes.
enum FrbCodes { FRB_E4M3 = 0, FRB_INT8 = 1 };

#define FRB_SMALLEST_ROW 1.2621774e-29f      // 2^-96

namespace frb_8bit {

// What a row's largest magnitude (its bits, so that NaN and infinity are the largest) gives: the factor of its entries
// before they are rounded, and the scale that is stored.
__device__ __forceinline__ void row_scale(uint32_t top_bits, int codes, float& factor, float& scale) {
    const float top = __uint_as_float(top_bits), limit = codes == FRB_E4M3 ? 448.f : 127.f;
    if (top_bits >= 0x7f800000u) { factor = 0.f; scale = __uint_as_float(0x7fc00000u); return; }
    if (top < FRB_SMALLEST_ROW) { factor = 0.f; scale = 0.f; return; }
    factor = __fdiv_rn(limit, top);
    scale = __fdiv_rn(top, limit);
}

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Four entries times `factor` as four codes, the first in the lowest byte.  A factor of zero gives codes of zero, whatever the entries.
__device__ __forceinline__ uint32_t four_codes(float4 x, float factor, int codes) {
    if (factor == 0.f) return 0u;
    const float a = x.x * factor, b = x.y * factor, c = x.z * factor, d = x.w * factor;
    if (codes == FRB_E4M3) {
        uint32_t out;
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
            "mov.b32 %0, {lo, hi};\n\t}"
            : "=r"(out) : "f"(a), "f"(b), "f"(c), "f"(d));
        return out;
    }
    uint32_t out;                     // (products of up to 127 (1 + 2^-23): none is rounded to another code than -127 .. 127)
    asm("{\n\t.reg .b32 upper;\n\t"
        "cvt.pack.sat.s8.s32.b32 upper, %4, %3, 0;\n\t"
        "cvt.pack.sat.s8.s32.b32 %0, %2, %1, upper;\n\t}"
        : "=r"(out) : "r"(__float2int_rn(a)), "r"(__float2int_rn(b)), "r"(__float2int_rn(c)), "r"(__float2int_rn(d)));
    return out;
}

// The codes of two halves of a register as float16 pairs: every code of either type is a float16 number.
// e4m3: bytes 0 and 1 as `lo`, bytes 2 and 3 as `hi`.
__device__ __forceinline__ void halves_of_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}

// int8: the codes in bytes 0 and 2 of w (what lies in bytes 1 and 3 does not matter).  Byte c with its sign bit turned is c + 128, and
// 0x6400 + n is the float16 1024 + n.
__device__ __forceinline__ uint32_t half_of_int8(uint32_t w) {
    const uint32_t biased = (w & 0x00ff00ffu) ^ 0x64806480u, offset = 0x64806480u;             // 1152 twice
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&biased), *reinterpret_cast<const __half2*>(&offset));
    return *reinterpret_cast<const uint32_t*>(&r);
}

// Four neighbouring codes times their row's scale.
__device__ __forceinline__ float4 four_values(uint32_t w, float scale, int codes) {
    if (codes == FRB_E4M3) {
        uint32_t lo, hi;
        halves_of_e4m3(w, lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        return make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
    }
    const auto value = [&](int byte) { return (float)(int8_t)(w >> (8 * byte)) * scale; };
    return make_float4(value(0), value(1), value(2), value(3));
}

}  // namespace frb_8bit

// Checks the head sizes that the 8-bit kernels are compiled for and calls LAUNCH(HD, VD).
#define FRB_8BIT_SIZES(what, head_dim, v_dim, LAUNCH)                                                                        \
    do {                                                                                                                      \
        if (head_dim == 32 && v_dim == 32) { LAUNCH(32, 32); }                                                                \
        else if (head_dim == 32 && v_dim == 64) { LAUNCH(32, 64); }                                                           \
        else if (head_dim == 64 && v_dim == 64) { LAUNCH(64, 64); }                                                           \
        else if (head_dim == 64 && v_dim == 128) { LAUNCH(64, 128); }                                                         \
        else if (head_dim == 96 && v_dim == 96) { LAUNCH(96, 96); }                                                           \
        else if (head_dim == 128 && v_dim == 128) { LAUNCH(128, 128); }                                                       \
        else { frb_set_error("%s: head_dim %d with value heads of %d is not built", what, head_dim, v_dim); return -1; }      \
    } while (0)

// Calls an entry point with its arguments read one after another from `packed`, each at its type's alignment, as they lie in a C struct of
// them.  (A call of thirty arguments costs the interpreter four microseconds argument by argument and one as a struct.)
template <typename... Args>
inline int call_packed(int (*entry)(Args...), const void* packed, cudaStream_t stream) {
    size_t at = 0;
    const auto next = [&](auto* type) {
        typedef std::remove_pointer_t<decltype(type)> T;
        if constexpr (std::is_same_v<T, cudaStream_t>) return stream;             // the last one
        else {
            at = (at + alignof(T) - 1) / alignof(T) * alignof(T);
            T value;
            memcpy(&value, static_cast<const char*>(packed) + at, sizeof(T));
            at += sizeof(T);
            return value;
        }
    };
    const std::tuple<Args...> args{next(static_cast<Args*>(nullptr))...};         // (braces: from the first to the last)
    return std::apply(entry, args);
}
