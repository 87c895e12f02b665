// Microscaled 4-bit floats (MXFP4 of the OCP Microscaling Formats specification v1.0): 32 consecutive features of a
// row share a power of two (E8M0: 2^(code - 127), 255 is NaN), and each is held as E2M1 (sign, 0 .5 1 1.5 2 3 4 6).
// A block's codes are 16 bytes, feature 2 i in the low half of byte i; a row's last block is filled with zeros.
#pragma once

#include "device.hpp"

namespace mbrt {

constexpr int MXFP4 = 5;          // beside the codes of enum DT: an operand in this format
constexpr int kMxBlock = 32;


// The part of |x| that a block's scale goes by: the bits without the sign, which order like the values, with infinities
// and NaN above all of them.
__device__ __forceinline__ uint32_t mx_size(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Scale code of a block whose largest value has these bits: floor(log2) - 2, so that it falls into [4, 8); at least
// 2^-127 (subnormals and zeros have the exponent field 0), NaN where something is infinite or NaN.
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t size) {
    const uint32_t e = size >> 23;
    return e == 255u ? 255u : e < 2u ? 0u : e - 2u;
}

// The conversions take a scale as an f32 and look at its exponent field alone: 0 stands for 2^-127, 255 for NaN.
__device__ __forceinline__ float mx_scale_operand(uint32_t code) { return __uint_as_float(code << 23); }

// Eight consecutive values in 4 bits: x 2^-s rounded to nearest, ties to even, past 6 to 6.
__device__ __forceinline__ uint32_t mx_pack8(const float (&x)[8], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
    return w;
}
__device__ __forceinline__ uint32_t mx_pack4(const float (&x)[4], float scale) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    return w;
}

// What eight codes stand for, as f32 and as bf16 (exact: two significant bits and a power of two).
__device__ __forceinline__ void mx_unpack8(uint32_t w, float scale, float (&x)[8]) {
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
}
__device__ __forceinline__ u32x4 mx_unpack8_bf16(uint32_t w, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3))};
}

// The largest of G consecutive lanes' sizes (G 4 or 8), in each of them; all lanes active.
template <int G>
__device__ __forceinline__ uint32_t mx_group_size(uint32_t v) {
    static_assert(G == 4 || G == 8, "the lanes of a block of 32");
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));
    v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));
    if (G == 8) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true));
    return v;
}

// Of the lanes l, l ^ 16, l ^ 32 and l ^ 48; all lanes active.
__device__ __forceinline__ uint32_t mx_rows_size(uint32_t v) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}

}  // namespace mbrt
