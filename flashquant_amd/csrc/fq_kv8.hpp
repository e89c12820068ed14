// Rows at 8 bits: e4m3 codes times a power of two of the row, whose E8M0 byte is kept beside them.
#pragma once

#include "fq_common.hpp"

namespace fq {

// Powers of two of a row.  The lowest keeps the smallest code times it, 2^-127, a float32; the highest is what rows near 2^128 need.
constexpr int kRowPowerMin = -118, kRowPowerMax = 120;

// Two codes of a word, as float32 and as the 16-bit types, all exact.
template <bool HIGH> __device__ __forceinline__ float2v codes_f32(uint32_t w) {
    return __builtin_bit_cast(float2v, __builtin_amdgcn_cvt_pk_f32_fp8(int(w), HIGH));
}
template <int DT, bool HIGH> __device__ __forceinline__ uint32_t codes_pair(uint32_t w) {
    if constexpr (DT == FQ_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
}

// 2^(byte - 127) of the byte at bits 8 K of w
template <int K> __device__ __forceinline__ float row_scale(uint32_t w) {
    if constexpr (K == 3) return bits_to_float((w >> 1) & 0x7f800000u);
    else return bits_to_float((w << (23 - 8 * K)) & 0x7f800000u);
}

}  // namespace fq
