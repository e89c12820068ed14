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

// The nearest number that the type holds.  A finite value near its end may have been rounded up to a code that stands for 2^16 (2^128):
// it comes back as the largest of the type, not as an infinity, which no code stands for.  (NaN stays.)
template <int DT> __device__ __forceinline__ float held(float x) {
    constexpr float most = DT == FQ_BF16 ? 0x1.fep127f : 65504.0f;
    return __builtin_fabsf(x) > most ? __builtin_copysignf(most, x) : x;
}

}  // namespace fq
