// What the kernels that apply rotary positions share.
#pragma once

#include "fq_device.hpp"

namespace fq {

// i / d for i d < 2^32, with magic = ceil(2^32 / d)
__device__ __forceinline__ uint32_t divide(uint32_t i, uint32_t d, uint32_t magic) { return d == 1 ? i : __umulhi(i, magic); }

// cos and sin of 2 pi x: the nearest quarter turn is taken off exactly and the rest, at most an eighth of a turn, turned into
// radians in 64 bits; then the Taylor series in 32, whose next terms are below 2^-28.  sin as t + t (t^2 ...), cos as 1 + t^2 ...,
// so that the roundings inside count little: within 1.6 2^-24.
__device__ __forceinline__ float2v turn_cos_sin(double x) {
    const double quarter = __builtin_rint(4.0 * x);
    const float t = float(__builtin_fma(-0.25, quarter, x) * 6.283185307179586476925287);
    const float z = t * t;
    const float s = __builtin_fmaf(t, z * __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), t);
    const float c = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const int k = int(quarter - 4.0 * __builtin_floor(0.25 * quarter));      // 0 .. 3
    const float a = (k & 1) ? s : c, b = (k & 1) ? c : s;
    return float2v{k == 1 || k == 2 ? -a : a, k >= 2 ? -b : b};
}

// (x0, x1) turned.  Which product is rounded is spelled out: the same bits at every alignment.
__device__ __forceinline__ float2v turned_pair(float x0, float x1, float2v cs) {
    return float2v{__builtin_fmaf(x0, cs.x, -(x1 * cs.y)), __builtin_fmaf(x1, cs.x, x0 * cs.y)};
}

// Two float32 values as a word of 16-bit ones.
template <int DT> __device__ __forceinline__ uint32_t rounded_words(float x, float y) {
    if constexpr (DT == FQ_F16) asm("" : "+v"(x), "+v"(y));      // two roundings everywhere: no v_fma_mixlo_f16 here and there
    return round_pair<DT>(x, y);
}

}  // namespace fq

namespace {

inline uint32_t magic_of(int d) { return uint32_t(((uint64_t(1) << 32) + uint32_t(d) - 1) / uint32_t(d)); }

// whether rows at `ptr` with these strides can be read and written 16 bytes at a time
inline bool wide_rows(const void* ptr, const int64_t* strides, int n, int vec) {
    if (!fq_host::aligned(ptr, 16)) return false;
    for (int i = 0; i < n; ++i)
        if (strides[i] % vec != 0) return false;
    return true;
}

inline int check_rotary(int64_t tokens, int H_Q, int H_K, int half, int D, int position_bytes) {
    if (tokens < 0 || H_Q < 0 || H_K < 0 || H_Q + int64_t(H_K) == 0 || H_Q > 4096 || H_K > 4096) return FQ_ERR_BAD_SHAPE;
    if (half < 1 || D < 2 * half || D > 1024) return FQ_ERR_BAD_SHAPE;
    if (position_bytes != 4 && position_bytes != 8) return FQ_ERR_UNSUPPORTED_DTYPE;
    return FQ_OK;
}

// strides but those of a batch or a block are 32-bit in the kernel
inline bool fits(const int64_t* strides, int n) {
    for (int i = 0; i < n; ++i)
        if (strides[i] > 0x7fffffffLL || strides[i] < -0x7fffffffLL) return false;
    return true;
}

}  // namespace
