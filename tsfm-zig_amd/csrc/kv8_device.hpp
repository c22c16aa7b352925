// Device helpers shared by the 8-bit serving kernels: scales, codes, and where a request's tokens are.
#pragma once

#include "common.hpp"
#include "kv8.hpp"

namespace tsfm {

__device__ __forceinline__ u32x4 ld16(const void* p) { return *reinterpret_cast<const u32x4*>(p); }
__device__ __forceinline__ u32x2 ld8(const void* p) { return *reinterpret_cast<const u32x2*>(p); }

template <bool BF16>
__device__ __forceinline__ float half_to_f32(uint32_t x) {  // the low 16 bits
    if constexpr (BF16) return __uint_as_float(x << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
}

// The smallest power of two s >= 2^-126 with amax / s <= 448 = 1.75 * 2^8, from amax's bits (finite, not
// negative); 1 for 0. A power of two costs e4m3 nothing of its relative precision, and x / s is exact: a code
// is rounded once.
__device__ __forceinline__ float e4m3_scale(float amax) {
    const uint32_t b = __float_as_uint(amax);
    if (b == 0) return 1.f;
    const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);  // biased
    return __uint_as_float((uint32_t)max(e, 1) << 23);
}

// Scale and multiplier of a cache block: code = round(x * mul).
template <int CODE>
__device__ __forceinline__ void block_scale(float amax, float& scale, float& mul) {
    if constexpr (CODE == kCodeE4m3) {
        scale = e4m3_scale(amax);
        mul = __uint_as_float((254u << 23) - __float_as_uint(scale));  // 1 / 2^e, exactly (e > -127)
    } else {
        const float top = fmaxf(amax, 0x1p-100f);
        scale = amax > 0.f ? top * (1.f / 127.f) : 1.f;
        mul = 127.f * (1.f / top);
    }
}

// Four values to four code bytes.
template <int CODE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (CODE == kCodeE4m3) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    } else {
        auto q = [](float x) { return (uint32_t)(int)fminf(fmaxf(__builtin_rintf(x), -127.f), 127.f) & 0xffu; };
        return q(a) | (q(b) << 8) | (q(c) << 16) | (q(d) << 24);
    }
}

// Eight codes to eight 16-bit values (exact: both codes fit the mantissas of bf16 and f16).
template <int CODE, bool BF16>
__device__ __forceinline__ u32x4 decode8(uint32_t lo, uint32_t hi) {
    u32x4 r;
    if constexpr (CODE == kCodeE4m3) {
        if constexpr (BF16) {
            r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
            r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
            r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
            r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
        } else {
            r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
            r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
            r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
            r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t w = i ? hi : lo;
            if constexpr (BF16) {
                const float f0 = (float)(int)(int8_t)w, f1 = (float)(int)(int8_t)(w >> 8);
                const float f2 = (float)(int)(int8_t)(w >> 16), f3 = (float)((int)w >> 24);
                r[2 * i] = pack2<true>(f0, f1);
                r[2 * i + 1] = pack2<true>(f2, f3);
            } else {
                // u = code + 128 as the low byte of the half 0x6400 | u = 1024 + u; less 1152: the code, exactly.
                const uint32_t u = w ^ 0x80808080u;
                const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
                const uint32_t a = __builtin_amdgcn_perm(u, 0x64646464u, 0x00050004u) ;
                const uint32_t b = __builtin_amdgcn_perm(u, 0x64646464u, 0x00070006u);
                r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) - off);
                r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, b) - off);
            }
        }
    }
    return r;
}

// The new tokens of request r: packed rows [t0, t0 + n), positions [before, total). Whatever the device's
// counts hold, [t0, t0 + n) lies within max_tokens and total within the request's table row.
struct Span {
    int t0, n, total, before;
};
__device__ __forceinline__ Span request_span(const int32_t* cu, const int32_t* len, int r, int max_tokens, int width) {
    Span s;
    s.t0 = min(max(cu[r], 0), max_tokens);
    s.n = min(max(cu[r + 1] - s.t0, 0), max_tokens - s.t0);
    s.total = (int)min((int64_t)max(len[r], 0), (int64_t)width * kKvBlock);
    s.before = s.total - s.n;
    return s;
}

}  // namespace tsfm
