// Codes of the 8-bit K/V caches (e4m3 and int8) and what the gfx950 kernels do
// with them. A cache holds codes [num_pages, page_size, Hkv, D] and one fp32
// scale per block of tokens and kv head; a value is code * scale.
#pragma once

#include "common.h"

namespace mtlattn {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Four codes (one dword) as two packed pairs of T, exactly: an e4m3 value has
// 4 significant bits, an int8 one 8, and both types' exponents hold them. One
// conversion per pair for e4m3; int8 goes through fp32 (a byte select each),
// or, for fp16, by setting the code's byte (with its sign bit flipped) under the
// exponent of 1024 and subtracting 1152, one instruction each per pair.
struct E4M3 {
    static constexpr int code = 3;
    template <typename T>
    __device__ static inline u32x2_t unpack4(uint32_t w);
    // 1 in each byte whose code is a NaN
    __device__ static inline uint32_t nans(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u; }
    __device__ static inline void to_float4(uint32_t w, float* f) {
        const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
    }
};
template <>
__device__ inline u32x2_t E4M3::unpack4<BF16>(uint32_t w) {
    return u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
}
template <>
__device__ inline u32x2_t E4M3::unpack4<F16>(uint32_t w) {
    return u32x2_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
}

struct I8 {
    static constexpr int code = 4;
    template <typename T>
    __device__ static inline u32x2_t unpack4(uint32_t w);
    __device__ static inline void to_float4(uint32_t w, float* f) {
        f[0] = (float)(int8_t)w;
        f[1] = (float)(int8_t)(w >> 8);
        f[2] = (float)(int8_t)(w >> 16);
        f[3] = (float)(int8_t)(w >> 24);
    }
};
template <>
__device__ inline u32x2_t I8::unpack4<BF16>(uint32_t w) {
    float f[4];
    to_float4(w, f);
    return u32x2_t{BF16::pack2(f[0], f[1]), BF16::pack2(f[2], f[3])};
}
template <>
__device__ inline u32x2_t I8::unpack4<F16>(uint32_t w) {
    const uint32_t u = w ^ 0x80808080u;
    const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
    const f16x2_t a = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    const f16x2_t b = __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    return u32x2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

}  // namespace mtlattn
