// Device helpers of the e4m3 KV cache, shared by its append / read kernels and
// the attention that reads it.
#pragma once

#include "q3k_common.hpp"

namespace q3k
{
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

    // The value a scale byte stands for, 2^(byte - 127) for bytes 1 .. 254 (the
    // append writes no other).
    __device__ __forceinline__ float e4m3_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

    // The value of one code.
    __device__ __forceinline__ float e4m3_value(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(code), 0); }

    // Codes 2 HI and 2 HI + 1 of a word times a power-of-two scale, as bf16 (exact
    // down to bf16's subnormals).
    template <bool HI>
    __device__ __forceinline__ uint32_t decode2(uint32_t codes, float scale)
    {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HI));
    }

    __device__ __forceinline__ Vec8 decode8(uint2 codes, float scale)
    {
        Vec8 r;
        r.d[0] = decode2<false>(codes.x, scale);
        r.d[1] = decode2<true>(codes.x, scale);
        r.d[2] = decode2<false>(codes.y, scale);
        r.d[3] = decode2<true>(codes.y, scale);
        return r;
    }
} // namespace q3k
