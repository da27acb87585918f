// Numbers as terms of 16-bit types for the matrix cores, and the products of those
// (paged_attention.hip, paged_attention_q4.hip, prompt_attention.hip).
#pragma once

#include "serving.hpp"

namespace tml {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 16 rows, 16 columns, k of 32.
template <int CT>
__device__ __forceinline__ floatx4 mma16(const srv_u32x4 &x, const srv_u32x4 &y, floatx4 c) {
    if constexpr (CT == TML_TYPE_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, x), __builtin_bit_cast(halfx8, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

// v in N terms of type CT, each the rounding of what those before it leave.
template <int CT, int N>
__device__ __forceinline__ void to_terms(float (&v)[8], srv_u32x4 (&t)[N]) {
    constexpr float kMost = CT == TML_TYPE_F16 ? 65504.0f : 0x1.fep127f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float x = v[e], y = v[e + 1];
            if (n == 0 && N > 1) {  // a finite value stays one
                x = __builtin_amdgcn_fmed3f(x, -kMost, kMost);
                y = __builtin_amdgcn_fmed3f(y, -kMost, kMost);
            }
            const uint32_t d = CT == TML_TYPE_F16 ? srv_pack_f16(x, y) : srv_pack_bf16(x, y);
            t[n][e / 2] = d;
            if (n + 1 < N) {
                v[e] -= CT == TML_TYPE_F16 ? tml_half_bits(d & 0xFFFFu) : __uint_as_float(d << 16);
                v[e + 1] -= CT == TML_TYPE_F16 ? tml_half_bits(d >> 16) : __uint_as_float(d & 0xFFFF0000u);
            }
        }
}

}  // namespace
}  // namespace tml
