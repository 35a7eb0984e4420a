// tl_attn.h -- what the kernels of paged attention share: its matrix products, the
// 16-bit forms of INT8 values and probabilities, and the parts that a shared prefix leaves.
#pragma once

#include "tl_rows.h"

namespace tl {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

template <bool BF>
TL_DEV v4f mfma32(v4i a, v4i b, v4f c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// two INT8 values (one in each 16-bit half, zero extended) as float16: 0x6400 | u
// is 1024 + u for u < 1024, and u = x ^ 0x80 is x + 128, so 1152 less is x exactly
TL_DEV int i8_pair_f16(unsigned halves) {
    const h2 v = __builtin_bit_cast(h2, halves ^ 0x64806480u);
    return __builtin_bit_cast(int, v - h2{(_Float16)1152.0f, (_Float16)1152.0f});
}

// two floats to the 16-bit type: bfloat16 truncated, float16 to nearest
template <bool BF>
TL_DEV int pack2(float a, float b) {
    if constexpr (BF) return (int)__builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    else return __builtin_bit_cast(int, h2{(_Float16)a, (_Float16)b});
}

TL_DEV float pair_max(float v) {   // maximum over the four 16-lane groups
    const unsigned u = __float_as_uint(v);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const float w = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const unsigned x = __float_as_uint(w);
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

constexpr float kLog2e = 1.44269504088896340736f;

// A shared prefix's part of a query head in scratch: O [head_dim], m and l, of split s
TL_DEV int64_t prefix_part(const PagedAttnArgs& a, int s, int row, int head) {
    return ((int64_t)s * a.rows + row) * a.n_heads + head;
}

}  // namespace tl
