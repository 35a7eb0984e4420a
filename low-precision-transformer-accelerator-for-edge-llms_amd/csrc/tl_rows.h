// tl_rows.h -- rows of float32, bfloat16 or float16 read and written by the
// serving operators' kernels.
#pragma once

#include "tl_device.h"
#include "tl_serving.h"

namespace tl {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));

TL_DEV float bf16_bits(unsigned u) { return __uint_as_float(u << 16); }
TL_DEV float f16_bits(unsigned u) { return (float)__builtin_bit_cast(_Float16, (unsigned short)u); }
TL_DEV unsigned to_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
TL_DEV unsigned to_f16(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

TL_DEV v4f unpack4(v2i w, int dt) {
    const unsigned a = (unsigned)w[0], b = (unsigned)w[1];
    if (dt == DT_BF16) return v4f{bf16_bits(a & 0xFFFFu), bf16_bits(a >> 16), bf16_bits(b & 0xFFFFu), bf16_bits(b >> 16)};
    return v4f{f16_bits(a & 0xFFFFu), f16_bits(a >> 16), f16_bits(b & 0xFFFFu), f16_bits(b >> 16)};
}

// four consecutive values of a row (16-byte aligned for float32, 8 for the
// 16-bit types)
TL_DEV v4f load4(const void* p, int64_t i, int dt) {
    if (dt == DT_F32) return *(const v4f*)((const float*)p + i);
    return unpack4(*(const v2i*)((const unsigned short*)p + i), dt);
}

TL_DEV float load1(const void* p, int64_t i, int dt) {
    if (dt == DT_F32) return ((const float*)p)[i];
    const unsigned u = ((const unsigned short*)p)[i];
    return dt == DT_BF16 ? bf16_bits(u) : f16_bits(u);
}

// values rounded once to a float type
TL_DEV void store4(void* p, int64_t i, int dt, v4f v) {
    if (dt == DT_F32) {
        *(v4f*)((float*)p + i) = v;
        return;
    }
    const bool bf = dt == DT_BF16;
    const unsigned a = bf ? to_bf16(v[0]) | (to_bf16(v[1]) << 16) : to_f16(v[0]) | (to_f16(v[1]) << 16);
    const unsigned b = bf ? to_bf16(v[2]) | (to_bf16(v[3]) << 16) : to_f16(v[2]) | (to_f16(v[3]) << 16);
    *(v2i*)((unsigned short*)p + i) = v2i{(int)a, (int)b};
}

TL_DEV void store1(void* p, int64_t i, int dt, float v) {
    if (dt == DT_F32) ((float*)p)[i] = v;
    else ((unsigned short*)p)[i] = (unsigned short)(dt == DT_BF16 ? to_bf16(v) : to_f16(v));
}

}  // namespace tl
