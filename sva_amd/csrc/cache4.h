// The 4-bit KV cache's row format, shared by the kernels that write and read it.
#pragma once
#include "common.cuh"

namespace sva {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// Row r of KV head g: codes at ((g * rows + r) * 2 + kv) * D / 2, scale bytes
// at ((g * rows + r) * 2 + kv) * D / 32, kv = 0 for K and 1 for V: a row's K
// and V halves are neighbours, so a row that is looked up alone is one or two
// lines.  32 consecutive elements share the scale 2^(byte - 127); byte 255
// marks a block that held an infinity or a NaN, and reads as NaN.
constexpr int kCache4Block = 32;
constexpr int kCache4Nan = 255;

// 2^(byte - 127); the conversions below read only its exponent field, which
// for 255 is that of a NaN: the products are NaN.
SVA_DEV float cache4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The eight codes of a word as floats, or as bf16 pairs (every code times a
// power of two is exact in bf16).
SVA_DEV void cache4_unpack8(uint32_t codes, float scale, float (&x)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
}
SVA_DEV bf16x8 cache4_unpack8_bf16(uint32_t codes, float scale) {
  union {
    bf16x2 p[4];
    bf16x8 v;
  } u;
  u.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0);
  u.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1);
  u.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2);
  u.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3);
  return u.v;
}

}  // namespace sva
