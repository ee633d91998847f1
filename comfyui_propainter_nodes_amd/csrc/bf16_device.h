// bf16_device.h -- bf16 storage for the norm and attention kernels that take it (the convolutions and the video model know f16 and
// f32 only).  A bf16 value travels as its 16 bits; f32 -> bf16 rounds to nearest even (at most half a step,
// 2^-8 of the value), NaN stays NaN.
#pragma once
#include "pp_device.h"

namespace pp {

struct bf16_t {
  unsigned short bits;
};

__device__ __forceinline__ float to_f32(bf16_t v) { return __builtin_bit_cast(float, (unsigned)v.bits << 16); }

#ifndef PP_EMU
typedef __bf16 pp_hw_bf2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {  // one v_cvt_pk_bf16_f32
  return __builtin_bit_cast(unsigned, pp_hw_bf2{(__bf16)a, (__bf16)b});
}
#else
inline unsigned pack_bf16(float a, float b) {
  auto one = [](float f) -> unsigned {
    const unsigned u = __builtin_bit_cast(unsigned, f);
    if (f != f) return (u >> 16) | 0x40u;
    return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
  };
  return one(a) | (one(b) << 16);
}
#endif
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
  return bf16_t{(unsigned short)pack_bf16(v, 0.f)};
}
__device__ __forceinline__ void ld8(const bf16_t* p, float* f) {
  const u4 v = *reinterpret_cast<const u4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __builtin_bit_cast(float, v[i] << 16);
    f[2 * i + 1] = __builtin_bit_cast(float, v[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void st8(bf16_t* p, const float* f) {
  *reinterpret_cast<u4*>(p) = u4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
}

}  // namespace pp
