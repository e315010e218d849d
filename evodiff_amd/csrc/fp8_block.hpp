// Blocks of 128 values in 8 bits (OCP e4m3) with a power-of-two scale: what the kernels that write them share.
#pragma once
#include <hip/hip_runtime.h>

namespace ed {

// E8M0 byte of the scale for a block whose largest magnitude has these bits: 448 = 2^8 * (1 + 0x600000 / 2^23).
__device__ __forceinline__ int scale_byte(unsigned amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 1 ? 1 : e > 254 ? 254 : e;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }  // 2^(127 - byte)

// largest finite magnitude (as bits) of eight values; infinities become NaN (a NaN does not count by itself, and stays one)
__device__ __forceinline__ unsigned amax8(float (&v)[8]) {
  float a = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
  if (a == __builtin_huge_valf()) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (fabsf(v[i]) == __builtin_huge_valf()) v[i] = __builtin_nanf("");
      a = fmaxf(a, fabsf(v[i]));
    }
  }
  return a != a ? 0u : __float_as_uint(a);  // (all NaN: none)
}
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv) {
  uint2 r;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  r.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
  r.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, w, true);
  return r;
}

// largest of 16 neighbouring lanes (a row of the data-parallel moves), in every one of them
__device__ __forceinline__ unsigned max16(unsigned a) {
  auto step = [](unsigned v, unsigned o) { return o > v ? o : v; };
  a = step(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xf, 0xf, true));   // quad_perm [1,0,3,2]
  a = step(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xf, 0xf, true));   // quad_perm [2,3,0,1]
  a = step(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x141, 0xf, 0xf, true));  // row_half_mirror
  return step(a, (unsigned)__builtin_amdgcn_update_dpp(0, (int)a, 0x140, 0xf, 0xf, true));  // row_mirror
}

}  // namespace ed
