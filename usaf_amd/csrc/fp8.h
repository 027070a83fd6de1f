// What the 8-bit block-scaled kernels share (fp8.hip, fp8_gemm.hip, few.hip).
#pragma once

#include "moe_gemm.h"

namespace usaf {

constexpr int FP8_BLOCK = 128;  // values of one scale along a row; rows of one scale of a weight

// E8M0 byte of a block's largest finite magnitude.
__device__ __forceinline__ int e8m0_of(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u);  // 448 = 1.75 * 2^8
  return (e < -120 ? -120 : e > 120 ? 120 : e) + 127;
}
__device__ __forceinline__ float inv_scale(int e8m0) { return __uint_as_float((uint32_t)(254 - e8m0) << 23); }

__device__ __forceinline__ float finite_abs(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7FFFFFFFu;
  return b < 0x7F800000u ? __uint_as_float(b) : 0.f;
}

// Four scaled values -> four codes.
__device__ __forceinline__ uint32_t to_codes(const float (&v)[4], float inv) {
  uint32_t o = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  o = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, (int)o, true);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if ((__float_as_uint(v[j]) & 0x7F800000u) == 0x7F800000u) o = (o & ~(0xFFu << (8 * j))) | (0x7Fu << (8 * j));
  return o;
}

// Over 16 neighbouring lanes, by rotations of such a row inside the vector instruction (__shfl_xor goes through LDS for two
// of the four).
template <int N>
__device__ __forceinline__ float max_rot(float v) {
  return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false)));
}
__device__ __forceinline__ float max16(float v) { return max_rot<1>(max_rot<2>(max_rot<4>(max_rot<8>(v)))); }

// Eight 16-bit values of a register quadruple.
template <int DT>
__device__ __forceinline__ void unpack8(const uint4 q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f32x2 f = unpack2<DT>(w[j]);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

// 8 neighbouring values of a 16-bit row; `left` of them exist.
template <int DT>
__device__ __forceinline__ void load8(const uint16_t* p, bool vec, int left, float (&v)[8]) {
  if (vec && left >= 8) {
    unpack8<DT>(*reinterpret_cast<const uint4*>(p), v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < left ? load_as_f32<DT>(p, j) : 0.f;
  }
}

// Quantizes 16 lanes' 8 values each (one block of a row) and stores them: the codes
// at q, the scale byte at s.
__device__ __forceinline__ void store_block(const float (&v)[8], int lane16, uint8_t* q, uint8_t* s) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[j]));
  const int e = e8m0_of(max16(m));
  const float inv = inv_scale(e);
  const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
  *reinterpret_cast<uint2*>(q) = uint2{to_codes(a, inv), to_codes(b, inv)};
  if (lane16 == 0) *s = (uint8_t)e;
}

// 32 codes of a lane -> four bf16 fragment registers of their values, exact.
__device__ __forceinline__ void values16(const u32x4 lo, const u32x4 hi, int e8m0, u32x4 (&o)[4]) {
  const int b = e8m0 & 0xFF;
  const float s = __uint_as_float(b == 0 ? 0x00400000u : (uint32_t)b << 23);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t w = j < 4 ? lo[j] : hi[j - 4];
    o[j >> 1][2 * (j & 1)] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false));
    o[j >> 1][2 * (j & 1) + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true));
  }
}

// Raises the 8-bit product's dynamic-LDS limit, once per process (usaf_hip_init, or its first use).
void prepare_fp8_kernels();

// The product of up to 32 rows, quantized in the same launch (fp8_small.hip).
bool fp8_small_ok(int64_t M, int64_t K);
int fp8_small(const void* x, int dtype, int64_t M, int64_t K, int64_t ld, const uint8_t* w, const uint8_t* w_scale, int64_t N,
              void* out, hipStream_t st);

}  // namespace usaf
