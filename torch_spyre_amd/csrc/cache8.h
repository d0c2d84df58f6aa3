// The 8-bit paged cache: pages of 64 tokens, per (page, KV head)
//   K  [D/16, 64 tok, 16]    16-feature units, a token's unit 16 bytes
//   V  [4, D, 16 tok]        16-token units, a feature's unit 16 bytes
//   scales  [64] fp32 each   value = code * scale of its token
// Both products of attention reduce over the dimension of a unit, so an MFMA
// operand is whole units, and 64 lanes that each load one unit read runs of
// 512 contiguous bytes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/spyre_hip.h"

namespace spyre_hip {

typedef _Float16 c8_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 c8_f16x8 __attribute__((ext_vector_type(8)));
typedef float c8_f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t c8_u32x4 __attribute__((ext_vector_type(4)));

// Four codes -> four fp16 numbers, exactly (e4m3's 4 significant bits and
// int8's 8 both fit fp16's 11).  int8: the byte, its sign bit flipped, as the
// low mantissa bits of 1024 is 1024 + 128 + code.
template <int KIND>
__device__ __forceinline__ void codes_to_f16(uint32_t w, c8_f16x2& lo, c8_f16x2& hi) {
  if constexpr (KIND == SPYRE_CODES_E4M3) {
    lo = __builtin_bit_cast(c8_f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, false));
    hi = __builtin_bit_cast(c8_f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, true));
  } else {
    const uint32_t x = w ^ 0x80808080u;
    const c8_f16x2 off = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
    lo = __builtin_bit_cast(c8_f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x07010700u)) - off;
    hi = __builtin_bit_cast(c8_f16x2, __builtin_amdgcn_perm(0x64646464u, x, 0x07030702u)) - off;
  }
}

template <int KIND>
__device__ __forceinline__ c8_f16x8 codes_to_f16x8(uint32_t w0, uint32_t w1) {
  c8_f16x2 a, b, c, d;
  codes_to_f16<KIND>(w0, a, b);
  codes_to_f16<KIND>(w1, c, d);
  return c8_f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four codes -> four floats, exactly.
template <int KIND>
__device__ __forceinline__ void codes_to_f32(uint32_t w, float (&x)[4]) {
  if constexpr (KIND == SPYRE_CODES_E4M3) {
    const c8_f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
    const c8_f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = lo[0], x[1] = lo[1], x[2] = hi[0], x[3] = hi[1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = static_cast<float>(static_cast<int8_t>(w >> (8 * e)));
  }
}

// 4 x 4 bytes transposed: word e of the result holds byte e of each word.
__device__ __forceinline__ void transpose4x4_b8(uint32_t (&x)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);  // x0.0 x1.0 x0.1 x1.1
  const uint32_t b = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);  // x0.2 x1.2 x0.3 x1.3
  const uint32_t c = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
  const uint32_t d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
  x[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  x[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  x[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  x[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// The 4 x 4 words that the lanes l, l + 16, l + 32, l + 48 (group g = l / 16)
// hold, transposed: word i of group g becomes word g of group i.
__device__ __forceinline__ void transpose4x4_groups(uint32_t (&x)[4]) {
  auto swap32 = [](uint32_t& a, uint32_t& b) {  // a's upper half of the wave <-> b's lower half
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  auto swap16 = [](uint32_t& a, uint32_t& b) {  // a's odd rows of 16 lanes <-> b's even rows
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0], b = r[1];
  };
  swap32(x[0], x[2]);
  swap32(x[1], x[3]);
  swap16(x[0], x[1]);
  swap16(x[2], x[3]);
}

}  // namespace spyre_hip
