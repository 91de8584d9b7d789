// Shared pieces of the block-scaled 8-bit operators.
//
// Format.  A matrix [R, C] is held as 8-bit floating-point codes (e4m3, or e5m2 for gradients), row-major with the
// row stride rounded up to 16 bytes, and one scale for every 128 consecutive elements of a row.  A scale is a power
// of two 2^e, kept as the byte e + 127; e is the smallest exponent >= -126 for which the largest finite magnitude of
// the block is at most FMAX * 2^e (FMAX = 448 or 57344, both 1.75 * 2^TOP).  Powers of two because the tensor core
// multiplies by such bytes itself (kind::mxf8f6f4), and because scaling by one is exact: a code is one rounding of
// x * 2^-e, whatever the order of the arithmetic.
//
// Scale layout.  The tensor core reads scales from tensor memory, 128 rows at a time: row r of the 128 sits in lane
// r % 32, column r / 32, and the four bytes of that 32-bit cell belong to four consecutive K blocks.  The global
// layout is the image of those cells, so that a 512-byte copy per 128 rows and 512 elements of K is all that moves:
//   byte(r, b) = ((r / 128) * ceil(nb / 4) + b / 4) * 512 + (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4
#pragma once
#include "ptx.cuh"

namespace cvb {

enum : int { FP8_E4M3 = 0, FP8_E5M2 = 1 };  // also the operand type codes of the MMA's instruction descriptor

__device__ __forceinline__ long long fp8_sf_offset(long long row, int b, int kgroups) {
  return ((row >> 7) * kgroups + (b >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (b & 3);
}

// A block's maximum is carried as the upper 16 bits of the magnitude, rounded up: what the scale asks of it, its
// exponent and whether its mantissa is above 1.75, is the same, and two blocks' maxima fit a register.
__device__ __forceinline__ uint32_t fp8_max16(uint32_t mag_bits) { return (mag_bits + 0xFFFFu) >> 16; }

// scale byte of a block from the largest finite magnitude: the exponent field, one more where the mantissa is above
// 1.75, less TOP.  Integer arithmetic: subnormal magnitudes (field 0) end at the smallest scale.
template <int FMT>
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t max16) {
  constexpr int TOP = FMT == FP8_E4M3 ? 8 : 15;
  return static_cast<uint32_t>(max(static_cast<int>((max16 + 0x1Fu) >> 7) - TOP, 1));
}
// 2^-e as a float; byte <= 247, so the exponent field stays positive
__device__ __forceinline__ float fp8_inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// product without the flush of subnormal inputs that this library is otherwise compiled with
__device__ __forceinline__ float fp8_mul(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int FMT>
__device__ __forceinline__ uint32_t fp8_pack2(float lo, float hi) {
  uint16_t r;
  if (FMT == FP8_E4M3)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// code of an infinity: e4m3 has none and takes NaN; e5m2 keeps it (the conversion itself would saturate)
template <int FMT>
__device__ __forceinline__ uint32_t fp8_inf_code(uint32_t bits) {
  return (FMT == FP8_E4M3 ? 0x7Fu : 0x7Cu) | ((bits >> 24) & 0x80u);
}

// eight values times `inv` as eight codes.  `odd` says that one of them may be infinite.
template <int FMT>
__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8], float inv, bool odd) {
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = fp8_mul(v[i], inv);
  uint2 o;
  o.x = fp8_pack2<FMT>(s[0], s[1]) | (fp8_pack2<FMT>(s[2], s[3]) << 16);
  o.y = fp8_pack2<FMT>(s[4], s[5]) | (fp8_pack2<FMT>(s[6], s[7]) << 16);
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t bits = __float_as_uint(v[i]);
      if ((bits & 0x7FFFFFFFu) == 0x7F800000u) {
        uint32_t& word = i < 4 ? o.x : o.y;
        const int at = (i & 3) * 8;
        word = (word & ~(0xFFu << at)) | (fp8_inf_code<FMT>(bits) << at);
      }
    }
  }
  return o;
}

// maximum of |v| over the finite ones of n values, as bits; *odd says that there were others.  The common case costs
// one maximum a value: fmaxf passes over NaN, and an infinity shows in the result and is then left out.
template <int N>
__device__ __forceinline__ uint32_t fp8_finite_max(const float (&v)[N], bool* odd) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) m = fmaxf(m, fabsf(v[i]));
  uint32_t bits = __float_as_uint(m);
  if (bits >= 0x7F800000u) {
    *odd = true;
    bits = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
      if (b < 0x7F800000u) bits = max(bits, b);
    }
  }
  return bits;
}

// eight consecutive elements from `p`, of which the first `n` exist (the others read as zero)
__device__ __forceinline__ void fp8_load8(const __nv_bfloat16* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = i < n ? __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << 16) : 0.f;
  }
}
__device__ __forceinline__ void fp8_load8(const float* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
  }
}

}  // namespace cvb
