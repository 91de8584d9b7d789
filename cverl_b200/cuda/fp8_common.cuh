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

// Scale bytes of two blocks from their maxima (one in each half of the word): the exponent field, one more where the
// mantissa is above 1.75, less TOP, at least 1.  Subnormal magnitudes (field 0) end at the smallest scale too.
template <int FMT>
__device__ __forceinline__ uint32_t fp8_scale_bytes(uint32_t max16x2) {
  constexpr uint32_t TOP = FMT == FP8_E4M3 ? 8 : 15;
  const uint32_t e = ((max16x2 + 0x001F001Fu) >> 7) & 0x01FF01FFu;
  return __vmaxu2(e, (TOP + 1) * 0x00010001u) - TOP * 0x00010001u;
}
// 2^-e of each as a bf16, whose exponent field is 254 - byte (7 or more: the byte is at most 247)
__device__ __forceinline__ uint32_t fp8_inverse_scales(uint32_t bytes) { return (0x00FE00FEu - bytes) << 7; }
__device__ __forceinline__ float fp8_low(uint32_t bf16x2) { return __uint_as_float(bf16x2 << 16); }
__device__ __forceinline__ float fp8_high(uint32_t bf16x2) { return __uint_as_float(bf16x2 & 0xFFFF0000u); }

// product without the flush of subnormal inputs that this library is otherwise compiled with
__device__ __forceinline__ float fp8_mul(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// four values as codes, saturating: infinities come out as the largest finite code here, see fp8_fix_inf
template <int FMT>
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d) {
  uint32_t r;
  if (FMT == FP8_E4M3)
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  else
    asm("{\n\t.reg .b16 lo, hi;\n\t"
        "cvt.rn.satfinite.e5m2x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e5m2x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// two bf16 by a power of two each: exact, or so small that its code is zero; subnormal inputs count
__device__ __forceinline__ uint32_t fp8_mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <int FMT>
__device__ __forceinline__ uint2 fp8_pack8(const float (&v)[8], float inv) {
  uint2 o;
  o.x = fp8_pack4<FMT>(fp8_mul(v[0], inv), fp8_mul(v[1], inv), fp8_mul(v[2], inv), fp8_mul(v[3], inv));
  o.y = fp8_pack4<FMT>(fp8_mul(v[4], inv), fp8_mul(v[5], inv), fp8_mul(v[6], inv), fp8_mul(v[7], inv));
  return o;
}
// the codes of infinite values among eight, put in afterwards by the few threads that hold one: e4m3 has no infinity
// and takes NaN; e5m2 keeps it
template <int FMT>
__device__ __forceinline__ void fp8_fix_inf(const float (&v)[8], uint8_t* codes, int n) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = __float_as_uint(v[i]);
    if (i < n && (bits & 0x7FFFFFFFu) == 0x7F800000u)
      codes[i] = static_cast<uint8_t>((FMT == FP8_E4M3 ? 0x7Fu : 0x7Cu) | ((bits >> 24) & 0x80u));
  }
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

// eight bf16 as read, of which the first n exist.  VEC: rows are whole 16-byte vectors, n is 0 or 8; the load is then
// one predicated instruction, and those of a row are all in flight before the first is used.
template <bool VEC>
__device__ __forceinline__ uint4 load_raw8(const __nv_bfloat16* p, int n) {
  uint4 u = make_uint4(0u, 0u, 0u, 0u);
  if (VEC) {
    if (n > 0) u = *reinterpret_cast<const uint4*>(p);
  } else {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
    u.x = (n > 0 ? e[0] : 0u) | ((n > 1 ? e[1] : 0u) << 16);
    u.y = (n > 2 ? e[2] : 0u) | ((n > 3 ? e[3] : 0u) << 16);
    u.z = (n > 4 ? e[4] : 0u) | ((n > 5 ? e[5] : 0u) << 16);
    u.w = (n > 6 ? e[6] : 0u) | ((n > 7 ? e[7] : 0u) << 16);
  }
  return u;
}
__device__ __forceinline__ void widen8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}

}  // namespace cvb
