// The FP8 block format: E4M3 codes with one fp32 scale per 128 consecutive columns of a row
// (activations) or per 128 x 128 block (weights).  Device functions shared by the cast, the product's
// small-batch kernel and the gated residual norm, so that all three write the same codes.
//
//   amax' = max(amax |x|, 1e-12),   scale = RN(amax' / 448),   code = e4m3(RN(448 x / amax'))
//
// The code is the rounding of 448 x / amax', not of x / scale: ratios x / amax' that fall exactly
// between two codes are common with bf16 inputs, and the rounded scale would tip them either way.
#pragma once

#include "vf4_common.cuh"

namespace vf4 {

// What a block's elements are multiplied with.  q = RN((x * mul) / div) comes from one Markstein step
// on inv = RN(1 / div) (div_markstein).  Above 2^96 both sides are scaled by 2^-32 (exactly), so
// 448 x stays finite for every finite x.  `plain` selects the true division: amax' infinite or NaN,
// where the step would turn 0 * inf into NaN (the formula gives 0 for finite x, NaN for x infinite).
struct Fp8Block {
  float mul, div, inv, scale;
  bool plain;
};

// RN(a / 448) for normal a >= 1e-12 by one Markstein step on y = RN(1 / 448); checked against the
// correctly rounded division for every significand (both sides scale exactly by powers of two).
VF4_DEV float div448_rn(float a) {
  const float y = 0.00223214295692741870880126953125f;   // RN(1/448) = 0x3B124925
  const float q = __fmul_rn(a, y);
  return __fmaf_rn(__fmaf_rn(-q, 448.0f, a), y, q);
}

VF4_DEV Fp8Block fp8_block(uint32_t amax_bits) {
  float a = __uint_as_float(amax_bits);
  a = a < 1e-12f ? 1e-12f : a;   // keeps a NaN
  Fp8Block b;
  b.scale = div448_rn(a);
  const bool big = a >= 0x1p96f;
  b.mul = big ? 448.f * 0x1p-32f : 448.f;
  b.div = big ? a * 0x1p-32f : a;
  b.plain = !(a < __uint_as_float(0x7F800000u));
  if (b.plain) b.scale = a;
  b.inv = __frcp_rn(b.div);
  return b;
}

VF4_DEV float fp8_quotient(float x, const Fp8Block& b) {
  const float v = __fmul_rn(x, b.mul);
  return b.plain ? __fdiv_rn(v, b.div) : div_markstein(v, b.div, b.inv);
}

// Eight values -> eight E4M3 codes (nearest even, saturating at +-448; NaN -> 0x7F), by pairs.
VF4_DEV uint2 fp8_encode8(const float* x, const Fp8Block& b) {
  uint32_t w[4];
  if (!b.plain) {
    const unsigned long long mul2 = f32x2_pack(b.mul, b.mul), inv2 = f32x2_pack(b.inv, b.inv);
    const unsigned long long nd2 = f32x2_pack(-b.div, -b.div);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long v = mul_f32x2(f32x2_pack(x[2 * i], x[2 * i + 1]), mul2);
      const unsigned long long q = mul_f32x2(v, inv2);
      const unsigned long long r = fma_f32x2(q, nd2, v);
      float q0, q1;
      f32x2_unpack(fma_f32x2(r, inv2, q), &q0, &q1);
      w[i] = e4m3x2(q0, q1);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = e4m3x2(fp8_quotient(x[2 * i], b), fp8_quotient(x[2 * i + 1], b));
  }
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// |x| as bits: their unsigned order is the order of the magnitudes, with NaN above infinity, so the
// maximum of a block with a NaN is a NaN as torch's amax gives it.
VF4_DEV uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

VF4_DEV uint32_t amax8_bits(const float* x) {
  uint32_t m = abs_bits(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max(m, abs_bits(x[i]));
  return m;
}

// Eight consecutive elements from p (nv of them valid; the others become 0).  kVec: p is 16-byte
// aligned and nv is 0 or 8.
template <typename T, bool kVec>
VF4_DEV void load8(const T* p, int nv, float* v) {
  if constexpr (kVec) {
    if (nv <= 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.f;
    } else if constexpr (sizeof(T) == 2) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
    } else {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < nv ? (float)p[i] : 0.f;
  }
}

// The same eight elements kept as they were loaded (bf16: four registers instead of eight).
template <typename T, bool kVec>
struct Raw8 {
  float v[8];
  VF4_DEV void load(const T* p, int nv) { load8<T, kVec>(p, nv, v); }
  VF4_DEV uint32_t amax_bits() const { return amax8_bits(v); }
  VF4_DEV void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
};

template <>
struct Raw8<__nv_bfloat16, true> {
  uint4 w;
  VF4_DEV void load(const __nv_bfloat16* p, int nv) {
    w = nv > 0 ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
  }
  VF4_DEV uint32_t amax_bits() const {   // two 16-bit lanes: the magnitudes' order is their bits' order
    const uint32_t k = 0x7FFF7FFFu;
    const uint32_t m = umax_u16x2(umax_u16x2(w.x & k, w.y & k), umax_u16x2(w.z & k, w.w & k));
    return max(m << 16, m & 0x7FFF0000u);
  }
  VF4_DEV void get(float* f) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
};

}  // namespace vf4
