// Values in 8 bits with a scale per 32 channels, on the device: pieces of 8 channels, the group's scale, codes, and the split of bf16
// values into two planes.  A lane owns a piece, the four lanes of a group are neighbours, and all lanes of a warp take part.
#pragma once
#include "uq_common.cuh"

namespace mx8 {

constexpr int kPiece = 8;     // channels of a lane's load
constexpr int kGroup = 32;    // channels of a scale

// ---- pieces: 8 channels of a row as fp32 ----------------------------------------------------------------------------
template <typename T> struct Raw;
template <> struct Raw<float> {
  float4 a, b;
  UQ_DEV void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
  UQ_DEV void get(float* v) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w; }
  UQ_DEV static void store(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
};
template <> struct Raw<__nv_bfloat16> {
  uint4 a;
  UQ_DEV void load(const __nv_bfloat16* p) { a = *reinterpret_cast<const uint4*>(p); }
  UQ_DEV void get(float* v) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  UQ_DEV static void store(__nv_bfloat16* p, const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Raw<__half> {
  uint4 a;
  UQ_DEV void load(const __half* p) { a = *reinterpret_cast<const uint4*>(p); }
  UQ_DEV void get(float* v) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  UQ_DEV static void store(__half* p, const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// ---- the quantiser --------------------------------------------------------------------------------------------------
// Two operations per issue slot: these kernels run out of those first.
UQ_DEV void mul2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
UQ_DEV void add2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}
UQ_DEV void fma2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {   // d = a * b + c
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d0), "=f"(d1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
UQ_DEV float max3(float a, float b, float c) {   // (a NaN is left out: its own code says it)
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
UQ_DEV float piece_amax(const float* v) {
  const float a = max3(fabsf(v[0]), fabsf(v[1]), fabsf(v[2])), b = max3(fabsf(v[3]), fabsf(v[4]), fabsf(v[5]));
  return fmaxf(max3(a, fabsf(v[6]), fabsf(v[7])), b);
}
UQ_DEV float group_amax(float m) {   // over the four lanes of a group
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
// The scale byte E + 127 for a group's largest magnitude.  448 = 1.75 * 2^8: E = (exponent of amax) - 8, one more where its
// mantissa is above 1.75; -127 at the lower end (zero and amax below 448 * 2^-127), 121 at most.
UQ_DEV uint32_t scale_byte(float amax) {
  const uint32_t b = __float_as_uint(amax);
  return (uint32_t)max((int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}
// 2^-E of such a byte, byte <= 248: exponent field 254 - byte
UQ_DEV float inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
UQ_DEV uint32_t e4m3x2(float lo, float hi) {
  unsigned short d;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(d) : "f"(hi), "f"(lo));
  return d;
}
// Codes of a piece: e4m3(v * inv), NaN where `amax`, its group's, says that there is an infinity and it is this value (the
// conversion would saturate it).
UQ_DEV uint2 codes_of(const float* v, float inv, float amax) {
  float q[kPiece];
#pragma unroll
  for (int i = 0; i < kPiece; i += 2) mul2(q[i], q[i + 1], v[i], v[i + 1], inv, inv);
  if (__float_as_uint(amax) >= 0x7f800000u) {
#pragma unroll
    for (int i = 0; i < kPiece; i++) q[i] = fabsf(v[i]) <= 3.4028235e38f ? q[i] : __int_as_float(0x7fc00000);
  }
  return make_uint2(e4m3x2(q[0], q[1]) | (e4m3x2(q[2], q[3]) << 16), e4m3x2(q[4], q[5]) | (e4m3x2(q[6], q[7]) << 16));
}

// ---- split of bf16 values: x = hi * 2^E + lo * 2^E' ------------------------------------------------------------------
UQ_DEV void e4m3x2_to_f32(uint32_t v, float& lo, float& hi) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)v));
  lo = __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu)));
  hi = __half2float(__ushort_as_half((unsigned short)(h2 >> 16)));
}
// A piece v into a plane's codes and scale byte, which is at least 1 (zeros too; 2^-126 has the steps that a bf16's last bit needs, and 0 has another use).
UQ_DEV void plane_of(const float* v, uint2& codes, uint32_t& byte) {
  const float amax = group_amax(piece_amax(v));
  byte = max(scale_byte(amax), 1u);
  codes = codes_of(v, inverse_scale(byte), amax);
}
// What a plane leaves out of its piece, exactly: both are multiples of the value's last bit or of the plane's last step, and close together.
UQ_DEV void take_out(float* v, uint2 codes, uint32_t byte) {
  const float scale = -uq_scale_f32(byte);
  const uint32_t h[4] = {codes.x & 0xffffu, codes.x >> 16, codes.y & 0xffffu, codes.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float a, b;
    e4m3x2_to_f32(h[i], a, b);
    fma2(v[2 * i], v[2 * i + 1], a, b, scale, scale, v[2 * i], v[2 * i + 1]);
  }
}
// A piece into the leading plane and the remainder's (v is that remainder then).
UQ_DEV void split_piece(float* v, uint2& hi, uint2& lo, uint32_t& hi_byte, uint32_t& lo_byte) {
  plane_of(v, hi, hi_byte);
  take_out(v, hi, hi_byte);
  plane_of(v, lo, lo_byte);
}

// ---- groups of wide range ---------------------------------------------------------------------------------------------
// What two planes leave out of bf16 values lies under 2^-21 of the group's largest, in values below 2^-13 of it.  Where that is an ordinary group's smallest
// value it is nothing beside the others.  In a group of wide range - a few large channels, whose codes in the weight may be zero - it is not: the group is
// "wide" where a value loses more than 2^-14 of the group's typical magnitude, the geometric mean of the values that are not zero (a bf16's bits, read
// as a whole number, are its logarithm but for the mantissa's curve; no large channel moves that mean far).  (Normal or Laplace distributed values, or
// products of two such: not one group of 131 072.  32 values of which 1, 4 or 8 are 1000 times the others: 17 to 29 %, 16 384 times: 86 to 99.7 %.)
constexpr uint32_t kWideByte = 0;   // in place of such a group's scales, with codes of zero
// Whether a lane's group is wide: its piece with its codes and bytes (not for a group with NaN or infinity, whose own codes say it).
UQ_DEV bool wide_group(uint4 raw, uint2 hi, uint2 lo, uint32_t hi_byte, uint32_t lo_byte) {
  Raw<__nv_bfloat16> x;
  x.a = raw;
  float rest[kPiece];
  x.get(rest);
  take_out(rest, hi, hi_byte);
  take_out(rest, lo, lo_byte);
  const float left = group_amax(piece_amax(rest));
  const uint32_t w[4] = {raw.x & 0x7fff7fffu, raw.y & 0x7fff7fffu, raw.z & 0x7fff7fffu, raw.w & 0x7fff7fffu};
  uint32_t n = 0;   // sum of the logarithms, and from bit 24 on how many
  bool finite = true;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t a = w[i] & 0xffffu, b = w[i] >> 16;
    n += a + b + (a ? 1u << 24 : 0u) + (b ? 1u << 24 : 0u);
    finite &= max(a, b) < 0x7f80u;
  }
  n += __shfl_xor_sync(0xffffffffu, n, 1);
  n += __shfl_xor_sync(0xffffffffu, n, 2);
  const uint32_t others = __ballot_sync(0xffffffffu, !finite) >> (threadIdx.x & 28) & 15u;
  return !others && left > 6.103515625e-05f * __uint_as_float((n & 0xffffffu) / max(n >> 24, 1u) << 16);   // 2^-14
}
// Whether two planes leave anything of a piece, and whether that has to be looked at (any of a warp's groups may be wide).  They leave nothing of a value
// whose leading code is 2^-5 or more (it is 2^-6 * 2^E or more, its last bit 2^-13 * 2^E or more and so no less than the remainder plane's last step, whose
// scale is 2^(E - 4) at most, half a step of 448's binade being 16 < 448 * 2^-4; and what the leading plane leaves of it is at most 8 such bits), and
// at most 2^-14 * 2^E, or the value, of a smaller one.
UQ_DEV bool may_leave(uint2 hi) {   // (a byte with an exponent field of 0 or 1: adding 0x70 to its upper three bits does not reach bit 7)
  return (((hi.x & 0x70707070u) + 0x70707070u) & ((hi.y & 0x70707070u) + 0x70707070u) & 0x80808080u) != 0x80808080u;
}
// A code's bits are a logarithm as well, 8 to the binade with 56 for 1: where a lane's eight codes are 84 on average (2^3.5 * 2^E), and so all 32, at most
// 10 values are that small, and even they leave the geometric mean too high for the rule: with n of them at 2^-14 * 2^E it is 2^(3.5 + 0.219 n
// - 14 n / 32) * 2^E, above 1 for every n up to 10, and smaller ones lose no more than themselves.
UQ_DEV bool may_be_wide(uint2 hi) { return __dp4a(hi.x & 0x7f7f7f7fu, 0x01010101u, __dp4a(hi.y & 0x7f7f7f7fu, 0x01010101u, 0u)) < 8u * 84u; }
// A code's value, and the code of one value.
UQ_DEV float e4m3_value(uint32_t code) {
  float lo, hi;
  e4m3x2_to_f32(code, lo, hi);
  return lo;
}

}  // namespace mx8
