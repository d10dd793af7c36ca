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
// A piece v into the leading plane's and the remainder's codes and scale bytes (v is used up).
UQ_DEV void split_piece(float* v, uint2& hi, uint2& lo, uint32_t& hi_byte, uint32_t& lo_byte) {
  float amax = group_amax(piece_amax(v));
  hi_byte = scale_byte(amax);
  hi = codes_of(v, inverse_scale(hi_byte), amax);
  const float scale = -uq_scale_f32(hi_byte);
  const uint32_t h[4] = {hi.x & 0xffffu, hi.x >> 16, hi.y & 0xffffu, hi.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    float a, b;
    e4m3x2_to_f32(h[i], a, b);
    fma2(v[2 * i], v[2 * i + 1], a, b, scale, scale, v[2 * i], v[2 * i + 1]);   // exact: both are multiples of x's last bit, at most 8 bits apart
  }
  amax = group_amax(piece_amax(v));
  lo_byte = scale_byte(amax);
  lo = codes_of(v, inverse_scale(lo_byte), amax);
}

}  // namespace mx8
