// Rows of activations into 8 bits: e4m3 codes with one UE8M0 scale per 32 channels, the operand of the products with 4-bit
// weights (uq_linear.cu).  Three producers share the quantiser: the root-mean-square norm with the residual's addition, the gated
// activation, and the split of 16-bit rows into two such planes.  No counterpart in the reference.
//
//   quantiser   E = the least integer with amax <= 448 * 2^E (the cache's "ceil" rule with e4m3's largest value: nothing is
//               clipped), byte = E + 127, code = e4m3(y * 2^-E) to nearest, ties to even; a group of zeros has byte 0.
//               A value that is not finite has the NaN code (e4m3 has no infinity).
//   norm        s = x + r, y = s * rsqrt(mean(s^2) + eps) * w.  s is kept in fp32 for the norm; the sum that is handed on
//               (the next residual) is s rounded once to the input's type, as any other addition in that type would leave it.
//   gate        y = g / (1 + exp(-g)) * u
//   split       x = hi * 2^E + lo * 2^E', hi = e4m3(x * 2^-E), lo the remainder's e4m3 with the remainder's own scale: 4 + 4
//               significant bits hold a bf16 value exactly, save for what lies under 2^-21 of its group's largest.
//
// All three are bound by memory: a lane owns pieces of 8 channels (one 16-byte load of a 16-bit type), a group of 32 is four
// lanes, whose maximum takes two shuffles; a piece leaves as one 8-byte store.
#include <climits>

#include "uq_common.cuh"

namespace {

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
UQ_DEV float piece_amax(const float* v) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < kPiece; i++) m = fmaxf(m, fabsf(v[i]));   // (a NaN is left out: its own code says it)
  return m;
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
UQ_DEV uint2 codes_of(const float* v, float inv, float amax) {
  float q[kPiece];
#pragma unroll
  for (int i = 0; i < kPiece; i++) q[i] = v[i] * inv;
  if (__float_as_uint(amax) >= 0x7f800000u) {   // an infinity in the group: the conversion would saturate it
#pragma unroll
    for (int i = 0; i < kPiece; i++) q[i] = fabsf(v[i]) <= 3.4028235e38f ? q[i] : __int_as_float(0x7fc00000);
  }
  return make_uint2(e4m3x2(q[0], q[1]) | (e4m3x2(q[2], q[3]) << 16), e4m3x2(q[4], q[5]) | (e4m3x2(q[6], q[7]) << 16));
}

// ---- norm -----------------------------------------------------------------------------------------------------------
struct NormArgs {
  const void *x, *r, *w;   // r null: nothing to add; w null: ones
  void* sum;               // null with r null
  uint8_t *codes, *scales;
  long long rows;
  int H;
  float eps;
};

// Sum over the `lanes` threads of a row: they are `warps_row` whole warps of the block.
template <bool kOneWarp>
UQ_DEV float row_sum(float v, float* sums, int warps_row, int first_warp) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (kOneWarp) return v;
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < warps_row; i++) t += sums[first_warp + i];
  __syncthreads();
  return t;
}

// A row per block, or (kOneWarp) per warp; V pieces per lane, the row stays in registers between its two uses.
template <typename T, int V, bool kOneWarp>
__global__ void __launch_bounds__(kOneWarp ? 128 : 1024) uq_rms_norm_kernel(NormArgs a, int pdl) {
  __shared__ float sums[32];
  const int lanes = kOneWarp ? 32 : blockDim.x;
  const int pieces = a.H / kPiece;
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  const int t = kOneWarp ? (threadIdx.x & 31) : threadIdx.x;
  const long long row = kOneWarp ? (long long)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (kOneWarp && row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.H;
  const T* r = a.r ? static_cast<const T*>(a.r) + row * a.H : nullptr;
  const T* w = static_cast<const T*>(a.w);
  Raw<T> xr[V], rr[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int p = t + i * lanes;
    if (p < pieces) {
      xr[i].load(x + (size_t)p * kPiece);
      if (r) rr[i].load(r + (size_t)p * kPiece);
    }
  }
  float s[V][kPiece];
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int p = t + i * lanes;
    if (p < pieces) {
      xr[i].get(s[i]);
      if (r) {
        float o[kPiece];
        rr[i].get(o);
#pragma unroll
        for (int j = 0; j < kPiece; j++) s[i][j] += o[j];
        Raw<T>::store(static_cast<T*>(a.sum) + row * a.H + (size_t)p * kPiece, s[i]);
      }
      float q = 0.f;
#pragma unroll
      for (int j = 0; j < kPiece; j++) q = fmaf(s[i][j], s[i][j], q);
      sq += q;
    }
  }
  float total = row_sum<kOneWarp>(sq, sums, (lanes + 31) >> 5, 0);
  float inv = rsqrtf(total / (float)a.H + a.eps);
  if (__float_as_uint(total) == 0x7f800000u) {
    // the squares left fp32 (entries beyond 2^63): once more with the row scaled by 2^-80, whose eps is nothing beside it
    constexpr float kDown = 8.2718061255302767e-25f;   // 2^-80
    sq = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++)
      if (t + i * lanes < pieces)
#pragma unroll
        for (int j = 0; j < kPiece; j++) sq = fmaf(s[i][j] * kDown, s[i][j] * kDown, sq);
    total = row_sum<kOneWarp>(sq, sums, (lanes + 31) >> 5, 0);
    inv = rsqrtf(total / (float)a.H) * kDown;
  }
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int p = t + i * lanes;
    const bool in = p < pieces;
    if (in) {
      float wv[kPiece];
      if (w) {
        Raw<T> wr;
        wr.load(w + (size_t)p * kPiece);
        wr.get(wv);
      }
#pragma unroll
      for (int j = 0; j < kPiece; j++) s[i][j] = w ? s[i][j] * inv * wv[j] : s[i][j] * inv;
    }
    const float amax = group_amax(in ? piece_amax(s[i]) : 0.f);
    if (in) {
      const uint32_t byte = scale_byte(amax);
      *reinterpret_cast<uint2*>(a.codes + row * a.H + (size_t)p * kPiece) = codes_of(s[i], inverse_scale(byte), amax);
      if ((t & 3) == 0) a.scales[row * (a.H / kGroup) + p / 4] = (uint8_t)byte;
    }
  }
}

// ---- gated activation -----------------------------------------------------------------------------------------------
struct GateArgs {
  const void* x;   // [rows, 2 F]: gates, then the values they multiply
  uint8_t *codes, *scales;
  long long rows;
  int F;
};

constexpr int kGateThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kGateThreads) uq_silu_mul_kernel(GateArgs a, int pdl) {
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  const int pieces = a.F / kPiece;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const int p = blockIdx.x * kGateThreads + threadIdx.x;
    const bool in = p < pieces;
    float y[kPiece];
    if (in) {
      const T* x = static_cast<const T*>(a.x) + row * 2 * a.F + (size_t)p * kPiece;
      Raw<T> gr, ur;
      gr.load(x);
      ur.load(x + a.F);
      float g[kPiece], u[kPiece];
      gr.get(g);
      ur.get(u);
#pragma unroll
      for (int j = 0; j < kPiece; j++) y[j] = g[j] / (1.f + expf(-g[j])) * u[j];
    }
    const float amax = group_amax(in ? piece_amax(y) : 0.f);
    if (in) {
      const uint32_t byte = scale_byte(amax);
      *reinterpret_cast<uint2*>(a.codes + row * a.F + (size_t)p * kPiece) = codes_of(y, inverse_scale(byte), amax);
      if ((p & 3) == 0) a.scales[row * (a.F / kGroup) + p / 4] = (uint8_t)byte;
    }
  }
}

// ---- split of bf16 rows into two planes -------------------------------------------------------------------------------
// Rows are laid out as uq_linear.cu reads them: tiles of tile_rows rows, a tile's leading planes, then its remainder planes; what
// fills up the last tile is never written, its products never read.
UQ_DEV void e4m3x2_to_f32(uint32_t v, float& lo, float& hi) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((unsigned short)v));
  lo = __half2float(__ushort_as_half((unsigned short)(h2 & 0xFFFFu)));
  hi = __half2float(__ushort_as_half((unsigned short)(h2 >> 16)));
}
__global__ void __launch_bounds__(kGateThreads) uq_split_kernel(const __nv_bfloat16* x, uint8_t* codes, uint8_t* scales, long long rows, int K, int tile_rows, int pdl) {
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  const int pieces = K / kPiece;
  const int p = blockIdx.x * kGateThreads + threadIdx.x;
  const bool in = p < pieces;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const long long hi_row = row + row / tile_rows * tile_rows, lo_row = hi_row + tile_rows;
    float v[kPiece];
    if (in) {
      Raw<__nv_bfloat16> xr;
      xr.load(x + row * K + (size_t)p * kPiece);
      xr.get(v);
    }
    float amax = group_amax(in ? piece_amax(v) : 0.f);
    uint32_t byte = scale_byte(amax);
    const uint2 hi = in ? codes_of(v, inverse_scale(byte), amax) : make_uint2(0, 0);
    if (in) {
      *reinterpret_cast<uint2*>(codes + hi_row * K + (size_t)p * kPiece) = hi;
      if ((p & 3) == 0) scales[hi_row * (K / kGroup) + p / 4] = (uint8_t)byte;
      const float scale = uq_scale_f32(byte);
      const uint32_t h[4] = {hi.x & 0xffffu, hi.x >> 16, hi.y & 0xffffu, hi.y >> 16};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float a, b;
        e4m3x2_to_f32(h[i], a, b);
        v[2 * i] = fmaf(-a, scale, v[2 * i]);           // exact: both are multiples of x's last bit, at most 8 bits apart
        v[2 * i + 1] = fmaf(-b, scale, v[2 * i + 1]);
      }
    }
    amax = group_amax(in ? piece_amax(v) : 0.f);
    byte = scale_byte(amax);
    if (in) {
      *reinterpret_cast<uint2*>(codes + lo_row * K + (size_t)p * kPiece) = codes_of(v, inverse_scale(byte), amax);
      if ((p & 3) == 0) scales[lo_row * (K / kGroup) + p / 4] = (uint8_t)byte;
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

template <typename T, int V>
cudaError_t norm_launch(const NormArgs& a, int lanes, cudaStream_t s) {
  const bool pdl = uq_pdl_on();
  if (lanes == 32) return uq_launch(uq_rms_norm_kernel<T, V, true>, dim3((unsigned)((a.rows + 3) / 4)), 128u, 0, s, pdl, a, (int)pdl);
  return uq_launch(uq_rms_norm_kernel<T, V, false>, dim3((unsigned)a.rows), (unsigned)lanes, 0, s, pdl, a, (int)pdl);
}
template <typename T>
cudaError_t norm_by_size(const NormArgs& a, int sms, cudaStream_t s) {
  const int pieces = a.H / kPiece;
  (void)sms;
  const int v = pieces <= 32 ? 1 : (pieces <= 64 ? 2 : 4);
  const int lanes = ((pieces + v - 1) / v + 31) / 32 * 32;
  if (v == 1) return norm_launch<T, 1>(a, lanes, s);
  if (v == 2) return norm_launch<T, 2>(a, lanes, s);
  return norm_launch<T, 4>(a, lanes, s);
}

}  // namespace

// dtype: 0 fp32, 1 bf16, 2 fp16 (of x, r, w and the sum)
cudaError_t uq_rms_norm_dispatch(const void* x, const void* r, const void* w, void* sum, uint8_t* codes, uint8_t* scales, long long rows, int H, int dtype, float eps,
                                 int sms, cudaStream_t s) {
  if (rows < 0 || rows > INT_MAX || H < kGroup || H > 32768 || H % kGroup || dtype < 0 || dtype > 2 || !(eps > 0.f)) return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  if (!x || !codes || !scales || (r != nullptr) != (sum != nullptr)) return cudaErrorInvalidValue;
  if (!aligned16(x) || !aligned16(r) || !aligned16(w) || !aligned16(sum) || !aligned8(codes)) return cudaErrorInvalidValue;
  const NormArgs a{x, r, w, sum, codes, scales, rows, H, eps};
  switch (dtype) {
    case 0: return norm_by_size<float>(a, sms, s);
    case 1: return norm_by_size<__nv_bfloat16>(a, sms, s);
    default: return norm_by_size<__half>(a, sms, s);
  }
}

cudaError_t uq_silu_mul_dispatch(const void* x, uint8_t* codes, uint8_t* scales, long long rows, int F, int dtype, cudaStream_t s) {
  if (rows < 0 || rows > INT_MAX || F < kGroup || F > (1 << 20) || F % kGroup || dtype < 0 || dtype > 2) return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  if (!x || !codes || !scales || !aligned16(x) || !aligned8(codes)) return cudaErrorInvalidValue;
  const GateArgs a{x, codes, scales, rows, F};
  const bool pdl = uq_pdl_on();
  const dim3 grid((unsigned)((F / kPiece + kGateThreads - 1) / kGateThreads), (unsigned)(rows < 32768 ? rows : 32768));
  switch (dtype) {
    case 0: return uq_launch(uq_silu_mul_kernel<float>, grid, (unsigned)kGateThreads, 0, s, pdl, a, (int)pdl);
    case 1: return uq_launch(uq_silu_mul_kernel<__nv_bfloat16>, grid, (unsigned)kGateThreads, 0, s, pdl, a, (int)pdl);
    default: return uq_launch(uq_silu_mul_kernel<__half>, grid, (unsigned)kGateThreads, 0, s, pdl, a, (int)pdl);
  }
}

cudaError_t uq_split_dispatch(const void* x, uint8_t* codes, uint8_t* scales, long long rows, int K, int tile_rows, cudaStream_t s) {
  const bool pdl = uq_pdl_on();
  const dim3 grid((unsigned)((K / kPiece + kGateThreads - 1) / kGateThreads), (unsigned)(rows < 32768 ? rows : 32768));
  return uq_launch(uq_split_kernel, grid, (unsigned)kGateThreads, 0, s, pdl, (const __nv_bfloat16*)x, codes, scales, rows, K, tile_rows, (int)pdl);
}
