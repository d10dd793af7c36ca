// Rows of activations into 8 bits: e4m3 codes with one UE8M0 scale per 32 channels, the operand of the products with 4-bit
// weights (uq_linear.cu).  Three producers share the quantiser: the root-mean-square norm with the residual's addition, the gated
// activation, and the split of 16-bit rows into two such planes.  No counterpart in the reference.
//
//   quantiser   E = the least integer with amax <= 448 * 2^E (the cache's "ceil" rule with e4m3's largest value: nothing is
//               clipped), byte = E + 127, code = e4m3(y * 2^-E) to nearest, ties to even; a group of zeros has byte 0.
//               A y that is not finite has the NaN code (e4m3 has no infinity).
//   norm        s = x + r, y = s * rsqrt(mean(s^2) + eps) * w.  s is kept in fp32 for the norm; the sum that is handed on
//               (the next residual) is s rounded once to the input's type, as any other addition in that type would leave it.
//   gate        y = g / (1 + exp(-g)) * u
//   split       x = hi * 2^E + lo * 2^E', hi = e4m3(x * 2^-E), lo the remainder's e4m3 with the remainder's own scale: 4 + 4
//               significant bits hold a bf16 value exactly, save for what lies under 2^-21 of its group's largest.  A group of which that
//               leaves out too much (wide_group) has zeros in both planes and byte 0, which no other group has: the products' kernel comes back for it.
//
// A lane owns pieces of 8 channels (one 16-byte load of a 16-bit type), a group of 32 is four lanes, whose maximum takes two shuffles;
// a piece leaves as one 8-byte store.  Memory should bound all three, and does where a value brings 7 bytes (norm of 16384 x 8192 bf16 with a
// residual: 138 us from a graph, 6.8 TB/s); with 3 and 5 bytes the issue slots run out first (norm of 8191 x 4096 fp16 23 us, 4.4 TB/s, 16
// instructions per value; gate of 5001 x 11040 bf16 52 to 58 us on different boxes, 4.8 to 5.3 TB/s, 24), hence the paired arithmetic.  fp32: gate of 4096 x 8192 47 us,
// 6.5 TB/s; norm of 8192 x 4096 with a residual 79 us, 5.6 TB/s (four pieces of fp32 do not fit 64 registers: 72 bytes of stack).
#include <atomic>
#include <climits>

#include "uq_mx8.cuh"

namespace {

using namespace mx8;

// ---- norm -----------------------------------------------------------------------------------------------------------
struct NormArgs {
  const void *x, *r, *w;   // r null: nothing to add; w null: ones
  void* sum;               // null with r null
  uint8_t *codes, *scales;
  long long rows;
  int H;
  float inv_h, eps;        // 1 / H
};

// Sum over a row's threads: a warp, or the block, whose warps leave their sums in an array (zero behind the last warp).
template <bool kOneWarp>
UQ_DEV float row_sum(float v, float* sums) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if (kOneWarp) return v;
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < (int)blockDim.x; i += 128) {   // four warps' sums at a time
    const float4 q = *reinterpret_cast<const float4*>(sums + (i >> 5));
    t += (q.x + q.y) + (q.z + q.w);
  }
  return t;
}

UQ_DEV float inverse_root(float v) {   // (v is never subnormal: eps is not); a Newton step takes the hardware's 2 ulp to under one
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  const float e = fmaf(-(v * r), r, 1.f);
  return v < 3e38f ? fmaf(0.5f * r, e, r) : r;   // (infinity and NaN as they are)
}

// Rows whose reciprocal root is above this (entries of 2^-12 and less, with an eps below 2^-24) are scaled up first.
constexpr float kTinyRow = 4096.f;

// A row per block, or (kOneWarp) per warp; V pieces per lane, the row stays in registers between its two uses.
// With t = s * w, y = t * inv and amax(y) = amax(t) * inv (a product by one factor keeps the order), so that a value costs one
// multiplication by inv * 2^-E on its way to its code, a power of two times what y itself rounds to.
template <typename T, int V, bool kOneWarp>
__global__ void __launch_bounds__(kOneWarp ? 128 : 1024) uq_rms_norm_kernel(NormArgs a, int pdl) {
  __shared__ __align__(16) float sums[32];
  const int lanes = kOneWarp ? 32 : blockDim.x;
  const int pieces = a.H / kPiece;
  if (!kOneWarp && threadIdx.x < 32 && threadIdx.x >= blockDim.x >> 5) sums[threadIdx.x] = 0.f;   // (read behind the barrier in row_sum)
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  const int t = kOneWarp ? (threadIdx.x & 31) : threadIdx.x;
  const long long row = kOneWarp ? (long long)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const T *x = static_cast<const T*>(a.x), *r = static_cast<const T*>(a.r), *w = static_cast<const T*>(a.w);
  Raw<T> xr[V], rr[V];
  if (kOneWarp && row >= a.rows) return;
  {
    const T *px = x + row * a.H, *pr = r + row * a.H;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int p = t + i * lanes;
      if (p < pieces) {
        xr[i].load(px + p * kPiece);
        if (r) rr[i].load(pr + p * kPiece);
      }
    }
  }
  {
    float s[V][kPiece];
    float sq0 = 0.f, sq1 = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int p = t + i * lanes;
      if (p < pieces) {
        xr[i].get(s[i]);
        if (r) {
          float o[kPiece];
          rr[i].get(o);
#pragma unroll
          for (int j = 0; j < kPiece; j += 2) add2(s[i][j], s[i][j + 1], s[i][j], s[i][j + 1], o[j], o[j + 1]);
          Raw<T>::store(static_cast<T*>(a.sum) + row * a.H + p * kPiece, s[i]);
        }
#pragma unroll
        for (int j = 0; j < kPiece; j += 2) fma2(sq0, sq1, s[i][j], s[i][j + 1], s[i][j], s[i][j + 1], sq0, sq1);
      }
    }
    float total = row_sum<kOneWarp>(sq0 + sq1, sums);
    float inv = inverse_root(fmaf(total, a.inv_h, a.eps));
    if (__float_as_uint(total) == 0x7f800000u) {
      // the squares left fp32 (entries beyond 2^56): once more with the row scaled by 2^-72, whose eps is nothing beside it
      constexpr float kDown = 2.1175823681357508e-22f;   // 2^-72
      sq0 = 0.f;
#pragma unroll
      for (int i = 0; i < V; i++)
        if (t + i * lanes < pieces)
#pragma unroll
          for (int j = 0; j < kPiece; j++) {
            s[i][j] *= kDown;
            sq0 = fmaf(s[i][j], s[i][j], sq0);
          }
      if (!kOneWarp) __syncthreads();   // (the sums of this turn have been read)
      total = row_sum<kOneWarp>(sq0, sums);
      inv = inverse_root(total * a.inv_h);
    }
    if (inv > kTinyRow) {   // the row is brought near one, so that neither s * w nor inv * 2^-E leaves fp32: by a power of two, which changes no rounding
      const float up = __uint_as_float(__float_as_uint(inv) & 0x7f800000u);   // (inv is at most 2^63, a row's entries at most sqrt(H) / inv)
      inv *= __uint_as_float(0x7f000000u - __float_as_uint(up));   // 1 / up
#pragma unroll
      for (int i = 0; i < V; i++)
        if (t + i * lanes < pieces)
#pragma unroll
          for (int j = 0; j < kPiece; j++) s[i][j] *= up;
    }
    uint8_t *pc = a.codes + row * a.H, *ps = a.scales + row * (a.H / kGroup);
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int p = t + i * lanes;
      const bool in = p < pieces;
      if (in && w) {
        float wv[kPiece];
        Raw<T> wr;
        wr.load(w + p * kPiece);
        wr.get(wv);
#pragma unroll
        for (int j = 0; j < kPiece; j += 2) mul2(s[i][j], s[i][j + 1], s[i][j], s[i][j + 1], wv[j], wv[j + 1]);
      }
      const float amax = group_amax(in ? piece_amax(s[i]) : 0.f) * inv;
      if (in) {
        const uint32_t byte = scale_byte(amax);
        float f = inv * inverse_scale(byte);
        if (byte < 32u) {   // y below 2^-86: inv * 2^-E may leave fp32 (from 32 on it is at most 2^12 * 2^95), so one after the other
          f = inverse_scale(byte);
#pragma unroll
          for (int j = 0; j < kPiece; j++) s[i][j] *= inv;
        }
        *reinterpret_cast<uint2*>(pc + p * kPiece) = codes_of(s[i], f, amax);
        if ((t & 3) == 0) ps[p >> 2] = (uint8_t)byte;
      }
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
constexpr int kGatePieces = 2;   // pieces of a thread whose loads are issued together

// g * sigmoid(g) * u for two pairs, through t = exp(-|g|), which does not overflow: g * (g < 0 ? t : 1) / (1 + t) * u.
// t = 2^(h + l) with h = -|g| * log2(e) rounded and l what the rounding and log2(e)'s own end lose (a product's error is exact in
// one fused multiplication): 2^h by the hardware, times 1 + l * ln(2).  1 + t is in [1, 2], where a Newton step brings the
// hardware's reciprocal to the last bit but one.  Under 2^-126 (gates below -87) t is zero.
UQ_DEV void silu_mul2(float& y0, float& y1, float u0, float u1) {
  constexpr float kLog2e = 1.44269504f, kLog2eRest = 1.92596303e-08f, kLn2 = 0.693147181f;   // log2(e) = kLog2e + kLog2eRest
  const float g0 = y0, g1 = y1, a0 = fmaxf(-fabsf(g0), -200.f), a1 = fmaxf(-fabsf(g1), -200.f);
  float h0, h1, l0, l1, t0, t1, d0, d1, r0, r1;
  mul2(h0, h1, a0, a1, kLog2e, kLog2e);
  fma2(l0, l1, a0, a1, kLog2e, kLog2e, -h0, -h1);
  fma2(l0, l1, a0, a1, kLog2eRest, kLog2eRest, l0, l1);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t0) : "f"(h0));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t1) : "f"(h1));
  mul2(l0, l1, l0, l1, kLn2, kLn2);
  fma2(t0, t1, t0, t1, l0, l1, t0, t1);
  add2(d0, d1, t0, t1, 1.f, 1.f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(d0));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(d1));
  fma2(d0, d1, -d0, -d1, r0, r1, 1.f, 1.f);
  fma2(r0, r1, r0, r1, d0, d1, r0, r1);
  mul2(y0, y1, g0, g1, g0 < 0.f ? t0 : 1.f, g1 < 0.f ? t1 : 1.f);
  mul2(y0, y1, y0, y1, r0, r1);
  mul2(y0, y1, y0, y1, u0, u1);
}

// Five blocks per SM for 16-bit types (us at 5001 x 11040 bf16: four 55.8, five 53.4, six 60.4; one piece in flight 55.4 to 61, four 53.4 to 61).
// The rows' pieces are one sequence, cut into runs of a block's threads: a group's four lanes never leave their row (F is a
// multiple of 32, runs start at multiples of 4), and no lane is idle for a row's odd end.  A thread's place moves on by a
// constant number of rows and pieces, so that nothing is divided on the way.
template <typename T>
__global__ void __launch_bounds__(kGateThreads, sizeof(T) == 4 ? 4 : 5) uq_silu_mul_kernel(GateArgs a, int pdl) {
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  const int pieces = a.F / kPiece;
  const long long all = a.rows * pieces, step = (long long)gridDim.x * kGateThreads;
  // (the grid is no larger than what the device holds: a block's first piece and the step are small numbers)
  const unsigned first_piece = blockIdx.x * kGateThreads + threadIdx.x, first_row = first_piece / (unsigned)pieces, step_row = (unsigned)step / (unsigned)pieces;
  long long at = first_piece;
  int p = (int)(first_piece - first_row * pieces);
  const T* x = static_cast<const T*>(a.x) + (long long)first_row * 2 * a.F + p * kPiece;
  const int step_piece = (int)((unsigned)step - step_row * pieces);
  const long long step_x = (long long)step_row * 2 * a.F + step_piece * kPiece;
  while (__any_sync(0xffffffffu, at < all)) {   // (a warp's lanes leave together: the shuffles need all of them)
    Raw<T> gr[kGatePieces], ur[kGatePieces];
    const long long first = at;
#pragma unroll
    for (int i = 0; i < kGatePieces; i++) {
      if (at < all) {
        gr[i].load(x);
        ur[i].load(x + a.F);
      }
      at += step;
      x += step_x;
      p += step_piece;
      if (p >= pieces) {   // the next row: its gates begin F values behind this one's factors
        p -= pieces;
        x += a.F;
      }
    }
#pragma unroll
    for (int i = 0; i < kGatePieces; i++) {
      const long long here = first + i * step;
      const bool in = here < all;
      float y[kPiece];
      if (in) {
        float u[kPiece];
        gr[i].get(y);
        ur[i].get(u);
#pragma unroll
        for (int j = 0; j < kPiece; j += 2) silu_mul2(y[j], y[j + 1], u[j], u[j + 1]);
      }
      const float amax = group_amax(in ? piece_amax(y) : 0.f);
      if (in) {
        const uint32_t byte = scale_byte(amax);
        *reinterpret_cast<uint2*>(a.codes + here * kPiece) = codes_of(y, inverse_scale(byte), amax);
        if ((threadIdx.x & 3) == 0) a.scales[here >> 2] = (uint8_t)byte;
      }
    }
  }
}

// ---- split of bf16 rows into two planes -------------------------------------------------------------------------------
// Rows are laid out as uq_linear.cu reads them: tiles of tile_rows rows, a tile's leading planes, then its remainder planes; what
// fills up the last tile is never written, its products never read.
__global__ void __launch_bounds__(kGateThreads) uq_split_kernel(const __nv_bfloat16* x, uint8_t* codes, uint8_t* scales, long long rows, int K, int tile_rows, int pdl) {
  // Released before its own wait, unlike the others: what follows is always the products' kernel of the same call, which lets nobody in before
  // this one is done, and may set its CTAs up meanwhile (8 rows x 4096 x 4096 6.62 -> 6.28 us, x 10240 x 8192 13.4 -> 13.2).
  if (pdl) uq_pdl_release();
  uq_pdl_wait();
  const int pieces = K / kPiece;
  const int p = blockIdx.x * kGateThreads + threadIdx.x;
  const bool in = p < pieces;
  for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
    const long long hi_row = row + row / tile_rows * tile_rows, lo_row = hi_row + tile_rows;
    float v[kPiece];
#pragma unroll
    for (int j = 0; j < kPiece; j++) v[j] = 0.f;
    Raw<__nv_bfloat16> xr;
    xr.a = make_uint4(0, 0, 0, 0);
    if (in) {
      xr.load(x + row * K + (size_t)p * kPiece);
      xr.get(v);
    }
    uint2 hi, lo;
    uint32_t hi_byte, lo_byte;
    split_piece(v, hi, lo, hi_byte, lo_byte);
    // (one step after the other: 8 rows x 10240 x 8192 13.4 us; without the first 13.5, without both 13.9)
    if (__builtin_expect(__any_sync(0xffffffffu, may_leave(hi) && in) && __any_sync(0xffffffffu, may_be_wide(hi) && in), 0)) {
      if (wide_group(xr.a, hi, lo, hi_byte, lo_byte)) {
        hi = lo = make_uint2(0, 0);
        hi_byte = lo_byte = kWideByte;
      }
    }
    if (in) {
      *reinterpret_cast<uint2*>(codes + hi_row * K + (size_t)p * kPiece) = hi;
      *reinterpret_cast<uint2*>(codes + lo_row * K + (size_t)p * kPiece) = lo;
      if ((p & 3) == 0) {
        scales[hi_row * (K / kGroup) + p / 4] = (uint8_t)hi_byte;
        scales[lo_row * (K / kGroup) + p / 4] = (uint8_t)lo_byte;
      }
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7) == 0; }

// Blocks that the device holds at once (looked up once per kernel and block size, the same on every device of the box).
template <typename K>
int resident_blocks(K kern, int threads, int sms, std::atomic<int>* cached) {
  int n = cached[threads / 32].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) != cudaSuccess || n < 1) { cudaGetLastError(); n = 1; }
    cached[threads / 32].store(n, std::memory_order_relaxed);
  }
  return n * sms;
}

template <typename T, int V, bool kOneWarp>
cudaError_t norm_launch(const NormArgs& a, cudaStream_t s) {
  const int pieces = a.H / kPiece, lanes = kOneWarp ? 32 : ((pieces + V - 1) / V + 31) / 32 * 32;
  const bool pdl = uq_pdl_on();
  return uq_launch(uq_rms_norm_kernel<T, V, kOneWarp>, dim3((unsigned)(kOneWarp ? (a.rows + 3) / 4 : a.rows)), (unsigned)(kOneWarp ? 128 : lanes), 0, s, pdl, a, (int)pdl);
}
template <typename T>
cudaError_t norm_by_size(const NormArgs& a, int sms, cudaStream_t s) {
  const int pieces = a.H / kPiece;
  if (pieces <= 32) return norm_launch<T, 1, true>(a, s);
  if (pieces <= 64) return norm_launch<T, 2, true>(a, s);
  if (pieces <= 128) return norm_launch<T, 4, true>(a, s);
  // A piece per thread while all rows fit the device at once, four from there on (us with one / four, bf16 with a residual:
  // 4096 channels, 8 rows 1.76 / 2.62, 296 rows 2.33 / 3.15, 1184 rows 5.90 / 5.04; 8192 channels, 8 rows 2.33 / 2.86, 296 rows 3.69 / 3.81,
  // 592 rows 6.64 / 4.79).
  const bool few = a.rows * pieces <= 2048ll * sms;
  if (pieces <= 1024 && few) return norm_launch<T, 1, false>(a, s);
  if (pieces <= 2048 && few) return norm_launch<T, 2, false>(a, s);
  return norm_launch<T, 4, false>(a, s);
}
template <typename T>
cudaError_t gate_launch(const GateArgs& a, int sms, cudaStream_t s) {
  static std::atomic<int> cached[33];
  const long long all = a.rows * (a.F / kPiece), want = (all + kGateThreads - 1) / kGateThreads;
  const long long most = resident_blocks(uq_silu_mul_kernel<T>, kGateThreads, sms, cached);
  const bool pdl = uq_pdl_on();
  return uq_launch(uq_silu_mul_kernel<T>, dim3((unsigned)(want < most ? want : most)), (unsigned)kGateThreads, 0, s, pdl, a, (int)pdl);
}

}  // namespace

// dtype: 0 fp32, 1 bf16, 2 fp16 (of x, r, w and the sum)
cudaError_t uq_rms_norm_dispatch(const void* x, const void* r, const void* w, void* sum, uint8_t* codes, uint8_t* scales, long long rows, int H, int dtype, float eps,
                                 int sms, cudaStream_t s) {
  if (rows < 0 || rows > INT_MAX || H < kGroup || H > 32768 || H % kGroup || dtype < 0 || dtype > 2 || !(eps >= 1.17549435e-38f)) return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  if (!x || !codes || !scales || (r != nullptr) != (sum != nullptr)) return cudaErrorInvalidValue;
  if (!aligned16(x) || !aligned16(r) || !aligned16(w) || !aligned16(sum) || !aligned8(codes)) return cudaErrorInvalidValue;
  const NormArgs a{x, r, w, sum, codes, scales, rows, H, 1.f / (float)H, eps};
  switch (dtype) {
    case 0: return norm_by_size<float>(a, sms, s);
    case 1: return norm_by_size<__nv_bfloat16>(a, sms, s);
    default: return norm_by_size<__half>(a, sms, s);
  }
}

cudaError_t uq_silu_mul_dispatch(const void* x, uint8_t* codes, uint8_t* scales, long long rows, int F, int dtype, int sms, cudaStream_t s) {
  if (rows < 0 || rows > INT_MAX || F < kGroup || F > (1 << 20) || F % kGroup || dtype < 0 || dtype > 2) return cudaErrorInvalidValue;
  if (rows == 0) return cudaSuccess;
  if (!x || !codes || !scales || !aligned16(x) || !aligned8(codes)) return cudaErrorInvalidValue;
  const GateArgs a{x, codes, scales, rows, F};
  switch (dtype) {
    case 0: return gate_launch<float>(a, sms, s);
    case 1: return gate_launch<__nv_bfloat16>(a, sms, s);
    default: return gate_launch<__half>(a, sms, s);
  }
}

cudaError_t uq_split_dispatch(const void* x, uint8_t* codes, uint8_t* scales, long long rows, int K, int tile_rows, cudaStream_t s) {
  const bool pdl = uq_pdl_on();
  const dim3 grid((unsigned)((K / kPiece + kGateThreads - 1) / kGateThreads), (unsigned)(rows < 32768 ? rows : 32768));
  return uq_launch(uq_split_kernel, grid, (unsigned)kGateThreads, 0, s, pdl, (const __nv_bfloat16*)x, codes, scales, rows, K, tile_rows, (int)pdl);
}
