// Products with a weight in 4 bits: y[m, n] = sum_k x[m, k] * code[n, k] * 2^(s[n, k / 32] - 127), for the few rows of a decode or
// verify step.  No counterpart in the reference.
//
// The weight is laid out as one stream of the paged cache with 128-token pages at head_dim 128 (codes [tiles, K/128, 128, 64],
// scales [tiles, K/128, 128, 4]: a tile is 128 output channels, a "head" 128 input channels), so the cache's own encoder writes it.
// Activations are e4m3 codes with one UE8M0 scale per 32 channels; bf16 rows are split into two such planes first (uq_rows.cu),
// whose products are added.
#include <climits>

#include "uq_common.cuh"

namespace {

constexpr int kSplitRows = 64;   // rows of bf16 activations in one tile of planes

struct LinearArgs {
  const uint8_t *x, *xs, *wc, *ws;
  void* out;
  long long M;
  int N, K, ksteps;
  int planes, tile_rows;   // 1: x is [M, K]; 2: the planes that uq_split_kernel writes, tiles of tile_rows
  int out_dtype;
};

UQ_DEV float e4m3_byte(uint32_t b) { return uq_e4m3_f32(b & 0xffu); }

// A warp per output channel, 8 input channels per lane at a time.
__global__ void __launch_bounds__(128) uq_fp4_linear_kernel(LinearArgs a, int pdl) {
  uq_pdl_wait();
  if (pdl) uq_pdl_release();
  const int lane = threadIdx.x & 31;
  const long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  for (long long m = blockIdx.y; m < a.M; m += gridDim.y) {
    float acc = 0.f;
    for (int k = lane * 8; k < a.K; k += 256) {
      const size_t row = ((size_t)(n / 128) * a.ksteps + k / 128) * 128 + n % 128;
      const uint32_t c = *reinterpret_cast<const uint32_t*>(a.wc + row * 64 + (k % 128) / 2);
      const float wscale = uq_scale_f32(a.ws[row * 4 + (k % 128) / 32]);
      for (int pl = 0; pl < a.planes; pl++) {
        long long xr = m;
        if (a.planes == 2) {
          const long long tile = m / a.tile_rows, left = a.M - tile * a.tile_rows;
          xr = tile * 2 * a.tile_rows + m % a.tile_rows + (pl ? (min(left, (long long)a.tile_rows) + 7) / 8 * 8 : 0);
        }
        const uint2 v = *reinterpret_cast<const uint2*>(a.x + xr * a.K + k);
        float part = 0.f;
        for (int i = 0; i < 8; i++) part = fmaf(e4m3_byte((i < 4 ? v.x : v.y) >> (8 * (i & 3))), uq_e2m1_f32((c >> (4 * i)) & 15u), part);
        acc = fmaf(part * uq_scale_f32(a.xs[xr * (a.K / 32) + k / 32]), wscale, acc);
      }
    }
    for (int d = 16; d; d >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, d);
    if (lane == 0) {
      const size_t o = (size_t)m * a.N + n;
      if (a.out_dtype == 0) static_cast<float*>(a.out)[o] = acc;
      else if (a.out_dtype == 1) static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16(acc);
      else static_cast<__half*>(a.out)[o] = __float2half(acc);
    }
  }
}

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

long long plane_rows(long long M) { return (M + kSplitRows - 1) / kSplitRows * 2 * kSplitRows; }

}  // namespace

cudaError_t uq_split_dispatch(const void*, uint8_t*, uint8_t*, long long, int, int, cudaStream_t);

// Bytes of scratch for bf16 activations: both planes' codes, then their scales.
size_t uq_fp4_linear_scratch(long long M, int K) { return M < 1 || K < 32 || K % 32 ? 0 : (size_t)plane_rows(M) * ((size_t)K + K / 32); }

// xs null: x is bf16 [M, K], scratch holds uq_fp4_linear_scratch bytes; else x is e4m3 [M, K] with scale bytes xs [M, K / 32].
// launches: kernels enqueued.
cudaError_t uq_fp4_linear_dispatch(const void* x, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, void* out, void* scratch, long long M, int N, int K, int out_dtype,
                                   unsigned int* status, cudaStream_t s, int* launches) {
  *launches = 0;
  if (M < 0 || M > (1 << 24) || N < 1 || N > (1 << 24) || K < 32 || K > (1 << 24) || K % 32 || out_dtype < 0 || out_dtype > 2) return cudaErrorInvalidValue;
  if (M == 0) return cudaSuccess;
  if (!x || !wc || !ws || !out || (!xs && !scratch)) return cudaErrorInvalidValue;
  if (!aligned_to(x, 16) || !aligned_to(wc, 32) || !aligned_to(ws, 16) || !aligned_to(out, 16) || (xs ? !aligned_to(xs, 4) : !aligned_to(scratch, 16))) return cudaErrorInvalidValue;
  (void)status;
  LinearArgs a{static_cast<const uint8_t*>(x), xs, wc, ws, out, M, N, K, (K + 127) / 128, 1, 0, out_dtype};
  if (!xs) {
    uint8_t* codes = static_cast<uint8_t*>(scratch);
    uint8_t* scales = codes + (size_t)plane_rows(M) * K;
    const cudaError_t e = uq_split_dispatch(x, codes, scales, M, K, kSplitRows, s);
    if (e != cudaSuccess) return e;
    *launches += 1;
    a.x = codes;
    a.xs = scales;
    a.planes = 2;
    a.tile_rows = kSplitRows;
  }
  const bool pdl = uq_pdl_on();
  const cudaError_t e = uq_launch(uq_fp4_linear_kernel, dim3((unsigned)((N + 3) / 4), (unsigned)(M < 32768 ? M : 32768)), 128u, 0, s, pdl, a, (int)pdl);
  if (e == cudaSuccess) *launches += 1;
  return e;
}
