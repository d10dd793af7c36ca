// Products with a weight in 4 bits: y[m, n] = sum_k x[m, k] * code[n, k] * 2^(s[n, k / 32] - 127), for the few rows of a decode or
// verify step.  No counterpart in the reference.
//
// The weight is laid out as one stream of the paged cache with 128-token pages at head_dim 128 (codes [tiles, K/128, 128, 64],
// scales [tiles, K/128, 128, 4]: a tile is 128 output channels, a "head" 128 input channels), so the cache's own encoder writes it
// and every 128 x 128 block is 8 KB of codes and 512 bytes of scales, both contiguous.
// Activations are e4m3 codes with one UE8M0 scale per 32 channels; bf16 rows are split into two such planes, whose products are
// added: up to 4 rows by the CTAs themselves, on their way into shared memory, more by a kernel of their own first (uq_rows.cu), so
// that not every tile of the weight does it again.  A group of wide range, of which two planes would leave out too
// much (mx8::wide_group), takes four: each 128 channels that hold one get two steps of their own, behind the others (ExtraSteps).
//
// What bounds it: reading the weight, N * K * 17 / 32 bytes, up to about 128 rows; so nothing is decoded by threads.  The block-scaled
// tensor instruction (kind::mxf8f6f4, one UE8M0 scale per 32 elements of K) takes the weight's codes and scale bytes as they are,
// with the 128 output channels as its M and the rows of x as its N (128 of them and a wide weight: the other way round, below):
//
//   y^T[n, m] += W[n, k] * X[m, k]     M = 128 channels, N = NB in {16, 32, 64, 128} rows, K = 32 per instruction
//
// The copy engine unpacks the 4-bit codes on the way into shared memory (16 codes = 8 bytes, then 8 bytes of padding: 128 codes
// are one 128-byte row of the swizzled tile).  The instruction wants the scales of rows l, 32 + l, 64 + l, 96 + l beside one another,
// the layout has those of 4 l .. 4 l + 3: the tensor map therefore brings the rows in the order 4 l + j -> 32 j + l (two
// dimensions of 32 and 4 rows, the outer one first in memory), and the scale bytes are copied as they lie.
//
// One CTA per (128 channels, NB rows, range of K); the ranges of one tile are a cluster, each of whose CTAs adds the fp32 partial tiles
// of all up for its share of the rows, in the order of the ranks: one launch, no scratch, the same bits every time.  The partials are
// pushed: stored straight from registers into the owner's shared memory and counted on its barrier (read by the owners between two
// cluster barriers, they took 1.8 of the 4.1 us of a 4-step CTA).  Few rows have a buffer beside the ring; more go over the ring once
// every CTA of the cluster is done with its own.
// Two CTAs fit an SM, so that their copies overlap and a grid need not be a multiple of the SMs.
//
// From a graph, weights larger than L2, beside the weight's bytes at the copy rate of 6.47 TB/s: 1 x 4096 x 4096 4.8 us (1.4), 8 bf16 rows
// x 10240 x 8192 13.4 (6.9), 17 8-bit rows x 8192 x 32768 25.6 (22), 1 x 65536 x 8192 47.6 (44), 64 bf16 rows x 65536 x 8192 68 to 71 (44).  Fill and drain are
// about 4 us of each: launch, first copies (1 us), the cluster's sum, and CTAs that start late because the last call's still hold an SM's halves.
#include <climits>

#include <algorithm>
#include <atomic>

#include "uq_mx8.cuh"
#include "uq_sm100.cuh"

namespace tc {

// warps 0-3: scales of x (or x itself, split), then the epilogue; 4: instructions; 5, 6: copies of the weight; 7, 8: copies of x and of the weight's scales.
// A copy holds its thread for some 300 cycles and a step's scales for as many, about what a step may take on an SM: the steps go
// round the warps of a role.
constexpr int kThreads = 9 * 32;
constexpr int kWarpMma = 4, kWarpW = 5, kWarpX = 7;
constexpr int kMaxSplit = 8;       // CTAs of a cluster
// Rows of bf16 that every CTA splits for itself, without the kernel that does it first (us with it / split in the CTAs: 4096 x 4096 1 row 6.55 / 5.05,
// 4 rows 6.76 / 5.12, 8 rows 6.83 / 6.35; 28672 x 8192 1 row 25.1 / 23.9, 4 rows 25.2 / 24.6, 6 rows 25.1 / 28.3, 8 rows 25.2 / 33.1).
constexpr int kDirectRows = 4;
constexpr uint32_t kNoTmem = 0xffffffffu;   // no address of tensor memory

struct LinearParams {
  const uint8_t* xs;    // [rows of the x map, K / 32]
  const __nv_bfloat16* x16;   // [M, K] bf16 rows: those that the CTAs split themselves, or those that the planes were made of
  const uint8_t* wc;
  const uint8_t* ws;
  void* out;
  unsigned int* status;
  long long M, xrows;
  int N, K, tiles, ksteps, mtiles;
  int out_dtype;
  int words;            // x's scale bytes of 128 channels are aligned words
  int pdl;
  int expire;           // for the test of the give-up path: the first step's scales of x are never announced (1: by any CTA, 2: by the last of each cluster)
};

// Steps behind a CTA's nk own: two for each of them in which a row has a group of wide range (marked by kWideByte, its planes are zeros), for that group's
// two planes and for the planes of what those leave out.  A bit per step in shared memory, or per run of steps where they are more than the bits; set
// while x's scales are brought, read once they all are (oBarMap), in ascending order: sums stay the same whoever came first.
struct ExtraSteps {
  static constexpr int kWords = 32, kBytes = 4 * kWords + 4;
  uint32_t at;   // of the words, and of one more that says whether there is a bit at all
  int nk, shift;
  UQ_DEV ExtraSteps(uint32_t at_, int nk_) : at(at_), nk(nk_), shift(0) {
    while ((nk - 1) >> shift >= 32 * kWords) shift++;
  }
  UQ_DEV uint32_t word(int w) const {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at + 4 * w) : "memory");
    return v;
  }
  UQ_DEV bool any() const { return __builtin_expect(word(kWords) != 0u, 0); }
  UQ_DEV int bit(int i) const { return i >> shift; }
  UQ_DEV void mark(int w, uint32_t bits) const {
    asm volatile("red.shared.or.b32 [%0], %1;" ::"r"(at + 4 * w), "r"(bits) : "memory");
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 4 * kWords), "r"(1) : "memory");
  }
  // f(i, k), until it says no: steps i and i + 1, from nk on, are for step k's channels
  template <typename F>
  UQ_DEV void each(F f) const {
    int i = nk;
    for (int w = 0; w <= (nk - 1) >> shift >> 5; w++)
      for (uint32_t m = word(w); m; m &= m - 1) {
        const int first = (32 * w + __ffs(m) - 1) << shift;
        for (int k = first; k < min(nk, first + (1 << shift)); k++, i += 2)
          if (!f(i, k)) return;
      }
  }
};

UQ_DEV void rows_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }   // of the first four warps
UQ_DEV bool wait_bar(uint32_t b, uint32_t parity, volatile int* abort_flag, unsigned int* status, int id, int k) {
  bool r = mbar_test(b, parity);
  if (!r) r = mbar_try(b, parity);
  if (!r) r = bounded_wait(b, parity, abort_flag, status, id, k);
  return r;
}

// One thread's marks: it takes the scale words of a row as they come and looks for kWideByte.
struct Marks {
  const ExtraSteps& extra;
  int word;
  uint32_t bits = 0;
  UQ_DEV Marks(const ExtraSteps& e, int i) : extra(e), word(e.bit(i) >> 5) {}
  UQ_DEV void flush() {
    if (bits) extra.mark(word, bits);
    bits = 0;
  }
  UQ_DEV void step(int i, uint32_t w) {
    const int b = extra.bit(i);
    if (b >> 5 != word) {
      flush();
      word = b >> 5;
    }
    static_assert(mx8::kWideByte == 0, "a zero byte, found by its borrow");
    if ((w - 0x01010101u) & ~w & 0x80808080u) bits |= 1u << (b & 31);
  }
};

template <int NB, int PLANES>
struct LinCfg {
  static constexpr int kRows = NB / PLANES;                  // rows of x per CTA
  // The partials' buffer lies beside the ring, not over it, where that costs no stage (16 bf16 rows x 10240 x 8192: beside a ring of four
  // stages 14.9 us, over one of five 13.2).
  static constexpr bool kBeside = NB == 16;
  static constexpr int kStages = NB <= 32 ? 5 : (NB == 64 ? 4 : 3);   // what half an SM's shared memory holds
  static constexpr int kA = 128 * 128, kB = NB * 128, kSf = 512;
  static constexpr int oB = kA, oSfa = oB + kB, oSfb = oSfa + kSf, kStage = oSfb + kSf;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kPRow = 512;                          // bytes of one row of a partial tile
  static constexpr int kP = (kRows + kMaxSplit - 1) * kPRow;   // (an owner's rows x the ranks: at most that many)
  static constexpr int oP = kBeside ? kRing : 0;
  static constexpr int kBody = oP + kP > kRing ? oP + kP : kRing;
  static constexpr int oBarIn = kBody, oBarTmem = oBarIn + 8, oBarDone = oBarTmem + 8, oBarF = oBarDone + 8, oBarE = oBarF + 8 * kStages;
  static constexpr int oBarLast = oBarE + 8 * kStages, oBarDone2 = oBarLast + 8, oBarMap = oBarDone2 + 8, oTmem = oBarMap + 8, oAbort = oTmem + 4, oExtra = oAbort + 4;
  static constexpr int kSmem = oExtra + ExtraSteps::kBytes;
  static constexpr int cSf = NB;                             // first column of the scales: 8 per stage (4 of the weight, 4 of x)
  static constexpr int kColsUsed = cSf + 8 * kStages;
  static constexpr int kCols = kColsUsed <= 64 ? 64 : (kColsUsed <= 128 ? 128 : 256);   // two CTAs' share an SM's 512
  // The ring's stages start on 1024-byte boundaries as long as a stage is a multiple of 1024 bytes (the swizzled tiles need it).
  static_assert(kStage % 1024 == 0 && kB % 1024 == 0, "swizzled tiles sit on 1024-byte boundaries");
  static_assert(2 * (kSmem + 1024) <= 228 * 1024, "two CTAs per SM");
};

// shared-memory matrix descriptor without a swizzle, for the copy of 32 rows of 16 bytes (8-row groups 128 bytes apart)
UQ_DEV uint64_t sf_desc(uint32_t addr) { return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | (1ull << 46); }
// 32 rows of 16 bytes -> 4 columns of the 32 lanes, the same in all four lane quarters; ordered with this thread's tensor instructions
UQ_DEV void tmem_copy_sf(uint32_t taddr, uint64_t desc) { asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory"); }
UQ_DEV void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x0, int x1, int x2, int x3, uint32_t bar, uint64_t pol) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;"
               ::"r"(dst), "l"(map), "r"(x0), "r"(x1), "r"(x2), "r"(x3), "r"(bar), "l"(pol) : "memory");
}
UQ_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
UQ_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// four bytes into a CTA of the cluster, counted on the barrier there
UQ_DEV void st_async(uint32_t addr, float v, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr), "r"(__float_as_uint(v)), "r"(bar) : "memory");
}
UQ_DEV uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Four consecutive channels n.. of a row of N: one store where the rows' boundaries allow it, else those inside the row one by one.
UQ_DEV void store4(float* o, const float* v, int n, int N) {
  if (N % 4 == 0) {
    if (n < N) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (n + j < N) o[j] = v[j];
  }
}
UQ_DEV uint32_t pack2(float a, float b, __nv_bfloat16) { return pack_bf16x2(a, b); }
UQ_DEV uint32_t pack2(float a, float b, __half) { return pack_f16x2(a, b); }
template <typename T>
UQ_DEV void store4(T* o, const float* v, int n, int N) {
  const uint32_t a = pack2(v[0], v[1], T{}), b = pack2(v[2], v[3], T{});
  if (N % 4 == 0) {
    if (n < N) *reinterpret_cast<uint2*>(o) = make_uint2(a, b);
  } else {
    const uint32_t w[4] = {a & 0xffffu, a >> 16, b & 0xffffu, b >> 16};
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (n + j < N) reinterpret_cast<unsigned short*>(o)[j] = (unsigned short)w[j];
  }
}

// (for the CTAs that split x: what seldom runs stays out of their loop)
static __device__ __noinline__ bool wide_group_far(uint4 raw, uint2 hi, uint2 lo, uint32_t hi_byte, uint32_t lo_byte) { return mx8::wide_group(raw, hi, lo, hi_byte, lo_byte); }

// x for a pair of extra steps, into the operands t0, t1 and their scales s0, s1: 128 channels (step k) of the tile's rows, the planes of wide groups into
// rows r and ROWS + r, zeros for all other groups (a row's sums do not depend on its neighbours).  A warp of WARPS has ROWS / WARPS rows and takes a group
// at a time, a channel per lane: few registers, which all launches of these kernels pay for (with eight channels per lane the kernel had 91 of them instead
// of 56, and 8 rows x 10240 x 8192, two CTAs per SM, took 13.8 us instead of 13.3).
template <int ROWS, int WARPS, bool kDirect>
UQ_DEV void extra_rows(const LinearParams& p, int m0, int rows, int k, int warp, uint8_t* t0, uint8_t* t1, uint8_t* s0, uint8_t* s1) {
  constexpr int n = ROWS / WARPS;
  const int lane = threadIdx.x & 31, r0 = warp * n;
  for (int i = lane; i < 8 * n; i += 32) {
    const int at = (r0 + i / 8) * 128 + i % 8 * 16;
    *reinterpret_cast<uint4*>(t0 + at) = *reinterpret_cast<uint4*>(t0 + ROWS * 128 + at) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(t1 + at) = *reinterpret_cast<uint4*>(t1 + ROWS * 128 + at) = make_uint4(0, 0, 0, 0);
  }
  auto scales_of = [](int r) { return (r & 31) * 16 + (r >> 5) * 4; };
  uint32_t groups = 0;   // of row r0 + lane, the wide ones
  if constexpr (kDirect) {   // as they were found before: eight channels per lane, two rows at a time
    uint32_t mine = 0;
#pragma unroll 1
    for (int j = 0; j < kDirectRows / 2; j++) {
      const int r = 2 * j + (lane >> 4), c = 128 * k + 8 * (lane & 15);
      mx8::Raw<__nv_bfloat16> x;
      x.a = make_uint4(0, 0, 0, 0);
      if (r < rows && c < p.K) x.load(p.x16 + (long long)(m0 + r) * p.K + c);
      float v[8];
      x.get(v);
      uint2 hi, lo;
      uint32_t hi_byte, lo_byte;
      mx8::split_piece(v, hi, lo, hi_byte, lo_byte);
      const uint32_t wide = __ballot_sync(0xffffffffu, wide_group_far(x.a, hi, lo, hi_byte, lo_byte));
      if (lane >> 1 == j) mine = wide >> 16 * (lane & 1);
    }
    groups = (mine & 1u) | (mine >> 3 & 2u) | (mine >> 6 & 4u) | (mine >> 9 & 8u);   // (four lanes a group)
  }
  if (lane < n) {
    const int r = r0 + lane;
    *reinterpret_cast<uint32_t*>(s0 + scales_of(r)) = *reinterpret_cast<uint32_t*>(s0 + scales_of(ROWS + r)) = 0x01010101u;
    *reinterpret_cast<uint32_t*>(s1 + scales_of(r)) = *reinterpret_cast<uint32_t*>(s1 + scales_of(ROWS + r)) = 0x01010101u;
    if (!kDirect && r < rows) {
      const uint8_t* bytes = p.xs + (long long)(2 * m0 + r) * (p.K / 32) + 4 * k;   // (m0: a multiple of ROWS)
      const uint32_t four = p.words ? *reinterpret_cast<const uint32_t*>(bytes) : 0u;
      for (int g = 0; g < 4 && 4 * k + g < p.K / 32; g++)
        if ((p.words ? four >> 8 * g & 0xffu : (uint32_t)bytes[g]) == mx8::kWideByte) groups |= 1u << g;
    }
  }
  __syncwarp();
  int r = -1;
  uint32_t left = 0;
  auto next = [&]() -> int {   // the next group, its row in r; -1: no more
    while (!left) {
      if (++r >= n) return -1;
      left = __shfl_sync(0xffffffffu, groups, r);
    }
    const int g = __ffs(left) - 1;
    left &= left - 1;
    return g;
  };
  auto load = [&](int g) -> uint32_t { return *reinterpret_cast<const unsigned short*>(p.x16 + (long long)(m0 + r0 + r) * p.K + 128 * k + 32 * g + lane); };
  int g = next();
  uint32_t x = g < 0 ? 0u : load(g);
#pragma unroll 1
  while (g >= 0) {
    const int row = r0 + r, c = 32 * g + lane;
    float v = __uint_as_float(x << 16);
    uint8_t* at0 = t0 + row * 128 + (((c >> 4) ^ (row & 7)) << 4) + (c & 15);
    const int to1 = (int)(t1 - t0), sf = scales_of(row) + g, sf2 = scales_of(ROWS + row) + g;
    g = next();
    if (g >= 0) x = load(g);
    uint32_t codes = 0;   // four planes' and their bytes
    uint32_t bytes = 0;
#pragma unroll 1
    for (int i = 0; i < 32; i += 8) {
      const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(v))));
      const uint32_t byte = max(mx8::scale_byte(amax), 1u), code = mx8::e4m3x2(__fmul_rn(v, mx8::inverse_scale(byte)), 0.f) & 0xffu;
      v = fmaf(mx8::e4m3_value(code), -uq_scale_f32(byte), v);
      codes |= code << i;
      bytes |= byte << i;
    }
    at0[0] = (uint8_t)codes;
    at0[ROWS * 128] = (uint8_t)(codes >> 8);
    at0[to1] = (uint8_t)(codes >> 16);
    at0[to1 + ROWS * 128] = (uint8_t)(codes >> 24);
    if (lane == 0) {
      s0[sf] = (uint8_t)bytes;
      s0[sf2] = (uint8_t)(bytes >> 8);
      s1[sf] = (uint8_t)(bytes >> 16);
      s1[sf2] = (uint8_t)(bytes >> 24);
    }
  }
}

// The extra steps of the kernel below, for its first four warps, which bring them whole, and for its issuing thread.
template <typename C, int kScaleWarps, bool kDirect>
__device__ __noinline__ bool bring_extra(const LinearParams& p, const CUtensorMap& map_w, uint32_t sm, uint8_t* smem, int nk, int k0, int tile_n, int m0, int rows) {
  constexpr int kGroups = 4 / kScaleWarps;
  static_assert(C::kStages >= 3, "a pair of steps, and whoever waits for a stage has seen the turn before the last one's end");
  const int warp = threadIdx.x >> 5;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::oAbort);
  bool ok = true;
  int issued = nk;
  auto free_stage = [&](int i) -> bool {
    const int s = i % C::kStages;
    return ok = __all_sync(0xffffffffu, i < C::kStages || wait_bar(sm + C::oBarE + 8 * s, ((i / C::kStages) & 1) ^ 1, abort_flag, p.status, 45, i));
  };
  ExtraSteps(sm + C::oExtra, nk).each([&](int i, int k) -> bool {
    const int mine = i + ((i ^ warp) & 1);   // two warps take turns at the weight's codes, two at its scales
    if (!free_stage(mine)) return false;
    if (elect_one()) {
      const uint32_t st = sm + mine % C::kStages * C::kStage, b = sm + C::oBarF + 8 * (mine % C::kStages);
      const size_t block = (size_t)tile_n * p.ksteps + k0 + k;
      mbar_expect_tx(b, warp < 2 ? 8192 : C::kSf);
      if (warp < 2) tma_load_4d(st, &map_w, 0, 0, 0, (int)block, b, l2_policy());
      else bulk_load(st + C::oSfa, p.ws + block * 512, 512, b, l2_policy());
      issued = mine + 1;
    }
    __syncwarp();
    if (((i - nk) >> 1) % kGroups == warp / kScaleWarps) {
      if (!free_stage(i) || !free_stage(i + 1)) return false;
      uint8_t *st0 = smem + i % C::kStages * C::kStage, *st1 = smem + (i + 1) % C::kStages * C::kStage;
      extra_rows<C::kRows, kScaleWarps, kDirect>(p, m0, rows, k0 + k, warp % kScaleWarps, st0 + C::oB, st1 + C::oB, st0 + C::oSfb, st1 + C::oSfb);
      fence_async_smem();
      __syncwarp();
      if ((threadIdx.x & 31) < 2) mbar_arrive(sm + C::oBarF + 8 * ((i + (threadIdx.x & 31)) % C::kStages));
    }
    return true;
  });
  ok = __all_sync(0xffffffffu, ok && wait_bar(sm + C::oBarDone2, 0, abort_flag, p.status, 46, nk));
  if (!ok)   // gave up: what this thread has copied lands before the CTA may end (where such a stage has been filled again, the wait runs out)
    for (int j = issued - 1; j >= nk && j >= issued - 2 * C::kStages; j -= 2) wait_bar(sm + C::oBarF + 8 * (j % C::kStages), (j / C::kStages) & 1, abort_flag, p.status, 41, j);
  __syncwarp();
  return ok;
}
template <typename C, int NB>
UQ_DEV void multiply_step(uint32_t sm, uint32_t tmem, int s, bool first) {
  tc_fence_after();
  const uint32_t st = sm + s * C::kStage, sf = tmem + C::cSf + 8 * s;
  tmem_copy_sf(sf, sf_desc(st + C::oSfa));
  tmem_copy_sf(sf + 4, sf_desc(st + C::oSfb));
  const uint64_t a = smem_desc(st, 16, 1024), b = smem_desc(st + C::oB, 16, 1024);
#pragma unroll
  for (int kb = 0; kb < 4; kb++)
    mma_bs(tmem, a + (uint64_t)(kb * 2), b + (uint64_t)(kb * 2), instr_desc_bs(128, NB, 5, 0, kb, kb), sf, sf + 4, (!first || kb) ? 1u : 0u);
}
template <typename C, int NB>
__device__ __noinline__ bool multiply_extra(uint32_t sm, volatile int* abort_flag, unsigned int* status, uint32_t tmem, int nk) {
  bool ok = true;
  for (int j = max(nk - C::kStages, 0); j < nk; j++) tc_commit(sm + C::oBarE + 8 * (j % C::kStages));   // the last stages of the steps before, which nobody has waited for
  ExtraSteps(sm + C::oExtra, nk).each([&](int first, int) -> bool {
    for (int i = first; i < first + 2; i++) {
      const int s = i % C::kStages;
      if (!(ok = wait_bar(sm + C::oBarF + 8 * s, (i / C::kStages) & 1, abort_flag, status, 42, i))) return false;
      multiply_step<C, NB>(sm, tmem, s, false);
      tc_commit(sm + C::oBarE + 8 * s);
    }
    return true;
  });
  if (ok) tc_commit(sm + C::oBarDone2);
  return ok;
}

template <int NB, int PLANES, bool kDirect>
__global__ void __launch_bounds__(kThreads, 2) uq_fp4_linear_kernel(const __grid_constant__ LinearParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
  using C = LinCfg<NB, PLANES>;
  extern __shared__ __align__(1024) uint8_t smem_lin[];
  const uint32_t sm = smem_u32(smem_lin);
  if (sm & 1023u) {   // never expected; the swizzled layouts below would be wrong
    uq_pdl_wait();
    if (threadIdx.x == 0) uq_report(p.status, 2u, sm, 1u);
    return;           // (every CTA of a cluster alike: the offset is the kernel's)
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = gridDim.y, rank = blockIdx.y;
  const int tile_n = blockIdx.x / p.mtiles, tile_m = blockIdx.x % p.mtiles;
  const int k0 = (int)((long long)p.ksteps * rank / split), nk = (int)((long long)p.ksteps * (rank + 1) / split) - k0;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_lin + C::oAbort);
  auto stage_at = [&](int s) { return sm + s * C::kStage; };
  auto bar = [&](int o, int s) { return sm + o + 8 * s; };
  auto wait = [&](uint32_t b, uint32_t parity, int id, int k) -> bool { return wait_bar(b, parity, abort_flag, p.status, id, k); };
  const size_t block0 = (size_t)tile_n * p.ksteps + k0;   // first 128 x 128 block of this CTA's range
  // A step's stage has one barrier for all that comes into it (weight, x with the weight's scales, x's scales): every barrier looked at
  // costs the issuing thread 30 of the 460 cycles that a step took it with three.
  auto full_bar = [&](int i) { return bar(C::oBarF, i % C::kStages); };
  // (A wait by parity tells a phase from its neighbours only: the warps of a role that take turns are no more than the stages, so that
  // a warp's step before this one has seen the phase before the one that it now waits for.)
  auto wait_free = [&](int i, int id) -> bool { return i < C::kStages || wait(bar(C::oBarE, i % C::kStages), ((i / C::kStages) & 1) ^ 1, id, i); };
  constexpr int kScaleWarps = (NB + 31) / 32, kGroups = 4 / kScaleWarps;   // warps that bring a step's scales (or x itself), and how many such groups take turns
  static_assert(kGroups <= C::kStages && 2 <= C::kStages, "no more turns than stages");
  constexpr bool kExtra = PLANES == 2;
  const ExtraSteps extra(sm + C::oExtra, nk);
  static_assert(ExtraSteps::kWords == 32, "a word per lane");

  const long long m0 = (long long)tile_m * C::kRows;
  const int rows = (int)min((long long)C::kRows, p.M - m0);   // of this tile
  const int mine = (rows - rank + split - 1) / split;         // rows rank, rank + split, .. are this CTA's to add up
  const bool expire = p.expire == 1 || (p.expire == 2 && rank == split - 1);

  if (warp == 0) {   // a barrier per lane
    constexpr int kBars = 6 + 2 * C::kStages;
    static_assert(kBars <= 32 && C::oBarE == C::oBarIn + 8 * (3 + C::kStages), "barriers lie side by side");
    if (lane < kBars) mbar_init(sm + C::oBarIn + 8 * lane, lane >= 3 && lane < 3 + C::kStages ? 2 + kScaleWarps : (lane == kBars - 1 ? 4 : 1));
    if (kExtra) *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oExtra + 4 * lane) = 0;
    fence_barrier_init();
    if (lane == 0) {
      *abort_flag = 0;
      *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem) = kNoTmem;
      *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oExtra + 4 * ExtraSteps::kWords) = 0;
    }
    __syncwarp();
    if (split > 1 && lane == 0) mbar_expect_tx(bar(C::oBarIn, 0), (uint32_t)(mine * split * C::kPRow));   // (no rows: complete at once)
  } else if (warp >= kWarpW && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(warp < kWarpX ? &map_w : &map_x) : "memory");   // (launch arguments, not global memory)
  }
  __syncthreads();
  if (C::kBeside && split > 1) cluster_arrive();   // every CTA's barriers stand before the first push
  uq_pdl_wait();   // from here on global memory is read and written
  if (p.pdl) uq_pdl_release();

  int issued = 0;   // by a copying thread: every other step below it
  if (warp >= kWarpW) {
    // ---- copies: two threads each for the weight's codes, and for x with the weight's scales
    const bool weights = warp < kWarpX;
    const int turn = weights ? warp - kWarpW : warp - kWarpX;
    if (elect_one()) {
      const uint64_t pol = l2_policy();
      uint64_t keep;
      asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));   // (x is read by every tile; 4096 x 4096: 5.2 us, 6.0 without)
      int i = turn;
      for (; i < nk; i += 2) {
        if (!wait_free(i, 40)) break;
        const uint32_t st = stage_at(i % C::kStages), b = full_bar(i);
        if (weights) {
          mbar_expect_tx(b, 8192);   // the packed bytes are counted
          tma_load_4d(st, &map_w, 0, 0, 0, (int)(block0 + i), b, pol);
        } else {
          mbar_expect_tx(b, (kDirect ? 0 : C::kB) + C::kSf);
          if (!kDirect) tma_load_2d(st + C::oB, &map_x, (k0 + i) * 128, tile_m * NB, b, keep);
          bulk_load(st + C::oSfa, p.ws + (block0 + i) * 512, 512, b, pol);
        }
      }
      issued = i;
    }
  } else if (warp == kWarpMma) {
    // (tensor memory is taken after the wait: see the verify kernel)
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm + C::oTmem), "n"(C::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    uint32_t tmem = kNoTmem;   // (the address is written before the allocation returns: the first read has it)
    for (int i = 0; i < (1 << 20) && tmem == kNoTmem; i++) tmem = *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem);
    if (elect_one()) {
      bool ok = tmem != kNoTmem;
      if (ok) {
        tc_fence_before();
        mbar_arrive(bar(C::oBarTmem, 0));
      } else {
        *abort_flag = 1;
        uq_report(p.status, 1u, 49u, 0u);
      }
      // The next step's barrier is looked at before this step's instructions are issued.
      int s = 0;
      uint32_t parity = 0, here = mbar_test(bar(C::oBarF, 0), 0);
      for (int i = 0; i < nk && ok; i++) {
        if (!here && !(ok = wait(bar(C::oBarF, s), parity, 42, i))) break;
        const int s1 = s + 1 == C::kStages ? 0 : s + 1;
        const uint32_t parity1 = parity ^ (s1 == 0 ? 1u : 0u);
        here = mbar_test(bar(C::oBarF, s1), parity1);
        multiply_step<C, NB>(sm, tmem, s, i == 0);
        if (i + C::kStages < nk) tc_commit(bar(C::oBarE, s));   // (nobody waits for the last ones, but for the steps behind them)
        s = s1;
        parity = parity1;
      }
      if (ok) tc_commit(bar(C::oBarDone, 0));
      if (kExtra && ok && (ok = wait(bar(C::oBarMap, 0), 0, 44, nk)) && extra.any()) ok = multiply_extra<C, NB>(sm, abort_flag, p.status, tmem, nk);
      if (!ok && tmem != kNoTmem) {   // gave up: what has been issued ends before tensor memory goes back
        tc_commit(bar(C::oBarLast, 0));
        ended_wait(bar(C::oBarLast, 0), 0);
      }
    }
  } else {
    int i = warp / kScaleWarps;
    if constexpr (kDirect) {
      // ---- x itself: a warp splits a step's 4 rows x 128 channels (lane: piece lane % 16 of rows lane / 16 and 2 + lane / 16) into the two planes of the
      // tile, rows r and 8 + r of 128 bytes with the 128-byte swizzle, and their scale bytes; the next step's loads are on their way.
      static_assert(!kDirect || (NB == 16 && PLANES == 2), "rows of both planes");
      constexpr int kPer = kDirectRows / 2;   // pieces of a lane
      const int piece = lane & 15, r0 = lane >> 4;
      mx8::Raw<__nv_bfloat16> next[kPer];
      auto load = [&](int i) {
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          const int k = (k0 + i) * 128 + piece * 8;
          if (2 * j >= rows) break;   // (the tile's rows behind the last one are never written, their products never read)
          if (i < nk && 2 * j + r0 < rows && k < p.K) next[j].load(p.x16 + (m0 + 2 * j + r0) * p.K + k);
          else next[j].a = make_uint4(0, 0, 0, 0);
        }
      };
      load(warp);
      for (; i < nk; i += 4) {
        const int s = i % C::kStages;
        uint2 hi[kPer], lo[kPer];
        uint32_t hi_byte[kPer], lo_byte[kPer];
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          if (2 * j >= rows) break;
          float v[8];
          next[j].get(v);
          mx8::split_piece(v, hi[j], lo[j], hi_byte[j], lo_byte[j]);
        }
        bool look = false;
#pragma unroll
        for (int j = 0; j < kPer; j++) look |= 2 * j + r0 < rows && mx8::may_leave(hi[j]);
        if (__builtin_expect(__any_sync(0xffffffffu, look), 0)) {   // (a step in ten of normally distributed values; with may_be_wide at once: 4 rows x 4096 x 4096 5.19 us, not 5.05)
          bool any = false;
#pragma unroll
          for (int j = 0; j < kPer; j++) {
            if (2 * j >= rows) break;
            if (__any_sync(0xffffffffu, mx8::may_be_wide(hi[j])) && wide_group_far(next[j].a, hi[j], lo[j], hi_byte[j], lo_byte[j])) {
              hi[j] = lo[j] = make_uint2(0, 0);
              hi_byte[j] = lo_byte[j] = mx8::kWideByte;
              any = true;
            }
          }
          if (any) extra.mark(extra.bit(i) >> 5, 1u << (extra.bit(i) & 31));
        }
        load(i + 4);
        if (!__all_sync(0xffffffffu, wait_free(i, 45))) break;
        uint8_t *tile = smem_lin + s * C::kStage + C::oB, *sf = smem_lin + s * C::kStage + C::oSfb + (piece >> 2);
#pragma unroll
        for (int j = 0; j < kPer; j++) {
          if (2 * j >= rows) break;
          const int r = 2 * j + r0, at = (((piece >> 1) ^ r) << 4) + (piece & 1) * 8;   // (r < 8: rows r and 8 + r have the same swizzle)
          *reinterpret_cast<uint2*>(tile + r * 128 + at) = hi[j];
          *reinterpret_cast<uint2*>(tile + (8 + r) * 128 + at) = lo[j];
          if ((piece & 3) == 0) {
            sf[r * 16] = (uint8_t)hi_byte[j];
            sf[(8 + r) * 16] = (uint8_t)lo_byte[j];
          }
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && (i > 0 || !expire)) mbar_arrive(full_bar(i));
      }
    } else {
      // ---- x's scales: thread r of a group of warps has row r's four bytes of the group's steps, two loads ahead
      const int r = (warp % kScaleWarps) * 32 + lane, groups = p.K / 32;
      const long long row = (long long)tile_m * NB + r;
      const bool have = r < NB && row < p.xrows && (!kExtra || r % C::kRows < rows);   // (what lies behind the last row was never written)
      const uint8_t* src = p.xs + row * groups;
      auto load = [&](int i) -> uint32_t {
        uint32_t w = 0x7f7f7f7fu;
        if (have && i < nk) {
          const int g = (k0 + i) * 4;
          if (p.words) return *reinterpret_cast<const uint32_t*>(src + g);
#pragma unroll
          for (int j = 0; j < 4; j++)
            if (g + j < groups) w = (w & ~(0xffu << (8 * j))) | ((uint32_t)src[g + j] << (8 * j));
        }
        return w;
      };
      uint32_t w0 = load(i), w1 = load(i + kGroups);
      Marks marks(extra, i);
      for (; i < nk; i += kGroups) {
        const int s = i % C::kStages;
        if (!__all_sync(0xffffffffu, wait_free(i, 45))) break;
        if (r < NB) *reinterpret_cast<uint32_t*>(smem_lin + s * C::kStage + C::oSfb + lane * 16 + (r >> 5) * 4) = w0;
        fence_async_smem();
        __syncwarp();
        if (lane == 0 && (i > 0 || !expire)) mbar_arrive(full_bar(i));
        if (kExtra) marks.step(i, w0);
        w0 = w1;
        w1 = load(i + 2 * kGroups);
      }
      if (kExtra) marks.flush();
    }
    bool more = false;
    if (kExtra) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::oBarMap, 0));
      rows_barrier();
      more = extra.any();
    }
    // ---- epilogue, first half: the accumulator's lane 32 j + l is channel 4 l + j of the tile.  A row of a partial tile is four runs of
    // 32 floats, one per warp.  Pushed, row t goes to the CTA of rank t % split, place (t / split, this rank).
    bool ok = __all_sync(0xffffffffu, wait(bar(C::oBarDone, 0), 0, 46, nk) && wait(bar(C::oBarTmem, 0), 0, 47, nk));
    if (more && ok) ok = bring_extra<C, kScaleWarps, kDirect>(p, map_w, sm, smem_lin, nk, k0, tile_n, (int)m0, rows);
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem);
    if (ok) tc_fence_after();
    if (split > 1) {
      if (!C::kBeside) cluster_arrive();   // this CTA's ring is free
      cluster_wait();
    }
    int owner = 0;
    uint32_t place = sm + C::oP + rank * C::kPRow + tid * 4;   // (row / split, rank)
#pragma unroll
    for (int c = 0; c < C::kRows; c += 8) {
      uint32_t v[8];
      if (ok) {
        tmem_ld8(tmem + ((uint32_t)(warp * 32) << 16) + c, v);
        if (PLANES == 2) {
          uint32_t u[8];
          tmem_ld8(tmem + ((uint32_t)(warp * 32) << 16) + C::kRows + c, u);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u[j]));
        } else {
          tc_wait_ld();
        }
      } else {   // gave up: the failure shows in the output
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0x7fc00000u;
      }
      if (split > 1) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          if (c + j < rows) st_async(cluster_addr(place, owner), __uint_as_float(v[j]), cluster_addr(bar(C::oBarIn, 0), owner));
          if (++owner == split) {
            owner = 0;
            place += split * C::kPRow;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) *reinterpret_cast<float*>(smem_lin + C::oP + (c + j) * C::kPRow + tid * 4) = __uint_as_float(v[j]);
      }
    }
    if (ok) tc_fence_before();
  }
  __syncwarp();
  bool in = true;
  if (split > 1) {
    if (warp >= kWarpMma) {   // (every thread of the cluster takes part)
      if (!C::kBeside) cluster_arrive();
      cluster_wait();
    }
    in = wait(bar(C::oBarIn, 0), 0, 48, nk);
  } else {
    __syncthreads();
  }
  in = in && !*abort_flag;
  // ---- second half: this CTA's share of the rows, the partial tiles in the order of the ranks.  A warp per row, four consecutive
  // channels per lane; the loads of all ranks are issued before the first addition.
  for (int i = warp; i < mine; i += kThreads / 32) {
    const int t = rank + i * split, n = tile_n * 128 + 4 * lane;
    float u[kMaxSplit][4];
#pragma unroll
    for (int r = 0; r < kMaxSplit; r++)
      if (r < split) {
        const uint8_t* at = smem_lin + C::oP + (i * split + r) * C::kPRow + lane * 4;
#pragma unroll
        for (int j = 0; j < 4; j++) u[r][j] = *reinterpret_cast<const float*>(at + j * 128);
      }
    float v[4] = {u[0][0], u[0][1], u[0][2], u[0][3]};
#pragma unroll
    for (int r = 1; r < kMaxSplit; r++)
      if (r < split)
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] += u[r][j];
    if (!in) v[0] = v[1] = v[2] = v[3] = __int_as_float(0x7fc00000);
    const size_t o = (size_t)(m0 + t) * p.N + n;
    if (p.out_dtype == 0) store4(static_cast<float*>(p.out) + o, v, n, p.N);
    else if (p.out_dtype == 1) store4(static_cast<__nv_bfloat16*>(p.out) + o, v, n, p.N);
    else store4(static_cast<__half*>(p.out) + o, v, n, p.N);
  }
  __syncthreads();
  if (warp == kWarpMma) {
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem);
    if (tmem != kNoTmem) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kCols) : "memory");
  } else if (*abort_flag) {
    // Somebody here gave up, and the CTA ends behind all that reaches its shared memory.  Pushes: it is sent all of them, and soon, since a CTA that gives up
    // pushes NaN behind its last limited wait (a barrier of the whole cluster at the end of every call instead: 0.14 us).  Copies: the stages' last
    // turns, and those before them, of which nobody may have taken notice (where such a stage has been filled again, the wait runs out).
    if (split > 1) ended_wait(bar(C::oBarIn, 0), 0);
    for (int j = issued - 2; j >= 0 && j >= issued - 2 * C::kStages; j -= 2) wait(full_bar(j), (j / C::kStages) & 1, 41, j);
  }
}

// ---------------------------------------------------------------------------------------------- 128 operand rows, wide weights
// More than 64 operand rows (33 to 64 rows of bf16 a tile, 65 to 128 of 8-bit values) and more tiles than SMs.  With the weight as the
// instruction's 128 rows a step brings 8.5 KB of weight and 16 KB of x, for one use, and writes and reads 64 KB of shared memory (512
// cycles of its 128 bytes).  Here x's 128 rows are the instruction's M and 256 channels its N: x comes, and is read, once per 256
// channels: 48 KB per 128 x 128 block of the weight.  One CTA per SM (the accumulators take half of tensor memory), the result is laid out over
// the ring at the end.
//
//   y[m, n] += X[m, k] * W[n, k]     M = 128 rows, N = 256 channels, K = 32 per instruction
template <int PLANES>
struct WideCfg {
  static constexpr int kRows = 128 / PLANES;
  static constexpr int kStages = 4;
  static constexpr int kW = 128 * 128, kX = 128 * 128, kSf = 512;   // bytes of one block of the weight, of x, of one block's scales
  static constexpr int oX = 2 * kW, oSfw = oX + kX, oSfx = oSfw + 2 * kSf, kStage = (oSfx + kSf + 1023) / 1024 * 1024;
  static constexpr int kRing = kStages * kStage;
  static constexpr int kPRow = 257 * 4;                             // bytes of a row of the result, one per operand row (odd in words: a lane per row writes it)
  static constexpr int oBarDone = kRing, oBarTmem = oBarDone + 8, oBarW = oBarTmem + 8, oBarX = oBarW + 8 * kStages, oBarS = oBarX + 8 * kStages, oBarE = oBarS + 8 * kStages;
  static constexpr int oBarLast = oBarE + 8 * kStages, oBarDone2 = oBarLast + 8, oBarMap = oBarDone2 + 8, oTmem = oBarMap + 8, oAbort = oTmem + 4, oExtra = oAbort + 4;
  static constexpr int kSmem = oExtra + ExtraSteps::kBytes;
  static constexpr int cSf = 256, kCols = 512;                      // columns of the scales: 12 per stage (4 of x, 8 of the weight)
  static_assert(128 * kPRow <= kRing && cSf + 12 * kStages <= kCols && kSmem + 1024 <= 228 * 1024, "fits an SM");
};

// Its extra steps, as above: every warp has a role in each.
template <typename C>
__device__ __noinline__ bool bring_extra_wide(const LinearParams& p, const CUtensorMap& map_w, uint32_t sm, uint8_t* smem, int nk, int pair, int m0, int rows) {
  const int role = threadIdx.x >> 5;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::oAbort);
  bool ok = true;
  int issued = nk;
  ExtraSteps(sm + C::oExtra, nk).each([&](int first, int k) -> bool {
    for (int i = first; i < first + 2; i++) {
      const int s = i % C::kStages;
      if (!(ok = __all_sync(0xffffffffu, i < C::kStages || wait_bar(sm + C::oBarE + 8 * s, ((i / C::kStages) & 1) ^ 1, abort_flag, p.status, 55, i)))) return false;
      if (elect_one()) {
        const uint32_t st = sm + s * C::kStage, b = sm + (role < 2 ? C::oBarW : C::oBarX) + 8 * s;
        const size_t block0 = (size_t)(2 * pair) * nk + k, block1 = (size_t)min(2 * pair + 1, p.tiles - 1) * nk + k;
        if (role == 2) {
          mbar_arrive(b);
        } else if (role < 2) {
          mbar_expect_tx(b, 8192);
          tma_load_4d(st + role * C::kW, &map_w, 0, 0, 0, (int)(role ? block1 : block0), b, l2_policy());
        } else {
          mbar_expect_tx(b, 2 * C::kSf);
          bulk_load(st + C::oSfw, p.ws + block0 * 512, 512, b, l2_policy());
          bulk_load(st + C::oSfw + C::kSf, p.ws + block1 * 512, 512, b, l2_policy());
        }
        issued = i + 1;
      }
      __syncwarp();
    }
    uint8_t *st0 = smem + first % C::kStages * C::kStage, *st1 = smem + (first + 1) % C::kStages * C::kStage;
    extra_rows<C::kRows, 4, false>(p, m0, rows, k, role, st0 + C::oX, st1 + C::oX, st0 + C::oSfx, st1 + C::oSfx);
    fence_async_smem();
    __syncwarp();
    if ((threadIdx.x & 31) < 2) mbar_arrive(sm + C::oBarS + 8 * ((first + (threadIdx.x & 31)) % C::kStages));
    return true;
  });
  ok = __all_sync(0xffffffffu, ok && wait_bar(sm + C::oBarDone2, 0, abort_flag, p.status, 56, nk));
  if (!ok)
    for (int j = issued - 1; j >= nk && j >= issued - C::kStages; j--)
      wait_bar(sm + (role < 2 ? C::oBarW : C::oBarX) + 8 * (j % C::kStages), (j / C::kStages) & 1, abort_flag, p.status, 51, j);
  __syncwarp();
  return ok;
}
template <typename C>
UQ_DEV bool multiply_step_wide(uint32_t sm, volatile int* abort_flag, unsigned int* status, uint32_t tmem, int i) {
  const int s = i % C::kStages;
  const uint32_t parity = (i / C::kStages) & 1;
  if (!(wait_bar(sm + C::oBarX + 8 * s, parity, abort_flag, status, 52, i) && wait_bar(sm + C::oBarS + 8 * s, parity, abort_flag, status, 53, i) &&
        wait_bar(sm + C::oBarW + 8 * s, parity, abort_flag, status, 54, i)))
    return false;
  tc_fence_after();
  const uint32_t st = sm + s * C::kStage, sf = tmem + C::cSf + 12 * s;
  tmem_copy_sf(sf, sf_desc(st + C::oSfx));
  tmem_copy_sf(sf + 4, sf_desc(st + C::oSfw));
  tmem_copy_sf(sf + 8, sf_desc(st + C::oSfw + C::kSf));
  const uint64_t a = smem_desc(st + C::oX, 16, 1024), b = smem_desc(st, 16, 1024);
#pragma unroll
  for (int kb = 0; kb < 4; kb++)
    mma_bs(tmem, a + (uint64_t)(kb * 2), b + (uint64_t)(kb * 2), instr_desc_bs(128, 256, 0, 5, kb, kb), sf, sf + 4, (i || kb) ? 1u : 0u);
  return true;
}
template <typename C>
__device__ __noinline__ bool multiply_extra_wide(uint32_t sm, volatile int* abort_flag, unsigned int* status, uint32_t tmem, int nk) {
  bool ok = true;
  for (int j = max(nk - C::kStages, 0); j < nk; j++) tc_commit(sm + C::oBarE + 8 * (j % C::kStages));
  ExtraSteps(sm + C::oExtra, nk).each([&](int first, int) -> bool {
    for (int i = first; i < first + 2 && ok; i++) {
      ok = multiply_step_wide<C>(sm, abort_flag, status, tmem, i);
      if (ok) tc_commit(sm + C::oBarE + 8 * (i % C::kStages));
    }
    return ok;
  });
  if (ok) tc_commit(sm + C::oBarDone2);
  return ok;
}

template <int PLANES>
__global__ void __launch_bounds__(kThreads, 1) uq_fp4_linear_wide_kernel(const __grid_constant__ LinearParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
  using C = WideCfg<PLANES>;
  extern __shared__ __align__(1024) uint8_t smem_lin[];
  const uint32_t sm = smem_u32(smem_lin);
  if (sm & 1023u) {   // never expected; the swizzled layouts below would be wrong
    uq_pdl_wait();
    if (threadIdx.x == 0) uq_report(p.status, 2u, sm, 1u);
    return;
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pair = blockIdx.x / p.mtiles, tile_m = blockIdx.x % p.mtiles, nk = p.ksteps;
  const long long m0 = (long long)tile_m * C::kRows;
  const int rows = (int)min((long long)C::kRows, p.M - m0);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_lin + C::oAbort);
  auto stage_at = [&](int s) { return sm + s * C::kStage; };
  auto bar = [&](int o, int s) { return sm + o + 8 * s; };
  auto wait = [&](uint32_t b, uint32_t parity, int id, int k) -> bool { return wait_bar(b, parity, abort_flag, p.status, id, k); };
  constexpr bool kExtra = PLANES == 2;
  const ExtraSteps extra(sm + C::oExtra, nk);
  // first blocks of the pair's two tiles (an odd number of tiles: the last one twice, its second copy is never stored)
  const size_t block[2] = {(size_t)(2 * pair) * nk, (size_t)min(2 * pair + 1, p.tiles - 1) * nk};

  if (warp == 0) {   // a barrier per lane
    constexpr int kBars = 5 + 4 * C::kStages;
    static_assert(kBars <= 32 && C::oBarE == C::oBarDone + 8 * (2 + 3 * C::kStages), "barriers lie side by side");
    if (lane < kBars) mbar_init(sm + C::oBarDone + 8 * lane, lane == kBars - 1 ? 4 : (lane < 2 || lane >= 2 + 3 * C::kStages ? 1 : (lane < 2 + 2 * C::kStages ? 2 : 4)));
    if (kExtra) *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oExtra + 4 * lane) = 0;
    fence_barrier_init();
    if (lane == 0) {
      *abort_flag = 0;
      *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem) = kNoTmem;
      *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oExtra + 4 * ExtraSteps::kWords) = 0;
    }
  } else if (warp >= kWarpW && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(warp < kWarpX ? &map_w : &map_x) : "memory");   // (launch arguments, not global memory)
  }
  __syncthreads();
  uq_pdl_wait();   // from here on global memory is read and written
  if (p.pdl) uq_pdl_release();

  if (warp >= kWarpW) {
    // ---- copies: a thread each for the two blocks of the weight, for x, and for the weight's scales
    const int role = warp - kWarpW;
    if (elect_one()) {
      const uint64_t pol = l2_policy();
      uint64_t keep;
      asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
      const int full = role < 2 ? C::oBarW : C::oBarX;
      int i = 0;
      for (; i < nk; i++) {
        const int s = i % C::kStages;
        if (i >= C::kStages && !wait(bar(C::oBarE, s), ((i / C::kStages) & 1) ^ 1, 50, i)) break;
        const uint32_t st = stage_at(s), b = bar(full, s);
        if (role < 2) {
          mbar_expect_tx(b, 8192);   // the packed bytes are counted
          tma_load_4d(st + role * C::kW, &map_w, 0, 0, 0, (int)(block[role] + i), b, pol);
        } else if (role == 2) {
          mbar_expect_tx(b, C::kX);
          tma_load_2d(st + C::oX, &map_x, i * 128, tile_m * 128, b, keep);
        } else {
          mbar_expect_tx(b, 2 * C::kSf);
          bulk_load(st + C::oSfw, p.ws + (block[0] + i) * 512, 512, b, pol);
          bulk_load(st + C::oSfw + C::kSf, p.ws + (block[1] + i) * 512, 512, b, pol);
        }
      }
      // What this thread has in flight lands before the CTA may end (it fills every stage itself: all but the last turns have been seen to land).
      for (int j = i - 1; j >= 0 && j >= i - C::kStages; j--) wait(bar(full, j % C::kStages), (j / C::kStages) & 1, 51, j);
    }
  } else if (warp == kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm + C::oTmem), "n"(C::kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    uint32_t tmem = kNoTmem;   // (the address is written before the allocation returns: the first read has it)
    for (int i = 0; i < (1 << 20) && tmem == kNoTmem; i++) tmem = *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem);
    if (elect_one()) {
      bool ok = tmem != kNoTmem;
      if (ok) {
        tc_fence_before();
        mbar_arrive(bar(C::oBarTmem, 0));
      } else {
        *abort_flag = 1;
        uq_report(p.status, 1u, 59u, 0u);
      }
      for (int i = 0; i < nk && ok; i++) {
        ok = multiply_step_wide<C>(sm, abort_flag, p.status, tmem, i);
        if (ok && i + C::kStages < nk) tc_commit(bar(C::oBarE, i % C::kStages));   // (nobody waits for the last ones, but for the steps behind them)
      }
      if (ok) tc_commit(bar(C::oBarDone, 0));
      if (kExtra && ok && (ok = wait(bar(C::oBarMap, 0), 0, 52, nk)) && extra.any()) ok = multiply_extra_wide<C>(sm, abort_flag, p.status, tmem, nk);
      if (!ok && tmem != kNoTmem) {   // gave up: what has been issued ends before tensor memory goes back
        tc_commit(bar(C::oBarLast, 0));
        ended_wait(bar(C::oBarLast, 0), 0);
      }
    }
  } else {
    // ---- x's scales: thread r has row r's four bytes of every step, two loads ahead
    const int groups = p.K / 32;
    const long long row = (long long)tile_m * 128 + tid;
    const bool have = row < p.xrows && (!kExtra || tid % C::kRows < rows);   // (what lies behind the last row was never written)
    const uint8_t* src = p.xs + row * groups;
    auto load = [&](int i) -> uint32_t {
      uint32_t w = 0x7f7f7f7fu;
      if (have && i < nk) {
        const int g = i * 4;
        if (p.words) return *reinterpret_cast<const uint32_t*>(src + g);
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (g + j < groups) w = (w & ~(0xffu << (8 * j))) | ((uint32_t)src[g + j] << (8 * j));
      }
      return w;
    };
    uint32_t w0 = load(0), w1 = load(1);
    Marks marks(extra, 0);
    int i = 0;
    auto free_stage = [&](int i) -> bool {
      return __all_sync(0xffffffffu, i < C::kStages || wait(bar(C::oBarE, i % C::kStages), ((i / C::kStages) & 1) ^ 1, 55, i));
    };
    for (; i < nk; i++) {
      const int s = i % C::kStages;
      if (!free_stage(i)) break;
      *reinterpret_cast<uint32_t*>(smem_lin + s * C::kStage + C::oSfx + lane * 16 + warp * 4) = w0;
      fence_async_smem();
      __syncwarp();
      if (lane == 0 && (i > 0 || !p.expire)) mbar_arrive(bar(C::oBarS, s));
      if (kExtra) marks.step(i, w0);
      w0 = w1;
      w1 = load(i + 2);
    }
    bool more = false;
    if (kExtra) {
      marks.flush();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(C::oBarMap, 0));
      rows_barrier();
      more = extra.any();
    }
    // ---- epilogue, first half: lane = row of the operand, column = channel (in the order of the tensor map)
    bool ok = __all_sync(0xffffffffu, wait(bar(C::oBarDone, 0), 0, 56, nk) && wait(bar(C::oBarTmem, 0), 0, 57, nk));
    if (more && ok) ok = bring_extra_wide<C>(p, map_w, sm, smem_lin, nk, pair, (int)m0, rows);
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem) + ((uint32_t)(warp * 32) << 16);
    if (ok) {
      tc_fence_after();
      float* part = reinterpret_cast<float*>(smem_lin + tid * C::kPRow);
#pragma unroll 2
      for (int c = 0; c < 256; c += 32) {
        uint32_t v[32];
        tmem_ld16(tmem + c, v);
        tmem_ld16(tmem + c + 16, v + 16);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; j++) part[c + j] = __uint_as_float(v[j]);
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (*abort_flag) {   // gave up (the copies in flight have been waited for): the failure shows in the output
    for (int i = tid; i < 128 * C::kPRow / 4; i += kThreads) reinterpret_cast<uint32_t*>(smem_lin)[i] = 0x7fc00000u;
    __syncthreads();
  }
  // ---- second half, a warp per row: the planes of a row of bf16 are added
  for (int t = warp; t < rows; t += kThreads / 32) {
    const float* at = reinterpret_cast<const float*>(smem_lin + t * C::kPRow) + lane;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = PLANES == 2 ? at[32 * j] + at[32 * j + C::kRows * C::kPRow / 4] : at[32 * j];
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const int n = (2 * pair + b) * 128 + 4 * lane;
      const size_t o = (size_t)(m0 + t) * p.N + n;
      if (p.out_dtype == 0) store4(static_cast<float*>(p.out) + o, v + 4 * b, n, p.N);
      else if (p.out_dtype == 1) store4(static_cast<__nv_bfloat16*>(p.out) + o, v + 4 * b, n, p.N);
      else store4(static_cast<__half*>(p.out) + o, v + 4 * b, n, p.N);
    }
  }
  if (warp == kWarpMma) {
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem_lin + C::oTmem);
    if (tmem != kNoTmem) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kCols) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------- host
// The weight's codes: 128 codes of a row, rows 4 l + j of a block as (l, j), blocks.
bool weight_map(CUtensorMap* map, const uint8_t* wc, long long blocks) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[4] = {128, 32, 4, (cuuint64_t)blocks};
  const cuuint64_t strides[3] = {256, 64, 8192};
  const cuuint32_t box[4] = {128, 32, 4, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 4, const_cast<uint8_t*>(wc), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// x's codes: K channels (zeros behind them), rows of which a box takes nb.
bool x_map(CUtensorMap* map, const uint8_t* x, long long rows, int K, int nb) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)K};
  const cuuint32_t box[2] = {128, (cuuint32_t)nb};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K>
cudaError_t linear_launch(K kern, int smem, std::atomic<bool>* ready, const LinearParams& p, const uint8_t* x, int nb, long long blocks, int split, cudaStream_t s) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {   // per device: the attribute belongs to the device's copy of the kernel
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) { cudaGetLastError(); return e; }
    ready[dev].store(true, std::memory_order_release);
  }
  CUtensorMap mw, mx;
  if (!weight_map(&mw, p.wc, (long long)p.tiles * p.ksteps)) return cudaErrorInvalidValue;
  if (!x) mx = mw;   // (not used)
  else if (!x_map(&mx, x, p.xrows, p.K, nb)) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)split);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = p.pdl;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = (unsigned)split;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, mw, mx);
  if (e != cudaSuccess) cudaGetLastError();
  return e;
}
template <int NB, int PLANES, bool kDirect = false>
cudaError_t narrow_launch(const LinearParams& p, const uint8_t* x, int split, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  return linear_launch(uq_fp4_linear_kernel<NB, PLANES, kDirect>, LinCfg<NB, PLANES>::kSmem, ready, p, x, NB, (long long)p.tiles * p.mtiles, split, s);
}
template <int PLANES>
cudaError_t wide_launch(const LinearParams& p, const uint8_t* x, cudaStream_t s) {
  static std::atomic<bool> ready[64];
  return linear_launch(uq_fp4_linear_wide_kernel<PLANES>, WideCfg<PLANES>::kSmem, ready, p, x, 128, (long long)(p.tiles + 1) / 2 * p.mtiles, 1, s);
}

}  // namespace tc

namespace {

bool aligned_to(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// rows of an instruction's operand that serve r rows of x
int operand_rows(long long r) { return r <= 16 ? 16 : (r <= 32 ? 32 : (r <= 64 ? 64 : 128)); }
// rows of both planes of M bf16 rows: tiles of 64, one smaller tile for fewer
int plane_tile(long long M) { return operand_rows(2 * std::min(M, 64ll)); }
long long plane_rows(long long M) { return (M + 63) / 64 * plane_tile(M); }

// CTAs along K (the cluster) for so many tiles of so many steps.  Calls follow one another on a stream, each kernel's CTAs set up while
// the one before still runs: with at most a CTA per SM that costs nothing, with more a CTA has to wait for an SM's half to fall
// free, about 1.4 us; a step less per CTA gains 0.14 to 0.25 us.  So: the most CTAs that leave the second halves free, or, where that
// saves a CTA more than ten steps, the most that fit both.  (Not quite all: clusters need their SMs in one part of the chip, and from 7/8
// on some CTAs wait; clusters of seven and eight from half on.)  us from a graph, tiles x steps, first / second choice:
//   32 x 32 (4096 x 4096) split 4 / 6  5.05 / 6.06     24 x 64 5 / 8  6.19 / 7.21     48 x 32 2 / 5  7.01 / 6.88
//   64 x 64 2 / 4  11.5 / 10.5     80 x 64 1 / 3  18.5 / 12.1     112 x 32 1 / 2  11.0 / 10.0     64 x 256 2 / 4  36.3 / 25.9
//   64 bf16 rows: 32 x 32 4 / 5  10.7 / 12.0     64 x 64 2 / 4  21.4 / 18.6
//   and past the limits: 48 x 32 6 9.0     40 x 40 3 / 7  6.46 / 9.06     16 x 16 6 / 8  3.14 / 4.51
int pick_split(long long tiles, int steps, int sms) {
  const int most = std::min(tc::kMaxSplit, steps);
  int one = 1, two = 1;
  for (int s = 2; s <= most; s++) {
    if (8 * tiles * s <= (s >= 7 ? 4 : 7) * sms) one = s;
    if (8 * tiles * s <= (s == 2 ? 16 : 14) * sms) two = s;
  }
  return two > one && (long long)steps * (two - one) > 10ll * one * two ? two : one;
}

}  // namespace

cudaError_t uq_split_dispatch(const void*, uint8_t*, uint8_t*, long long, int, int, cudaStream_t);

// Bytes of scratch for bf16 activations: both planes' codes, then their scales (none for rows that the CTAs split themselves).
size_t uq_fp4_linear_scratch(long long M, int K) { return M <= tc::kDirectRows || K < 32 || K % 32 ? 0 : (size_t)plane_rows(M) * ((size_t)K + K / 32); }

// xs null: x is bf16 [M, K], scratch holds uq_fp4_linear_scratch bytes; else x is e4m3 [M, K] with scale bytes xs [M, K / 32].
// launches: kernels enqueued.
cudaError_t uq_fp4_linear_dispatch(const void* x, const uint8_t* xs, const uint8_t* wc, const uint8_t* ws, void* out, void* scratch, long long M, int N, int K, int out_dtype,
                                   unsigned int* status, int sms, int expire, cudaStream_t s, int* launches) {
  *launches = 0;
  if (M < 0 || M > (1 << 24) || N < 1 || N > (1 << 24) || K < 32 || K > (1 << 24) || K % 32 || out_dtype < 0 || out_dtype > 2) return cudaErrorInvalidValue;
  if (M == 0) return cudaSuccess;
  const bool direct = !xs && M <= tc::kDirectRows;
  if (!x || !wc || !ws || !out || (!xs && !direct && !scratch)) return cudaErrorInvalidValue;
  if (!aligned_to(x, 16) || !aligned_to(wc, 32) || !aligned_to(ws, 16) || !aligned_to(out, (N % 4 == 0 ? 4 : 1) * (out_dtype == 0 ? 4 : 2)) || (xs ? !aligned_to(xs, 4) : !direct && !aligned_to(scratch, 16))) return cudaErrorInvalidValue;
  const long long tiles = (N + 127) / 128, ksteps = (K + 127) / 128;
  const int planes = xs ? 1 : 2;
  const int nb = planes == 2 ? plane_tile(M) : operand_rows(M);
  const long long mtiles = (M + nb / planes - 1) / (nb / planes);
  if (tiles * ksteps > INT_MAX || tiles * mtiles > INT_MAX) return cudaErrorInvalidValue;
  if (!status || !tc::encode_fn()) return cudaErrorInitializationError;
  tc::LinearParams p{};
  const uint8_t* codes = static_cast<const uint8_t*>(x);
  p.xs = xs;
  p.xrows = M;
  if (!xs) p.x16 = static_cast<const __nv_bfloat16*>(x);
  if (direct) {
    codes = nullptr;
  } else if (planes == 2) {
    p.xrows = plane_rows(M);
    uint8_t* c = static_cast<uint8_t*>(scratch);
    uint8_t* sc = c + (size_t)p.xrows * K;
    const cudaError_t e = uq_split_dispatch(x, c, sc, M, K, nb / 2, s);
    if (e != cudaSuccess) return e;
    *launches += 1;
    codes = c;
    p.xs = sc;
  }
  p.wc = wc;
  p.ws = ws;
  p.out = out;
  p.status = status;
  p.M = M;
  p.N = N;
  p.K = K;
  p.ksteps = (int)ksteps;
  p.mtiles = (int)mtiles;
  p.out_dtype = out_dtype;
  p.words = K % 128 == 0 && aligned_to(p.xs, 4);
  p.pdl = uq_pdl_on() ? 1 : 0;
  p.expire = expire;
  p.tiles = (int)tiles;
  // 128 operand rows: 256 channels a CTA where the tiles are more than the SMs (64 bf16 rows, us with 128 / 256 channels: 14336 x 4096
  // 16.5 / 18.2, 16384 x 8192 24.5 / 31.1, 20000 x 4096 22.9 / 18.6, 28672 x 8192 39.8 / 33.9, 65536 x 8192 83 / 72; 128 8-bit rows,
  // 65536 x 8192 88 / 71): the narrow kernel can then not split K, and with fewer the wide one leaves SMs without work.
  const bool wide = nb == 128 && tiles * mtiles > sms;
  const int split = pick_split(tiles * mtiles, (int)ksteps, sms);
  cudaError_t e;
  switch (nb * 2 + planes) {
    case 33: e = tc::narrow_launch<16, 1>(p, codes, split, s); break;
    case 34: e = direct ? tc::narrow_launch<16, 2, true>(p, codes, split, s) : tc::narrow_launch<16, 2>(p, codes, split, s); break;
    case 65: e = tc::narrow_launch<32, 1>(p, codes, split, s); break;
    case 66: e = tc::narrow_launch<32, 2>(p, codes, split, s); break;
    case 129: e = tc::narrow_launch<64, 1>(p, codes, split, s); break;
    case 130: e = tc::narrow_launch<64, 2>(p, codes, split, s); break;
    case 257: e = wide ? tc::wide_launch<1>(p, codes, s) : tc::narrow_launch<128, 1>(p, codes, split, s); break;
    default: e = wide ? tc::wide_launch<2>(p, codes, s) : tc::narrow_launch<128, 2>(p, codes, split, s); break;
  }
  if (e == cudaSuccess) *launches += 1;
  return e;
}
