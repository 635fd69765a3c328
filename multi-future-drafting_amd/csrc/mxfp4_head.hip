// Draft LM head with a 4-bit weight for gfx950: logits = bf16(x W^T) over the drafted rows,
//   W[n][k] = e2m1(codes[n][k / 2], half k % 2) * 2^(exps[n][k / 32] - 127),
// the weight as in the OCP microscaling format MXFP4 (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives; an e8m0 scale for 32
// weights), row-major, low half of a byte first. An e2m1 value has two significant bits and the scale is a power of two, so
// W is exact in bf16 and gfx950 makes it there in one instruction for two weights, scale included: products are exact in
// fp32, sums are fp32 (v_mfma_f32_16x16x32_bf16), and the only rounding is the logit's own.
//
// The weight (4.25 bits each: 207 MB at 151936 x 2560) streams once per 128 drafted rows, straight to registers: a lane takes
// 16 bytes, 32 weights of one row under one scale, and the four lane groups of a 16-row tile take 128 k together. Which k a
// lane holds is free as long as both operands agree, so the four MFMAs of such a step use k = 32 (lane / 16) + 8 j + 0 .. 7.
//  * Wide form: a workgroup of eight waves takes a share of the vocabulary, a wave up to VT 16-row tiles of it against all
//    of the launch's drafted rows (MTL 16-row tiles), which come through LDS in blocks of 32 to 64 KB by direct loads, double
//    buffered, one barrier per block. Bound by the weight's way from memory with few drafted rows (151936 x 2560, 15 rows: 47
//    us, 4.5 TB/s; a plain read of the weight alone 32), by the matrix pipes with 128 (98304 x 2560, 120 rows: 61 us, 1.06
//    PFLOP/s with the padding to 128; a large library product reaches 1.24).
//  * K-split form, for vocabularies that leave a wave of the wide form without a tile: a workgroup takes one tile, each of its
//    four waves every fourth step of k; the drafted rows come from L2 straight to registers, the partial sums meet in LDS
//    and are added in wave order. Bound by latency.
#include <algorithm>
#include <type_traits>

#include "mfd_common.h"

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int MT = 128;   // drafted rows of one launch
constexpr int KS = 128;   // k per step
constexpr int NW = 8;     // waves of the wide form
constexpr int KNW = 4;    // waves of the k-split form

struct HeadArgs {
  const uint16_t* x;  // drafted row m at x + (m / rpg) * group_stride + (m % rpg) * row_stride
  int64_t row_stride, group_stride;
  int rpg, row0;      // the launch's drafted rows are row0 .. row0 + M - 1
  const uint8_t* codes;  // [N][K / 2]
  const uint8_t* exps;   // [N][K / 32]
  uint16_t* out;      // [M][out_stride], row 0 = drafted row row0
  int64_t out_stride;
  int M, N, K;
  // wide form: workgroups; of more than one round also those of the whole ones and their vocabulary rows, and the others' rows
  int nwg, full_wgs, full_rows, last_rows;
};

// One direct-to-LDS load: lane l's 16 bytes at g land at LDS byte address lds_byte + 16 l (lds_byte wave-uniform). Inline asm:
// the compiler does not count it among its own loads; the kernel waits for it explicitly.
__device__ __forceinline__ void dma16(const void* g, uint32_t lds_byte) {
  const uint32_t l = __builtin_amdgcn_readfirstlane(lds_byte);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Workgroup barrier that is also a compiler memory barrier, with this wave's LDS operations done; loads in flight go on
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const uint8_t* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), (short)0, (int)bytes, 0x00020000);
}

__device__ __forceinline__ const uint16_t* drafted_row(const HeadArgs& a, int r) {
  const int m = a.row0 + min(r, a.M - 1);  // rows past the last repeat it and are not stored
  return a.x + (int64_t)(m / a.rpg) * a.group_stride + (int64_t)(m % a.rpg) * a.row_stride;
}
// An operand read takes chunk 4 g4 + j of 16 rows: four rows apart the low bits differ, within four the high ones
__device__ __forceinline__ int swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
// First vocabulary row of workgroup g. One round: an even split in multiples of 8 rows. More: full ranges for the whole rounds,
// equal ones that are no larger for the last.
template <bool ROUNDS>
__host__ __device__ __forceinline__ int wg_row0(const HeadArgs& a, int g) {
  if (!ROUNDS) return g >= a.nwg ? a.N : (int)(((int64_t)g * a.N / a.nwg) & ~(int64_t)7);
  const int64_t row = (int64_t)(g < a.full_wgs ? g : a.full_wgs) * a.full_rows +
                      (int64_t)(g < a.full_wgs ? 0 : g - a.full_wgs) * a.last_rows;
  return (int)(row < a.N ? row : a.N);
}

// Eight codes times the scale as bf16: exact
__device__ __forceinline__ bf16x8 widen(uint32_t c, float s) {
  const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3)};
  return __builtin_bit_cast(bf16x8, v);
}
// The scale of lane group g4 among a step's four (the conversion reads the float's exponent alone: 0 is 2^-127, as in the format)
__device__ __forceinline__ float scale_of(uint32_t e4, int g4) { return __uint_as_float(((e4 >> (8 * g4)) & 0xffu) << 23); }

// C registers of a tile pair to bf16 and out: weight rows n .. n + 3 of the range, the drafted row's output at orow
__device__ __forceinline__ void store4(uint16_t* orow, int n, int rows, const f32x4& c) {
  const u32x2 pk = {__builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){c[0], c[1]}, bf16x2)),
                    __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){c[2], c[3]}, bf16x2))};
  if (n + 4 <= rows) {
    *reinterpret_cast<u32x2*>(orow + n) = pk;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < rows) orow[n + e] = (uint16_t)(pk[e >> 1] >> (16 * (e & 1)));
  }
}

// Sizes of the wide form by MTL (3 and 6 beside the powers of two: 40 drafted rows 55 us against 62 with 64, 90 rows 87 against
// 97 with 128, both 151936 x 2560). VT_MAX: as many as the accumulators and two steps' weights leave registers for.
template <int MTL>
struct Wide {
  static constexpr int BLOCK = (MTL <= 2 ? 32 : MTL % 3 == 0 ? 48 : 64) * 1024;  // bytes of a drafted-row block
  static constexpr int WPC = MTL <= 2 ? 2 : 1;   // workgroups per CU
  static constexpr int VT_MAX = MTL == 3 || MTL == 4 ? 5 : MTL == 6 ? 4 : 3;
};

// ROUNDS: more than one round of workgroups; those of the last one have any number of tiles up to VT, else it is VT or VT - 1
template <int VT, int MTL, bool ROUNDS>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2 * Wide<MTL>::WPC, 2 * Wide<MTL>::WPC)))
void mxfp4_wide_kernel(HeadArgs a) {
  constexpr int FEWEST = ROUNDS ? 0 : VT - 1;
  constexpr int BLOCK = Wide<MTL>::BLOCK, HPS = 2;  // 128-k halves per step
  constexpr int HB = BLOCK / (32 * MTL);  // k per drafted block
  constexpr int CPR = HB / 8;             // 16-byte chunks of a row's block
  constexpr int SPB = HB / (KS * HPS);    // steps per block
  constexpr int LPW = BLOCK / 1024 / NW;  // direct loads of a wave per block
  static_assert(SPB == 1 || SPB % 2 == 0, "steps go in pairs");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R0 = wg_row0<ROUNDS>(a, blockIdx.x);
  const int rows = wg_row0<ROUNDS>(a, blockIdx.x + 1) - R0;
  if (rows <= 0) return;
  const int K = a.K, S = (K + KS * HPS - 1) / (KS * HPS);
  const int l16 = lane & 15, g4 = lane >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;

  // direct loads of drafted block b: chunk c of row r goes to c ^ swz(r) of the row's block, so that the lanes of an operand
  // read hit all banks; chunks past the last k repeat the last one and are never read
  auto issue_x = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int at = (i * NW + w) * 64 + lane;
      const int r = at / CPR, c = (at % CPR) ^ swz(r);
      dma16(drafted_row(a, r) + min(b * HB + 8 * c, K - 8), lds0 + (uint32_t)(b & 1) * BLOCK + (uint32_t)(i * NW + w) * 1024u);
    }
  };
  // this wave's tiles: t0 .. t0 + vtv - 1 (an even split of at most 8 VT tiles), the loop compiled for each number of them: a
  // test per product would cost more than the product. Rows past the range read as zero by the buffers' bounds.
  const int T = (rows + 15) / 16;
  const int t0 = __builtin_amdgcn_readfirstlane(w * T / NW);
  const int vtv = __builtin_amdgcn_readfirstlane((w + 1) * T / NW) - t0;
  const __amdgpu_buffer_rsrc_t rc = buffer_of(a.codes + (int64_t)R0 * (K / 2), (uint32_t)rows * (uint32_t)(K / 2));
  const __amdgpu_buffer_rsrc_t re = buffer_of(a.exps + (int64_t)R0 * (K / 32), (uint32_t)rows * (uint32_t)(K / 32));
  const uint32_t coff = (uint32_t)(16 * t0 + l16) * (uint32_t)(K / 2) + 16u * g4;
  const uint32_t eoff = (uint32_t)(16 * t0 + l16) * (uint32_t)(K / 32);
  auto walk = [&](auto tiles) __attribute__((always_inline)) {
    constexpr int V = decltype(tiles)::value;
    f32x4 acc[V + 1][MTL];
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < MTL; ++j) acc[i][j] = (f32x4){};
    u32x4 wf[2][V + 1][HPS];
    u32x2 ef[2][V + 1];
    // (past the last step: the last one, not used. The scheduler leaves a step's loads where they are: sunk to the next
    // step's, they would be waited for together.)
    auto load_w = [&](int p, int v) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t u = (uint32_t)min(v, S - 1);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ef[p][i] = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_raw_buffer_load_b64(re, eoff, (uint32_t)i * (uint32_t)(K / 2) + u * (4u * HPS), 0));
#pragma unroll
        for (int h = 0; h < HPS; ++h)
          wf[p][i][h] = __builtin_bit_cast(
              u32x4,
              __builtin_amdgcn_raw_buffer_load_b128(rc, coff, (uint32_t)i * (uint32_t)(8 * K) + u * (64u * HPS) + 64u * h, 0));
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    // A step's products in slots of V MFMAs: slot q is drafted tile q % MTL of the half's k chunk q / MTL. The drafted
    // operand is read FD slots ahead (left alone, the compiler reads it just before its products), and a chunk's weights
    // are widened in the slot before its first. A scheduling barrier closes each slot.
    constexpr int FD = MTL <= 2 ? 2 : 4;
    auto step = [&](int p, int v) __attribute__((always_inline)) {
      const uint8_t* base = smem + ((v / SPB) & 1) * BLOCK + l16 * (HB * 2);
#pragma unroll
      for (int h = 0; h < HPS; ++h) {
        if (h > 0 && (v * HPS + h) * KS >= K) break;  // K is an odd number of halves
        const int c0 = ((v % SPB) * HPS + h) * (KS / 8) + 4 * g4;
        auto fetch = [&](int q) __attribute__((always_inline)) {
          return *reinterpret_cast<const bf16x8*>(base + 16 * (q % MTL) * (HB * 2) + (((c0 + q / MTL) ^ swz(l16)) << 4));
        };
        float sc[V + 1];
        bf16x8 f[2][V + 1], xf[4 * MTL];
#pragma unroll
        for (int i = 0; i < V; ++i) sc[i] = scale_of(ef[p][i][h], g4);
#pragma unroll
        for (int q = 0; q < FD; ++q) xf[q] = fetch(q);
#pragma unroll
        for (int i = 0; i < V; ++i) f[0][i] = widen(wf[p][i][h][0], sc[i]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < 4 * MTL; ++q) {
          const int j = q / MTL, m = q % MTL;
          if (q + FD < 4 * MTL) xf[q + FD] = fetch(q + FD);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[i][m] = mfma16(f[j & 1][i], xf[q], acc[i][m]);
          if (m == MTL - 1 && j < 3) {
#pragma unroll
            for (int i = 0; i < V; ++i) f[(j + 1) & 1][i] = widen(wf[p][i][h][j + 1], sc[i]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    // Block b's direct loads have landed in every wave (the weight loads of one or two steps, V (HPS + 1) each, are
    // younger), block b - 1 is read, and its half takes block b + 1.
    auto next_block = [&](int b) __attribute__((always_inline)) {
      wait_vmcnt<(SPB == 1 ? 1 : 2) * V * (HPS + 1)>();
      lds_barrier();
      if ((b + 1) * SPB < S) issue_x(b + 1);
    };
    issue_x(0);
    load_w(0, 0);
    load_w(1, 1);
#pragma unroll 1
    for (int v = 0; v < S; v += 2) {
      if (SPB <= 2 || v % SPB == 0) next_block(v / SPB);
      step(0, v);
      load_w(0, v + 2);
      if (v + 1 < S) {
        if (SPB == 1) next_block(v + 1);
        step(1, v + 1);
      }
      load_w(1, v + 3);
    }
    wait_vmcnt<0>();
    // C register r of accumulator (i, m): weight row 16 (t0 + i) + 4 g4 + r of the range, drafted row 16 m + l16
#pragma unroll
    for (int m = 0; m < MTL; ++m) {
      const int mm = 16 * m + l16;
      if (mm >= a.M) continue;
      uint16_t* orow = a.out + (int64_t)mm * a.out_stride + R0;
#pragma unroll
      for (int i = 0; i < V; ++i) store4(orow, 16 * (t0 + i) + 4 * g4, rows, acc[i][m]);
    }
  };
  auto pick = [&](auto self, auto tiles) __attribute__((always_inline)) {
    constexpr int V = decltype(tiles)::value;
    if (V == FEWEST || vtv == V) walk(tiles);
    else if constexpr (V > FEWEST) self(self, std::integral_constant<int, V - 1>{});
  };
  pick(pick, std::integral_constant<int, VT>{});
}

template <int MTL>
__global__ __launch_bounds__(KNW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void mxfp4_ksplit_kernel(HeadArgs a) {
  static_assert(MTL <= 2, "two steps' operands in registers");
  __shared__ f32x4 part[KNW * MTL * 64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R0 = blockIdx.x * 16;
  const int rows = min(16, a.N - R0);
  const int K = a.K, S = K / KS;
  const int l16 = lane & 15, g4 = lane >> 4;
  const int64_t row = R0 + min(l16, rows - 1);
  const uint8_t* cp = a.codes + row * (K / 2) + 16 * g4;
  const uint8_t* ep = a.exps + row * (K / 32);
  const uint16_t* xp[MTL];
#pragma unroll
  for (int m = 0; m < MTL; ++m) xp[m] = drafted_row(a, 16 * m + l16) + 32 * g4;
  f32x4 acc[MTL];
#pragma unroll
  for (int m = 0; m < MTL; ++m) acc[m] = (f32x4){};
  u32x4 wf[2];
  uint32_t ef[2];
  bf16x8 xf[2][MTL][4];
  auto load = [&](int s, int v) __attribute__((always_inline)) {
    wf[s] = *reinterpret_cast<const u32x4*>(cp + 64 * v);
    ef[s] = *reinterpret_cast<const uint32_t*>(ep + 4 * v);
#pragma unroll
    for (int m = 0; m < MTL; ++m)
#pragma unroll
      for (int j = 0; j < 4; ++j) xf[s][m][j] = *reinterpret_cast<const bf16x8*>(xp[m] + KS * v + 8 * j);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto products = [&](int s) __attribute__((always_inline)) {
    const float sc = scale_of(ef[s], g4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bf16x8 f = widen(wf[s][j], sc);
#pragma unroll
      for (int m = 0; m < MTL; ++m) acc[m] = mfma16(f, xf[s][m][j], acc[m]);
    }
  };
  if (w < S) load(0, w);
  for (int v = w; v < S; v += 2 * KNW) {
    if (v + KNW < S) load(1, v + KNW);
    products(0);
    if (v + KNW < S) {
      if (v + 2 * KNW < S) load(0, v + 2 * KNW);
      products(1);
    }
  }
#pragma unroll
  for (int m = 0; m < MTL; ++m) part[(w * MTL + m) * 64 + lane] = acc[m];
  __syncthreads();
  if (w < MTL) {
    f32x4 c = part[w * 64 + lane];
#pragma unroll
    for (int x = 1; x < KNW; ++x) {
      const f32x4 d = part[(x * MTL + w) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] += d[e];
    }
    const int mm = 16 * w + l16;
    if (mm < a.M) store4(a.out + (int64_t)mm * a.out_stride + R0, 4 * g4, rows, c);
  }
}

template <int VT, int MTL, bool ROUNDS = false>
int launch_wide(const HeadArgs& a, hipStream_t st) {
  if constexpr (VT <= Wide<MTL>::VT_MAX) {
    constexpr int lds = 2 * Wide<MTL>::BLOCK;
    const int rc = mfd_set_max_lds(reinterpret_cast<const void*>(&mxfp4_wide_kernel<VT, MTL, ROUNDS>), lds);
    if (rc != MFD_OK) return rc;
    hipLaunchKernelGGL((mxfp4_wide_kernel<VT, MTL, ROUNDS>), dim3((unsigned)a.nwg), dim3(NW * 64), lds, st, a);
  }
  return MFD_OK;
}
template <int MTL>
int launch_rows(HeadArgs a, int cus, hipStream_t st) {
  // k-split: up to a tile per CU and 32 drafted rows (hidden 2560: 4000 x 32 rows 9.1 us against the wide form's 10.9, 4000 x 4
  // 5.8 against 8.9; beyond either, 8000 x 16 rows 10.3 against 9.5, 4000 x 96 19.0 against 17.2, 16000 x 96 60.6 against 20.8)
  if constexpr (MTL <= 2)
    if (a.N <= 16 * cus) {
      hipLaunchKernelGGL(mxfp4_ksplit_kernel<MTL>, dim3((unsigned)((a.N + 15) / 16)), dim3(KNW * 64), 0, st, a);
      return MFD_OK;
    }
  const int slots = Wide<MTL>::WPC * cus;  // workgroups that run together
  a.full_rows = NW * Wide<MTL>::VT_MAX * 16;
  a.nwg = slots;
  if (a.N / slots + 8 > a.full_rows) {
    // whole rounds of full workgroups, then one that shares the rest: a wave's tiles come whole, and an even split over the
    // rounds leaves more waves with a part of one (98304 rows, 120 drafted ones: 61 us in one round, 73 in two even ones)
    a.full_wgs = (int)(a.N / ((int64_t)slots * a.full_rows)) * slots;
    const int64_t rest = a.N - (int64_t)a.full_wgs * a.full_rows;
    a.last_rows = (int)((rest + 8 * slots - 1) / (8 * slots)) * 8;
    a.nwg += a.full_wgs;
    return launch_wide<Wide<MTL>::VT_MAX, MTL, true>(a, st);
  }
  const int vt = (a.N / a.nwg + 8 + 16 * NW - 1) / (16 * NW);  // tiles of a wave
  switch (vt) {
    case 1: return launch_wide<1, MTL>(a, st);
    case 2: return launch_wide<2, MTL>(a, st);
    case 3: return launch_wide<3, MTL>(a, st);
    case 4: return launch_wide<4, MTL>(a, st);
    default: return launch_wide<5, MTL>(a, st);
  }
}

int head_gemm(const uint16_t* x, int64_t row_stride, int rows_per_group, int64_t group_stride, const uint8_t* codes,
              const uint8_t* exps, int M, int N, int K, uint16_t* out, int64_t out_stride, void* stream, const char* who) {
  if (M < 0 || N < 1 || K < 1 || rows_per_group < 1 || row_stride < 0 || group_stride < 0)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad sizes M=%d N=%d K=%d rows_per_group=%d", who, M, N, K, rows_per_group);
  if (K % KS != 0) return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: needs K %% %d == 0 (K=%d)", who, KS, K);
  // a workgroup's share of the weight, up to 672 rows of K / 2 bytes with its last tile's padding, has 32-bit offsets
  if (K > (1 << 23)) return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: hidden size %d above 2^23", who, K);
  if (M == 0) return MFD_OK;
  if (!x || !codes || !exps || !out) return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null pointer", who);
  if (row_stride % 8 != 0 || group_stride % 8 != 0 || out_stride < N || out_stride % 4 != 0 ||
      (reinterpret_cast<uintptr_t>(x) & 15) || (reinterpret_cast<uintptr_t>(codes) & 15) ||
      (reinterpret_cast<uintptr_t>(exps) & 3) || (reinterpret_cast<uintptr_t>(out) & 7))
    return mfd_set_error(MFD_ERR_UNSUPPORTED,
                         "%s: x and codes need 16-byte alignment, exps 4, output rows 8 (row_stride=%lld group_stride=%lld "
                         "out_stride=%lld)",
                         who, (long long)row_stride, (long long)group_stride, (long long)out_stride);
  const int cus = mfd_num_cus();
  const hipStream_t st = static_cast<hipStream_t>(stream);
  for (int m0 = 0; m0 < M; m0 += MT) {
    const HeadArgs a{x, row_stride, group_stride, rows_per_group, m0, codes, exps, out + (int64_t)m0 * out_stride, out_stride,
                     std::min(MT, M - m0), N, K, 0, 0, 0, 0};
    const int rc = a.M <= 16   ? launch_rows<1>(a, cus, st)
                   : a.M <= 32 ? launch_rows<2>(a, cus, st)
                   : a.M <= 48 ? launch_rows<3>(a, cus, st)
                   : a.M <= 64 ? launch_rows<4>(a, cus, st)
                   : a.M <= 96 ? launch_rows<6>(a, cus, st)
                               : launch_rows<8>(a, cus, st);
    if (rc != MFD_OK) return rc;
    MFD_CHECK_LAUNCH();
  }
  return MFD_OK;
}

}  // namespace

extern "C" int mfd_draft_head_mxfp4(const uint16_t* x, int64_t row_stride, int rows_per_group, int64_t group_stride,
                                    const uint8_t* codes, const uint8_t* exps, int M, int N, int K, uint16_t* out,
                                    int64_t out_stride, void* stream) {
  return head_gemm(x, row_stride, rows_per_group, group_stride, codes, exps, M, N, K, out, out_stride, stream,
                   "mfd_draft_head_mxfp4");
}

extern "C" int mfd_draft_topk_head_mxfp4(const uint16_t* x, int64_t row_stride, int rows_per_group, int64_t group_stride,
                                         const uint8_t* codes, const uint8_t* exps, int M, int N, int K, uint16_t* logits,
                                         int64_t logits_stride, int k, float* out_logp, void* out_ids, int ids_int64,
                                         float* out_logz, const int32_t* vocab_ids, void* workspace, int64_t workspace_bytes,
                                         void* stream) {
  const int rc = head_gemm(x, row_stride, rows_per_group, group_stride, codes, exps, M, N, K, logits, logits_stride, stream,
                           "mfd_draft_topk_head_mxfp4");
  if (rc != MFD_OK || M == 0) return rc;
  return vocab_ids ? mfd_topk_logz_vocab(logits, M, N, logits_stride, k, out_logp, out_ids, ids_int64, out_logz, vocab_ids,
                                         workspace, workspace_bytes, stream)
                   : mfd_topk_logz(logits, M, N, logits_stride, k, out_logp, out_ids, ids_int64, out_logz, workspace,
                                   workspace_bytes, stream);
}
