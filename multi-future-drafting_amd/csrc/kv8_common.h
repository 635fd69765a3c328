// The 8-bit draft KV cache: e4m3 codes (OCP, 448 the largest) and a power-of-two float32 scale per page and KV head.
//
// A power-of-two scale costs nothing over a free one here: e4m3 has the same three mantissa bits in every binade, so a
// free scale only moves the largest value up to 448 from at worst 224.2, and in return decoding, encoding and a page's
// rescaling are exact shifts of the exponent (the conversions of gfx950 take such a scale along for free).
#pragma once
#include "mfd_common.h"

namespace kv8 {

constexpr int D = 128;        // head dim
constexpr int MIN_EXP = -40;  // scales lie in [2^-40, 2^40]: their quotients and products stay inside fp32
constexpr int MAX_EXP = 40;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Where the tokens of a batch's requests lie. Request b's token t: slot table[row][t / page] * page + t % page with
// row = req_idx ? req_idx[b] : b. Every id is checked against its bound before it is used.
struct Pages {
  const int32_t* table;
  int64_t table_stride;
  int table_rows, table_width;
  const int64_t* req_idx;
  int num_pages;
  int page_shift;  // log2(page size), 4 .. 8
};

// A request's table row, or NULL where its index lies outside the table.
__device__ __forceinline__ const int32_t* table_row(const Pages& p, int b) {
  const int64_t row = p.req_idx ? p.req_idx[b] : b;
  return row >= 0 && row < p.table_rows ? p.table + row * p.table_stride : nullptr;
}
// A request's length, as far as its table row reaches.
__device__ __forceinline__ int bounded_len(const Pages& p, int64_t len) {
  const int64_t cap = min((int64_t)p.table_width << p.page_shift, (int64_t)0x7fffff00);
  return (int)max((int64_t)0, min(len, cap));
}

__device__ __forceinline__ void raise(int32_t* err_flag, int bit) {
  if (err_flag) atomicOr(err_flag, bit);
}

// Inclusive prefix sum over a wave's lanes, by DPP: within rows of 16, then a row's last lane to the rows behind it
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast 15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast 31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int wave_sum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }

// Smallest 2^e with amax / 2^e <= 448 = 0.875 * 2^9, e within the range (amax finite, not negative).
__device__ __forceinline__ float page_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  int e = (int)(bits >> 23) - 126 - 9 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);  // amax = m 2^(exp - 126), m in [0.5, 1)
  e = max(MIN_EXP, min(MAX_EXP, e));
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// 1 / s of a power of two within the range
__device__ __forceinline__ float inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// |x|, with infinities and NaN as 0: they set neither a page's scale nor a partial row's
__device__ __forceinline__ float finite_abs(float x) {
  const float v = fabsf(x);
  return v < INFINITY ? v : 0.f;
}
// x clamped to the type's range; NaN stays NaN (both comparisons fail)
__device__ __forceinline__ float clamp448(float x) { return x > 448.f ? 448.f : (x < -448.f ? -448.f : x); }

// Four scaled values -> four codes (round to nearest even; x already divided by the scale, which is exact)
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(x0), clamp448(x1), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamp448(x2), clamp448(x3), w, true);
}
// Four codes -> four values times s
__device__ __forceinline__ void decode4(uint32_t c, float s, float (&x)[4]) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  x[0] = lo[0] * s;
  x[1] = lo[1] * s;
  x[2] = hi[0] * s;
  x[3] = hi[1] * s;
}

// Host-side checks that every entry point of the cache makes; 0 or an error code with its message.
inline int check_cache(const char* who, const void* k_cache, const void* v_cache, int64_t kc_ss, int64_t kc_sh,
                       int64_t vc_ss, int64_t vc_sh, int page_size, int Hkv, int D_, const void* table, int table_rows,
                       int table_width, int num_pages) {
  if (D_ != D) return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: head dim %d (only %d)", who, D_, D);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64, 128 or 256)", who, page_size);
  if (Hkv < 1 || Hkv > 1024 || table_rows < 0 || table_width < 0 || num_pages < 0)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad sizes Hkv=%d table %d x %d pages=%d", who, Hkv, table_rows,
                         table_width, num_pages);
  if (!table && table_rows > 0 && table_width > 0)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null page table", who);
  if (((reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache)) & 15) ||
      ((kc_ss | kc_sh | vc_ss | vc_sh) & 15))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: cache rows need 16-byte alignment (bases and strides)", who);
  // slot ids and strides are 32-bit in the kernels, and so is a tile's row offset: 63 strides
  if ((int64_t)num_pages * page_size > 0x7fffffff || (int64_t)num_pages * Hkv > 0x7fffffff || kc_ss < 0 || vc_ss < 0 ||
      kc_ss > (1 << 25) || vc_ss > (1 << 25))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: needs fewer than 2^31 slots and scales, and slot strides in [0, 2^25]", who);
  return MFD_OK;
}

}  // namespace kv8
