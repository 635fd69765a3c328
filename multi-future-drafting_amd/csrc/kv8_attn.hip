// Mode attention over the 8-bit draft KV cache (kv8_common.h) for gfx950, and the attention weight that each cached
// token received.
//
//   o[row] = sum_t p[row, t] v_t,  p = softmax(scale q k_t)  over the request's cached tokens (k_t = code * k_scale,
//   v_t = code * v_scale of the token's page) and, where they are given, the bf16 keys of the row's own mode block;
//   lse[row] = log sum exp, natural;   w[h][t] = decay w[h][t] + sum over KV head h's query rows of
//   exp(scale q k_t - lse[row]).
//
// A KV head's query rows (G query heads x K L queries, head-major) are packed into units of 32, the column count of
// v_mfma_f32_32x32x16: only the last unit of a KV head is padded, whatever K L is. Scores are S^T = K Q^T in bf16 (a code
// has four significant bits and the scale is a power of two, so k is exact in bf16 and every product in fp32) and
// O^T += V^T P^T in fp16: V as bare codes (exact), P rounded to fp16 (2^-11 at most, an eighth of the bf16 output's own
// rounding), times the quotient of the page's v_scale and the accumulators' unit: a power of two, which the exponential
// takes along in its argument and the row sum leaves out again, both exactly. The accumulators are brought to another unit
// only where that quotient leaves [2^-2, 2^6] (P stays below 2^14 and mostly above fp16's subnormals; a probability among
// them is off by 2^-23 of the row's sum at most). Statistics are fp32.
//
// Two kernels, by the units of a KV head:
//  * tile kernel: the waves of a workgroup (a unit each) share 64-key tiles. The codes come from memory to registers, two
//    tiles ahead, and are widened on their way into LDS (K to bf16 with its scale folded in by the conversion, V to
//    fp16), so that each code is widened once per workgroup and the products find plain MFMA operands: two buffers each
//    of K and V, one barrier per tile. Scores of tile t + 1 and the products of tile t run interleaved in 32 slots.
//    Bound by the issue of matrix and vector instructions (32 % and 37 % of the cycles) and by how the grid fills (1.5 waves
//    per SIMD on average of the two that fit: 384 workgroups on 256 places, waves without rows, the longest request's outlast
//    the others): 16 requests of 1187 .. 8033 tokens, 40 heads, 8 x 16 queries: 236 us, 0.80 PFLOP/s; over pages of 16 or 32
//    tokens, with a look-up per thread, 246. One request of 4096 tokens, 32 heads: 22 us and 5.3 of merge; a workgroup's 5 tiles
//    take 11 of them, the look-ups and first loads in front 3.4.
//  * stream kernel, for one unit per KV head (plain decoding): nothing is shared, so each wave walks 32-key tiles of its
//    own through its own LDS, without barriers, and the waves' results meet at the end. Bound by the cache's way from
//    memory: 16 requests of 4748 .. 32132 tokens 137 us with the merge, 4.3 TB/s (a plain read of as much 6.7, a copy 4.9). One
//    request of 1187 tokens: 8.7 us and 4.0 of merge, latency.
// Both split a context over workgroups (a fixed number of keys each, so that a batch's long contexts become more
// workgroups, not longer ones) and merge by log-sum-exp.
#include <algorithm>
#include <type_traits>

#include "kv8_common.h"

namespace {

using kv8::D;
using kv8::Pages;
using kv8::u32x4;

constexpr int TK = 64;         // keys per tile of the tile kernel
constexpr int UROWS = 32;      // query rows per unit
constexpr int SK = 32;         // keys per tile of the stream kernel
constexpr float LN2 = 0.6931471805599453f;

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct Args {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* kn;  // NULL: no block keys
  const uint16_t* vn;
  int64_t kn_st, kn_sh, vn_st, vn_sh;
  const uint8_t* kc;
  const uint8_t* vc;
  int64_t kc_ss, kc_sh, vc_ss, vc_sh;
  const float* ks;  // [pages][Hkv]
  const float* vs;
  Pages pages;
  const int64_t* ctx_lens;
  uint16_t* out;
  int64_t o_st, o_sh;
  float* lse;      // [bs K L][H] or NULL
  uint16_t* ws_o;  // [S][bs][Hkv][rows][D] fp16: the partial output row divided by 2^ws_exp
  float* ws_lse;   // [S][bs][Hkv][rows], base 2
  float* ws_exp;   // [S][bs][Hkv][rows] the row's power-of-two scale exponent
  int bs, K, L, H, Hkv, G, KL, rows;  // rows = G K L: query rows of a KV head
  int SC, S, split_keys;              // context splits; partials (tile kernel: one more for the block keys)
  int pairs, min_tiles;               // split_keys 0: (request, partial) pairs of the grid, and a split's fewest 64-key tiles
  int32_t* ws_n;                      // [bs] a request's context splits
  int causal, ngroups;
  float scale_log2;
  int32_t* err_flag;
};

__device__ __forceinline__ void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(0xC07F); }
__device__ __forceinline__ void wait_vmcnt0() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// One direct-to-LDS load: lane l's 16 bytes at g land at LDS byte address lds_byte + 16 l (lds_byte wave-uniform)
__device__ __forceinline__ void dma16(const uint16_t* g, uint32_t lds_byte) {
  const uint32_t l = __builtin_amdgcn_readfirstlane(lds_byte);
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(l), "v"(g) : "memory", "m0");
}
// Workgroup barrier that is also a compiler memory barrier, with this wave's LDS operations done. Global loads in
// flight are not waited for: the next tiles' codes stay on their way across it.
__device__ __forceinline__ void lds_barrier() {
  wait_lgkmcnt0();
  asm volatile("s_barrier" ::: "memory");
}

// The value of the other 32-lane half beside the own (see v_permlane32_swap; the copy is opaque, or the compiler would
// take the two results for equal).
__device__ __forceinline__ int2 both_halves(float x) {
  int y;
  asm volatile("v_mov_b32 %0, %1" : "=v"(y) : "v"(__builtin_bit_cast(int, x)));
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, x), y, false, false);
  return make_int2(r[0], r[1]);
}
__device__ __forceinline__ float half_max(float x) {
  const int2 r = both_halves(x);
  return fmaxf(__builtin_bit_cast(float, r.x), __builtin_bit_cast(float, r.y));
}
__device__ __forceinline__ float half_sum(float x) {
  const int2 r = both_halves(x);
  return __builtin_bit_cast(float, r.x) + __builtin_bit_cast(float, r.y);
}
__device__ __forceinline__ uint32_t f2h2_bits(float x0, float x1) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x0, x1}, f16x2));
}
__device__ __forceinline__ uint32_t f2bf2_bits(float x0, float x1) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){x0, x1}, bf16x2));
}
__device__ __forceinline__ f32x2 h2_to_f2(uint32_t h) {
  return __builtin_convertvector(__builtin_bit_cast(f16x2, h), f32x2);
}
__device__ __forceinline__ f32x16 mfma32_f16(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Eight codes -> eight bf16 values times s (exact); eight codes -> eight fp16 values (exact)
__device__ __forceinline__ u32x4 widen_k(uint32_t c0, uint32_t c1, float s) {
  return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, s, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, s, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, s, true))};
}
__device__ __forceinline__ u32x4 widen_v(uint32_t c0, uint32_t c1) {
  return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c0, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c0, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c1, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c1, 1.f, true))};
}
// A widened tile in LDS is [key][d] with padded rows, so that every operand read is a lane's base plus a constant: K rows of
// 272 bytes (16 lanes read 16 bytes of 16 rows: 16 bytes apart modulo 256, all banks once), V rows of 288 (the transpose
// read takes 32 bytes of each of four rows: 32 bytes apart).
constexpr int KROW = 272, VROW = 288;
// 16-byte chunks 2 part and 2 part + 1 of a row. Parts 4 .. 7 write the upper one first: the eight lanes of a row then hit
// all banks at once.
__device__ __forceinline__ void put_chunks(uint8_t* row, int part, const u32x4& first, const u32x4& second) {
  const int c0 = 2 * part + (part >> 2);
  *reinterpret_cast<u32x4*>(row + 16 * c0) = first;
  *reinterpret_cast<u32x4*>(row + 16 * (c0 ^ 1)) = second;
}
__device__ __forceinline__ void put_row(uint8_t* row, int part, const u32x4& lo, const u32x4& hi) {
  const bool up = part >= 4;
  put_chunks(row, part, up ? hi : lo, up ? lo : hi);
}
__device__ __forceinline__ void put_k_codes(uint8_t* row, int part, const u32x4& c, float s) {
  const bool up = part >= 4;
  put_chunks(row, part, widen_k(up ? c[2] : c[0], up ? c[3] : c[1], s), widen_k(up ? c[0] : c[2], up ? c[1] : c[3], s));
}
__device__ __forceinline__ void put_v_codes(uint8_t* row, int part, const u32x4& c) {
  const bool up = part >= 4;
  put_chunks(row, part, widen_v(up ? c[2] : c[0], up ? c[3] : c[1]), widen_v(up ? c[0] : c[2], up ? c[1] : c[3]));
}
// Byte offsets of a lane's operands within a tile. K: row l32 (+ 32 rows for the second subtile), d chunk 2 c + half: + 32 c.
// V^T fragment of d block db and 16-key chunk c (ds_read_b64_tr_b16): + 64 db + 16 c rows, and eight rows further the chunk's
// second 4-key group. The k order within a chunk is the row order of S^T's accumulators, so P needs no move.
__device__ __forceinline__ int k_operand(int lane) { return (lane & 31) * KROW + (lane >> 5) * 16; }
__device__ __forceinline__ int v_operand(int lane) {
  const int sl = lane & 15;
  return (4 * (lane >> 5) + (sl >> 2)) * VROW + ((lane >> 4) & 1) * 32 + (sl & 3) * 8;
}
__device__ __forceinline__ u32x4 v_fragment(const uint8_t* p) {
  const v4i16 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)p);
  const v4i16 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(p + 8 * VROW));
  const v4i16 v[2] = {x0, x1};
  return __builtin_bit_cast(u32x4, v);
}
// Row `slot` of a cache (ids and strides below 2^31: one 32 x 32 + 64 bit instruction)
__device__ __forceinline__ const uint8_t* slot_row(const uint8_t* cache, int slot, uint32_t ss) {
  return cache + (uint64_t)(uint32_t)slot * ss;
}

// Quotient a / b of two scales given as bits: powers of two; and its logarithm
__device__ __forceinline__ float scale_quotient(uint32_t a, uint32_t b) { return __uint_as_float(a - b + 0x3f800000u); }
__device__ __forceinline__ int quotient_log2(uint32_t a, uint32_t b) { return (int)(a - b) >> 23; }
// The accumulators' unit for values of scale vs (bits): kept while vs / unit is in [2^-2, 2^6], else a quarter of vs
__device__ __forceinline__ uint32_t unit_for(uint32_t vs, uint32_t unit) {
  const int q = quotient_log2(vs, unit);
  return q < -2 || q > 6 ? vs - (2u << 23) : unit;
}
// The accumulators brought to unit `to` (wave-uniform)
__device__ __forceinline__ void set_unit(uint32_t to, uint32_t& unit, f32x16 (&oacc)[D / 32]) {
  if (to != unit) {
    const float f = scale_quotient(unit, to);
#pragma unroll
    for (int db = 0; db < D / 32; ++db) oacc[db] *= f;
    unit = to;
  }
}

// Request of scheduling rank rho: requests by context length, longest first (ties by index), so that the longest
// workgroups start first and short ones fill in behind them. Up to MAX_RANKED of them, a lane each; larger batches go in their
// own order: every workgroup compares all pairs, which soon takes longer than what it could save (plain decoding of up to 2048
// tokens, 64 requests: 44.1 us ranked, 44.5 not; 128: 88 and 80, 512: 1241 and 254; 92 of 200 tokens and, behind them, four of
// 8000: 94 and 94; thousands would hold the GPU for minutes).
constexpr int MAX_RANKED = 64;
__device__ __forceinline__ int request_of_rank(const int64_t* ctx_lens, int bs, int rho) {
  if (bs <= 1 || bs > MAX_RANKED) return rho;
  const int b = threadIdx.x & 63;
  int rank = -1;
  if (b < bs) {
    const int64_t cb = ctx_lens[b];
    rank = 0;
    for (int j = 0; j < bs; ++j) {
      const int64_t cj = ctx_lens[j];
      rank += (cj > cb || (cj == cb && j < b)) ? 1 : 0;
    }
  }
  const uint64_t hit = __builtin_amdgcn_ballot_w64(rank == rho);
  return hit ? __builtin_ctzll(hit) : rho;  // (none: lengths written while they were read; the index stays in range)
}

// Program p: (KV head, request b, split s of `parts` of `keys` keys); false where there is none. KV heads fastest: with eight of
// them each XCD (workgroup id modulo 8) has one.
//
// split_keys given: every request SC splits; requests by rank, and with fewer heads the turn of the splits with the rank keeps
// a split from meeting the same XCDs in every request (short requests have only the first splits: a fixed pairing of splits
// and XCDs measured 462 us against 276).
// Not given: the splits' length, the same for all requests, is the shortest for which the requests' partials together are no
// more than the grid has pairs, so that a batch of mixed lengths fills it as well as one of equal ones; each workgroup finds it
// from the lengths (a lane per request, a search by halves).
__device__ __forceinline__ bool program_of(const Args& a, int p, int& s, int& kvh, int& b, int& parts, int& keys) {
  kvh = p % a.Hkv;
  const int q = p / a.Hkv;
  if (a.split_keys > 0 || a.SC == 1) {
    const int rho = q / a.S;
    s = (q + rho) % a.S;
    b = __builtin_amdgcn_readfirstlane(request_of_rank(a.ctx_lens, a.bs, rho));
    parts = a.SC;
    keys = a.split_keys;
    return true;
  }
  const int lane = threadIdx.x & 63;
  const bool mine = lane < a.bs;
  const int tiles = mine ? (kv8::bounded_len(a.pages, a.ctx_lens[lane]) + TK - 1) / TK : 0;
  const int extra = a.S - a.SC, want = a.pairs - extra * a.bs;
  const int total = kv8::wave_sum(tiles);
  auto count = [&](int k) { return mine ? max(1, (tiles + k - 1) / k) : 0; };
  // (at hi, total / hi + bs of them at most)
  int lo = max(a.min_tiles, (total + want - 1) / want);
  int hi = max(lo, max(total / (want - a.bs), total / a.SC) + 1);
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2, c = count(mid);
    const bool fits = __builtin_amdgcn_ballot_w64(c > a.SC) == 0 && kv8::wave_sum(c) <= want;
    hi = fits ? mid : hi;
    lo = fits ? lo : mid + 1;
  }
  const int c = count(lo), n = mine ? c + extra : 0;
  const int end = kv8::wave_scan(n);
  const uint64_t hit = __builtin_amdgcn_ballot_w64(q >= end - n && q < end);
  if (hit == 0) return false;
  b = __builtin_ctzll(hit);
  parts = __builtin_amdgcn_readlane(c, b);
  s = q - __builtin_amdgcn_readlane(end - n, b);
  if (s == parts) s = a.SC;  // the block keys' partial
  keys = lo * TK;
  return true;
}

// The keys [lo, hi) of context split s of `parts`
__device__ __forceinline__ void split_range(int s, int parts, int keys, int ctx, int& lo, int& hi) {
  lo = 0;
  hi = ctx;
  if (parts > 1) {
    lo = (int)min((int64_t)s * keys, (int64_t)ctx);
    if (s < parts - 1) hi = lo + min(keys, ctx - lo);  // (the last split takes what a longer context has left)
  }
}

// Infinities and NaN among the block's values: a product with them would be NaN in every row that shares the tile, also where
// the key is masked (0 times infinity). They are staged as zeros, and the rows that see them take them by themselves.
__device__ __forceinline__ bool has_nonfinite(const u32x4& x) {
  bool any = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) any |= (x[e] & 0x7f80u) == 0x7f80u || (x[e] & 0x7f800000u) == 0x7f800000u;
  return any;
}
__device__ __forceinline__ void drop_nonfinite(u32x4& x) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] &= (x[e] & 0x7f80u) == 0x7f80u ? 0xffff0000u : 0xffffffffu;
    x[e] &= (x[e] & 0x7f800000u) == 0x7f800000u ? 0xffffu : 0xffffffffu;
  }
}
// .. added to the accumulators of the rows (columns of O^T) that see the key; v: the key's values, from this half's d = 0
__device__ __forceinline__ void add_nonfinite(const uint16_t* v, bool sees, f32x16 (&oacc)[D / 32]) {
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const u16x4 x = *reinterpret_cast<const u16x4*>(v + db * 32 + gq * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float f = bf2f(x[e]);
        oacc[db][gq * 4 + e] += sees && !(fabsf(f) < INFINITY) ? f : 0.f;
      }
    }
}

// Index of a query row in the partials
__device__ __forceinline__ int64_t partial_row(const Args& a, int s, int b, int kvh, int r) {
  return (((int64_t)s * a.bs + b) * a.Hkv + kvh) * a.rows + r;
}

// ------------------------------------------------------------------------------------------------ tile kernel

// WHOLE: pages of at least 64 tokens, so that a tile lies in one page: its page id, address and scales are wave-uniform. Else
// each thread looks up its own keys' pages.
template <int NW, bool WHOLE>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv8_attn_tile_kernel(Args a) {
  static_assert(NW == 4 || NW == 8, "workgroups of 4 or 8 waves");
  constexpr int NPT = 8 / NW;   // 16-code pieces of a K or V tile per thread
  constexpr int RSTEP = NW * 8;
  __shared__ __attribute__((aligned(16))) uint8_t lds_k[2 * TK * KROW], lds_v[2 * TK * VROW];
  __shared__ uint32_t lds_vs[WHOLE ? 1 : 2 * TK];
  __shared__ uint32_t lds_nf[2][TK / 32];  // block keys with infinities or NaN among their values, of this and the next tile
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, l32 = lane & 31;
  const int KL = a.KL, Lb = a.L, rows = a.rows;
  const bool causal = a.causal != 0;
  const float scale = a.scale_log2;

  // workgroup -> (program, unit group); the unit groups of a program read the same keys: consecutive on one XCD (workgroup
  // id modulo 8), they share its L2
  const int P = (a.pairs ? a.pairs : a.bs * a.S) * a.Hkv;
  const int jx = blockIdx.x >> 3;
  const int ug = jx % a.ngroups;
  const int pidx = (jx / a.ngroups) * 8 + (blockIdx.x & 7);
  if (pidx >= P) return;
  int s, kvh, b, parts, keys;
  if (!program_of(a, pidx, s, kvh, b, parts, keys)) return;

  // this lane's query row; a padding row computes a copy of the last one and stores nothing
  const int u0 = (ug * NW + w) * UROWS;
  const bool active = u0 < rows;  // the wave has a row
  const bool row_ok = u0 + l32 < rows;
  const int r = min(u0 + l32, rows - 1);
  const int head = kvh * a.G + r / KL;
  const int qi = r % KL;
  const int64_t token = (int64_t)b * KL + qi;
  const int mode_lo = (qi / Lb) * Lb;  // first block key of this row's mode

  bf16x8 qf[D / 16];  // Q^T: B operand, k = d = 16 c + 8 half + e
  {
    const uint16_t* qp = a.q + token * a.q_st + (int64_t)head * a.q_sh + half * 8;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = as_bf16x8(*reinterpret_cast<const u16x8*>(qp + c * 16));
  }
  const int64_t given_len = a.ctx_lens[b];
  const int32_t* trow = kv8::table_row(a.pages, b);
  const int shift = a.pages.page_shift, pmask = (1 << shift) - 1, num_pages = a.pages.num_pages;
  const int ctx = __builtin_amdgcn_readfirstlane(trow && num_pages > 0 ? kv8::bounded_len(a.pages, given_len) : 0);
  int lo, hi;
  split_range(s, parts, keys, ctx, lo, hi);
  bool with_block = a.kn != nullptr;
  if (a.S > a.SC) {  // split: the block keys are a partial of their own
    if (s == a.SC) lo = hi = ctx;
    else with_block = false;
  }
  const int ntiles = (hi - lo + TK - 1) / TK;
  const int last = ntiles - 1;
  if (tid == 0 && s == 0 && ug == 0 && kvh == 0) {
    if (ctx != given_len || !trow) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
    if (a.S > 1) a.ws_n[b] = parts;
  }
  if (a.S > 1 && ntiles == 0 && !with_block) {  // an empty split
    if (row_ok && half == 0) a.ws_lse[partial_row(a, s, b, kvh, r)] = -INFINITY;
    return;
  }

  float m_run = -INFINITY, l_run = 0.f;
  f32x16 oacc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) oacc[db] = (f32x16){};
  uint32_t unit = 0x3f800000u;  // of the accumulators: bits of a power of two

  const uint8_t* const kb = lds_k + k_operand(lane);
  const uint8_t* const vb = lds_v + v_operand(lane);
  // S^T of the tile in K buffer 0: keys 32 ks + 8 (x / 4) + 4 half + x % 4 (x: register), column = this lane's row
  auto scores = [&](f32x16 (&sv)[2]) __attribute__((always_inline)) {
    sv[0] = sv[1] = (f32x16){};
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const u16x8 k0f = *reinterpret_cast<const u16x8*>(kb + 32 * c);
      const u16x8 k1f = *reinterpret_cast<const u16x8*>(kb + 32 * c + 32 * KROW);
      sv[0] = mfma32(as_bf16x8(k0f), qf[c], sv[0]);
      sv[1] = mfma32(as_bf16x8(k1f), qf[c], sv[1]);
    }
  };
  // Online softmax, first part: keys outside [klo, khi) of the tile masked, the row maximum, and the running reference
  // moved (with a rescale) only when a score exceeds it by more than 2^8; returns the reference.
  auto softmax_max = [&](bool masked, int klo, int khi, f32x16 (&sv)[2]) __attribute__((always_inline)) {
    if (masked) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const int key = ks * 32 + 8 * (x >> 2) + 4 * half + (x & 3);
          sv[ks][x] = (key >= klo && key < khi) ? sv[ks][x] : -INFINITY;
        }
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int x = 0; x < 16; ++x) tmax = fmaxf(tmax, sv[ks][x]);
    const float tm = half_max(tmax) * scale;
    if (__builtin_amdgcn_ballot_w64(tm > m_run + 8.f) != 0) {
      const float m_new = fmaxf(m_run, tm);
      const float alpha = (m_run == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) oacc[db] *= alpha;
      m_run = m_new;
    }
    return (m_run == -INFINITY) ? 0.f : m_run;
  };

  // ---- staging: thread (row tid / 8 + i RSTEP, 16 codes tid % 8) of a tile. Keys past the range repeat its last one
  //      (probability 0).
  const int r0 = tid >> 3, part = tid & 7;
  const uint8_t* kc_h = a.kc + (int64_t)kvh * a.kc_sh;
  const uint8_t* vc_h = a.vc + (int64_t)kvh * a.vc_sh;
  const float* ks_h = a.ks + kvh;
  const float* vs_h = a.vs + kvh;
  const uint32_t kc_ss = (uint32_t)a.kc_ss, vc_ss = (uint32_t)a.vc_ss;
  const int Hkv = a.Hkv;
  int bad = 0;
  // A wave-uniform word by a vector load all the same: a scalar one shares its counter with LDS and returns out of order, so
  // that the next wait for an LDS operand would wait for it too.
  int lane0 = 0;
  asm("v_mov_b32 %0, 0" : "=v"(lane0));
  constexpr int NE = WHOLE ? 1 : NPT;  // page ids of a tile that a thread keeps
  auto key_of = [&](int t, int i) __attribute__((always_inline)) { return min(lo + t * TK + r0 + i * RSTEP, hi - 1); };
  // Page ids are asked for an iteration before they are used, and looked at (their bounds) only then: a test next to the
  // load would wait for it.
  auto pages_of = [&](int t, int (&e)[NE]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      if constexpr (WHOLE) e[i] = trow[((lo + t * TK) >> shift) + lane0];
      else e[i] = trow[key_of(t, i) >> shift];
    }
  };
  auto checked = [&](int e) __attribute__((always_inline)) {
    const bool ok = (uint32_t)e < (uint32_t)num_pages;
    bad |= ok ? 0 : 1;
    return ok ? e : 0;
  };
  auto load = [&](const uint8_t* cache, uint32_t ss, const float* scales, int t, const int (&e)[NE], u32x4 (&c)[NPT],
                  float (&sc)[NE]) __attribute__((always_inline)) {
    if constexpr (WHOLE) {
      const int k0 = lo + t * TK, pg = checked(__builtin_amdgcn_readfirstlane(e[0]));
      const uint8_t* base = slot_row(cache, __builtin_amdgcn_readfirstlane((pg << shift) + (k0 & pmask)), ss);
      const int nv = hi - k0;
      if (nv >= TK) {
#pragma unroll
        for (int i = 0; i < NPT; ++i)
          c[i] = *reinterpret_cast<const u32x4*>(base + i * RSTEP * ss + ((uint32_t)r0 * ss + (uint32_t)part * 16));
      } else {
#pragma unroll
        for (int i = 0; i < NPT; ++i)
          c[i] = *reinterpret_cast<const u32x4*>(
              base + ((uint32_t)min(r0 + i * RSTEP, nv - 1) * ss + (uint32_t)part * 16));
      }
      sc[0] = scales[pg * Hkv + lane0];
    } else {
#pragma unroll
      for (int i = 0; i < NPT; ++i) {
        const int pg = checked(e[i]);
        c[i] = *reinterpret_cast<const u32x4*>(slot_row(cache, (pg << shift) + (key_of(t, i) & pmask), ss) + part * 16);
        sc[i] = scales[pg * Hkv];
      }
    }
  };
  auto put_k = [&](int j, const u32x4 (&c)[NPT], const float (&sc)[NE]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NPT; ++i) put_k_codes(lds_k + (j * TK + r0 + i * RSTEP) * KROW, part, c[i], sc[WHOLE ? 0 : i]);
  };
  auto put_v = [&](int j, const u32x4 (&c)[NPT], const float (&sc)[NE]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NPT; ++i) {
      put_v_codes(lds_v + (j * TK + r0 + i * RSTEP) * VROW, part, c[i]);
      if constexpr (!WHOLE)
        if (part == 0) lds_vs[j * TK + r0 + i * RSTEP] = __float_as_uint(sc[i]);
    }
  };

  if (ntiles > 0) {
    // Tile t of K and of V goes through buffer t % 2. When iteration t starts, K(t + 1) and V(t) are in LDS, K(t + 2) and
    // V(t + 1) in (or on their way to) registers and S(t) is computed; it writes those two into the buffers that
    // iteration t - 1 read last, asks for K(t + 3) and V(t + 2), and computes S(t + 1) and O += V(t) P(t).
    u32x4 kr[NPT], vr[NPT];
    float ksc[NE], vsc[NE];
    int ev[NE], ek[NE];  // pages of tiles t + 2 and t + 3
    uint32_t vs_t;       // WHOLE: scale of V(t)
    {
      u32x4 k0[NPT], v0[NPT];
      float k0s[NE], v0s[NE];
      int e0[NE], e1[NE];
      pages_of(0, e0);
      pages_of(min(1, last), e1);
      pages_of(min(2, last), ev);
      pages_of(min(3, last), ek);
      load(kc_h, kc_ss, ks_h, 0, e0, k0, k0s);
      load(vc_h, vc_ss, vs_h, 0, e0, v0, v0s);
      load(kc_h, kc_ss, ks_h, min(1, last), e1, kr, ksc);
      put_k(0, k0, k0s);
      put_v(0, v0, v0s);
      put_k(1, kr, ksc);
      vs_t = __builtin_amdgcn_readfirstlane(__float_as_uint(v0s[0]));
      load(kc_h, kc_ss, ks_h, min(2, last), ev, kr, ksc);
      load(vc_h, vc_ss, vs_h, min(1, last), e1, vr, vsc);
    }
    f32x16 s_a[2], s_b[2];
    lds_barrier();
    scores(s_a);
    lds_barrier();  // every wave is done with K buffer 0

    // The 32 MFMAs of an iteration as a fixed sequence of slots: s < 8 is S^T subtile 0 of tile t + 1 (d chunk s), 8 .. 15
    // P V of key chunks 0 and 1 of tile t (d block s % 4), 16 .. 23 S^T subtile 1, 24 .. 31 P V of chunks 2 and 3. LDS
    // operands are read FD slots ahead, a pair of probabilities is formed in each S^T slot, and a scheduling barrier
    // closes every slot (left alone, the compiler hoists all reads and spills, or sinks them next to their products).
    constexpr int FD = 2;
    auto slot_is_qk = [](int sl) __attribute__((always_inline)) { return sl < 8 || (sl >= 16 && sl < 24); };
    auto chunk_of = [](int sl) __attribute__((always_inline)) { return sl < 12 ? 0 : sl < 16 ? 1 : sl < 28 ? 2 : 3; };
    // (j: the buffer of V(t); K(t + 1) is in the other one)
    auto fetch = [&](int sl, int j) __attribute__((always_inline)) {
      if (slot_is_qk(sl))
        return *reinterpret_cast<const u32x4*>(kb + (j ^ 1) * (TK * KROW) + 32 * (sl & 7) + (sl >= 16 ? 32 * KROW : 0));
      return v_fragment(vb + j * (TK * VROW) + 64 * (sl & 3) + 16 * VROW * chunk_of(sl));
    };
    auto iteration = [&](int t, auto parity, f32x16 (&s_cur)[2], f32x16 (&s_nxt)[2]) __attribute__((always_inline)) {
      constexpr int j = decltype(parity)::value;  // t % 2: LDS addresses become constants
      put_k(j, kr, ksc);
      put_v(j ^ 1, vr, vsc);
      const uint32_t vs_next = __builtin_amdgcn_readfirstlane(__float_as_uint(vsc[0]));
      if (t + 2 < ntiles) {
        load(vc_h, vc_ss, vs_h, t + 2, ev, vr, vsc);
        load(kc_h, kc_ss, ks_h, min(t + 3, last), ek, kr, ksc);
#pragma unroll
        for (int i = 0; i < NE; ++i) ev[i] = ek[i];
        pages_of(min(t + 4, last), ek);
      }
      if (active) {
        const int khi = hi - (lo + t * TK);
        const float msub = softmax_max(khi < TK, 0, khi, s_cur);
        // each 16-key chunk's quotient of scale and unit: in the exponent, and out of the row sum
        constexpr int NC = WHOLE ? 1 : 4;  // chunks with a scale of their own
        float sub[NC], back[NC];
        uint32_t units[NC];
        {
          uint32_t vs_l = vs_t;
          if constexpr (!WHOLE) vs_l = lds_vs[j * TK + 16 * (lane & 3)];
          uint32_t u = unit;
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const uint32_t vs = WHOLE ? vs_t : (uint32_t)__builtin_amdgcn_readlane(vs_l, c);
            u = unit_for(vs, u);
            units[c] = u;
            sub[c] = msub - (float)quotient_log2(vs, u);
            back[c] = scale_quotient(u, vs);
          }
        }
        u32x4 opnd[32];
#pragma unroll
        for (int sl = 0; sl < FD; ++sl) opnd[sl] = fetch(sl, j);
        u32x4 pv[4];  // P^T B fragments (fp16 pairs) of the chunks
        float psum = 0.f;
        f32x16 acc0 = {}, acc1 = {};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int sl = 0; sl < 32; ++sl) {
          if (sl == 8 || (!WHOLE && (sl == 12 || sl == 24 || sl == 28))) set_unit(units[WHOLE ? 0 : chunk_of(sl)], unit, oacc);
          if (sl + FD < 32) opnd[sl + FD] = fetch(sl + FD, j);
          if (slot_is_qk(sl)) {
            if (sl < 8) acc0 = mfma32(__builtin_bit_cast(bf16x8, opnd[sl]), qf[sl & 7], acc0);
            else acc1 = mfma32(__builtin_bit_cast(bf16x8, opnd[sl]), qf[sl & 7], acc1);
            // key pair y of chunk c: S^T registers x, x + 1 of subtile c / 2
            const int c = (sl < 8 ? 0 : 2) + ((sl & 7) >> 2), y = sl & 3;
            const int x = (c & 1) * 8 + 2 * y;
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s_cur[c >> 1][x], scale, -sub[WHOLE ? 0 : c]));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s_cur[c >> 1][x + 1], scale, -sub[WHOLE ? 0 : c]));
            psum += p0 + p1;
            asm volatile("" : "+v"(psum));  // keeps the add in this slot
            pv[c][y] = f2h2_bits(p0, p1);
            if (!WHOLE && y == 3) {
              l_run = __builtin_fmaf(psum, back[c], l_run);
              psum = 0.f;
            }
          } else {
            const int c = chunk_of(sl), db = sl & 3;
            oacc[db] = mfma32_f16(__builtin_bit_cast(f16x8, opnd[sl]), __builtin_bit_cast(f16x8, pv[c]), oacc[db]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (WHOLE) l_run = __builtin_fmaf(psum, back[0], l_run);
        s_nxt[0] = acc0;
        s_nxt[1] = acc1;
      }
      vs_t = vs_next;
      lds_barrier();
    };
    for (int t = 0;;) {
      iteration(t, std::integral_constant<int, 0>{}, s_a, s_b);
      if (++t >= ntiles) break;
      iteration(t, std::integral_constant<int, 1>{}, s_b, s_a);
      if (++t >= ntiles) break;
    }
  }
  if (bad) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);

  // ---- the request's block keys in bf16: tiles through buffer 0, P split into a bf16 pair hi + lo (2^-17) against V as
  //      it is. A workgroup whose rows lie in one query head needs only the keys of those rows' modes.
  if (with_block) {
    int blo = 0, bhi = KL;
    const int g0 = ug * NW * UROWS, g1 = min(g0 + NW * UROWS, rows) - 1;  // the workgroup's rows
    if (g0 / KL == g1 / KL) {
      blo = (g0 % KL) / Lb * Lb;
      bhi = ((g1 % KL) / Lb + 1) * Lb;
    }
    set_unit(0x3f800000u, unit, oacc);
    if (tid < TK / 32) lds_nf[0][tid] = 0;
    int turn = 0;
    for (int b0 = blo; b0 < bhi; b0 += TK, turn ^= 1) {
      lds_barrier();  // every wave is done with the buffers
#pragma unroll
      for (int i = 0; i < NPT; ++i) {
        const int rr = r0 + i * RSTEP;
        const int64_t tk = (int64_t)b * KL + min(b0 + rr, bhi - 1);
        const u32x4* kp = reinterpret_cast<const u32x4*>(a.kn + tk * a.kn_st + (int64_t)kvh * a.kn_sh + part * 16);
        const u32x4* vp = reinterpret_cast<const u32x4*>(a.vn + tk * a.vn_st + (int64_t)kvh * a.vn_sh + part * 16);
        const u32x4 kx = kp[0], ky = kp[1];
        u32x4 vx = vp[0], vy = vp[1];
        if (has_nonfinite(vx) || has_nonfinite(vy)) {
          drop_nonfinite(vx);
          drop_nonfinite(vy);
          atomicOr(&lds_nf[turn][rr >> 5], 1u << (rr & 31));
        }
        put_row(lds_k + rr * KROW, part, kx, ky);
        put_row(lds_v + rr * VROW, part, vx, vy);
      }
      lds_barrier();
      if (tid < TK / 32) lds_nf[turn ^ 1][tid] = 0;  // (read last in front of this tile's first barrier)
      const int klo = mode_lo - b0, khi = min(mode_lo + (causal ? qi - mode_lo + 1 : Lb), bhi) - b0;
      if (active && __builtin_amdgcn_ballot_w64(klo < TK && khi > 0) != 0) {
        f32x16 sv[2];
        scores(sv);
        const float msub = softmax_max(true, klo, khi, sv);
        float psum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          u32x4 ph, pl;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int x = (c & 1) * 8 + 2 * y;
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[c >> 1][x], scale, -msub));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[c >> 1][x + 1], scale, -msub));
            psum += p0 + p1;
            ph[y] = f2bf2_bits(p0, p1);
            pl[y] = f2bf2_bits(p0 - __uint_as_float(ph[y] << 16), p1 - __uint_as_float(ph[y] & 0xffff0000u));
          }
#pragma unroll
          for (int db = 0; db < D / 32; ++db) {
            const bf16x8 vf = __builtin_bit_cast(bf16x8, v_fragment(vb + 64 * db + 16 * VROW * c));
            oacc[db] = mfma32(vf, __builtin_bit_cast(bf16x8, ph), oacc[db]);
            oacc[db] = mfma32(vf, __builtin_bit_cast(bf16x8, pl), oacc[db]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        l_run += psum;
#pragma unroll 1
        for (int x = 0; x < TK / 32; ++x) {
          uint32_t nf = __builtin_amdgcn_readfirstlane(lds_nf[turn][x]);
#pragma unroll 1
          for (; nf; nf &= nf - 1) {
            const int key = x * 32 + __builtin_ctz(nf);
            const uint16_t* vp = a.vn + ((int64_t)b * KL + min(b0 + key, bhi - 1)) * a.vn_st + (int64_t)kvh * a.vn_sh;
            add_nonfinite(vp + half * 4, key >= klo && key < khi, oacc);
          }
        }
      }
    }
  }
  lds_barrier();  // every wave is done with the buffers
  if (!active) return;

  // The rows leave through LDS (a unit's part of the K or V buffers, padded rows), so that a store takes whole rows and not 16
  // bytes of each of 32 (one request of 32768 tokens 85 us against 87).
  uint8_t* const rows_lds = w < 4 ? lds_k + w * (UROWS * KROW) : lds_v + (w - 4) * (UROWS * VROW);
  const int pitch = w < 4 ? KROW : VROW;
  const int valid = min(rows - u0, UROWS);
  auto put = [&](int db, int gq, uint32_t lo2, uint32_t hi2) __attribute__((always_inline)) {
    *reinterpret_cast<u32x2*>(rows_lds + l32 * pitch + db * 64 + gq * 16 + half * 8) = (u32x2){lo2, hi2};
  };
  const int piece = lane & 15;  // of 16 bytes; four rows per store
  auto take = [&](int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(rows_lds + (4 * i + (lane >> 4)) * pitch + piece * 16);
  };
  const float l_tot = half_sum(l_run);
  const float inv = l_tot > 0.f ? __uint_as_float(unit) / l_tot : (l_tot == 0.f ? 0.f : l_tot);  // (NaN stays NaN)
  const float lse2 = l_tot > 0.f ? m_run + __log2f(l_tot) : (l_tot == 0.f ? -INFINITY : l_tot);
  if (a.S == 1) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        put(db, gq, f2bf2_bits(oacc[db][gq * 4 + 0] * inv, oacc[db][gq * 4 + 1] * inv),
            f2bf2_bits(oacc[db][gq * 4 + 2] * inv, oacc[db][gq * 4 + 3] * inv));
    asm volatile("" ::: "memory");  // (a wave's LDS operations complete in order)
#pragma unroll
    for (int i = 0; i < UROWS / 4; ++i) {
      const int at = 4 * i + (lane >> 4);
      if (at < valid) {
        const int rr = u0 + at;
        uint16_t* op = a.out + ((int64_t)b * KL + rr % KL) * a.o_st + (int64_t)(kvh * a.G + rr / KL) * a.o_sh;
        *reinterpret_cast<u32x4*>(op + piece * 8) = take(i);
      }
    }
    if (a.lse && row_ok && half == 0) a.lse[token * a.H + head] = lse2 * LN2;
    return;
  }
  // partial row in fp16, its finite components scaled by a power of two into (-1, 1): half the bytes of fp32 for the merge to
  // read back, at 2^-11 of a component, or 2^-24 of the row's largest where that is more
  float mx = 0.f;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int x = 0; x < 16; ++x) mx = fmaxf(mx, fabsf(oacc[db][x] * inv));
  mx = half_max(mx);
  if (__builtin_amdgcn_ballot_w64(mx == INFINITY) != 0) {  // (hardly ever: the test per component would cost 1 us)
    mx = 0.f;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) mx = fmaxf(mx, kv8::finite_abs(oacc[db][x] * inv));
    mx = half_max(mx);
  }
  const int ex = mx > 0.f ? __builtin_amdgcn_frexp_expf(mx) : 0;
  const float down = __builtin_ldexpf(inv, -ex);
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq)
      put(db, gq, f2h2_bits(oacc[db][gq * 4 + 0] * down, oacc[db][gq * 4 + 1] * down),
          f2h2_bits(oacc[db][gq * 4 + 2] * down, oacc[db][gq * 4 + 3] * down));
  asm volatile("" ::: "memory");
  const int64_t first = partial_row(a, s, b, kvh, u0);
  uint16_t* const op = a.ws_o + first * D + lane * 8;  // (a partial's rows lie side by side)
#pragma unroll
  for (int i = 0; i < UROWS / 4; ++i)
    if (4 * i + (lane >> 4) < valid) *reinterpret_cast<u32x4*>(op + i * (4 * D)) = take(i);
  if (row_ok && half == 0) {
    a.ws_lse[first + l32] = lse2;
    a.ws_exp[first + l32] = (float)ex;
  }
}

// ---------------------------------------------------------------------------------------------- stream kernel

// SNW waves: four, and two workgroups on a CU; or eight, where the grid has no more workgroups than there are CUs
template <int SNW>
__global__ __launch_bounds__(SNW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv8_attn_stream_kernel(Args a) {
  static_assert(SNW == 4 || SNW == 8, "a row's results are joined by 8 or 16 threads");
  constexpr int WLDS = SK * (KROW + VROW);  // bytes of a wave's widened K and V tile (17.5 KB)
  static_assert(UROWS * D * 4 <= WLDS, "a wave's result fits its tiles");
  __shared__ __attribute__((aligned(16))) uint8_t lds[SNW * WLDS];
  __shared__ float lds_m[SNW][UROWS], lds_l[SNW][UROWS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, l32 = lane & 31;
  const int KL = a.KL, Lb = a.L, rows = a.rows;
  const float scale = a.scale_log2;
  int s, kvh, b, parts, keys;
  if (!program_of(a, blockIdx.x, s, kvh, b, parts, keys)) return;
  const int32_t* trow = kv8::table_row(a.pages, b);
  const int shift = a.pages.page_shift, pmask = (1 << shift) - 1, num_pages = a.pages.num_pages;
  const int ctx = __builtin_amdgcn_readfirstlane(trow && num_pages > 0 ? kv8::bounded_len(a.pages, a.ctx_lens[b]) : 0);
  int lo, hi;
  split_range(s, parts, keys, ctx, lo, hi);
  const bool with_block = a.kn != nullptr && s == 0;
  if (tid == 0 && s == 0 && kvh == 0) {
    if (ctx != a.ctx_lens[b] || !trow) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
    if (a.S > 1) a.ws_n[b] = parts;
  }
  if (lo >= hi && !with_block && a.S > 1) {  // an empty split
    if (tid < rows) a.ws_lse[partial_row(a, s, b, kvh, tid)] = -INFINITY;
    return;
  }
  const int r = min(l32, rows - 1);
  const int qi = r % KL;
  const int mode_lo = (qi / Lb) * Lb;
  bf16x8 qf[D / 16];
  {
    const uint16_t* qp =
        a.q + ((int64_t)b * KL + qi) * a.q_st + (int64_t)(kvh * a.G + r / KL) * a.q_sh + half * 8;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) qf[c] = as_bf16x8(*reinterpret_cast<const u16x8*>(qp + c * 16));
  }
  uint8_t* const lds_k = lds + w * WLDS;
  uint8_t* const lds_v = lds_k + SK * KROW;
  const uint8_t* const kb = lds_k + k_operand(lane);
  const uint8_t* const vb = lds_v + v_operand(lane);
  float m_run = -INFINITY, l_run = 0.f;
  f32x16 oacc[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) oacc[db] = (f32x16){};
  uint32_t unit = 0x3f800000u;  // of the accumulators: bits of a power of two

  auto scores = [&]() __attribute__((always_inline)) {
    f32x16 acc = {};
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      acc = mfma32(as_bf16x8(*reinterpret_cast<const u16x8*>(kb + 32 * c)), qf[c], acc);
    return acc;
  };
  // register x of a 32-key score tile is key 8 (x / 4) + 4 half + x % 4
  auto softmax_max = [&](bool masked, int klo, int khi, f32x16& sv) __attribute__((always_inline)) {
    if (masked) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const int key = 8 * (x >> 2) + 4 * half + (x & 3);
        sv[x] = (key >= klo && key < khi) ? sv[x] : -INFINITY;
      }
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int x = 0; x < 16; ++x) tmax = fmaxf(tmax, sv[x]);
    const float tm = half_max(tmax) * scale;
    if (__builtin_amdgcn_ballot_w64(tm > m_run + 8.f) != 0) {
      const float m_new = fmaxf(m_run, tm);
      const float alpha = (m_run == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) oacc[db] *= alpha;
      m_run = m_new;
    }
    return (m_run == -INFINITY) ? 0.f : m_run;
  };

  // ---- this wave's tiles: w, w + SNW, ..; a lane holds 16 codes (lane % 8) of rows lane / 8 + 8 i
  const int r0 = lane >> 3, part = lane & 7;
  const uint8_t* kc_h = a.kc + (int64_t)kvh * a.kc_sh + part * 16;
  const uint8_t* vc_h = a.vc + (int64_t)kvh * a.vc_sh + part * 16;
  const int Hkv = a.Hkv;
  const float* ks_h = a.ks + kvh;
  const float* vs_h = a.vs + kvh;
  const uint32_t kc_ss = (uint32_t)a.kc_ss, vc_ss = (uint32_t)a.vc_ss;
  const int ntiles = (hi - lo + SK - 1) / SK;
  int bad = 0;
  auto key_of = [&](int t, int i) __attribute__((always_inline)) { return min(lo + t * SK + r0 + 8 * i, hi - 1); };
  auto page_of = [&](int t, int i) __attribute__((always_inline)) { return trow[key_of(t, i) >> shift]; };
  if (w < ntiles) {
    u32x4 kr[4], vr[4];
    float ksc[4], vsc[4];
    int en[4];
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool ok = (uint32_t)en[i] < (uint32_t)num_pages;  // (looked at here: the ids were asked for a tile ago)
        bad |= ok ? 0 : 1;
        const int pg = ok ? en[i] : 0;
        const int slot = (pg << shift) + (key_of(t, i) & pmask);
        kr[i] = *reinterpret_cast<const u32x4*>(slot_row(kc_h, slot, kc_ss));
        vr[i] = *reinterpret_cast<const u32x4*>(slot_row(vc_h, slot, vc_ss));
        ksc[i] = ks_h[pg * Hkv];
        vsc[i] = vs_h[pg * Hkv];
      }
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) en[i] = page_of(w, i);
    load(w);
    if (w + SNW < ntiles) {
#pragma unroll
      for (int i = 0; i < 4; ++i) en[i] = page_of(w + SNW, i);
    }
    for (int t = w; t < ntiles; t += SNW) {
      // (a wave's LDS operations complete in order: nothing of the last tile is still to be read)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        put_k_codes(lds_k + (r0 + 8 * i) * KROW, part, kr[i], ksc[i]);
        put_v_codes(lds_v + (r0 + 8 * i) * VROW, part, vr[i]);
      }
      const uint32_t vs_t[2] = {(uint32_t)__builtin_amdgcn_readfirstlane(__float_as_uint(vsc[0])),
                                (uint32_t)__builtin_amdgcn_readfirstlane(__float_as_uint(vsc[2]))};
      if (t + SNW < ntiles) {
        load(t + SNW);
        if (t + 2 * SNW < ntiles) {
#pragma unroll
          for (int i = 0; i < 4; ++i) en[i] = page_of(t + 2 * SNW, i);
        }
      }
      asm volatile("" ::: "memory");
      f32x16 sv = scores();
      const int khi = hi - (lo + t * SK);
      const float msub = softmax_max(khi < SK, 0, khi, sv);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        set_unit(unit_for(vs_t[c], unit), unit, oacc);
        const float sub = msub - (float)quotient_log2(vs_t[c], unit);
        u32x4 pv;
        float psum = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[8 * c + 2 * y], scale, -sub));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[8 * c + 2 * y + 1], scale, -sub));
          psum += p0 + p1;
          pv[y] = f2h2_bits(p0, p1);
        }
        l_run = __builtin_fmaf(psum, scale_quotient(unit, vs_t[c]), l_run);
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
          oacc[db] = mfma32_f16(__builtin_bit_cast(f16x8, v_fragment(vb + 64 * db + 16 * VROW * c)),
                                __builtin_bit_cast(f16x8, pv), oacc[db]);
      }
      asm volatile("" ::: "memory");
    }
  }
  if (bad) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
  // ---- the block keys (rows <= 32, so K L <= 32: one tile), in bf16 with P as a bf16 pair, by the last wave
  if (with_block && w == SNW - 1) {
    set_unit(0x3f800000u, unit, oacc);
    uint32_t nf = 0;  // keys with infinities or NaN among their values
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = r0 + 8 * i;
      const int64_t tk = (int64_t)b * KL + min(rr, KL - 1);
      const u32x4* kp = reinterpret_cast<const u32x4*>(a.kn + tk * a.kn_st + (int64_t)kvh * a.kn_sh + part * 16);
      const u32x4* vp = reinterpret_cast<const u32x4*>(a.vn + tk * a.vn_st + (int64_t)kvh * a.vn_sh + part * 16);
      const u32x4 kx = kp[0], ky = kp[1];
      u32x4 vx = vp[0], vy = vp[1];
      uint64_t lanes = __builtin_amdgcn_ballot_w64(has_nonfinite(vx) || has_nonfinite(vy));
      if (lanes) {
        drop_nonfinite(vx);
        drop_nonfinite(vy);
        for (; lanes; lanes &= lanes - 1) nf |= 1u << (8 * i + __builtin_ctzll(lanes) / 8);
      }
      put_row(lds_k + rr * KROW, part, kx, ky);
      put_row(lds_v + rr * VROW, part, vx, vy);
    }
    asm volatile("" ::: "memory");
    f32x16 sv = scores();
    const int khi = a.causal ? qi + 1 : mode_lo + Lb;
    const float msub = softmax_max(true, mode_lo, khi, sv);
    float psum = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4 ph, pl;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[8 * c + 2 * y], scale, -msub));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[8 * c + 2 * y + 1], scale, -msub));
        psum += p0 + p1;
        ph[y] = f2bf2_bits(p0, p1);
        pl[y] = f2bf2_bits(p0 - __uint_as_float(ph[y] << 16), p1 - __uint_as_float(ph[y] & 0xffff0000u));
      }
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        const bf16x8 vf = __builtin_bit_cast(bf16x8, v_fragment(vb + 64 * db + 16 * VROW * c));
        oacc[db] = mfma32(vf, __builtin_bit_cast(bf16x8, ph), oacc[db]);
        oacc[db] = mfma32(vf, __builtin_bit_cast(bf16x8, pl), oacc[db]);
      }
    }
    l_run += psum;
#pragma unroll 1
    for (; nf; nf &= nf - 1) {
      const int key = __builtin_ctz(nf);
      const uint16_t* vp = a.vn + ((int64_t)b * KL + min(key, KL - 1)) * a.vn_st + (int64_t)kvh * a.vn_sh;
      add_nonfinite(vp + half * 4, key >= mode_lo && key < khi, oacc);
    }
  }
  // ---- the waves' results: each brings its accumulators to the common reference and into its part of LDS as [row][d] fp32
  //      (16 KB); TPR threads per row add them in wave order
  constexpr int TPR = SNW * 64 / UROWS, DPT = D / TPR;  // 8 or 16 threads, of 16 or 8 d's
  const float l_w = half_sum(l_run);
  if (half == 0) {
    lds_m[w][l32] = m_run;
    lds_l[w][l32] = l_w;
  }
  lds_barrier();
  float m_tot = lds_m[0][l32];
#pragma unroll
  for (int x = 1; x < SNW; ++x) m_tot = fmaxf(m_tot, lds_m[x][l32]);
  const float fac = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m_tot) * __uint_as_float(unit);
  float* const own = reinterpret_cast<float*>(lds + w * WLDS);
  // 16-byte piece c of row r at c ^ r, so that the lanes of a write or a read spread over the banks
  auto has_keys = [&](int x) __attribute__((always_inline)) { return x < ntiles || (with_block && x == SNW - 1); };
  if (has_keys(w)) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const int c = db * 8 + gq * 2 + half;
        *reinterpret_cast<f32x4*>(own + l32 * D + ((c ^ l32) & 31) * 4) =
            (f32x4){oacc[db][gq * 4 + 0] * fac, oacc[db][gq * 4 + 1] * fac, oacc[db][gq * 4 + 2] * fac,
                    oacc[db][gq * 4 + 3] * fac};
      }
  }
  lds_barrier();
  const int row = tid / TPR, piece = tid % TPR, d0 = piece * DPT;
  f32x4 o[DPT / 4] = {};
  float mt = -INFINITY, lt = 0.f;
#pragma unroll
  for (int x = 0; x < SNW; ++x) mt = fmaxf(mt, lds_m[x][row]);
#pragma unroll
  for (int x = 0; x < SNW; ++x) {
    if (!has_keys(x)) continue;
    const float mw = lds_m[x][row], lw = lds_l[x][row];
    lt += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f(mw - mt);  // (-inf: no key, 0, or NaN)
#pragma unroll
    for (int c = 0; c < DPT / 4; ++c)
      o[c] += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + x * WLDS) + row * D +
                                              (((d0 / 4 + c) ^ row) & 31) * 4);
  }
  if (row >= rows) return;  // (whole groups of threads)
  const float inv = lt > 0.f ? 1.f / lt : (lt == 0.f ? 0.f : lt);
  const float lse2 = lt > 0.f ? mt + __log2f(lt) : (lt == 0.f ? -INFINITY : lt);
  if (a.S == 1) {
    const int64_t token = (int64_t)b * KL + row % KL;
    const int head = kvh * a.G + row / KL;
    uint16_t* op = a.out + token * a.o_st + (int64_t)head * a.o_sh + d0;
#pragma unroll
    for (int c = 0; c < DPT / 8; ++c) {
      u16x8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = f2bf_bits(o[2 * c + (e >> 2)][e & 3] * inv);
      *reinterpret_cast<u16x8*>(op + 8 * c) = v;
    }
    if (a.lse && piece == 0) a.lse[token * a.H + head] = lse2 * LN2;
    return;
  }
  float mx = 0.f;
#pragma unroll
  for (int c = 0; c < DPT / 4; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) mx = fmaxf(mx, kv8::finite_abs(o[c][e] * inv));
#pragma unroll
  for (int x = 1; x < TPR; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
  const int ex = mx > 0.f ? __builtin_amdgcn_frexp_expf(mx) : 0;
  const float down = __builtin_ldexpf(inv, -ex);
  const int64_t prow = partial_row(a, s, b, kvh, row);
#pragma unroll
  for (int c = 0; c < DPT / 8; ++c) {
    u32x4 hv;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      hv[e] = f2h2_bits(o[2 * c + (e >> 1)][2 * (e & 1)] * down, o[2 * c + (e >> 1)][2 * (e & 1) + 1] * down);
    *reinterpret_cast<u32x4*>(a.ws_o + prow * D + d0 + 8 * c) = hv;
  }
  if (piece == 0) {
    a.ws_lse[prow] = lse2;
    a.ws_exp[prow] = (float)ex;
  }
}

// ------------------------------------------------------------------------------------------------------- merge

// 16 threads per row, 8 d's each; the partials in batches of 8, all loads of a batch in flight together, joined with a
// running log-sum-exp. An empty partial (lse -inf) wrote no row: what is read of it is not used. Latency: 4 to 6 us (four
// groups of threads per row that share the partials: 32.2 us against 31.0 at one request of 4096 tokens).
__global__ __launch_bounds__(256) void kv8_attn_merge_kernel(Args a) {
  constexpr int SB = 8;
  const int64_t per = (int64_t)a.bs * a.Hkv * a.rows;
  const int64_t prow = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (prow >= per) return;
  const int d0 = (threadIdx.x & 15) * 8;
  const int parts = a.split_keys > 0 ? a.SC : a.ws_n[prow / a.rows / a.Hkv], S = parts + a.S - a.SC;
  float m = -INFINITY, tot = 0.f;
  float acc[8] = {};
  for (int s0 = 0; s0 < S; s0 += SB) {
    float l[SB], ex[SB];
    u32x4 oh[SB];
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      l[j] = -INFINITY;
      ex[j] = 0.f;
      oh[j] = (u32x4){};
      if (s0 + j < S) {
        const int64_t at = (s0 + j < parts ? s0 + j : a.SC) * per + prow;
        l[j] = a.ws_lse[at];
        ex[j] = a.ws_exp[at];
        oh[j] = *reinterpret_cast<const u32x4*>(a.ws_o + at * D + d0);
      }
    }
    float mb = l[0];
#pragma unroll
    for (int j = 1; j < SB; ++j) mb = fmaxf(mb, l[j]);
    const float mn = fmaxf(m, mb);
    const float sc = m == -INFINITY ? 0.f : exp2f(m - mn);
    tot *= sc;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= sc;
    m = mn;
#pragma unroll
    for (int j = 0; j < SB; ++j) {
      if (l[j] == -INFINITY) continue;
      const float wgt = exp2f(l[j] - m);  // NaN stays NaN
      const float wo = __builtin_ldexpf(wgt, (int)ex[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x2 x = h2_to_f2(oh[j][e]);
        acc[2 * e] += x[0] * wo;
        acc[2 * e + 1] += x[1] * wo;
      }
      tot += wgt;
    }
  }
  const float inv = tot > 0.f ? 1.f / tot : (tot == 0.f ? 0.f : tot);
  const int r = (int)(prow % a.rows);
  const int kvh = (int)(prow / a.rows % a.Hkv);
  const int64_t b = prow / a.rows / a.Hkv;
  const int64_t token = b * a.KL + r % a.KL;
  const int head = kvh * a.G + r / a.KL;
  u16x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = f2bf_bits(acc[e] * inv);
  *reinterpret_cast<u16x8*>(a.out + token * a.o_st + (int64_t)head * a.o_sh + d0) = v;
  if (a.lse && d0 == 0) a.lse[token * a.H + head] = tot > 0.f ? (m + log2f(tot)) * LN2 : (tot == 0.f ? -INFINITY : tot);
}

// ----------------------------------------------------------------------------------------------------- weights

// Attention weight per cached token. A workgroup takes 256 (or 128) keys of one (request, KV head), 64 a wave: the wave's keys
// are widened once through LDS into MFMA operands (64 registers) and stay there, while the KV head's query rows stream by in
// units of 32 through a double buffer in LDS that the waves share. A lane then holds, for its query row, the 32 keys of its
// half; p = exp2(s scale - lse) is added up per key over the units in registers, and once at the end over the 32 lanes.
// Every sum has one owner and one order: no atomics. Bound by issue, mostly the exponentials' (one per product of 256 flops):
// 16 requests of 1187 .. 8033 tokens, 40 heads, 8 x 16 queries: 125 us, 0.76 PFLOP/s; one request of 4096, 32 heads: 10.9 us,
// look-ups and latency. Plain decoding reads the keys and little else, by 1.2 waves per SIMD: the 16 requests 31.5 us (2.5 TB/s),
// one of 4096 tokens 5.9.
//
// KW: the workgroup's 64-key parts. RS: waves per part, each of which takes every RS-th share of the units, their sums joined in
// LDS in wave order. One wave per part where that leaves each CU more than a workgroup; else two, and four on half as many keys
// where that is still one round (one request of 4096 tokens 12.1 us against 14.9 with two, of 5000 20.3 against 15.1; 16 requests
// 183 us with two against 131 with one). QS: units of a wave per stage; one where a KV head has one unit (3 requests of up
// to 12151 tokens, 4 rows: 14.3 us against 16.7).
struct WArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const float* lse;  // [bs K L][H], natural
  const uint8_t* kc;
  int64_t kc_ss, kc_sh;
  const float* ks;
  Pages pages;
  const int64_t* ctx_lens;
  float* w;  // [rows][Hkv][width]
  int64_t w_sr, w_sh;
  int w_rows, width;
  int bs, H, Hkv, G, KL, rows;
  float scale_log2, decay;
  int32_t* err_flag;
};

template <int KW, int RS, int QS>
__global__ __launch_bounds__(KW * RS * 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void kv8_weights_kernel(WArgs a) {
  static_assert((KW == 2 || KW == 4) && QS <= 2, "whole loads per stage");
  constexpr int NWV = KW * RS, WKEYS = KW * TK;
  // widened keys (32 of each wave at a time) and two stages of query rows, each with a place of its own: the first stage is
  // on its way while the keys are looked up
  constexpr int KLDS = NWV * SK * KROW, STAGE = RS * QS * UROWS * D * 2;
  static_assert(KLDS % 1024 == 0, "the stages are aligned");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[KLDS + 2 * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, l32 = lane & 31;
  const int wk = w % KW, wr = w / KW;  // the wave's 64 keys, and its share of the units
  // KV heads fastest, key ranges slowest: with eight heads each XCD (workgroup id modulo 8) has one, whose query rows stay in
  // its L2, and ranges that only the longest requests reach are spread over all of them
  const int kvh = blockIdx.x % a.Hkv, b = blockIdx.x / a.Hkv % a.bs, range = blockIdx.x / a.Hkv / a.bs;
  const int32_t* trow = kv8::table_row(a.pages, b);
  const int64_t wrow = a.pages.req_idx ? a.pages.req_idx[b] : b;
  const int shift = a.pages.page_shift, pmask = (1 << shift) - 1;
  int ctx = trow && a.pages.num_pages > 0 && wrow < a.w_rows ? kv8::bounded_len(a.pages, a.ctx_lens[b]) : 0;
  if (tid == 0 && range == 0 && kvh == 0 && (ctx > a.width || ctx != a.ctx_lens[b] || !trow || wrow >= a.w_rows))
    kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
  ctx = __builtin_amdgcn_readfirstlane(min(ctx, a.width));
  const int lo = range * WKEYS;
  if (lo >= ctx) return;

  // Query rows come by direct-to-LDS loads, a stage of RS QS units at a time, double buffered. A load moves four whole rows:
  // load i of wave w takes rows 4 NWV i + 4 w + lane / 16 of the stage, and chunk c of row r lands at c ^ (r % 16) of the row
  // (the lane at position p asks for chunk p ^ (r % 16)). Rows past the last repeat the first.
  const int stages = (a.rows + RS * QS * UROWS - 1) / (RS * QS * UROWS);
  constexpr int QSTEP = 4 * NWV;  // rows from one of a wave's loads to its next
  const int qr = 4 * w + (lane >> 4);
  const int dg = QSTEP / a.KL, dq = QSTEP % a.KL;
  const uint32_t q_st = (uint32_t)a.q_st, q_sh = (uint32_t)a.q_sh;  // (a request's queries span less than 2^30 elements)
  const uint32_t q_step = dg * q_sh + dq * q_st, q_wrap = q_sh - a.KL * q_st;
  const uint16_t* const q_b = a.q + (int64_t)b * a.KL * a.q_st + (int64_t)kvh * a.G * a.q_sh;
  int rr = qr, rq = qr % a.KL;  // the next load's row, and its query
  const uint32_t q_first = ((lane & 15) ^ (qr & 15)) * 8;
  uint32_t qo = q_first + (uint32_t)(qr / a.KL) * q_sh + (uint32_t)rq * q_st;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)(lds + KLDS);
  auto load_q = [&](int st) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < RS * QS * UROWS / QSTEP; ++i) {
      dma16(q_b + (rr < a.rows ? qo : q_first), lds0 + (uint32_t)((st & 1) * STAGE + (QSTEP * i + 4 * w) * (D * 2)));
      rr += QSTEP;
      rq += dq;
      const bool wrap = rq >= a.KL;
      rq -= wrap ? a.KL : 0;
      qo += q_step + (wrap ? q_wrap : 0);
    }
  };
  // lse of row l32 of the wave's units of the next stage; padding rows get +inf (probability 0), and so do rows whose lse is
  // -inf (they saw no key)
  constexpr int LSTEP = RS * QS * UROWS;
  const int lg = LSTEP / a.KL, lq = LSTEP % a.KL;
  const uint32_t l_step = lg + lq * a.H, l_wrap = 1 - a.KL * a.H;
  const float* const lse_b = a.lse + (int64_t)b * a.KL * a.H + kvh * a.G;
  int lr[QS], lrq[QS];
  uint32_t lof[QS];
#pragma unroll
  for (int x = 0; x < QS; ++x) {
    lr[x] = (wr * QS + x) * UROWS + l32;
    lrq[x] = lr[x] % a.KL;
    lof[x] = (uint32_t)lrq[x] * a.H + lr[x] / a.KL;
  }
  float l_nxt[QS];
  auto load_lse = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < QS; ++x) {
      l_nxt[x] = INFINITY;
      if (lr[x] < a.rows) l_nxt[x] = lse_b[lof[x]];
      lr[x] += LSTEP;
      lrq[x] += lq;
      const bool wrap = lrq[x] >= a.KL;
      lrq[x] -= wrap ? a.KL : 0;
      lof[x] += l_step + (wrap ? l_wrap : 0);
    }
  };

  load_q(0);
  load_lse();
  const int base = l32 * 128 + ((((half ^ l32) & 1) | (l32 & 14)) << 3);
  bf16x8 kf[2][D / 16];
  const uint8_t* const kc_h = a.kc + (int64_t)kvh * a.kc_sh + (lane & 7) * 16;
  int bad = 0;
  auto load_key = [&](int key, u32x4& c, float& s) __attribute__((always_inline)) {
    int e = trow[min(key, ctx - 1) >> shift];
    if ((uint32_t)e >= (uint32_t)a.pages.num_pages) {
      bad = 1;
      e = 0;
    }
    c = *reinterpret_cast<const u32x4*>(slot_row(kc_h, (e << shift) + (min(key, ctx - 1) & pmask), (uint32_t)a.kc_ss));
    s = a.ks[e * a.Hkv + kvh];
  };
  auto read_keys = [&](int ks, const uint8_t* tile) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) kf[ks][d] = as_bf16x8(*reinterpret_cast<const u16x8*>(tile + k_operand(lane) + 32 * d));
  };
  {
    // 64 rows, a lane 16 codes (lane % 8) of rows lane / 8 + 8 i, 32 rows through the wave's part of LDS at a time
    uint8_t* tile = lds + w * (SK * KROW);
    u32x4 c[8];
    float sc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) load_key(lo + wk * TK + (lane >> 3) + 8 * i, c[i], sc[i]);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int i = 0; i < 4; ++i) put_k_codes(tile + ((lane >> 3) + 8 * i) * KROW, lane & 7, c[4 * ks + i], sc[4 * ks + i]);
      asm volatile("" ::: "memory");  // (a wave's LDS operations complete in order)
      read_keys(ks, tile);
      asm volatile("" ::: "memory");
    }
  }
  if (bad) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
  float acc[32];
#pragma unroll
  for (int x = 0; x < 32; ++x) acc[x] = 0.f;
  float l_st[QS];  // of the stage that is read, base 2
  // Stage st has landed in every wave and the one before is read: its buffer takes the one behind
  auto next_stage = [&](int st) __attribute__((always_inline)) {
    wait_vmcnt0();
    lds_barrier();
#pragma unroll
    for (int x = 0; x < QS; ++x) {
      asm volatile("" : "+v"(l_nxt[x]));  // (opaque: formed where it was asked for instead, l_st would wait for it there)
      l_st[x] = l_nxt[x] == -INFINITY ? INFINITY : l_nxt[x] * 1.4426950408889634f;
    }
    if (st + 1 < stages) {
      load_q(st + 1);
      load_lse();
    }
  };
  // S^T of the wave's unit n (n / QS: its stage), and meanwhile the probabilities of the one before: a wave's matrix and vector
  // instructions overlap where they alternate (16 of v_mfma_f32_32x32x16, then 128 FMAs: 971 cycles, 776 with three waves per
  // SIMD; each followed by 8 of them: 680 and 624). Slots 2 c and 2 c + 1 are the two 32-key subtiles against d chunk c, read FD
  // chunks ahead; a scheduling barrier closes each slot. Units past the last are padding rows' (probability 0).
  constexpr int FD = 2;
  auto unit_step = [&](int n, bool first, bool more, float l, f32x16 (&cur)[2], f32x16 (&nxt)[2])
                       __attribute__((always_inline)) {
    // rows that add nothing (lse -inf, padding): scores of infinities and NaN in their q must not make them NaN
    if (!first && __builtin_amdgcn_ballot_w64(l == INFINITY) != 0) {
#pragma unroll
      for (int x = 0; x < 32; ++x) cur[x >> 4][x & 15] = l == INFINITY ? 0.f : cur[x >> 4][x & 15];
    }
    const uint16_t* qb =
        reinterpret_cast<const uint16_t*>(lds + KLDS + (n / QS & 1) * STAGE) + (wr * QS + n % QS) * (UROWS * D);
    bf16x8 qf[D / 16];
    if (more) {
#pragma unroll
      for (int c = 0; c < FD; ++c) qf[c] = as_bf16x8(*reinterpret_cast<const u16x8*>(qb + (base ^ (c << 4))));
      nxt[0] = nxt[1] = (f32x16){};
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int sl = 0; sl < 16; ++sl) {
      const int c = sl >> 1, ks = sl & 1;
      if (more) {
        if (ks == 0 && c + FD < D / 16)
          qf[c + FD] = as_bf16x8(*reinterpret_cast<const u16x8*>(qb + (base ^ ((c + FD) << 4))));
        nxt[ks] = mfma32(kf[ks][c], qf[c], nxt[ks]);
      }
      if (!first) {
        asm volatile("" : "+v"(l));  // this and the one behind the sums keep the exponentials in this slot
        acc[2 * sl] += __builtin_amdgcn_exp2f(__builtin_fmaf(cur[c >> 2][2 * (sl & 7)], a.scale_log2, -l));
        acc[2 * sl + 1] += __builtin_amdgcn_exp2f(__builtin_fmaf(cur[c >> 2][2 * (sl & 7) + 1], a.scale_log2, -l));
        asm volatile("" : "+v"(acc[2 * sl]), "+v"(acc[2 * sl + 1]));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  f32x16 s_a[2], s_b[2];
  next_stage(0);
  unit_step(0, true, true, 0.f, s_b, s_a);
  const int n_units = stages * QS;
  float l_cur = l_st[0];
  // unit n - 1's probabilities are formed while unit n's products run
  auto advance = [&](int n, f32x16 (&cur)[2], f32x16 (&nxt)[2]) __attribute__((always_inline)) {
    const float l = l_cur;
    if (QS == 1 || n % QS == 0) next_stage(n / QS);
    l_cur = l_st[n % QS];
    unit_step(n, false, true, l, cur, nxt);
  };
  int n = 1;
  for (; n + 1 < n_units; n += 2) {
    advance(n, s_a, s_b);
    advance(n + 1, s_b, s_a);
  }
  if (n < n_units) {
    advance(n, s_a, s_b);
    unit_step(0, false, false, l_cur, s_b, s_a);
  } else {
    unit_step(0, false, false, l_cur, s_a, s_b);
  }
  lds_barrier();
  // Sum over the 32 lanes of a half, halving the registers as the lanes are joined: in step m a lane keeps the half of its
  // registers that its bit m names and gives the other half to lane ^ m. Register x ends in the lane whose bits 4 .. 0
  // (m = 16, 8, 4, 2, 1) spell x.
  auto join = [&](auto step) __attribute__((always_inline)) {
    constexpr int n = decltype(step)::value;
    const bool up = (l32 & n) != 0;
#pragma unroll
    for (int x = 0; x < n; ++x) {
      const float give = up ? acc[x] : acc[x + n], keep = up ? acc[x + n] : acc[x];
      acc[x] = keep + __shfl_xor(give, n);
    }
  };
  join(std::integral_constant<int, 16>{});
  join(std::integral_constant<int, 8>{});
  join(std::integral_constant<int, 4>{});
  join(std::integral_constant<int, 2>{});
  join(std::integral_constant<int, 1>{});
  const int x = l32 & 15, in_tile = (l32 >> 4) * 32 + 8 * (x >> 2) + 4 * half + (x & 3);
  float sum = acc[0];
  if constexpr (RS > 1) {
    float* const part = reinterpret_cast<float*>(lds) + wk * TK + in_tile;
    if (wr > 0) part[(wr - 1) * WKEYS] = sum;
    lds_barrier();
    if (wr > 0) return;
#pragma unroll
    for (int y = 0; y < RS - 1; ++y) sum += part[y * WKEYS];
  }
  const int key = lo + wk * TK + in_tile;
  if (key < ctx) {
    float* p = a.w + wrow * a.w_sr + (int64_t)kvh * a.w_sh + key;
    *p = a.decay != 0.f ? a.decay * *p + sum : sum;  // (a decay of 0 does not read the old sum)
  }
}

}  // namespace

static int64_t partials(int with_block, int num_ctx_splits, int rows) {
  if (num_ctx_splits <= 1) return 1;
  return num_ctx_splits + (with_block && rows > UROWS ? 1 : 0);
}

extern "C" int64_t mfd_kv8_attn_workspace_bytes(int bs, int num_modes, int block_size, int H, int Hkv, int with_block,
                                                int num_ctx_splits) {
  if (num_ctx_splits <= 1 || bs < 1 || num_modes < 1 || block_size < 1 || H < 1 || Hkv < 1) return 0;
  const int64_t rows = (int64_t)bs * H * num_modes * block_size;
  return partials(with_block, num_ctx_splits, (int)(H / Hkv * (int64_t)num_modes * block_size)) * rows * (D * 2 + 4 + 4) +
         (int64_t)bs * 4;
}

static int check_attn(const char* who, int bs, int num_modes, int block_size, int H, int Hkv, float scale,
                      const void* q, int64_t q_st, int64_t q_sh) {
  if (bs < 0 || bs > 65535 || num_modes < 1 || block_size < 1 || H < 1 || Hkv < 1 || H % Hkv != 0)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad sizes bs=%d K=%d L=%d H=%d Hkv=%d", who, bs, num_modes, block_size,
                         H, Hkv);
  if ((int64_t)num_modes * block_size > (1 << 16) || (int64_t)H / Hkv * num_modes * block_size > (1 << 24))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: num_modes * block_size = %lld above 65536 (or 2^24 rows per KV head)",
                         who, (long long)num_modes * block_size);
  if (!(scale > 0.f)) return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: scale must be positive", who);
  if ((reinterpret_cast<uintptr_t>(q) & 15) || ((q_st | q_sh) & 7))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: q needs 16-byte aligned rows", who);
  return MFD_OK;
}

extern "C" int mfd_kv8_attn(const uint16_t* q, int64_t q_st, int64_t q_sh, const uint16_t* k_new, const uint16_t* v_new,
                            int64_t kn_st, int64_t kn_sh, int64_t vn_st, int64_t vn_sh, const uint8_t* k_cache,
                            const uint8_t* v_cache, int64_t kc_ss, int64_t kc_sh, int64_t vc_ss, int64_t vc_sh,
                            const float* k_scale, const float* v_scale, int num_pages, const int32_t* page_table,
                            int64_t table_stride, int table_rows, int table_width, int page_size,
                            const int64_t* req_idx, const int64_t* ctx_lens, int bs, int num_modes, int block_size,
                            int H, int Hkv, int D_, float scale, int causal_in_block, int num_ctx_splits,
                            int split_keys, uint16_t* out, int64_t o_st, int64_t o_sh, float* lse, void* workspace,
                            int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  const char* who = "mfd_kv8_attn";
  int rc = kv8::check_cache(who, k_cache, v_cache, kc_ss, kc_sh, vc_ss, vc_sh, page_size, Hkv, D_, page_table, table_rows,
                            table_width, num_pages);
  if (rc == MFD_OK) rc = check_attn(who, bs, num_modes, block_size, H, Hkv, scale, q, q_st, q_sh);
  if (rc != MFD_OK) return rc;
  if (num_ctx_splits < 1 || num_ctx_splits > 1024 ||
      (num_ctx_splits > 1 && (split_keys < 0 || split_keys % TK != 0 || (split_keys == 0 && bs > 64))))
    return mfd_set_error(MFD_ERR_INVALID_ARG,
                         "%s: num_ctx_splits %d (1..1024) of split_keys %d (a multiple of %d, 0 for up to 64 requests)", who,
                         num_ctx_splits, split_keys, TK);
  if (bs == 0) return MFD_OK;
  if (!q || !out || !ctx_lens || (!k_new) != (!v_new) ||
      (num_pages > 0 && table_rows > 0 && table_width > 0 && (!k_cache || !v_cache || !k_scale || !v_scale)))
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null tensor pointer", who);
  if (((reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new) | reinterpret_cast<uintptr_t>(out)) & 15) ||
      ((kn_st | kn_sh | vn_st | vn_sh | o_st | o_sh) & 7))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: tensors need 16-byte aligned rows (strides in multiples of 8)", who);
  const int64_t need = mfd_kv8_attn_workspace_bytes(bs, num_modes, block_size, H, Hkv, k_new != nullptr, num_ctx_splits);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: 16-byte aligned workspace of %lld bytes needed", who, (long long)need);
  Args a{};
  a.q = q; a.q_st = q_st; a.q_sh = q_sh;
  a.kn = k_new; a.vn = v_new; a.kn_st = kn_st; a.kn_sh = kn_sh; a.vn_st = vn_st; a.vn_sh = vn_sh;
  a.kc = k_cache; a.vc = v_cache; a.kc_ss = kc_ss; a.kc_sh = kc_sh; a.vc_ss = vc_ss; a.vc_sh = vc_sh;
  a.ks = k_scale; a.vs = v_scale;
  a.pages = {page_table, table_stride, table_rows, table_width, req_idx, num_pages, __builtin_ctz((unsigned)page_size)};
  a.ctx_lens = ctx_lens;
  a.out = out; a.o_st = o_st; a.o_sh = o_sh; a.lse = lse;
  a.bs = bs; a.K = num_modes; a.L = block_size; a.H = H; a.Hkv = Hkv; a.G = H / Hkv;
  a.KL = num_modes * block_size;
  a.rows = a.G * a.KL;
  a.SC = num_ctx_splits; a.split_keys = num_ctx_splits > 1 ? split_keys : 0;
  a.S = (int)partials(k_new != nullptr, num_ctx_splits, a.rows);
  a.causal = causal_in_block ? 1 : 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.err_flag = err_flag;
  const int64_t prows = (int64_t)bs * H * a.KL;
  a.ws_o = static_cast<uint16_t*>(workspace);
  a.ws_lse = workspace ? reinterpret_cast<float*>(a.ws_o + a.S * prows * D) : nullptr;
  a.ws_exp = workspace ? a.ws_lse + a.S * prows : nullptr;
  a.ws_n = workspace ? reinterpret_cast<int32_t*>(a.ws_exp + a.S * prows) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int units = (a.rows + UROWS - 1) / UROWS;
  // Eight waves share a tile's widening where they all have a unit, and in a batch that half fills the chip even where some
  // idle (16 requests of 4000 tokens: 12 units 134 us against 169 with four, 20 units 245 against 268; 4 requests, 12 units 65
  // against 60). kv8_cache.py counts by the same rule.
  const int64_t by8 = (int64_t)bs * Hkv * ((units + 7) / 8);
  const int NW = units % 8 == 0 || (units > 4 && 2 * by8 >= mfd_num_cus()) ? 8 : 4;
  a.ngroups = (units + NW - 1) / NW;
  if (num_ctx_splits > 1 && split_keys == 0) {
    // whole rounds of the workgroups that run together, as few as leave a request two splits on average
    const int64_t slots = (int64_t)mfd_num_cus() * (NW == 8 && units > 1 ? 1 : 2), per = (int64_t)Hkv * a.ngroups;
    const int64_t need = (int64_t)bs * (2 + a.S - a.SC);
    a.pairs = (int)std::max(need, (need * per + slots - 1) / slots * slots / per);
    a.min_tiles = units == 1 ? 2 : 3;  // (shorter splits cost more in partials than they save)
  }
  const int64_t programs = (a.pairs ? a.pairs : (int64_t)bs * a.S) * Hkv;
  const int64_t grid = units == 1 ? programs : (programs + 7) / 8 * 8 * a.ngroups;
  if (grid > 0x7fffffff || (prows + 15) / 16 > 0x7fffffff)
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  // stream kernel: eight waves where a CU has one workgroup (1187 tokens 12.8 us against 13.7, 4 requests of 2000 and two
  // workgroups per CU 21.8 against 17.9)
  if (units == 1 && grid <= mfd_num_cus())
    hipLaunchKernelGGL(kv8_attn_stream_kernel<8>, dim3((unsigned)grid), dim3(512), 0, st, a);
  else if (units == 1)
    hipLaunchKernelGGL(kv8_attn_stream_kernel<4>, dim3((unsigned)grid), dim3(256), 0, st, a);
  else if (NW == 8 && page_size >= TK)
    hipLaunchKernelGGL((kv8_attn_tile_kernel<8, true>), dim3((unsigned)grid), dim3(512), 0, st, a);
  else if (NW == 8)
    hipLaunchKernelGGL((kv8_attn_tile_kernel<8, false>), dim3((unsigned)grid), dim3(512), 0, st, a);
  else if (page_size >= TK)
    hipLaunchKernelGGL((kv8_attn_tile_kernel<4, true>), dim3((unsigned)grid), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((kv8_attn_tile_kernel<4, false>), dim3((unsigned)grid), dim3(256), 0, st, a);
  MFD_CHECK_LAUNCH();
  if (a.S > 1) {
    hipLaunchKernelGGL(kv8_attn_merge_kernel, dim3((unsigned)((prows + 15) / 16)), dim3(256), 0, st, a);
    MFD_CHECK_LAUNCH();
  }
  return MFD_OK;
}

extern "C" int mfd_kv8_weights(const uint16_t* q, int64_t q_st, int64_t q_sh, const float* lse, const uint8_t* k_cache,
                               int64_t kc_ss, int64_t kc_sh, const float* k_scale, int num_pages,
                               const int32_t* page_table, int64_t table_stride, int table_rows, int table_width,
                               int page_size, const int64_t* req_idx, const int64_t* ctx_lens, int bs, int num_modes,
                               int block_size, int H, int Hkv, int D_, float scale, float decay, float* weights,
                               int64_t w_row_stride, int64_t w_head_stride, int w_rows, int width, int32_t* err_flag,
                               void* stream) {
  const char* who = "mfd_kv8_weights";
  int rc = kv8::check_cache(who, k_cache, k_cache, kc_ss, kc_sh, 0, 0, page_size, Hkv, D_, page_table, table_rows,
                            table_width, num_pages);
  if (rc == MFD_OK) rc = check_attn(who, bs, num_modes, block_size, H, Hkv, scale, q, q_st, q_sh);
  if (rc != MFD_OK) return rc;
  if (q_st < 0 || q_sh < 0 || (int64_t)num_modes * block_size * q_st + (int64_t)H * q_sh >= (1 << 30) ||
      (int64_t)num_modes * block_size * H >= (1 << 30))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: a request's queries must span less than 2^30 elements", who);
  if (w_rows < 0 || width < 0 || !(decay >= 0.f && decay <= 1.f))
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad weights rows=%d width=%d, or decay %g outside [0, 1]", who, w_rows,
                         width, (double)decay);
  if (bs == 0 || width == 0 || num_pages == 0 || table_width == 0 || table_rows == 0) return MFD_OK;
  if (!q || !lse || !k_cache || !k_scale || !weights || !ctx_lens)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null tensor pointer", who);
  WArgs a{};
  a.q = q; a.q_st = q_st; a.q_sh = q_sh; a.lse = lse;
  a.kc = k_cache; a.kc_ss = kc_ss; a.kc_sh = kc_sh; a.ks = k_scale;
  a.pages = {page_table, table_stride, table_rows, table_width, req_idx, num_pages, __builtin_ctz((unsigned)page_size)};
  a.ctx_lens = ctx_lens;
  a.w = weights; a.w_sr = w_row_stride; a.w_sh = w_head_stride; a.w_rows = w_rows; a.width = width;
  a.bs = bs; a.H = H; a.Hkv = Hkv; a.G = H / Hkv; a.KL = num_modes * block_size; a.rows = a.G * a.KL;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.decay = decay;
  a.err_flag = err_flag;
  const int64_t keys = std::min<int64_t>(width, (int64_t)table_width * page_size);
  auto grid_of = [&](int range) { return (keys + range - 1) / range * Hkv * bs; };
  const int64_t grid = grid_of(4 * TK);
  if (grid > 0x3fffffff) return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int cus = mfd_num_cus();
  if (a.rows <= UROWS)
    hipLaunchKernelGGL((kv8_weights_kernel<4, 1, 1>), dim3((unsigned)grid), dim3(256), 0, st, a);
  else if (grid > cus)
    hipLaunchKernelGGL((kv8_weights_kernel<4, 1, 2>), dim3((unsigned)grid), dim3(256), 0, st, a);
  else if (grid_of(2 * TK) > cus)
    hipLaunchKernelGGL((kv8_weights_kernel<4, 2, 2>), dim3((unsigned)grid), dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((kv8_weights_kernel<2, 4, 1>), dim3((unsigned)grid_of(2 * TK)), dim3(512), 0, st, a);
  MFD_CHECK_LAUNCH();
  return MFD_OK;
}
