// The 8-bit draft KV cache's own upkeep on gfx950: tokens stored into it, the tokens to keep chosen by the attention
// weight they received, and the kept ones moved to fresh pages. (Its attention is kv8_attn.hip.)
//
// Store. A page's scale s is the smallest power of two with amax / s <= 448 over what the page has held since its first
// token, and a code is e4m3(x / s): nearest even, half a step of three mantissa bits (2^-4 of the value) at most. One workgroup
// takes one (page, KV head) of K or of V: it holds the page's new rows in registers while the largest magnitude is found (one
// pass over the input), rounds the page's older rows again only if the scale grew (a shift of the exponent: exact except where
// a code becomes subnormal), and never touches the rows behind the new ones. Prompts (16476 tokens of four requests, 8 heads)
// are bound by memory: 22 us, 4.6 TB/s of the 4.9 that a large copy reaches. The tokens of a round (16 requests, 90 tokens)
// take 5 us, a launch and one chain of dependent loads, and their eager call 12.
//
// Selection. score[t] = the sum over KV heads of weights[h][t], formed in fp64 and rounded once to fp32, so that the order of
// the sum cannot decide which token stays. Scores become 32-bit keys whose unsigned order is the scores' (always-kept tokens at
// the top, NaN at the bottom); one workgroup per request finds the budget-th largest by three histogram passes over 11, 11 and
// 10 bits and writes the kept indices ascending by one prefix sum. Ties at the border go to the lowest index. 2048 of 8192
// tokens, 8 heads: 12.8 us, of which 4 are the sums' way into one CU, 1.1 each pass's chain of counts, prefix sum and barriers,
// 2 the indices; 32 requests at once the same. Rows wider than 16384 tokens take a kernel for the keys and one that reads them from
// memory, whatever the lengths: 2000 tokens in rows of 32768 17.6 us in a graph, in rows of 8192 17.2; 32768 tokens 3 + 23.
//
// Compaction. One workgroup per (destination page, KV head) of K or of V gathers its kept rows, finds their largest magnitude,
// and writes them with a scale of their own; the same launch moves the running sums (a workgroup per request and head, in
// place) and clears those of the freed tail. 32 requests to 1024 tokens each 36.3 us, 3.7 TB/s of gathered reads and writes (as
// much with the kept tokens side by side; four heads to a workgroup, with the look-ups made once: no gain). Vector instructions
// take 63 % of the cycles, two decodes, the maximum and an encode for each code, with 5.6 waves per SIMD under way. One request
// to 2048: 6.0 us, launch and latency.
#include <algorithm>

#include "kv8_common.h"

namespace {

using kv8::D;
using kv8::Pages;
using kv8::u32x4;

constexpr int NT = 256;          // threads of a store / compaction workgroup: 32 rows of 8 x 16 elements at a time
constexpr int ROWS = NT / 8;

// Largest of the workgroup's values, in every thread (one barrier).
__device__ __forceinline__ float group_max(float v, float* buf) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(buf[0], buf[1]), fmaxf(buf[2], buf[3]));
}

struct StoreArgs {
  const uint16_t* x[2];  // new keys, new values (bf16)
  int64_t x_st[2], x_sh[2];
  uint8_t* cache[2];
  int64_t c_ss[2], c_sh[2];
  float* scale[2];
  Pages pages;
  const int64_t* start_lens;
  const int32_t* cu_tokens;
  int N, Hkv, max_pages;
  int32_t* err_flag;
};

template <int PASSES>
__global__ __launch_bounds__(NT) void kv8_store_kernel(StoreArgs a) {
  __shared__ float buf[4];
  const int b = blockIdx.y, z = blockIdx.z;
  const int h = blockIdx.x % a.Hkv, pi = blockIdx.x / a.Hkv;
  const int shift = a.pages.page_shift, P = 1 << shift;
  const int n0 = a.cu_tokens[b], n1 = a.cu_tokens[b + 1];
  const int c0 = max(0, min(n0, a.N)), c1 = max(c0, min(n1, a.N));
  const int64_t start = max((int64_t)-1, min(a.start_lens[b], (int64_t)1 << 40));  // (beyond either: no table reaches there)
  const int64_t end = start + (c1 - c0);
  const int32_t* row = kv8::table_row(a.pages, b);
  if (blockIdx.x == 0 && z == 0 && threadIdx.x == 0 && (n0 < 0 || n1 < n0 || n1 > a.N || start < 0 || !row))
    kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
  if (c1 == c0) return;
  const int64_t p = (start >> shift) + pi;
  const int64_t p0 = p << shift;
  if (p0 >= end) return;
  // tokens behind the last page of the grid (more of them than the call said) are not stored either
  const bool cut = pi == a.max_pages - 1 && p0 + P < end;
  int page = -1;
  if (row && start >= 0 && p < a.pages.table_width) page = row[p];
  if (cut || page < 0 || page >= a.pages.num_pages) {
    if (threadIdx.x == 0) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
    if (page < 0 || page >= a.pages.num_pages) return;
  }
  const int first = (int)(max(start, p0) - p0), last = (int)(min(end, p0 + P) - p0);  // new rows of the page
  const int r0 = threadIdx.x >> 3, part = threadIdx.x & 7;

  const uint16_t* x = a.x[z] + (c0 + (p0 - start)) * a.x_st[z] + (int64_t)h * a.x_sh[z] + part * 16;
  u16x8 in[PASSES][2];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + ROWS * i;
    in[i][0] = in[i][1] = (u16x8){};
    if (r >= first && r < last) {
      const u16x8* xp = reinterpret_cast<const u16x8*>(x + r * a.x_st[z]);
      in[i][0] = xp[0];
      in[i][1] = xp[1];
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) amax = fmaxf(amax, kv8::finite_abs(bf2f(in[i][e >> 3][e & 7])));
  float* sp = a.scale[z] + (int64_t)page * a.Hkv + h;
  const float old = first > 0 ? *sp : 0.f;  // a page begun anew forgets its scale
  amax = group_max(amax, buf);              // every thread has read the old scale
  const float s = fmaxf(old, kv8::page_scale(amax));
  const float inv = kv8::inverse(s);
  if (threadIdx.x == 0) *sp = s;
  uint8_t* c = a.cache[z] + ((int64_t)page << shift) * a.c_ss[z] + (int64_t)h * a.c_sh[z] + part * 16;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + ROWS * i;
    u32x4* cp = reinterpret_cast<u32x4*>(c + r * a.c_ss[z]);
    if (r >= first && r < last) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = bf2f(in[i][e >> 1][4 * (e & 1) + j]) * inv;
        w[e] = kv8::encode4(f[0], f[1], f[2], f[3]);
      }
      *cp = w;
    } else if (r < first && s != old) {  // an older row of a page whose scale grew
      const u32x4 v = *cp;
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
        kv8::decode4(v[e], old * inv, f);
        w[e] = kv8::encode4(f[0], f[1], f[2], f[3]);
      }
      *cp = w;
    }
  }
}

// ------------------------------------------------------------------------------------------------- selection

struct SelectArgs {
  const float* w;  // [rows][Hkv][width]
  int64_t w_sr, w_sh;
  int w_rows, width, Hkv;
  const int64_t* req_idx;
  const int64_t* ctx_lens;
  int budget, sink, recent;
  int32_t* keep;  // [bs][budget]
  int64_t* new_lens;
  uint32_t* keys;  // [bs][key_stride]
  int64_t key_stride;
  int32_t* err_flag;
};

constexpr int ST = 1024;      // threads of a selection workgroup
constexpr int REG_KEYS = 16;  // keys of a thread that stay in registers, at most
constexpr uint32_t ALWAYS = 0xFFFFFFFFu;

__device__ __forceinline__ int select_len(const SelectArgs& a, int b) {
  const int64_t row = a.req_idx ? a.req_idx[b] : b;
  if (row < 0 || row >= a.w_rows) return 0;
  return (int)max((int64_t)0, min(a.ctx_lens[b], (int64_t)a.width));
}

// Key of token t of a request's row w: its score's, or the top one
__device__ __forceinline__ uint32_t key_of(const SelectArgs& a, const float* w, int t, int len) {
  double sum = 0.;
  int h = 0;
  for (; h + 8 <= a.Hkv; h += 8) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = w[(h + j) * a.w_sh + t];
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += (double)x[j];
  }
  for (; h < a.Hkv; ++h) sum += (double)w[h * a.w_sh + t];
  const float score = (float)sum + 0.f;  // -0 as +0
  const uint32_t key = score == score ? float_order_key(score) : 0u;
  return t < a.sink || t >= len - a.recent ? ALWAYS : key;
}
__device__ __forceinline__ const float* weight_row(const SelectArgs& a, int b) {
  return a.w + (a.req_idx ? a.req_idx[b] : b) * a.w_sr;
}

__global__ __launch_bounds__(256) void evict_score_kernel(SelectArgs a) {
  const int b = blockIdx.y;
  const int len = select_len(a, b);
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= len || len <= a.budget) return;  // (a request within the budget keeps everything)
  a.keys[b * a.key_stride + t] = key_of(a, weight_row(a, b), t, len);
}

// Exclusive prefix sum of v over the workgroup's ST threads; buf: ST / 64 words, other ones than the scan before took. One
// barrier.
__device__ __forceinline__ int group_scan(int v, int* buf) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int s = kv8::wave_scan(v);
  if (lane == 63) buf[w] = s;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int j = 0; j < ST / 64; ++j) before += j < w ? buf[j] : 0;
  return before + s - v;
}

// NK > 0: requests of at most NK ST tokens, whose keys are formed here and stay in registers (key i of a thread: token i ST +
// thread): one launch, and one read of the sums. 0: longer ones, whose keys evict_score_kernel left in the workspace.
template <int NK>
__global__ __launch_bounds__(ST) void evict_select_kernel(SelectArgs a) {
  constexpr int NW = ST / 64;
  // each bin COPIES times, one for every lane modulo COPIES: a wave's keys share few bins (the first digit is little more than
  // the exponent), and adds to one word go one after the other. The copies lie in other banks each (STRIDE), and neighbouring
  // bins side by side: with a bin as eight words in a row, choosing 2048 of 8192 tokens took 1.2 us more.
  constexpr int COPIES = 8, STRIDE = 2048 + 8;
  __shared__ __attribute__((aligned(16))) int hist[STRIDE * COPIES];
  __shared__ __attribute__((aligned(16))) int buf[2][NW];  // (of one scan and the next)
  __shared__ uint32_t found[2];  // digit, and how many of its bin are still wanted
  __shared__ int counts[NK > 0 ? 2 * NK * NW : 1];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int len = select_len(a, b);
  const int n = min(len, a.budget);
  int32_t* keep = a.keep + (int64_t)b * a.budget;
  if (tid == 0) {
    a.new_lens[b] = n;
    const int64_t row = a.req_idx ? a.req_idx[b] : b;
    if (row < 0 || row >= a.w_rows || a.ctx_lens[b] < 0 || a.ctx_lens[b] > a.width)
      kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
  }
  for (int i = n + tid; i < a.budget; i += ST) keep[i] = -1;
  if (len <= a.budget) {
    for (int i = tid; i < n; i += ST) keep[i] = i;
    return;
  }
  for (int i = 4 * tid; i < STRIDE * COPIES; i += 4 * ST) *reinterpret_cast<u32x4*>(hist + i) = (u32x4){};
  uint32_t key[NK > 0 ? NK : 1];
  if constexpr (NK > 0) {
    const float* w = weight_row(a, b);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int t = i * ST + tid;
      key[i] = t < len ? key_of(a, w, t, len) : 0u;
    }
  }
  const uint32_t* keys = a.keys + b * a.key_stride;
  // the n-th largest key, digit by digit: `prefix` holds the digits found, `want` how many keys with them are kept
  uint32_t prefix = 0, mask = 0;
  int want = n;
  __syncthreads();  // the bins are clear
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    auto bin_of = [&](uint32_t digit) { return &hist[(tid & (COPIES - 1)) * STRIDE + (digit & (bins - 1))]; };
    auto count = [&](bool in, uint32_t k) {
      if (in) atomicAdd(bin_of(k >> shift), 1);
    };
    if constexpr (NK > 0) {
#pragma unroll
      for (int i = 0; i < NK; ++i)
        count(i * ST + tid < len && (key[i] & mask) == prefix, key[i]);
    } else {
      for (int i = 4 * tid; i < len; i += 4 * ST) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);  // rows are padded to whole quads
#pragma unroll
        for (int e = 0; e < 4; ++e)
          count(i + e < len && (k[e] & mask) == prefix, k[e]);
      }
    }
    __syncthreads();
    const int hi = bins - 1 - 2 * tid;  // this thread's bins hi, hi - 1: descending over the threads
    int h0 = 0, h1 = 0;  // their copies added up, and cleared for the next pass
    if (hi >= 1) {
#pragma unroll
      for (int c = 0; c < COPIES; ++c) {
        int2* const h = reinterpret_cast<int2*>(hist + c * STRIDE + hi - 1);
        h0 += h->y;
        h1 += h->x;
        *h = make_int2(0, 0);
      }
    }
    const int before = group_scan(h0 + h1, buf[pass & 1]);
    if (before < want && want <= before + h0) {
      found[0] = hi;
      found[1] = want - before;
    } else if (before + h0 < want && want <= before + h0 + h1) {
      found[0] = hi - 1;
      found[1] = want - before - h0;
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    want = (int)found[1];
  }
  // kept: keys above the border `prefix`, and the first `want` of those equal to it
  if constexpr (NK > 0) {
    // token order is (register, wave, lane): the wave's counts of each register meet in LDS, one prefix sum over them
    const int lane = tid & 63, w = tid >> 6;
    uint64_t above[NK], same[NK];
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const bool in = i * ST + tid < len;
      above[i] = __builtin_amdgcn_ballot_w64(in && key[i] > prefix);
      same[i] = __builtin_amdgcn_ballot_w64(in && key[i] == prefix);
      if (lane == 0) {
        counts[i * NW + w] = __builtin_popcountll(above[i]);
        counts[(NK + i) * NW + w] = __builtin_popcountll(same[i]);
      }
    }
    __syncthreads();
    static_assert(2 * NK * NW <= ST, "a count per thread");
    const int c = tid < 2 * NK * NW ? counts[tid] : 0;
    const int before = group_scan(c, buf[1]);
    if (tid < 2 * NK * NW) counts[tid] = before;
    __syncthreads();
    const int gt_all = counts[NK * NW];  // (what lies before the first of the equal ones)
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const int gt0 = counts[i * NW + w] + __builtin_popcountll(above[i] & lower);
      const int eq0 = counts[(NK + i) * NW + w] - gt_all + __builtin_popcountll(same[i] & lower);
      const bool is_above = above[i] >> lane & 1, is_same = same[i] >> lane & 1;
      if (is_above || (is_same && eq0 < want)) keep[gt0 + min(eq0, want)] = i * ST + tid;
    }
  } else {
    // a thread takes a run of the row
    const int seg = ((len + ST - 1) / ST + 3) & ~3;
    const int lo = tid * seg, hi = min(lo + seg, len);
    int gt = 0, eq = 0;
    for (int i = lo; i < hi; i += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        gt += (i + e < hi && k[e] > prefix) ? 1 : 0;
        eq += (i + e < hi && k[e] == prefix) ? 1 : 0;
      }
    }
    const int gt0 = group_scan(gt, buf[1]);
    int eq0 = group_scan(eq, buf[0]);
    int at = gt0 + min(eq0, want);
    for (int i = lo; i < hi; i += 4) {
      const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (i + e >= hi) break;
        const bool same = k[e] == prefix;
        if (k[e] > prefix || (same && eq0 < want)) keep[at++] = i + e;
        eq0 += same ? 1 : 0;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ compaction

struct CompactArgs {
  const int32_t* keep;  // [bs][budget]
  int budget;
  const int64_t* new_lens;
  const int64_t* ctx_lens;
  uint8_t* cache[2];
  int64_t c_ss[2], c_sh[2];
  float* scale[2];
  Pages src, dst;
  float* w;
  int64_t w_sr, w_sh;
  int w_rows, width;
  int Hkv, dst_pages;
  int32_t* err_flag;
};

// Running sums of one (request, head): entry i <- entry keep[i]. keep ascends, so a chunk's sources lie at or behind
// its targets and behind every earlier chunk's; within a chunk all are read before any is written.
__device__ void move_weights(const CompactArgs& a, int b, int h, int n) {
  const int64_t row = a.dst.req_idx ? a.dst.req_idx[b] : b;
  if (!a.w || row < 0 || row >= a.w_rows) return;
  float* w = a.w + row * a.w_sr + h * a.w_sh;
  const int32_t* keep = a.keep + (int64_t)b * a.budget;
  const int len = (int)max((int64_t)0, min(a.ctx_lens[b], (int64_t)a.width));
  constexpr int U = 8;  // entries of a thread per chunk
  const int m = min(n, a.width);
  for (int i0 = 0; i0 < m; i0 += NT * U) {
    float x[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * NT + threadIdx.x;
      const int t = i < m ? keep[i] : -1;
      x[j] = t >= 0 && t < a.width ? w[t] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * NT + threadIdx.x;
      if (i < m) w[i] = x[j];
    }
    __syncthreads();
  }
  for (int i = m + threadIdx.x; i < len; i += NT) w[i] = 0.f;
}

template <int PASSES>
__global__ __launch_bounds__(NT) void evict_compact_kernel(CompactArgs a) {
  __shared__ float buf[4];
  const int b = blockIdx.y, z = blockIdx.z;
  const int h = blockIdx.x % a.Hkv, p = blockIdx.x / a.Hkv;
  const int shift = a.dst.page_shift;
  const int n = (int)max((int64_t)0, min(a.new_lens[b], (int64_t)a.budget));
  const int32_t *src_row = kv8::table_row(a.src, b), *dst_row = kv8::table_row(a.dst, b);
  const int len = kv8::bounded_len(a.src, a.ctx_lens[b]);
  if (p == a.dst_pages) {
    if (z != 0) return;
    if (h == 0 && threadIdx.x == 0) {  // what this request's workgroups cut, or leave out
      const int64_t row = a.dst.req_idx ? a.dst.req_idx[b] : b;
      if (n != a.new_lens[b] || len != a.ctx_lens[b] || !src_row || !dst_row || (a.w && (row >= a.w_rows || len > a.width)))
        kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
    }
    move_weights(a, b, h, n);
    return;
  }
  const int i0 = p << shift;
  if (i0 >= n) return;
  int page = -1;
  if (src_row && dst_row && p < a.dst.table_width) page = dst_row[p];
  if (page < 0 || page >= a.dst.num_pages) {
    if (threadIdx.x == 0) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
    return;
  }
  const int rows = min(n - i0, 1 << shift);
  const int r0 = threadIdx.x >> 3, part = threadIdx.x & 7;
  const int32_t* keep = a.keep + (int64_t)b * a.budget + i0;
  u32x4 in[PASSES];
  float s_in[PASSES];
  bool bad = false;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + ROWS * i;
    in[i] = (u32x4){};
    s_in[i] = 0.f;  // a row that cannot be read becomes zero
    if (r < rows) {
      const int t = keep[r];
      const int sp = t >= 0 && t < len ? src_row[t >> shift] : -1;
      if (sp >= 0 && sp < a.src.num_pages) {
        const int64_t slot = ((int64_t)sp << shift) + (t & ((1 << shift) - 1));
        in[i] = *reinterpret_cast<const u32x4*>(a.cache[z] + slot * a.c_ss[z] + (int64_t)h * a.c_sh[z] + part * 16);
        s_in[i] = a.scale[z][(int64_t)sp * a.Hkv + h];
      } else {
        bad = true;
      }
    }
  }
  if (bad) kv8::raise(a.err_flag, MFD_DEVERR_BAD_PAGE);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float f[4];
      kv8::decode4(in[i][e], s_in[i], f);
#pragma unroll
      for (int j = 0; j < 4; ++j) amax = fmaxf(amax, kv8::finite_abs(f[j]));
    }
  amax = group_max(amax, buf);
  const float s = kv8::page_scale(amax);
  const float inv = kv8::inverse(s);
  if (threadIdx.x == 0) a.scale[z][(int64_t)page * a.Hkv + h] = s;
  uint8_t* c = a.cache[z] + ((int64_t)page << shift) * a.c_ss[z] + (int64_t)h * a.c_sh[z] + part * 16;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + ROWS * i;
    if (r < rows) {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
        kv8::decode4(in[i][e], s_in[i] * inv, f);
        w[e] = kv8::encode4(f[0], f[1], f[2], f[3]);
      }
      // past the caches (nobody reads it soon: 32 requests to 1024 of up to 8033 tokens, 40.2 us against 44.3)
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(c + r * a.c_ss[z]));
    }
  }
}

}  // namespace

extern "C" int mfd_kv8_store(const uint16_t* k, const uint16_t* v, int64_t kn_st, int64_t kn_sh, int64_t vn_st,
                             int64_t vn_sh, uint8_t* k_cache, uint8_t* v_cache, int64_t kc_ss, int64_t kc_sh,
                             int64_t vc_ss, int64_t vc_sh, float* k_scale, float* v_scale, int num_pages,
                             const int32_t* page_table, int64_t table_stride, int table_rows, int table_width,
                             int page_size, const int64_t* req_idx, const int64_t* start_lens,
                             const int32_t* cu_tokens, int N, int bs, int max_tokens, int Hkv, int D_,
                             int32_t* err_flag, void* stream) {
  const char* who = "mfd_kv8_store";
  const int rc = kv8::check_cache(who, k_cache, v_cache, kc_ss, kc_sh, vc_ss, vc_sh, page_size, Hkv, D_, page_table,
                                  table_rows, table_width, num_pages);
  if (rc != MFD_OK) return rc;
  if (bs < 0 || bs > 65535 || N < 0 || max_tokens < 0)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad sizes bs=%d N=%d max_tokens=%d", who, bs, N, max_tokens);
  if (bs == 0 || N == 0 || max_tokens == 0) return MFD_OK;
  if (!k || !v || !k_cache || !v_cache || !k_scale || !v_scale || !start_lens || !cu_tokens)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null pointer", who);
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) ||
      ((kn_st | kn_sh | vn_st | vn_sh) & 7))
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: new rows need 16-byte alignment (strides in multiples of 8)", who);
  StoreArgs a{};
  a.x[0] = k; a.x[1] = v;
  a.x_st[0] = kn_st; a.x_st[1] = vn_st; a.x_sh[0] = kn_sh; a.x_sh[1] = vn_sh;
  a.cache[0] = k_cache; a.cache[1] = v_cache;
  a.c_ss[0] = kc_ss; a.c_ss[1] = vc_ss; a.c_sh[0] = kc_sh; a.c_sh[1] = vc_sh;
  a.scale[0] = k_scale; a.scale[1] = v_scale;
  a.pages = {page_table, table_stride, table_rows, table_width, req_idx, num_pages, __builtin_ctz((unsigned)page_size)};
  a.start_lens = start_lens; a.cu_tokens = cu_tokens;
  a.N = N; a.Hkv = Hkv; a.err_flag = err_flag;
  a.max_pages = (int)(((int64_t)std::min(max_tokens, N) + page_size - 2) / page_size + 1);  // from any first offset
  if ((int64_t)a.max_pages * Hkv > 0x7fffffff)
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: max_tokens=%d too large", who, max_tokens);
  const dim3 grid((unsigned)(a.max_pages * Hkv), (unsigned)bs, 2);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (page_size <= 32) hipLaunchKernelGGL(kv8_store_kernel<1>, grid, dim3(NT), 0, st, a);
  else if (page_size == 64) hipLaunchKernelGGL(kv8_store_kernel<2>, grid, dim3(NT), 0, st, a);
  else if (page_size == 128) hipLaunchKernelGGL(kv8_store_kernel<4>, grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL(kv8_store_kernel<8>, grid, dim3(NT), 0, st, a);
  MFD_CHECK_LAUNCH();
  return MFD_OK;
}

static int64_t key_stride_of(int width) { return ((int64_t)width + 3) & ~(int64_t)3; }

extern "C" int64_t mfd_evict_select_workspace_bytes(int bs, int width) {
  return bs > 0 && width > REG_KEYS * ST ? (int64_t)bs * key_stride_of(width) * 4 : 0;
}

extern "C" int mfd_evict_select(const float* weights, int64_t w_row_stride, int64_t w_head_stride, int w_rows,
                                int width, int Hkv, const int64_t* req_idx, const int64_t* ctx_lens, int bs,
                                int budget, int sink, int recent, int32_t* keep, int64_t* new_lens, void* workspace,
                                int64_t workspace_bytes, int32_t* err_flag, void* stream) {
  const char* who = "mfd_evict_select";
  if (bs < 0 || bs > 65535 || w_rows < 0 || width < 0 || width > (1 << 30) || Hkv < 1)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad sizes bs=%d rows=%d width=%d Hkv=%d", who, bs, w_rows, width, Hkv);
  if (sink < 0 || recent < 0 || budget < 1 || (int64_t)sink + recent > budget)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: budget %d must be positive and hold sink %d + recent %d", who, budget,
                         sink, recent);
  if (bs == 0) return MFD_OK;
  if (!ctx_lens || !keep || !new_lens || (!weights && w_rows > 0 && width > 0))
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null pointer", who);
  const int64_t need = mfd_evict_select_workspace_bytes(bs, width);
  if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: 16-byte aligned workspace of %lld bytes needed", who, (long long)need);
  SelectArgs a{weights, w_row_stride, w_head_stride, w_rows, width, Hkv, req_idx, ctx_lens, budget, sink, recent, keep,
               new_lens, static_cast<uint32_t*>(workspace), key_stride_of(width), err_flag};
  hipStream_t st = static_cast<hipStream_t>(stream);
  // keys in registers up to 16 per thread; beyond, a kernel of its own forms them (all CUs read the sums, not one per request)
  if (width <= 8 * ST) {
    hipLaunchKernelGGL(evict_select_kernel<8>, dim3((unsigned)bs), dim3(ST), 0, st, a);
  } else if (width <= REG_KEYS * ST) {
    hipLaunchKernelGGL(evict_select_kernel<REG_KEYS>, dim3((unsigned)bs), dim3(ST), 0, st, a);
  } else {
    if (width > budget) {  // (a shorter row holds no request above the budget: nothing to score)
      hipLaunchKernelGGL(evict_score_kernel, dim3((unsigned)((width + 255) / 256), (unsigned)bs), dim3(256), 0, st, a);
      MFD_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(evict_select_kernel<0>, dim3((unsigned)bs), dim3(ST), 0, st, a);
  }
  MFD_CHECK_LAUNCH();
  return MFD_OK;
}

extern "C" int mfd_evict_compact_kv8(const int32_t* keep, int budget, const int64_t* new_lens, const int64_t* ctx_lens,
                                     uint8_t* k_cache, uint8_t* v_cache, int64_t kc_ss, int64_t kc_sh, int64_t vc_ss,
                                     int64_t vc_sh, float* k_scale, float* v_scale, int num_pages,
                                     const int32_t* src_table, int64_t src_stride, int src_rows, int src_width,
                                     const int32_t* dst_table, int64_t dst_stride, int dst_rows, int dst_width,
                                     int page_size, const int64_t* req_idx, float* weights, int64_t w_row_stride,
                                     int64_t w_head_stride, int w_rows, int width, int bs, int Hkv, int D_,
                                     int32_t* err_flag, void* stream) {
  const char* who = "mfd_evict_compact_kv8";
  int rc = kv8::check_cache(who, k_cache, v_cache, kc_ss, kc_sh, vc_ss, vc_sh, page_size, Hkv, D_, src_table, src_rows,
                            src_width, num_pages);
  if (rc == MFD_OK)
    rc = kv8::check_cache(who, k_cache, v_cache, kc_ss, kc_sh, vc_ss, vc_sh, page_size, Hkv, D_, dst_table, dst_rows,
                          dst_width, num_pages);
  if (rc != MFD_OK) return rc;
  if (bs < 0 || bs > 65535 || budget < 1 || width < 0 || w_rows < 0)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: bad sizes bs=%d budget=%d width=%d", who, bs, budget, width);
  if (bs == 0) return MFD_OK;
  if (!keep || !new_lens || !ctx_lens || !k_cache || !v_cache || !k_scale || !v_scale)
    return mfd_set_error(MFD_ERR_INVALID_ARG, "%s: null pointer", who);
  CompactArgs a{};
  a.keep = keep; a.budget = budget; a.new_lens = new_lens; a.ctx_lens = ctx_lens;
  a.cache[0] = k_cache; a.cache[1] = v_cache;
  a.c_ss[0] = kc_ss; a.c_ss[1] = vc_ss; a.c_sh[0] = kc_sh; a.c_sh[1] = vc_sh;
  a.scale[0] = k_scale; a.scale[1] = v_scale;
  const int shift = __builtin_ctz((unsigned)page_size);
  a.src = {src_table, src_stride, src_rows, src_width, req_idx, num_pages, shift};
  a.dst = {dst_table, dst_stride, dst_rows, dst_width, req_idx, num_pages, shift};
  a.w = weights; a.w_sr = w_row_stride; a.w_sh = w_head_stride; a.w_rows = w_rows; a.width = width;
  a.Hkv = Hkv; a.err_flag = err_flag;
  a.dst_pages = (int)(((int64_t)budget + page_size - 1) / page_size);
  if (((int64_t)a.dst_pages + 1) * Hkv > 0x7fffffff)
    return mfd_set_error(MFD_ERR_UNSUPPORTED, "%s: budget=%d too large", who, budget);
  const dim3 grid((unsigned)((a.dst_pages + 1) * Hkv), (unsigned)bs, 2);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (page_size <= 32) hipLaunchKernelGGL(evict_compact_kernel<1>, grid, dim3(NT), 0, st, a);
  else if (page_size == 64) hipLaunchKernelGGL(evict_compact_kernel<2>, grid, dim3(NT), 0, st, a);
  else if (page_size == 128) hipLaunchKernelGGL(evict_compact_kernel<4>, grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL(evict_compact_kernel<8>, grid, dim3(NT), 0, st, a);
  MFD_CHECK_LAUNCH();
  return MFD_OK;
}
