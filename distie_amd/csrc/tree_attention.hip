// Attention over a paged cache in 8 bits, and attention of drafted tokens over a cache of any type, for one head size (compiled
// with -DDISTIE_HEAD_DIM like attention.hip, whose kernels read caches in the activation's type for undrafted tokens).
//
// out[t, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(q[t, h] . k_j * scale) over the entries j of the request's cache that t sees;
// zero if it sees none. Entry j lies in page table[j / P] at j % P of k [pages, kv_heads, P, D] and v [pages, kv_heads, D, P]. In an
// 8-bit cache k_j = 2^a_j c_j and v_j = 2^b_j d_j with codes c, d (e4m3) and powers kept as bytes a + 127, b + 127 [pages, kv_heads, P].
//
// Which entries a token sees: of a request with n tokens in the step and `kv_len` entries behind it (past = kv_len - n),
//  * without `visible`: j <= position(t), and position(t) - j < window where there is one;
//  * with `visible` (a tree of drafted tokens; uint64 words [tokens, words]): j < past (within the window of position(t)), and of
//    the entries past + i, i < n, those whose bit i is set in t's words (within the window of position(i-th token) too).
// What a token does not see has no part in its sums, whatever it holds: entries that no request has written, NaN and infinities.
//
//  * attn_any: one workgroup per (token, head), any types and sizes; the plainest form.
//  * attn_runs: few columns over long contexts (steps of single tokens, small trees): matrix cores straight from the cache, the context cut
//    into runs; attn_runs_merge and attn_runs_merge_narrow put the runs' sums together.
//  * attn_tiles: many columns (portions of prompts, wide trees): tiles of 64 entries shared by 128 or 256 columns through LDS.

#include "common.h"
#include <atomic>

#ifndef DISTIE_HEAD_DIM
#error "compile with -DDISTIE_HEAD_DIM=<head size>"
#endif

namespace {

constexpr int D = DISTIE_HEAD_DIM;
typedef unsigned long long word_t;
struct code_t { uint8_t bits; };          // e4m3

__device__ __forceinline__ float to_float(code_t x) { return __builtin_amdgcn_cvt_f32_fp8(static_cast<int>(x.bits), 0); }
using ::to_float;
__device__ __forceinline__ float power_of(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }      // 2^(byte - 127)

struct Call {
  const void* q;
  int64_t q_stride;
  const void* k;
  const void* v;
  const uint8_t* k_scale;            // null: the cache is not in 8 bits
  const uint8_t* v_scale;
  const int32_t* positions;
  const int32_t* token_request;
  const int32_t* cu_q;
  const int32_t* kv_len;
  const int32_t* table;
  int table_width;
  const int32_t* table_rows;
  const word_t* visible;             // null: no tree
  int words;
  void* out;
  int tokens, requests, heads, kv_heads, block_size;
  int64_t pages;
  float scale;
  int window;                        // 0: none
};

__device__ __forceinline__ const int32_t* table_of(const Call& c, int request) {
  return c.table + static_cast<int64_t>(c.table_rows != nullptr ? c.table_rows[request] : request) * c.table_width;
}

// Whether token t (at `pos`, of a request whose first token is `begin`) sees entry j < past + n.
__device__ __forceinline__ bool sees(const Call& c, int64_t t, int pos, int begin, int past, int j) {
  int at = j;
  if (c.visible != nullptr && j >= past) {
    const int i = j - past;
    if (i / 64 >= c.words || !(c.visible[t * c.words + i / 64] >> (i % 64) & 1)) return false;
    if (c.window == 0) return true;
    at = c.positions[begin + i];
  } else if (c.visible == nullptr && j > pos) {
    return false;
  }
  return c.window == 0 || pos - at < c.window;
}

constexpr int ANY_WAVES = 4;
constexpr int ANY_DIMS = (D + DISTIE_WAVE - 1) / DISTIE_WAVE;

// Wave w takes the chunks w, w + 4, ... of 64 entries, a lane an entry for the scores and a lane a dimension for the sums; the four
// running maxima, denominators and sums meet in LDS.
template <typename T, typename C>
__global__ __launch_bounds__(DISTIE_WAVE * ANY_WAVES) void attn_any_kernel(const Call c) {
  __shared__ float q_lds[D];
  __shared__ float weight[ANY_WAVES][DISTIE_WAVE];
  __shared__ int64_t place[ANY_WAVES][DISTIE_WAVE];
  __shared__ float sums[ANY_WAVES][D];
  __shared__ float tops[ANY_WAVES], totals[ANY_WAVES];
  const int64_t t = blockIdx.x;
  const int head = blockIdx.y, kh = head / (c.heads / c.kv_heads);
  const int lane = threadIdx.x % DISTIE_WAVE, wave = threadIdx.x / DISTIE_WAVE;
  const int request = c.token_request[t], begin = c.cu_q[request], kv_len = c.kv_len[request];
  const int past = kv_len - (c.cu_q[request + 1] - begin), pos = c.positions[t];
  const int32_t* table = table_of(c, request);
  const T* q = static_cast<const T*>(c.q) + t * c.q_stride + static_cast<int64_t>(head) * D;
  for (int d = threadIdx.x; d < D; d += DISTIE_WAVE * ANY_WAVES) q_lds[d] = to_float(q[d]);
  __syncthreads();
  const int end = c.visible != nullptr ? kv_len : min(pos + 1, kv_len);
  const int first = c.window > 0 ? max(0, (c.visible != nullptr ? min(pos, past) : pos) - c.window + 1) : 0;
  float top = -INFINITY, total = 0.f, sum[ANY_DIMS] = {};
  for (int chunk = first / DISTIE_WAVE * DISTIE_WAVE + wave * DISTIE_WAVE; chunk < end; chunk += ANY_WAVES * DISTIE_WAVE) {
    const int j = chunk + lane;
    int64_t at = -1;
    if (j < end && j / c.block_size < c.table_width && sees(c, t, pos, begin, past, j)) {
      const int64_t page = table[j / c.block_size];
      if (page >= 0 && page < c.pages) at = (page * c.kv_heads + kh) * c.block_size + j % c.block_size;
    }
    float score = -INFINITY;
    if (at >= 0) {
      const C* k = static_cast<const C*>(c.k) + at * D;
      float s = 0.f;
#pragma unroll 8
      for (int d = 0; d < D; ++d) s = fmaf(q_lds[d], to_float(k[d]), s);
      score = s * c.scale * (c.k_scale != nullptr ? power_of(c.k_scale[at]) : 1.f);
    }
    const float best = fmaxf(top, wave_max(score));
    const float keep = best == -INFINITY ? 1.f : expf(top - best);
    // (a score of plus infinity or NaN makes the row NaN, as it is in the formula)
    const float w = at < 0 ? 0.f : expf(score - (best == -INFINITY ? 0.f : best));
    total = total * keep + wave_sum(w);
    top = best;
    weight[wave][lane] = at >= 0 && c.v_scale != nullptr ? w * power_of(c.v_scale[at]) : w;
    place[wave][lane] = at;
    __builtin_amdgcn_wave_barrier();
    for (int u = 0; u < ANY_DIMS; ++u) sum[u] *= keep;
    const int count = min(DISTIE_WAVE, end - chunk);
    for (int i = 0; i < count; ++i) {
      const int64_t from = place[wave][i];
      if (from < 0) continue;
      const C* v = static_cast<const C*>(c.v) + from / c.block_size * c.block_size * D + from % c.block_size;
      for (int u = 0; u < ANY_DIMS; ++u) {
        const int d = lane + u * DISTIE_WAVE;
        if (d < D) sum[u] = fmaf(weight[wave][i], to_float(v[static_cast<int64_t>(d) * c.block_size]), sum[u]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  for (int u = 0; u < ANY_DIMS; ++u)
    if (lane + u * DISTIE_WAVE < D) sums[wave][lane + u * DISTIE_WAVE] = sum[u];
  if (lane == 0) tops[wave] = top, totals[wave] = total;
  __syncthreads();
  float best = -INFINITY, all = 0.f, factor[ANY_WAVES];
  for (int w = 0; w < ANY_WAVES; ++w) best = fmaxf(best, tops[w]);
  for (int w = 0; w < ANY_WAVES; ++w) {
    factor[w] = totals[w] == 0.f ? 0.f : tops[w] == best ? 1.f : expf(tops[w] - best);
    all += totals[w] * factor[w];
  }
  T* out = static_cast<T*>(c.out) + (t * c.heads + head) * D;
  for (int d = threadIdx.x; d < D; d += DISTIE_WAVE * ANY_WAVES) {
    float s = 0.f;
    for (int w = 0; w < ANY_WAVES; ++w) s += totals[w] == 0.f ? 0.f : factor[w] * sums[w][d];
    out[d] = from_float<T>(all == 0.f ? 0.f : s / all);
  }
}

template <typename T>
int launch_any(const Call& c, int cache_type, hipStream_t stream) {
  const dim3 grid(c.tokens, c.heads);
  switch (cache_type) {
    case DISTIE_F32: attn_any_kernel<T, float><<<grid, DISTIE_WAVE * ANY_WAVES, 0, stream>>>(c); break;
    case DISTIE_BF16: attn_any_kernel<T, bf16_t><<<grid, DISTIE_WAVE * ANY_WAVES, 0, stream>>>(c); break;
    case DISTIE_E4M3: attn_any_kernel<T, code_t><<<grid, DISTIE_WAVE * ANY_WAVES, 0, stream>>>(c); break;
    default: return DISTIE_BAD_ARGUMENT;
  }
  return launch_status();
}

#if DISTIE_HEAD_DIM % 32 == 0 && DISTIE_HEAD_DIM <= 256
#define DISTIE_FAST_CACHE_ATTENTION 1
// ===================================================================================================
//  The matrix-core kernels: head sizes of a multiple of 32 up to 256, pages of a multiple of 16 entries.
//
//  * attn_runs: a wave owns 16 "columns" (token after token of a request, the query heads of one kv head inside a token) and
//    a run of the request's entries, which it takes in chunks of 64:
//        S^T[entry, col] = K[entry, :] . q[col, :]       four tiles of 16 entries
//        O[col, d]      += P[col, entry] . V^T[d, entry]  two steps of 32 entries
//    A lane (r = lane % 16, g = lane / 16) holds, of a 16 x 16 tile of S^T, rows 4g..4g+3 of column r, and as an operand of a 32-deep
//    product eight values of row r. Row m of tile t is taken to be entry 16 (m / 4) + 4t + m % 4 of the chunk: the lane's 16 scores are
//    then entries 16g..16g+15 in their order, which is what it reads of V^T as one piece (16 bytes of codes), and nothing
//    but maxima moves between lanes. Codes become bfloat16 in registers, with the key's power in the same instruction; the value's power
//    goes into the weight, which it changes by an exponent only. Float32 queries and weights go through these products in three parts
//    (`Products`); over a float32 cache the same operands go through the 16 x 16 x 4 products, eight a step. The W waves of a workgroup take neighbouring runs and put their sums together in LDS, in
//    pairs; workgroups beyond one a tile leave parts that attn_runs_merge puts together, in order.
// ===================================================================================================
typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8;
typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
typedef __attribute__((__vector_size__(8 * sizeof(float)))) float floatx8;
typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float floatx2;
typedef __attribute__((__vector_size__(4 * sizeof(uint32_t)))) uint32_t uintx4;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int DK = D / 32;              // 32-deep steps of q . k
constexpr int DB = D / 16;              // 16-wide blocks of the output

template <typename T> struct Operand;
template <> struct Operand<bf16_t> { typedef bf16x8 type; };
template <> struct Operand<float> { typedef floatx8 type; };

__device__ __forceinline__ floatx4 product(const bf16x8& a, const bf16x8& b, floatx4 sum) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, sum, 0, 0, 0);
}
__device__ __forceinline__ floatx4 product(const floatx8& a, const floatx8& b, floatx4 sum) {
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], sum, 0, 0, 0);
  return sum;
}

// In what type products are taken, and in how many parts the float32 side of them. A value of an 8-bit cache is exact in bfloat16 (from
// powers of 2^-124 on), and a float32 number (of 2^-102 and more; below, the last parts leave bfloat16's range) is exactly the sum of three
// bfloat16 numbers (24 bits, 8 each: cut off, never rounded): three products in bfloat16 add up to the float32 one, each exact, with the
// same float32 sums, in a fifth of its time. Beside a float32 cache there is no such way.
template <typename T, typename C> struct Products { typedef T type; static constexpr int PARTS = 1; };
template <> struct Products<float, code_t> { typedef bf16_t type; static constexpr int PARTS = 3; };

// Element i of `parts` operands: x, or its three parts.
template <int PARTS, typename O>
__device__ __forceinline__ void place(O* out, int i, float x) {
  if constexpr (PARTS == 1) {
    out[0][i] = x;          // (rounded to the operand's type)
  } else {
#pragma unroll
    for (int a = 0; a < PARTS; ++a) {
      const float part = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
      out[a][i] = static_cast<__bf16>(part);
      x -= part;
    }
  }
}

// eight codes (two words) as values times `power`
__device__ __forceinline__ bf16x8 of_codes(uint32_t a, uint32_t b, float power) {
  uintx4 words;
  words[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, false));
  words[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, power, true));
  words[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, false));
  words[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, power, true));
  return __builtin_bit_cast(bf16x8, words);
}

// A row of K as a lane holds it: the values of its operands, in pieces of 16 bytes. Operand dk of lane group g holds the eight
// values from dim(dk, g) on; with codes one piece is two operands.
template <typename C> struct Row;
template <> struct Row<code_t> {
  static constexpr int PAIRS = D / 64;
  uint4 piece[PAIRS > 0 ? PAIRS : 1];
  uint2 last;
  static __device__ __forceinline__ int dim(int dk, int g) { return dk / 2 < PAIRS ? 64 * (dk / 2) + 16 * g + 8 * (dk % 2) : 32 * dk + 8 * g; }
  __device__ __forceinline__ void load(const code_t* row, int g) {
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) piece[i] = *reinterpret_cast<const uint4*>(row + 64 * i + 16 * g);
    if constexpr (D % 64 != 0) last = *reinterpret_cast<const uint2*>(row + D - 32 + 8 * g);
  }
  __device__ __forceinline__ bf16x8 operand(int dk, float power) const {
    if (dk / 2 >= PAIRS) return of_codes(last.x, last.y, power);
    const uint4 p = piece[dk / 2];
    return dk % 2 == 0 ? of_codes(p.x, p.y, power) : of_codes(p.z, p.w, power);
  }
};
template <> struct Row<bf16_t> {
  uint4 piece[DK];
  static __device__ __forceinline__ int dim(int dk, int g) { return 32 * dk + 8 * g; }
  __device__ __forceinline__ void load(const bf16_t* row, int g) {
#pragma unroll
    for (int i = 0; i < DK; ++i) piece[i] = *reinterpret_cast<const uint4*>(row + 32 * i + 8 * g);
  }
  __device__ __forceinline__ bf16x8 operand(int dk, float) const { return __builtin_bit_cast(bf16x8, piece[dk]); }
};
template <> struct Row<float> {
  uint4 piece[2 * DK];
  static __device__ __forceinline__ int dim(int dk, int g) { return 32 * dk + 8 * g; }
  __device__ __forceinline__ void load(const float* row, int g) {
#pragma unroll
    for (int i = 0; i < 2 * DK; ++i) piece[i] = *reinterpret_cast<const uint4*>(row + 32 * (i / 2) + 8 * g + 4 * (i % 2));
  }
  __device__ __forceinline__ floatx8 operand(int dk, float) const {
    struct { uint4 a, b; } both = {piece[2 * dk], piece[2 * dk + 1]};
    return __builtin_bit_cast(floatx8, both);
  }
};

// All bits of those values of a word that are not finite.
template <typename C>
__device__ __forceinline__ uint32_t odd_values(uint32_t w) {
  if constexpr (sizeof(C) == 1) return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
  else if constexpr (sizeof(C) == 2) return ((((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15) * 0xffffu;
  else return (w & 0x7f800000u) == 0x7f800000u ? 0xffffffffu : 0u;
}

// The value of dimension d at entry j, for the rare pass over single values.
template <typename C>
__device__ __forceinline__ float value_at(const Call& c, const int32_t* table, int kh, int j, int d) {
  const int64_t page = min(static_cast<int64_t>(max(table[min(j / c.block_size, c.table_width - 1)], 0)), c.pages - 1);
  return to_float(static_cast<const C*>(c.v)[((page * c.kv_heads + kh) * D + d) * c.block_size + j % c.block_size]);
}

// Sixteen entries of a row of V^T, as words.
template <typename C> struct Sixteen {
  static constexpr int WORDS = 4 * sizeof(C);
  uint32_t word[WORDS];
  __device__ __forceinline__ void load(const C* p) {
#pragma unroll
    for (int i = 0; i < WORDS / 4; ++i) {
      const uint4 x = reinterpret_cast<const uint4*>(p)[i];
      word[4 * i] = x.x, word[4 * i + 1] = x.y, word[4 * i + 2] = x.z, word[4 * i + 3] = x.w;
    }
  }
  // what `seen` (16 bits) does not name is cleared, and what is not finite; whether there was such
  __device__ __forceinline__ bool clear(uint32_t seen) {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) {
      uint32_t w = word[i];
      if constexpr (sizeof(C) == 1) w &= (((seen >> (4 * i) & 0xfu) * 0x00204081u) & 0x01010101u) * 0xffu;
      else if constexpr (sizeof(C) == 2) w &= (seen >> (2 * i) & 1u ? 0xffffu : 0u) | (seen >> (2 * i + 1) & 1u ? 0xffff0000u : 0u);
      else w = seen >> i & 1u ? w : 0u;
      const uint32_t odd = odd_values<C>(w);
      found |= odd;
      word[i] = w & ~odd;
    }
    return found != 0;
  }
  // entries 8 s .. 8 s + 7 as an operand
  template <typename O>
  __device__ __forceinline__ O operand(int s) const {
    if constexpr (sizeof(C) == 1) return of_codes(word[2 * s], word[2 * s + 1], 1.f);
    else {
      struct { uint32_t x[WORDS / 2]; } all;
#pragma unroll
      for (int i = 0; i < WORDS / 2; ++i) all.x[i] = word[s * (WORDS / 2) + i];
      return __builtin_bit_cast(O, all);
    }
  }
};

// bits low .. high of 16 (nothing outside 0 .. 15)
__device__ __forceinline__ uint32_t bits_between(int low, int high) {
  const uint32_t upto = high >= 15 ? 0xffffu : high < 0 ? 0u : (2u << high) - 1u;
  return low <= 0 ? upto : low > 15 ? 0u : upto & ~((1u << low) - 1u);
}

// Which of the entries j .. j + 15 token t (at `pos`) sees, of the request with `past` entries in front of its n tokens from `begin` on.
__device__ __forceinline__ uint32_t sixteen_seen(const Call& c, int64_t t, int pos, int begin, int past, int n, int j) {
  const int low = c.window > 0 ? pos - c.window + 1 - j : 0;
  if (c.visible == nullptr) return bits_between(low, min(pos, past + n - 1) - j);
  uint32_t seen = bits_between(low, past - 1 - j);
  const int o = j - past;
  if (o > -16 && o < n) {
    const word_t* words = c.visible + t * c.words;
    word_t x;
    if (o >= 0) {
      x = o / 64 < c.words ? words[o / 64] >> (o % 64) : 0;
      if (o % 64 > 48 && o / 64 + 1 < c.words) x |= words[o / 64 + 1] << (64 - o % 64);
    } else {
      x = words[0] << -o;
    }
    uint32_t drafted = static_cast<uint32_t>(x) & bits_between(past - j, past + n - 1 - j);
    if (c.window > 0)
      for (int i = 0; i < 16; ++i)
        if ((drafted >> i & 1u) && pos - c.positions[begin + o + i] >= c.window) drafted &= ~(1u << i);
    seen |= drafted;
  }
  return seen;
}

struct Runs {
  int shares;             // workgroups along the entries
  int length;             // entries of a wave (attn_runs) or workgroup (attn_tiles): a multiple of 64, the same for all requests, so that a
                          // long one gets more workgroups; shares (times waves) of it reach over every request's entries
  int tiles;              // of columns: attn_runs, a request at most; attn_tiles, all requests' times the walks of each, or more
  int least, most;        // requests with so many tokens are served
  int by_request;         // parts are kept by request (which brings one token), not by token
  int dense;              // every request brings one token and no entry of cu_q needs to be read: request i's token is token i
  int shift;              // log2 of the page size, or -1
  float* part_o;          // float32 [rows, heads, shares, D]
  float* part_ml;         // float32 [rows, heads, shares, 2]
};

template <typename T, typename C, int W, bool EARLY>
__global__ __launch_bounds__(DISTIE_WAVE * W, (D <= 128 && sizeof(T) == 2 ? 2 : 1)) void attn_runs_kernel(const Call c, const Runs u) {
  typedef typename Operand<typename Products<T, C>::type>::type operand_t;
  constexpr int PARTS = Products<T, C>::PARTS;
  const int lane = threadIdx.x % DISTIE_WAVE;
  const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / DISTIE_WAVE) : 0;
  const int r = lane % 16, g = lane / 16;
  const int group = c.heads / c.kv_heads;
  const float scale_log2 = c.scale * 1.4426950408889634f;
  const int request = blockIdx.z, kh = blockIdx.x % c.kv_heads, tile = blockIdx.x / c.kv_heads, share = blockIdx.y;
  const int32_t* table = table_of(c, request);
  const int begin = u.dense ? request : c.cu_q[request], n = u.dense ? 1 : c.cu_q[request + 1] - begin;
  const int past = c.kv_len[request] - n;
  const int col0 = tile * 16, columns = n * group;
  if (n < u.least || n > u.most || col0 >= columns) return;
  const bool tree = c.visible != nullptr;
  const int request_first = c.window > 0 ? max(0, (tree ? past : c.positions[begin]) - c.window + 1) : 0;
  const int run_begin = request_first / 64 * 64 + (share * W + wave) * u.length;
  // The page of a block of 16 entries. Blocks outside the run may have none: they read some page of the cache, and what they read is
  // dropped. (So the first pages are asked for without waiting for how long the request is.)
  const auto page_of = [&](int block) {
    const int slot = u.shift >= 0 ? (block * 16) >> u.shift : block * 16 / c.block_size;
    return table[min(slot, c.table_width - 1)];
  };
  int k_page = page_of(run_begin / 16 + r / 4), v_page = page_of(run_begin / 16 + g);
  // ---- the lane's columns
  const int own_col = min(col0 + r, columns - 1);            // columns past the end repeat the last; dropped later
  const int token = begin + own_col / group, pos = c.positions[token];
  operand_t q_reg[DK][PARTS];
  const T* q = static_cast<const T*>(c.q) + token * c.q_stride + static_cast<int64_t>(kh * group + own_col % group) * D;
#pragma unroll
  for (int dk = 0; dk < DK; ++dk) {
    const auto values = *reinterpret_cast<const typename Operand<T>::type*>(q + Row<C>::dim(dk, g));
    if constexpr (PARTS == 1) q_reg[dk][0] = values;
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) place<PARTS>(q_reg[dk], i, values[i]);
  }
  // ---- this wave's run of the request's entries, and what of it the tile's tokens see
  const int first_token = begin + col0 / group, last_token = begin + min(col0 + 15, columns - 1) / group;
  const int tile_first = tree ? request_first : c.window > 0 ? max(0, c.positions[first_token] - c.window + 1) : 0;
  const int tile_last = tree ? past + n - 1 : min(c.positions[last_token], past + n - 1);
  const int key_begin = max(run_begin, tile_first), key_end = min(run_begin + u.length - 1, tile_last);
  const int open_until = tree ? past - 1 : c.positions[first_token];          // every column sees the entries up to here that its window holds

  if (u.shares > 1 && run_begin - wave * u.length > tile_last) {          // no wave of the workgroup has an entry
    for (int col = col0 + threadIdx.x; col < min(col0 + 16, columns); col += DISTIE_WAVE * W) {
      const int64_t row = u.by_request ? request : begin + col / group;
      *reinterpret_cast<float2*>(u.part_ml + 2 * ((row * c.heads + kh * group + col % group) * u.shares + share)) = float2{-INFINITY, 0.f};
    }
    return;
  }
  floatx4 o_acc[DB];
  float m_run = -INFINITY, l_run = 0.f;
#pragma unroll
  for (int db = 0; db < DB; ++db) o_acc[db] = floatx4{0.f, 0.f, 0.f, 0.f};
  // (pages, kv heads) and places in the page: of the block, as the start of its rows in entries
  const auto entry_of = [&](int block, int page) {
    const int at = u.shift >= 0 ? (block * 16) & (c.block_size - 1) : block * 16 % c.block_size;
    const int64_t held = min(static_cast<int64_t>(max(page, 0)), c.pages - 1);
    return longlong2{(held * c.kv_heads + kh) * c.block_size, at};
  };
  const int chunk_begin = key_begin / 64 * 64;
  if (chunk_begin != run_begin) k_page = page_of(chunk_begin / 16 + r / 4), v_page = page_of(chunk_begin / 16 + g);          // (a window begins inside the run)
  Row<C> k_row[4];
  Sixteen<C> v_row[DB];
  uint4 k_powers = {0, 0, 0, 0}, v_powers = {0, 0, 0, 0};
  const auto fetch_k = [&](int block, int page) {
    const longlong2 at = entry_of(block, page);
    if constexpr (sizeof(C) == 1) k_powers = *reinterpret_cast<const uint4*>(c.k_scale + at.x + at.y);
    const C* from = static_cast<const C*>(c.k) + (at.x + at.y + r % 4) * D;
#pragma unroll
    for (int t = 0; t < 4; ++t) k_row[t].load(from + 4 * t * D, g);
  };
  const auto fetch_v = [&](int block, int page) {
    const longlong2 at = entry_of(block, page);
    if constexpr (sizeof(C) == 1) v_powers = *reinterpret_cast<const uint4*>(c.v_scale + at.x + at.y);
    const C* from = static_cast<const C*>(c.v) + at.x * D + at.y + static_cast<int64_t>(r) * c.block_size;
#pragma unroll
    for (int db = 0; db < DB; ++db) v_row[db].load(from + static_cast<int64_t>(16 * db) * c.block_size);
  };
  // EARLY: keys and values are asked for a chunk ahead, into the registers of those that have just been used (keys behind their products,
  // values behind theirs), so a wave always has half a chunk on its way; behind the last chunk the last block once more, which the caches
  // hold. Else a chunk's loads stand in front of it.
  const int last_block = max(key_end, 0) / 16;
  if constexpr (EARLY) {
    fetch_k(chunk_begin / 16 + r / 4, k_page);          // (under no condition: the results would be waited for where the branches meet)
    fetch_v(chunk_begin / 16 + g, v_page);
    k_page = page_of(min(chunk_begin / 16 + 4 + r / 4, last_block)), v_page = page_of(min(chunk_begin / 16 + 4 + g, last_block));
  }
  bool odd = false;
  for (int chunk = chunk_begin; chunk <= key_end; chunk += 64) {
    if constexpr (!EARLY) {
      fetch_k(chunk / 16 + r / 4, k_page);
      fetch_v(chunk / 16 + g, v_page);
      k_page = page_of(chunk / 16 + 4 + r / 4), v_page = page_of(chunk / 16 + 4 + g);            // of the next chunk, while these are on their way
    }
    // ---- scores
    floatx4 s[4];
    {
      const uint32_t words[4] = {k_powers.x, k_powers.y, k_powers.z, k_powers.w};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float power = sizeof(C) == 1 ? power_of(words[t] >> (8 * (r % 4)) & 0xffu) : 1.f;
        s[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int dk = 0; dk < DK; ++dk) {
          const operand_t k = k_row[t].operand(dk, power);
#pragma unroll
          for (int a = 0; a < PARTS; ++a) s[t] = product(k, q_reg[dk][a], s[t]);
        }
      }
    }
    const int v_page_next = v_page;
    if constexpr (EARLY) {
      __builtin_amdgcn_sched_barrier(0);
      fetch_k(min(chunk / 16 + 4 + r / 4, last_block), k_page);
      k_page = page_of(min(chunk / 16 + 8 + r / 4, last_block)), v_page = page_of(min(chunk / 16 + 8 + g, last_block));
      __builtin_amdgcn_sched_barrier(0);
    }
    // ---- which of them count: in most chunks all
    bool open = chunk + 63 <= min(open_until, key_end) && chunk >= key_begin;
    if (c.window > 0) open = open && __all(chunk > pos - c.window);
    if (!open) {
      const uint32_t in_run = bits_between(key_begin - (chunk + 16 * g), key_end - (chunk + 16 * g));
      const uint32_t seen = in_run & sixteen_seen(c, token, pos, begin, past, n, chunk + 16 * g);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(seen >> (4 * t + i) & 1u)) s[t][i] = -INFINITY;
      // What no column sees is cleared: it may be anything, and a weight of zero times NaN is NaN. So is what is not finite among the
      // rest, since some columns see it and others do not: the pass behind the walk puts it where it is seen.
      uint32_t by_any = seen;
#pragma unroll
      for (int step = 1; step < 16; step *= 2) by_any |= __shfl_xor(static_cast<int>(by_any), step, DISTIE_WAVE);
      bool found = false;
#pragma unroll
      for (int db = 0; db < DB; ++db) found |= v_row[db].clear(by_any);
      if constexpr (sizeof(C) == 1) {            // (their powers as well: the byte 255 would be an infinity)
        const auto keep = [&](uint32_t word, int i) { return word & ((((by_any >> (4 * i) & 0xfu) * 0x00204081u) & 0x01010101u) * 0xffu); };
        v_powers = uint4{keep(v_powers.x, 0), keep(v_powers.y, 1), keep(v_powers.z, 2), keep(v_powers.w, 3)};
      }
      odd |= __any(found);
    }
    // ---- softmax step of each column
    operand_t p_reg[2][PARTS];
    const uint32_t value_powers[4] = {v_powers.x, v_powers.y, v_powers.z, v_powers.w};
    float best = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) best = fmaxf(best, s[t][i]);
    best = lanes_max<32>(lanes_max<16>(best)) * scale_log2;          // the scale is positive: the largest stays the largest
    const float m_new = fmaxf(m_run, best);
    const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
    const float from = m_new == -INFINITY ? 0.f : -m_new;
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float p = fast_exp2(fmaf(s[t][i], scale_log2, from));
        sum += p;
        if constexpr (sizeof(C) == 1) p *= power_of(value_powers[t] >> (8 * i) & 0xffu);
        // (a weight has 8 bits in bfloat16, as every operand of these products; the denominator adds it unrounded)
        place<PARTS>(p_reg[t / 2], 4 * (t % 2) + i, p);
      }
    l_run = l_run * alpha + sum;          // the lanes of a column each keep a part of the sum
    m_run = m_new;
    float a4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a4[i] = __shfl(alpha, 4 * g + i, DISTIE_WAVE);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) o_acc[db][i] *= a4[i];
#pragma unroll
    for (int step = 0; step < 2; ++step)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const operand_t v = v_row[db].template operand<operand_t>(step);
#pragma unroll
        for (int a = 0; a < PARTS; ++a) o_acc[db] = product(p_reg[step][a], v, o_acc[db]);
      }
    if constexpr (EARLY) {
      __builtin_amdgcn_sched_barrier(0);
      fetch_v(min(chunk / 16 + 4 + g, last_block), v_page_next);
    }
  }
  if (odd) {
    // NaN and infinities among the values that not all columns see, one by one
#pragma unroll 1
    for (int j = key_begin; j <= key_end; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = begin + min(col0 + 4 * g + i, columns - 1) / group;
        const bool seen = sees(c, t, c.positions[t], begin, past, j);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const float v = value_at<C>(c, table, kh, j, 16 * db + r);
          if (seen && !(fabsf(v) < INFINITY)) o_acc[db][i] += v;
        }
      }
    }
  }
  l_run = lanes_sum<32>(lanes_sum<16>(l_run));

  // ---- the workgroup's runs, put together in pairs: the upper half of the waves leave theirs in LDS, the lower half take them up
  if constexpr (W > 1) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    constexpr int PIECES = DB;                                           // floatx4 a lane
    floatx4* sums = reinterpret_cast<floatx4*>(lds);                      // [W / 2][PIECES][64]
    float* states = lds + (W / 2) * PIECES * DISTIE_WAVE * 4;              // [W / 2][2][64]
#pragma unroll
    for (int half = W / 2; half > 0; half /= 2) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
        const int at = wave - half;
#pragma unroll
        for (int db = 0; db < DB; ++db) sums[(at * PIECES + db) * DISTIE_WAVE + lane] = o_acc[db];
        states[2 * at * DISTIE_WAVE + lane] = m_run;
        states[(2 * at + 1) * DISTIE_WAVE + lane] = l_run;
      }
      __syncthreads();
      if (wave < half) {
        const float m_other = states[2 * wave * DISTIE_WAVE + lane];
        const float l_other = states[(2 * wave + 1) * DISTIE_WAVE + lane];
        const float m_new = fmaxf(m_run, m_other);
        const float own = m_run == m_new ? 1.f : fast_exp2(m_run - m_new), other = m_other == m_new ? 1.f : fast_exp2(m_other - m_new);
        l_run = l_run * own + l_other * other;
        m_run = m_new;
        float own4[4], other4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) own4[i] = __shfl(own, 4 * g + i, DISTIE_WAVE), other4[i] = __shfl(other, 4 * g + i, DISTIE_WAVE);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const floatx4 o = sums[(wave * PIECES + db) * DISTIE_WAVE + lane];
#pragma unroll
          for (int i = 0; i < 4; ++i) o_acc[db][i] = o_acc[db][i] * own4[i] + o[i] * other4[i];
        }
      }
    }
    if (wave > 0) return;
  }
  // ---- the result, or this share's part of it
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int col = col0 + 4 * g + i;
    const float m_col = __shfl(m_run, 4 * g + i, DISTIE_WAVE), l_col = __shfl(l_run, 4 * g + i, DISTIE_WAVE);
    if (col >= columns) continue;
    const int64_t t = begin + col / group;
    const int head = kh * group + col % group;
    if (u.shares == 1) {
      const float inverse = l_col == 0.f ? 0.f : 1.f / l_col;
      T* out = static_cast<T*>(c.out) + (t * c.heads + head) * D;
#pragma unroll
      for (int db = 0; db < DB; ++db) out[16 * db + r] = static_cast<T>(o_acc[db][i] * inverse);
    } else {
      const int64_t part = ((u.by_request ? request : t) * c.heads + head) * u.shares + share;
#pragma unroll
      for (int db = 0; db < DB; ++db) u.part_o[part * D + 16 * db + r] = o_acc[db][i];
      if (r == 0) *reinterpret_cast<float2*>(u.part_ml + 2 * part) = float2{m_col, l_col};
    }
  }
}

// One wave a workgroup left as many more parts to the merge; eight fill a compute unit and end together: RUN_WAVES of 1 / 4 / 8, the best number of
// shares each, us with 28 heads of 128 on 4 and codes: 64 requests of 8,000 entries 83.5 / 76.8 / 80.6, 64 of 1,000 17.4 / 15.0 / 16.4, 16 of
// 4,000 17.7 / 17.7 / 18.0, 4 of 16,000 20.6 / 17.7 / 18.4, one of 32,000 21.5 / 16.2 / 16.6, one of 1,000 8.8 / 9.9 / 11.6.
constexpr int RUN_WAVES = 4;
constexpr int MOST_SHARES = DISTIE_WAVE;
constexpr int MERGE_WAVES = 4;
constexpr int MERGE_AHEAD = 8;

// One wave a (row, head): a lane a share for the weights, a lane two or more dimensions for the sums, which are added in order.
// EAGER: the first parts are asked for together with the shares' states, whether they hold anything or not (few rows: one trip to memory
// instead of two); else only those up to the last that does (many rows, where what is read counts).
template <typename T, bool EAGER>
__global__ __launch_bounds__(DISTIE_WAVE * MERGE_WAVES) void attn_runs_merge_kernel(const Call c, const Runs u, int64_t rows) {
  const int lane = threadIdx.x % DISTIE_WAVE;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * MERGE_WAVES + __builtin_amdgcn_readfirstlane(threadIdx.x / DISTIE_WAVE);
  if (pair >= rows * c.heads) return;
  const int64_t row = pair / c.heads;
  constexpr int PER = (D + DISTIE_WAVE - 1) / DISTIE_WAVE;
  const float* part_o = u.part_o + pair * u.shares * D;
  float part[MERGE_AHEAD][PER];
  const auto fetch = [&](int s, int last) {
#pragma unroll
    for (int a = 0; a < MERGE_AHEAD; ++a)
#pragma unroll
      for (int e = 0; e < PER; ++e) part[a][e] = part_o[static_cast<int64_t>(min(s + a, last)) * D + min(lane + e * DISTIE_WAVE, D - 1)];
  };
  const float2 ml = *reinterpret_cast<const float2*>(u.part_ml + 2 * (pair * u.shares + min(lane, u.shares - 1)));
  if constexpr (EAGER) {
    fetch(0, u.shares - 1);
    loads_first();
  }
  int64_t t = row;
  if (!u.dense) {
    const int request = u.by_request ? row : c.token_request[row];
    const int begin = c.cu_q[request], n = c.cu_q[request + 1] - begin;
    if (n < u.least || n > u.most) return;
    if (u.by_request) t = begin;
  }
  const bool there = lane < u.shares && ml.y != 0.f;            // a share without an entry left a denominator of zero, and no sums
  const unsigned long long any = __ballot(there);
  const int shares = any == 0 ? 0 : DISTIE_WAVE - __clzll(any);
  const float top = wave_max(there ? ml.x : -INFINITY);
  const float weight = !there ? 0.f : ml.x == top ? 1.f : fast_exp2(ml.x - top);
  const float total = wave_sum(there ? weight * ml.y : 0.f);
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  float sum[PER] = {};
  for (int s = 0; s < shares; s += MERGE_AHEAD) {
    if (!EAGER || s > 0) {
      fetch(s, shares - 1);
      loads_first();
    }
#pragma unroll
    for (int a = 0; a < MERGE_AHEAD; ++a) {
      const float w = __shfl(weight, min(s + a, shares - 1), DISTIE_WAVE);
#pragma unroll
      for (int e = 0; e < PER; ++e) sum[e] = s + a < shares && w != 0.f ? fmaf(w, part[a][e], sum[e]) : sum[e];
    }
  }
  T* out = static_cast<T*>(c.out) + (t * c.heads + pair % c.heads) * D;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (lane + e * DISTIE_WAVE < D) out[lane + e * DISTIE_WAVE] = from_float<T>(sum[e] * inverse);
}

constexpr int EAGER_PAIRS = 4096;          // (row, head)s: two rounds of waves at most

// Many rows of at most 16 shares: four (row, head)s a wave, 16 lanes each, so that a wave has four times as much on its way. 976 tokens of 28 heads with up
// to three shares: 11.7 us with one a wave, 7.8.
template <typename T>
__global__ __launch_bounds__(DISTIE_WAVE * MERGE_WAVES) void attn_runs_merge_narrow_kernel(const Call c, const Runs u, int64_t rows) {
  constexpr int LANES = 16, PER = D / LANES, STEP = PER % 4 == 0 ? 4 : 2, AT_ONCE = 4;
  typedef __attribute__((__vector_size__(STEP * sizeof(float)))) float piece_t;
  const int lane = threadIdx.x % LANES;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * (blockDim.x / LANES) + threadIdx.x / LANES;
  const bool inside = pair < rows * c.heads;
  const int64_t held = inside ? pair : 0, row = held / c.heads;
  const float2 ml = *reinterpret_cast<const float2*>(u.part_ml + 2 * (held * u.shares + min(lane, u.shares - 1)));
  const int request = u.by_request ? row : c.token_request[row];
  const int begin = c.cu_q[request], n = c.cu_q[request + 1] - begin;
  const bool served = inside && n >= u.least && n <= u.most;
  const bool there = served && lane < u.shares && ml.y != 0.f;
  const float top = lanes_max<8>(lanes_max<4>(lanes_max<2>(lanes_max<1>(there ? ml.x : -INFINITY))));
  const float weight = !there ? 0.f : ml.x == top ? 1.f : fast_exp2(ml.x - top);
  const float total = lanes_sum<8>(lanes_sum<4>(lanes_sum<2>(lanes_sum<1>(there ? weight * ml.y : 0.f))));
  const float inverse = total == 0.f ? 0.f : 1.f / total;
  // a lane's pieces lie LANES pieces apart, so 16 lanes read a run of memory at once
  const float* part_o = u.part_o + held * u.shares * D + STEP * lane;
  float sum[PER] = {};
  const unsigned any = static_cast<unsigned>(__ballot(there) >> (threadIdx.x % DISTIE_WAVE / LANES * LANES)) & 0xffffu;
  const int shares = any == 0 ? 0 : 32 - __clz(any);
  int most = shares;                        // of the wave's four: all lanes take part in the shuffles
  most = max(most, __shfl_xor(most, 16, DISTIE_WAVE));
  most = max(most, __shfl_xor(most, 32, DISTIE_WAVE));
  for (int s = 0; s < most; s += AT_ONCE) {
    piece_t part[AT_ONCE][PER / STEP];
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a)
#pragma unroll
      for (int e = 0; e < PER / STEP; ++e)
        part[a][e] = *reinterpret_cast<const piece_t*>(part_o + static_cast<int64_t>(max(0, min(s + a, shares - 1))) * D + STEP * LANES * e);
    loads_first();
#pragma unroll
    for (int a = 0; a < AT_ONCE; ++a) {
      const float w = __shfl(weight, min(s + a, LANES - 1), LANES);
#pragma unroll
      for (int e = 0; e < PER; ++e) sum[e] = s + a < shares && w != 0.f ? fmaf(w, part[a][e / STEP][e % STEP], sum[e]) : sum[e];
    }
  }
  if (!served) return;
  T* out = static_cast<T*>(c.out) + ((u.by_request ? static_cast<int64_t>(begin) : row) * c.heads + held % c.heads) * D + STEP * lane;
#pragma unroll
  for (int e = 0; e < PER / STEP; ++e)
#pragma unroll
    for (int i = 0; i < STEP; ++i) out[STEP * LANES * e + i] = from_float<T>(sum[STEP * e + i] * inverse);
}
template <typename T>
int launch_merge(const Call& c, const Runs& u, hipStream_t stream) {
  const int64_t rows = u.by_request ? c.requests : c.tokens;
  const unsigned blocks = static_cast<unsigned>((rows * c.heads + MERGE_WAVES - 1) / MERGE_WAVES);
  if (rows * c.heads <= EAGER_PAIRS) attn_runs_merge_kernel<T, true><<<blocks, DISTIE_WAVE * MERGE_WAVES, 0, stream>>>(c, u, rows);
  else if (u.shares <= 16) attn_runs_merge_narrow_kernel<T><<<(blocks + 3) / 4, DISTIE_WAVE * MERGE_WAVES, 0, stream>>>(c, u, rows);
  else attn_runs_merge_kernel<T, false><<<blocks, DISTIE_WAVE * MERGE_WAVES, 0, stream>>>(c, u, rows);
  return launch_status();
}

// From runs of so many entries on the loads go a chunk ahead (codes only: the other types' chunks leave no registers for the next addresses): 64
// requests of 1,050 to 3,150 entries 35.2 -> 31.6 us, 8 of 32,767 55.1 -> 53.3; runs of one or two chunks wait longer for the loads behind the last (one
// request of 517 8.7 -> 9.4).
constexpr int EARLY_FROM = 256;

template <typename T, typename C>
int launch_runs(const Call& c, const Runs& u, hipStream_t stream) {
  constexpr int W = RUN_WAVES;
  constexpr size_t lds = W == 1 ? 0 : static_cast<size_t>(W / 2) * DISTIE_WAVE * (DB * 4 + 2) * sizeof(float);
  static_assert(lds <= 65536, "no more LDS than a launch has without asking");
  const dim3 grid(c.kv_heads * u.tiles, u.shares, c.requests);
  constexpr bool AHEAD_TOO = sizeof(C) == 1 && sizeof(T) == 2;
  if (AHEAD_TOO && u.length >= EARLY_FROM) attn_runs_kernel<T, C, W, AHEAD_TOO><<<grid, DISTIE_WAVE * W, lds, stream>>>(c, u);
  else attn_runs_kernel<T, C, W, false><<<grid, DISTIE_WAVE * W, lds, stream>>>(c, u);
  int status = launch_status();
  if (status != 0 || u.shares == 1) return status;
  return launch_merge<T>(c, u, stream);
}
template <typename T, typename C>
int launch_runs_of(const Call& c, const Runs& u, hipStream_t stream) {
  if constexpr (sizeof(C) < 4 || D <= 128) return launch_runs<T, C>(c, u, stream);          // (beyond, the registers do not hold a chunk)
  else return DISTIE_BAD_ARGUMENT;
}
// ===================================================================================================
//  * attn_tiles: many columns (portions of prompts, wide trees; bfloat16). A workgroup of four waves owns 128 columns, of eight 256, and walks over
//    the request's entries 64 at a time: K rows and V^T rows lie in LDS in bfloat16 (codes are converted once on their way there,
//    keys with their power), in two places, so a tile is stored while the one before is used and the loop has one barrier. A wave multiplies its
//    32 columns against them with the 32 x 32 x 16 products:
//        S^T[entry, col] = K[entry, :] . q[col, :]        O^T[d, col] += V^T[d, entry] . P^T[entry, col]
//    A lane (c = lane % 32, h = lane / 32) holds, of a tile of 32 x 32 scores, rows 8i + 4h + j of column c. Entries lie in the rows of K
//    with bits 2 and 3 of their number swapped: the lane's scores are then eight neighbouring entries 16t + 8h .. + 7 each, which is what
//    an operand of the second product holds and what is read of V^T in one piece.
//    What bounds it: of a compute unit's time a third are the products, four tenths the vector ALU (exponentials, conversion, the weights'
//    powers), the rest LDS and waiting; they add up instead of hiding each other, at some 1.9 GHz. A portion of 2,048 tokens behind 2,051, 28 heads
//    of 128 on 4, codes: 131 us, 690 TFLOP/s; 4 trees of 200 tokens over 9,000 to 16,000 entries, bfloat16: 182 us, 790 (128 columns: 192). Tried
//    and slower: 64 columns a wave, so that an operand read from LDS serves two products (266 us, a wave a SIMD and nothing beside it); eight
//    waves in two groups that take products and softmax in turns (198).
// ===================================================================================================
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float floatx16;

constexpr int TILE = 64;                              // entries
constexpr int TK = D / 16;                            // steps of q . k
constexpr int TD = D / 32;                            // blocks of 32 output rows
constexpr int K_STRIDE = D + 8;                       // rows of an odd number of 16-byte pieces: free of bank conflicts
constexpr int V_STRIDE = TILE + 8;
constexpr float GROW = 8.f;                           // in units of log 2: how far a score may pass a column's reference
constexpr int AHEAD = D <= 128 ? 6 : 4;                              // reads from LDS in flight ahead of the products
struct TileLds {
  bf16_t k[TILE * K_STRIDE];
  bf16_t v[D * V_STRIDE];
  float powers[TILE];                                 // of the values
};

__device__ __forceinline__ word_t bits_between_64(int low, int high) {
  const word_t upto = high >= 63 ? ~0ull : high < 0 ? 0ull : (2ull << high) - 1ull;
  return low <= 0 ? upto : low > 63 ? 0ull : upto & ~((1ull << low) - 1ull);
}

// Which of the entries j .. j + 63 token t sees (`sixteen_seen` of more).
__device__ __forceinline__ word_t sixty_four_seen(const Call& c, int64_t t, int pos, int begin, int past, int n, int j) {
  const int low = c.window > 0 ? pos - c.window + 1 - j : 0;
  if (c.visible == nullptr) return bits_between_64(low, min(pos, past + n - 1) - j);
  word_t seen = bits_between_64(low, past - 1 - j);
  const int o = j - past;
  if (o > -64 && o < n) {
    const word_t* words = c.visible + t * c.words;
    word_t x;
    if (o >= 0) {
      x = o / 64 < c.words ? words[o / 64] >> (o % 64) : 0;
      if (o % 64 > 0 && o / 64 + 1 < c.words) x |= words[o / 64 + 1] << (64 - o % 64);
    } else {
      x = words[0] << -o;
    }
    x &= bits_between_64(past - j, past + n - 1 - j);
    if (c.window > 0)
      for (int i = 0; i < 64; ++i)
        if ((x >> i & 1ull) && pos - c.positions[begin + o + i] >= c.window) x &= ~(1ull << i);
    seen |= x;
  }
  return seen;
}

// Walks of u.length entries each (the host counts alike): of a request's longest tile, how many of them all its tiles have, how many tiles have
// the walk m behind those (the last ones, in a portion whose tokens see more and more), and of the tile whose last token is `last`.
__device__ __forceinline__ int walks_at_most(const Call& c, const Runs& u, int past, int n) {
  const int first = c.window > 0 ? max(0, past - c.window + 1) / TILE * TILE : 0;
  return max(1, min(u.shares, (past + n - first + u.length - 1) / u.length));
}
__device__ __forceinline__ int walks_of_all(const Call& c, const Runs& u, int past, int at_most) {
  return c.visible != nullptr || c.window > 0 ? at_most : min(at_most, past / u.length + 1);
}
__device__ __forceinline__ int tiles_with_walk(const Runs& u, int past, int group, int tiles, int wide, int m) {
  return tiles - static_cast<int>(static_cast<int64_t>(m * u.length - past) * group / wide);
}
__device__ __forceinline__ int walks_of_tile(const Call& c, const Runs& u, int past, int n, int last) {
  if (c.visible != nullptr || c.window > 0) return walks_at_most(c, u, past, n);
  return max(1, min(u.shares, (past + last + u.length) / u.length));
}

template <typename C, int WAVES>
__global__ __launch_bounds__(DISTIE_WAVE * WAVES, D <= 128 ? 2 : 1) void attn_tiles_kernel(const Call c, const Runs u) {
  constexpr int TILE_COLUMNS = 32 * WAVES;
  constexpr int SHARE = WAVES / 4;                      // waves that bring a block of 16 entries together
  extern __shared__ __attribute__((aligned(16))) char tile_lds[];
  TileLds* lds = reinterpret_cast<TileLds*>(tile_lds);
  int* odd = reinterpret_cast<int*>(lds + 2);          // some value that not all columns see is not finite
  const int lane = threadIdx.x % DISTIE_WAVE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / DISTIE_WAVE);
  const int col_lane = lane % 32, h = lane / 32;
  const int group = c.heads / c.kv_heads;
  const float scale_log2 = c.scale * 1.4426950408889634f;
  const bool tree = c.visible != nullptr;

  // ---- which columns and entries. The requests' work lies one behind the other, of each its (walk, tile) pairs, the late tiles first (the late
  // tokens of a portion see the most, and the longest work should start first): a lane a request finds the one of this workgroup.
  const int kh = blockIdx.x % c.kv_heads;
  int item = blockIdx.x / c.kv_heads, request = -1, tiles = 0;
  for (int first = 0; first < c.requests && request < 0; first += DISTIE_WAVE) {
    const int mine = min(first + lane, c.requests - 1);
    const int brought = c.cu_q[mine + 1] - c.cu_q[mine];
    const bool served = first + lane < c.requests && brought >= u.least && brought <= u.most;
    const int own_tiles = served ? (brought * group + TILE_COLUMNS - 1) / TILE_COLUMNS : 0;
    const int own_past = c.kv_len[mine] - brought, walks = walks_at_most(c, u, own_past, brought), of_all = walks_of_all(c, u, own_past, walks);
    int work = own_tiles * of_all;
    for (int m = of_all; served && m < walks; ++m) work += tiles_with_walk(u, own_past, group, own_tiles, TILE_COLUMNS, m);
    int upto = work;
#pragma unroll
    for (int step = 1; step < DISTIE_WAVE; step *= 2) {
      const int before = __shfl_up(upto, step, DISTIE_WAVE);
      upto += lane >= step ? before : 0;
    }
    const unsigned long long here = __ballot(upto > item);
    const int at = here != 0 ? __ffsll(here) - 1 : DISTIE_WAVE - 1;
    if (here != 0) {
      request = first + at;
      tiles = __shfl(own_tiles, at, DISTIE_WAVE);
      item -= __shfl(upto - work, at, DISTIE_WAVE);
    } else {
      item -= __shfl(upto, at, DISTIE_WAVE);
    }
  }
  request = __builtin_amdgcn_readfirstlane(request);
  if (request < 0) return;
  item = __builtin_amdgcn_readfirstlane(item);
  tiles = __builtin_amdgcn_readfirstlane(tiles);
  const int begin = c.cu_q[request], n = c.cu_q[request + 1] - begin, past = c.kv_len[request] - n;
  const int of_all = walks_of_all(c, u, past, walks_at_most(c, u, past, n));
  int share = min(item / tiles, of_all);
  item -= share * tiles;
  for (; share >= of_all && share < u.shares - 1; ++share) {
    const int with_it = tiles_with_walk(u, past, group, tiles, TILE_COLUMNS, share);
    if (item < with_it) break;
    item -= with_it;
  }
  const int tile = tiles - 1 - item;
  const int columns = n * group, col0 = tile * TILE_COLUMNS;
  const int32_t* table = table_of(c, request);
  const int first_token = begin + col0 / group, last_token = begin + min(col0 + TILE_COLUMNS, columns) / group - (min(col0 + TILE_COLUMNS, columns) % group == 0);
  const int first_pos = c.positions[first_token];
  const int key_first = c.window > 0 ? max(0, (tree ? past : first_pos) - c.window + 1) : 0;
  const int key_last = tree ? past + n - 1 : min(c.positions[last_token], past + n - 1);

  // ---- the lane's column
  const int wave_col0 = col0 + 32 * wave;
  const bool idle = wave_col0 >= columns;                       // the whole wave: it only brings its block of each tile
  const int col = min(wave_col0 + col_lane, columns - 1);        // columns past the end repeat the last; dropped later
  const int64_t token = begin + col / group;
  const int pos = c.positions[token];
  const int head = kh * group + col % group;
  bf16x8 q_reg[TK];
  {
    const bf16_t* q = static_cast<const bf16_t*>(c.q) + token * c.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
    for (int i = 0; i < TK; ++i) q_reg[i] = *reinterpret_cast<const bf16x8*>(q + 16 * i + 8 * h);
  }
  // what all columns of the wave see: entries up to `open_until` (within the windows of all of them)
  const int wave_first = begin + min(wave_col0, columns - 1) / group, wave_last = begin + min(wave_col0 + 31, columns - 1) / group;
  const int open_until = tree ? past - 1 : min(c.positions[wave_first], key_last);
  const int wave_until = tree ? key_last : min(c.positions[wave_last], key_last);
  floatx16 o_acc[TD];
#pragma unroll
  for (int db = 0; db < TD; ++db)
#pragma unroll
    for (int e = 0; e < 16; ++e) o_acc[db][e] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  const int block = wave / SHARE, of_block = wave % SHARE;
  // ---- one tile on its way: a wave brings a block of 16 entries of it, or half of one, one page lookup a wave; the 16 rows of K are one run
  // of bytes in their page, V^T is D runs of 16 entries. Every lane issues the same loads for every tile, under no condition: a block that
  // is outside the entries reads the start of the cache and is cleared when it is stored.
  constexpr int PIECES = D * static_cast<int>(sizeof(C));          // of 16 bytes, of K and of V^T
  constexpr int AT_ONCE = DISTIE_WAVE * SHARE;
  constexpr int PASSES = (PIECES + AT_ONCE - 1) / AT_ONCE;
  constexpr int OF_ROW = PIECES / 16;                              // pieces of a row of K
  constexpr int IN_PIECE = 16 / static_cast<int>(sizeof(C));       // entries or dimensions of a piece
  uint4 k_stage[PASSES], v_stage[PASSES];
  uint32_t k_power[PASSES];
  uint32_t v_power = 0;
  // where in its block a lane's pieces lie, in bytes: the same for every tile, beside a base that is the same for the wave. (Where all
  // lanes have a piece in every pass, a pass lies a fixed way behind the one before and needs no register of its own.)
  constexpr int EACH = static_cast<int>(sizeof(C));
  constexpr bool EVEN = PIECES % AT_ONCE == 0;
  const int first_piece = lane + DISTIE_WAVE * of_block;
  const auto piece_of = [&](int p) { return min(first_piece + p * AT_ONCE, PIECES - 1); };
  uint32_t k_off[EVEN ? 1 : PASSES], v_off[EVEN ? 1 : PASSES], k_power_off[PASSES];
#pragma unroll
  for (int p = 0; p < (EVEN ? 1 : PASSES); ++p) {
    const int j = piece_of(p);
    k_off[p] = 16 * j;
    v_off[p] = (j / EACH * c.block_size + IN_PIECE * (j % EACH)) * EACH;
  }
#pragma unroll
  for (int p = 0; p < PASSES; ++p) k_power_off[p] = piece_of(p) / OF_ROW;
  const uint32_t v_power_off = lane % 16;
  const auto live = [&](int entry) { return entry <= key_last && entry + 15 >= key_first; };
  const auto lookup = [&](int k0) {
    const int entry = k0 + 16 * block;
    const int slot = u.shift >= 0 ? entry >> u.shift : entry / c.block_size;
    // (a vector load: a scalar one, which the compiler would make of it, shares its counter with the reads of LDS, and each of those would wait for it)
    int lane_index = min(slot, c.table_width - 1);
    asm volatile("" : "+v"(lane_index));
    return table[lane_index];
  };
  const auto fetch = [&](int k0, int page_in_lanes) {
    const int page = __builtin_amdgcn_readfirstlane(page_in_lanes);
    const int entry = k0 + 16 * block;
    const bool there = live(entry);
    const int at = there ? (u.shift >= 0 ? entry & (c.block_size - 1) : entry % c.block_size) : 0;
    const int64_t held = there ? min(static_cast<int64_t>(max(page, 0)), c.pages - 1) : 0;
    const int64_t base = (held * c.kv_heads + kh) * c.block_size;
    const char* k_block = reinterpret_cast<const char*>(static_cast<const C*>(c.k) + (base + at) * D);
    const char* v_block = reinterpret_cast<const char*>(static_cast<const C*>(c.v) + base * D + at);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int64_t v_pass = static_cast<int64_t>(p) * AT_ONCE * c.block_size;          // of rows of V^T, AT_ONCE / EACH each
      k_stage[p] = *reinterpret_cast<const uint4*>(EVEN ? k_block + 16 * AT_ONCE * p + k_off[0] : k_block + k_off[p]);
      v_stage[p] = *reinterpret_cast<const uint4*>(EVEN ? v_block + v_pass + v_off[0] : v_block + v_off[p]);
      if constexpr (sizeof(C) == 1) k_power[p] = (c.k_scale + base + at)[k_power_off[p]];
    }
    if constexpr (sizeof(C) == 1) v_power = (c.v_scale + base + at)[v_power_off];
  };
  // whether every column of the workgroup sees all of a block
  const int last_pos = tree ? past + n - 1 : c.positions[last_token];
  const auto block_open = [&](int entry) {
    return (tree ? entry + 15 < past : entry + 15 <= first_pos) && (c.window == 0 || entry > last_pos - c.window);
  };
  const auto stash = [&](int k0, TileLds& to) {
    const int entry = k0 + 16 * block;                       // the same for the whole wave: the branches are uniform
    const bool there = live(entry), whole = there && entry + 15 <= key_last;
    const bool open = block_open(entry);
    uint32_t found = 0;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int j = first_piece + p * AT_ONCE;
      if (!EVEN && j >= PIECES) continue;
      const int row = j / OF_ROW;                           // its entry, with bits 2 and 3 swapped
      bf16_t* k_to = to.k + (16 * block + (row & 3) + (row & 4) * 2 + (row & 8) / 2) * K_STRIDE + IN_PIECE * (j % OF_ROW);
      bf16_t* v_to = to.v + j / static_cast<int>(sizeof(C)) * V_STRIDE + 16 * block + IN_PIECE * (j % static_cast<int>(sizeof(C)));
      uint4 k = k_stage[p], v = v_stage[p];
      if (!whole) {
        // behind the last entry is what no request has written, or another one has: cleared (a weight of zero times NaN is NaN)
        if (!there) k = uint4{0u, 0u, 0u, 0u};
        const int written = there ? key_last - (entry + IN_PIECE * (j % static_cast<int>(sizeof(C)))) + 1 : 0;          // of this piece's entries
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          constexpr int EACH = 4 / static_cast<int>(sizeof(C));
          const int left = written - EACH * i;
          w[i] = left >= EACH ? w[i] : left <= 0 ? 0u : w[i] & ((1u << (8 * static_cast<int>(sizeof(C)) * left)) - 1u);
        }
        v = uint4{w[0], w[1], w[2], w[3]};
      }
      if (!open) {
        // what is not finite among entries that not all columns see: the pass behind the walk puts it where it is seen
        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t values = odd_values<C>(w[i]);
          found |= values;
          w[i] &= ~values;
        }
        v = uint4{w[0], w[1], w[2], w[3]};
      }
      if constexpr (sizeof(C) == 1) {
        const float power = power_of(k_power[p]);
        reinterpret_cast<bf16x8*>(k_to)[0] = of_codes(k.x, k.y, power);
        reinterpret_cast<bf16x8*>(k_to)[1] = of_codes(k.z, k.w, power);
        reinterpret_cast<bf16x8*>(v_to)[0] = of_codes(v.x, v.y, 1.f);
        reinterpret_cast<bf16x8*>(v_to)[1] = of_codes(v.z, v.w, 1.f);
      } else {
        *reinterpret_cast<uint4*>(k_to) = k;
        *reinterpret_cast<uint4*>(v_to) = v;
      }
    }
    if constexpr (sizeof(C) == 1) {
      if (lane < 16 && of_block == 0) to.powers[16 * block + lane] = there && entry + lane <= key_last ? power_of(v_power) : 0.f;        // (255 would be an infinity)
    }
    if (__any(found != 0) && lane == 0) *odd = 1;
  };

  const auto compute = [&](int k0, const TileLds& from) {
    if (idle || k0 > wave_until) return;
    floatx16 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) s[kb][e] = 0.f;
    {
      bf16x8 a[2 * TK];
#pragma unroll
      for (int i = 0; i < 2 * TK; ++i) a[i] = *reinterpret_cast<const bf16x8*>(from.k + (32 * (i % 2) + col_lane) * K_STRIDE + 16 * (i / 2) + 8 * h);
#pragma unroll
      for (int i = 0; i < 2 * TK; ++i) s[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], q_reg[i / 2], s[i % 2], 0, 0, 0);
      constexpr int ahead = 2 * TK < AHEAD ? 2 * TK : AHEAD;
      __builtin_amdgcn_sched_group_barrier(0x100, ahead, 0);
#pragma unroll
      for (int i = 0; i < 2 * TK - ahead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, ahead, 0);
    }
    bool open = k0 + TILE - 1 <= open_until;
    if (c.window > 0) open = open && __all(k0 > pos - c.window);
    if (!open) {
      const word_t own = sixty_four_seen(c, token, pos, begin, past, n, k0) >> (8 * h);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (!(own >> (32 * kb + 16 * (e / 8) + e % 8) & 1ull)) s[kb][e] = -INFINITY;
    }
    // The running reference m of a column follows its largest score only when that has grown by more than GROW since m was set: then the
    // sums so far are scaled down, for all columns of the wave at once. In between a weight may reach 2^GROW, which float32 sums and
    // bfloat16 weights hold as well as they hold 1.
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[kb][e]);
    top = lanes_max<32>(top);
    const float best = top * scale_log2;                  // the scale is positive: the largest stays the largest
    if (__any(best > m_run + GROW)) {                     // also the first score of a column (m = -inf)
      const float m_new = fmaxf(m_run, best);
      const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int db = 0; db < TD; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) o_acc[db][e] *= alpha;
    }
    const float shift = m_run == -INFINITY ? 0.f : -m_run;
    bf16x8 p_reg[4];                                      // step t: entries 16 t + 8 h .. + 7
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      floatx4 powers[2];
      if constexpr (sizeof(C) == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) powers[i] = *reinterpret_cast<const floatx4*>(from.powers + 16 * t + 8 * h + 4 * i);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float p = fast_exp2(fmaf(s[t / 2][8 * (t % 2) + e], scale_log2, shift));
        sum += p;
        if constexpr (sizeof(C) == 1) p *= powers[e / 4][e % 4];
        p_reg[t][e] = static_cast<bf16_t>(p);
      }
    }
    l_run += sum;
    {
      bf16x8 vt[4 * TD];
#pragma unroll
      for (int i = 0; i < 4 * TD; ++i) vt[i] = *reinterpret_cast<const bf16x8*>(from.v + (32 * (i % TD) + col_lane) * V_STRIDE + 16 * (i / TD) + 8 * h);
#pragma unroll
      for (int i = 0; i < 4 * TD; ++i) o_acc[i % TD] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vt[i], p_reg[i / TD], o_acc[i % TD], 0, 0, 0);
      constexpr int ahead = 4 * TD < AHEAD ? 4 * TD : AHEAD;
      __builtin_amdgcn_sched_group_barrier(0x100, ahead, 1);
#pragma unroll
      for (int i = 0; i < 4 * TD - ahead; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 1);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, ahead, 1);
    }
  };

  // with several shares the entries are walked in parts, one workgroup each (the last takes what is left)
  const int walks = walks_of_tile(c, u, past, n, last_token - begin);
  const int walk_begin = key_first / TILE * TILE + share * u.length, walk_end = share == walks - 1 ? key_last : min(key_last, walk_begin + u.length - 1);
  if (u.shares > 1 && h == 0 && wave_col0 + col_lane < columns) {
    // parts without an entry: the merge reads no sums where the denominator is zero
    float* states = u.part_ml + 2 * (token * c.heads + head) * u.shares;
    if (walk_begin > walk_end) *reinterpret_cast<float2*>(states + 2 * share) = float2{-INFINITY, 0.f};
    if (share == walks - 1)
      for (int z = walks; z < u.shares; ++z) *reinterpret_cast<float2*>(states + 2 * z) = float2{-INFINITY, 0.f};
  }
  if (walk_begin > walk_end && u.shares > 1) return;
  if (threadIdx.x == 0) *odd = 0;
  __syncthreads();
  if (walk_begin <= walk_end) {
    fetch(walk_begin, lookup(walk_begin));
    int page = lookup(walk_begin + TILE);
    stash(walk_begin, lds[0]);
    fetch(walk_begin + TILE, page);
    page = lookup(walk_begin + 2 * TILE);
    int place = 0;
    for (int k0 = walk_begin; k0 <= walk_end; k0 += TILE, place ^= 1) {
      __syncthreads();                       // this tile is stored, and every wave is done with the one before
      if (k0 + TILE <= walk_end) stash(k0 + TILE, lds[place ^ 1]);
      fetch(k0 + 2 * TILE, page);            // (under a condition its results would be waited for where the branches meet)
      page = lookup(k0 + 3 * TILE);
      compute(k0, lds[place]);
    }
  }
  __syncthreads();
  if (*odd && !idle) {
#pragma unroll 1
    for (int j = max(walk_begin, key_first); j <= walk_end; ++j) {
      if (block_open(j / 16 * 16)) continue;
      const bool seen = sees(c, token, pos, begin, past, j);
#pragma unroll
      for (int db = 0; db < TD; ++db)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = value_at<C>(c, table, kh, j, 32 * db + 8 * (e / 4) + 4 * h + e % 4);
          if (seen && !(fabsf(v) < INFINITY)) o_acc[db][e] += v;
        }
    }
  }
  // ---- write: the lane holds, of its column, output rows 32 db + 8 i + 4 h + (0..3)
  l_run = lanes_sum<32>(l_run);
  if (wave_col0 + col_lane >= columns) return;
  if (u.shares == 1) {
    bf16_t* out = static_cast<bf16_t*>(c.out) + (token * c.heads + head) * D;
    const float inverse = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll
    for (int db = 0; db < TD; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bf16x2 pair[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) pair[j / 2][j % 2] = static_cast<bf16_t>(o_acc[db][4 * i + j] * inverse);
        *reinterpret_cast<uint2*>(out + 32 * db + 8 * i + 4 * h) = uint2{__builtin_bit_cast(uint32_t, pair[0]), __builtin_bit_cast(uint32_t, pair[1])};
      }
  } else {
    const int64_t part = (token * c.heads + head) * u.shares + share;
    float* out = u.part_o + part * D;
#pragma unroll
    for (int db = 0; db < TD; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<floatx4*>(out + 32 * db + 8 * i + 4 * h) = floatx4{o_acc[db][4 * i], o_acc[db][4 * i + 1], o_acc[db][4 * i + 2], o_acc[db][4 * i + 3]};
    if (h == 0) *reinterpret_cast<float2*>(u.part_ml + 2 * part) = float2{m_run, l_run};
  }
}

template <typename C, int WAVES>
int launch_tiles(const Call& c, const Runs& u, hipStream_t stream) {
  constexpr size_t lds = 2 * sizeof(TileLds) + 16;
  if constexpr (lds > 65536) {
    // (asked for once a device; asking twice does no harm)
    static std::atomic<uint64_t> asked{0};
    int device = 0;
    hipError_t status = hipGetDevice(&device);
    if (status != hipSuccess) return static_cast<int>(status);
    if (device >= 64 || !(asked.load() >> device & 1)) {
      status = hipFuncSetAttribute(reinterpret_cast<const void*>(attn_tiles_kernel<C, WAVES>), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
      if (status != hipSuccess) return static_cast<int>(status);
      if (device < 64) asked.fetch_or(1ull << device);
    }
  }
  attn_tiles_kernel<C, WAVES><<<c.kv_heads * u.tiles, DISTIE_WAVE * WAVES, lds, stream>>>(c, u);
  int status = launch_status();
  if (status != 0 || u.shares == 1) return status;
  return launch_merge<bf16_t>(c, u, stream);
}
#endif

}  // namespace

// The largest number of shares of `distie_cache_attention_runs`; 0: this head size has the plainest kernel only.
extern "C" int distie_cache_attention_shares() {
#ifdef DISTIE_FAST_CACHE_ATTENTION
  return MOST_SHARES;
#else
  return 0;
#endif
}

constexpr int MOST_PAGE = 1 << 20;          // entries: offsets inside a page are kept in 32 bits

static bool call_of(Call* c, const void* q, int64_t q_stride, const void* k, const void* v, const uint8_t* k_scale, const uint8_t* v_scale,
                    const int32_t* positions, const int32_t* token_request, const int32_t* cu_q, const int32_t* kv_len, const int32_t* table,
                    int table_width, const int32_t* table_rows, const void* visible, int words, void* out, int tokens, int requests, int heads,
                    int kv_heads, int block_size, int64_t pages, float scale, int window) {
  *c = Call{q, q_stride, k, v, k_scale, v_scale, positions, token_request, cu_q, kv_len, table, table_width, table_rows,
            static_cast<const word_t*>(visible), words, out, tokens, requests, heads, kv_heads, block_size, pages, scale, window};
  return heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && heads <= 65535 && block_size >= 1 && pages >= 1 && table_width >= 1 &&
         requests >= 1 && requests <= 65535 && block_size <= MOST_PAGE && window >= 0 && scale > 0.f && (visible == nullptr || words >= 1);
}

#define CALL_ARGUMENTS                                                                                                                    \
  const void *q, int dtype, int64_t q_stride, const void *k, const void *v, int cache_type, const uint8_t *k_scale, const uint8_t *v_scale, \
      const int32_t *positions, const int32_t *token_request, const int32_t *cu_q, const int32_t *kv_len, const int32_t *table,              \
      int table_width, const int32_t *table_rows, const void *visible, int words, void *out, int tokens, int requests, int heads,            \
      int kv_heads, int block_size, int64_t pages, float scale, int window
#define CALL_OF(c)                                                                                                                         \
  call_of(&c, q, q_stride, k, v, k_scale, v_scale, positions, token_request, cu_q, kv_len, table, table_width, table_rows, visible, words, \
          out, tokens, requests, heads, kv_heads, block_size, pages, scale, window)

extern "C" int distie_cache_attention_any(CALL_ARGUMENTS, hipStream_t stream) {
  Call c;
  if (tokens <= 0) return 0;
  if (!CALL_OF(c) || (cache_type == DISTIE_E4M3) != (k_scale != nullptr && v_scale != nullptr)) return DISTIE_BAD_ARGUMENT;
  DISTIE_DISPATCH(dtype, T, return launch_any<T>(c, cache_type, stream));
}

// Requests that bring `least` to `most` tokens, in tiles of 16 columns. `shares`
// workgroups of four waves along a request's entries, `length` entries a wave; with more than one, part_o (float32 [rows, heads, shares, D]) and part_ml ([rows, heads, shares, 2])
// hold the parts in between, a row a token or, with `by_request` (then least = most = 1), a request. `dense`: all requests bring one token.
extern "C" int distie_cache_attention_runs(CALL_ARGUMENTS, int least, int most, int shares, int length, int by_request, int dense, float* part_o,
                                           float* part_ml, hipStream_t stream) {
#ifdef DISTIE_FAST_CACHE_ATTENTION
  Call c;
  if (tokens <= 0) return 0;
  if (!CALL_OF(c) || (cache_type == DISTIE_E4M3) != (k_scale != nullptr && v_scale != nullptr) || block_size % 16 != 0 || least < 1 || most < least ||
      shares < 1 || shares > MOST_SHARES || (shares > 1 && (part_o == nullptr || part_ml == nullptr)) || ((by_request || dense) && most != 1) || (dense && (tokens != requests || visible != nullptr)) || length < 64 || length % 64 != 0 ||
      (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_scale) |
       reinterpret_cast<uintptr_t>(v_scale) | static_cast<uintptr_t>(q_stride * (dtype == DISTIE_F32 ? 4 : 2))) % 16 != 0)
    return DISTIE_BAD_ARGUMENT;
  const int64_t tiles = (static_cast<int64_t>(most) * (heads / kv_heads) + 15) / 16;
  if (tiles * kv_heads > 0x7fffffff) return DISTIE_BAD_ARGUMENT;
  const int shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  const Runs u{shares, length, static_cast<int>(tiles), least, most, by_request, dense, shift, part_o, part_ml};
  if (dtype == DISTIE_BF16 && cache_type == DISTIE_E4M3) return launch_runs_of<bf16_t, code_t>(c, u, stream);
  if (dtype == DISTIE_BF16 && cache_type == DISTIE_BF16) return launch_runs_of<bf16_t, bf16_t>(c, u, stream);
  if (dtype == DISTIE_F32 && cache_type == DISTIE_E4M3) return launch_runs_of<float, code_t>(c, u, stream);
  if (dtype == DISTIE_F32 && cache_type == DISTIE_F32) return launch_runs_of<float, float>(c, u, stream);
#endif
  return DISTIE_BAD_ARGUMENT;
}

// Requests that bring `least` to `most` tokens, in tiles of `columns` = 128 or (head sizes of up to 128) 256 columns; bfloat16. Shares (of `length` entries) and parts as above, a row a token.
extern "C" int distie_cache_attention_tiles(CALL_ARGUMENTS, int least, int most, int columns, int items, int shares, int length, float* part_o,
                                            float* part_ml, hipStream_t stream) {
#ifdef DISTIE_FAST_CACHE_ATTENTION
  Call c;
  if (tokens <= 0) return 0;
  if (!CALL_OF(c) || (cache_type == DISTIE_E4M3) != (k_scale != nullptr && v_scale != nullptr) || block_size % 16 != 0 || least < 1 || most < least ||
      shares < 1 || shares > MOST_SHARES || (shares > 1 && (part_o == nullptr || part_ml == nullptr)) || dtype != DISTIE_BF16 || kv_heads > 65535 || (columns != 128 && (columns != 256 || D > 128)) || length < TILE || length % TILE != 0 ||
      (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | static_cast<uintptr_t>(q_stride * 2)) % 16 != 0)
    return DISTIE_BAD_ARGUMENT;
  if (items < 1 || items > 0x7fffffff / kv_heads) return DISTIE_BAD_ARGUMENT;
  const int shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
  const Runs u{shares, length, items, least, most, 0, 0, shift, part_o, part_ml};
  if constexpr (D <= 128) {
    if (columns == 256 && cache_type == DISTIE_E4M3) return launch_tiles<code_t, 8>(c, u, stream);
    if (columns == 256 && cache_type == DISTIE_BF16) return launch_tiles<bf16_t, 8>(c, u, stream);
  }
  if (cache_type == DISTIE_E4M3) return launch_tiles<code_t, 4>(c, u, stream);
  if (cache_type == DISTIE_BF16) return launch_tiles<bf16_t, 4>(c, u, stream);
#endif
  return DISTIE_BAD_ARGUMENT;
}
