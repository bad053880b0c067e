// A cache of keys and values in 8 bits: written behind the rotation, read back, and (for a cache of any type) the entries of an
// accepted path of drafted tokens moved to their places.
//
// A row x of D values (the key or the value of one token and kv head) is kept as codes c (e4m3: 4 significant bits, largest 448)
// and one power of two: e is the smallest with max|x| <= 448 * 2^e (within -126..127), c = e4m3(x * 2^-e) rounded to nearest, ties
// to even, and the byte e + 127. x * 2^-e is exact, so the code's rounding is the only one, and c * 2^e is exact in bfloat16 (for e
// from -124 on: the smallest code is 2^-9, the smallest bfloat16 number 2^-133). A float scale would fill the code's range better, but a
// floating-point code gains nothing from that. Values that are not finite become the code NaN and are left out of the maximum.
//
// Layout: k [pages, kv_heads, P, D], v [pages, kv_heads, D, P] (one byte a value), powers [pages, kv_heads, P] each.

#include "vector_values.h"

typedef uint8_t code_t;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float floatx2;

constexpr int MOST_DIMS = 1024;
constexpr int MOST_WRITE_DIMS = 256;          // of the kernel that takes rows by groups of lanes

// e + 127 of a row whose largest finite magnitude has the bits `bits`: 448 = 1.75 * 2^8
__device__ __forceinline__ int power_byte(uint32_t bits) {
  const int e = static_cast<int>(bits >> 23) - 135 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -126), 127) + 127;
}
__device__ __forceinline__ float power_of(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }      // 2^(byte - 127)
// 2^-(byte - 127): byte 254 gives the subnormal 2^-127
__device__ __forceinline__ float inverse_power(int byte) { return byte < 254 ? power_of(254 - byte) : __uint_as_float(0x400000u); }
__device__ __forceinline__ float finite_size(float x) {
  const float size = fabsf(x);
  return size < INFINITY ? size : 0.f;            // (also of NaN)
}
__device__ __forceinline__ float no_infinity(float x) { return fabsf(x) < INFINITY ? x : __uint_as_float(0x7fc00000u); }
// four codes, the first in the lowest byte
__device__ __forceinline__ uint32_t codes_of(float a, float b, float c, float d) {
  int word = __builtin_amdgcn_cvt_pk_fp8_f32(no_infinity(a), no_infinity(b), 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(no_infinity(c), no_infinity(d), word, true));
}
__device__ __forceinline__ float value_of(uint32_t code) { return __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(code), false)[0]; }

// cos and sin of position * frequency: the angle in 64 bits (in 32 it is off by 2^-24 of itself, 0.004 at position 65,536), both
// rounded once
__device__ __forceinline__ float2 turn_of(int position, float frequency) {
  double s, c;
  sincos(static_cast<double>(position) * static_cast<double>(frequency), &s, &c);
  return float2{static_cast<float>(c), static_cast<float>(s)};
}
// each product rounded before the difference: the bits of the plain formula
__device__ __forceinline__ float turned(float own, float other, float cos, float sin, bool first) {
  return first ? __fsub_rn(__fmul_rn(own, cos), __fmul_rn(other, sin)) : __fadd_rn(__fmul_rn(own, cos), __fmul_rn(other, sin));
}

// Any head size and rotation: one wave a row (head of q, k or v of a token), its values in LDS.
template <typename S, typename T>
__global__ __launch_bounds__(DISTIE_WAVE) void rope_kv_write_e4m3_any_kernel(
    const S* __restrict__ qkv, int64_t row_stride, int slices, int64_t slice_stride, T* __restrict__ q_out, const int32_t* __restrict__ positions,
    const int32_t* __restrict__ slots, code_t* __restrict__ k_cache, code_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
    uint8_t* __restrict__ v_scale, const float* __restrict__ inv_freq, int pairs, int heads, int kv_heads, int dim, int block_size,
    int64_t places, int write) {
  __shared__ float row[MOST_DIMS];
  const int64_t token = blockIdx.x;
  const int part = blockIdx.y, lane = threadIdx.x;
  const S* from = qkv + token * row_stride + static_cast<int64_t>(part) * dim;
  for (int d = lane; d < dim; d += DISTIE_WAVE) row[d] = slices == 1 ? to_float(from[d]) : sum_strided(from + d, slices, slice_stride);
  __syncthreads();
  if (part < heads + kv_heads) {
    const int position = positions[token];
    for (int i = lane; i < pairs; i += DISTIE_WAVE) {
      const float2 t = turn_of(position, inv_freq[i]);
      const float a = row[i], b = row[i + pairs];
      row[i] = turned(a, b, t.x, t.y, true);
      row[i + pairs] = turned(b, a, t.x, t.y, false);
    }
    __syncthreads();
  }
  if (part < heads) {
    for (int d = lane; d < dim; d += DISTIE_WAVE) q_out[(token * heads + part) * dim + d] = from_float<T>(row[d]);
    return;
  }
  const int64_t slot = slots[token];
  if (!write || slot < 0 || slot >= places) return;
  float most = 0.f;
  for (int d = lane; d < dim; d += DISTIE_WAVE) most = fmaxf(most, finite_size(row[d]));
  const int byte = power_byte(__float_as_uint(wave_max(most)));
  const float inverse = inverse_power(byte);
  const bool key = part < heads + kv_heads;
  const int head = part - heads - (key ? 0 : kv_heads);
  const int64_t page = slot / block_size, at = slot % block_size, base = page * kv_heads + head;
  for (int d = lane; d < dim; d += DISTIE_WAVE) {
    const code_t code = static_cast<code_t>(codes_of(row[d] * inverse, 0.f, 0.f, 0.f) & 0xff);
    if (key) k_cache[(base * block_size + at) * dim + d] = code;
    else v_cache[(base * dim + d) * block_size + at] = code;
  }
  if (lane == 0) (key ? k_scale : v_scale)[base * block_size + at] = static_cast<uint8_t>(byte);
}

// Head sizes of a multiple of 8 up to 256, all of a head rotated or nothing: a row on 4 to 32 neighbouring lanes, a lane V = 8 (or 4) values
// of its first half and as many that they are turned with. Blocks take `tokens_each` tokens of all or some heads of q and k (cosine and sine of a
// token once for all of them, in LDS), or, behind those, 16 tokens of one head of v: their codes turn around in LDS, and a word of
// four entries of one dimension is stored at once where the entries are neighbours in a page.
// What bounds it is memory: 4,102 tokens of 28 heads of 128 and 4 kv heads (71 MB) take 18.1 us, 3.9 TB/s; with a wave a row 55.2, with four values a
// lane and eight tokens a block 23.5. Eight tokens take 4.8 us by themselves and 4.0 in a row of launches, 3.2 of these without angles.
constexpr int WRITE_THREADS = 256;
constexpr int V_TOKENS = 16;
struct WriteShape {
  int tokens_each, parts_each, part_blocks, qk_blocks, lanes, rows;          // rows: of a pass of the block
};

// the largest of `lanes` neighbouring lanes (4 to 32)
__device__ __forceinline__ float group_max(float v, int lanes) {
  v = lanes_max<2>(lanes_max<1>(v));
  if (lanes > 4) v = lanes_max<4>(v);
  if (lanes > 8) v = lanes_max<8>(v);
  if (lanes > 16) v = lanes_max<16>(v);
  return v;
}
template <int V>
__device__ __forceinline__ float most_of(const float x[V], const float y[V]) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) most = fmaxf(most, fmaxf(finite_size(x[i]), finite_size(y[i])));
  return most;
}
// V codes at a place of a multiple of V bytes
template <int V>
__device__ __forceinline__ void store_codes(void* to, const float x[V], float inverse) {
  uint32_t words[V / 4];
#pragma unroll
  for (int i = 0; i < V / 4; ++i) words[i] = codes_of(x[4 * i] * inverse, x[4 * i + 1] * inverse, x[4 * i + 2] * inverse, x[4 * i + 3] * inverse);
  if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = uint2{words[0], words[1]};
  else *reinterpret_cast<uint32_t*>(to) = words[0];
}

template <typename S, typename T, bool SLICED, int V>
__global__ __launch_bounds__(WRITE_THREADS) void rope_kv_write_e4m3_kernel(
    const S* __restrict__ qkv, int64_t row_stride, int slices, int64_t slice_stride, T* __restrict__ q_out, const int32_t* __restrict__ positions,
    const int32_t* __restrict__ slots, code_t* __restrict__ k_cache, code_t* __restrict__ v_cache, uint8_t* __restrict__ k_scale,
    uint8_t* __restrict__ v_scale, const float* __restrict__ inv_freq, int pairs, int tokens, int heads, int kv_heads, int dim, int block_size,
    int64_t places, int write, const WriteShape shape) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int half = dim / 2, lane = threadIdx.x % shape.lanes, at_row = threadIdx.x / shape.lanes;
  const bool works = V * lane < half;                                     // (a head of 96: 6 of 8 lanes)
  const int d = works ? V * lane : 0;
  const auto load = [&](const S* from, float out[V]) {
    if constexpr (SLICED) sum_values<V>(from, slices, slice_stride, out);
    else load_values<V>(from, out);
  };
  if (static_cast<int>(blockIdx.x) < shape.qk_blocks) {
    float2* turns = reinterpret_cast<float2*>(lds);                        // [tokens_each][half]
    const int token0 = blockIdx.x / shape.part_blocks * shape.tokens_each, part0 = blockIdx.x % shape.part_blocks * shape.parts_each;
    const int count = min(shape.tokens_each, tokens - token0), parts = min(shape.parts_each, heads + kv_heads - part0);
    const int rows = count * parts;
    // two rows on their way at once, the first pair in front of the angles
    float a[2][V], b[2][V];
    const auto fetch = [&](int first) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = min(first + u * shape.rows + at_row, rows - 1);
        const S* from = qkv + (token0 + row / parts) * row_stride + static_cast<int64_t>(part0 + row % parts) * dim + d;
        load(from, a[u]);
        load(from + half, b[u]);
      }
    };
    fetch(0);
    if (pairs > 0) {
      for (int i = threadIdx.x; i < count * half; i += WRITE_THREADS) turns[i] = turn_of(positions[token0 + i / half], inv_freq[i % half]);
      __syncthreads();
    }
    for (int first = 0; first < rows; first += 2 * shape.rows) {
      float x[2][V], y[2][V];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][i] = a[u][i], y[u][i] = b[u][i];
      if (first + 2 * shape.rows < rows) fetch(first + 2 * shape.rows);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = first + u * shape.rows + at_row;
        const bool there = row < rows && works;
        const int token = token0 + min(row, rows - 1) / parts, part = part0 + min(row, rows - 1) % parts;
        if (pairs > 0) {
          const float2* turn = turns + (token - token0) * half + d;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float first_half = x[u][i], second = y[u][i];
            x[u][i] = turned(first_half, second, turn[i].x, turn[i].y, true);
            y[u][i] = turned(second, first_half, turn[i].x, turn[i].y, false);
          }
        }
        const float most = group_max(works ? most_of<V>(x[u], y[u]) : 0.f, shape.lanes);
        if (part < heads) {
          T* to = q_out + (static_cast<int64_t>(token) * heads + part) * dim + d;
          if (there) {
            store_values<V>(to, x[u]);
            store_values<V>(to + half, y[u]);
          }
        } else {
          const int64_t slot = slots[token];
          const int byte = power_byte(__float_as_uint(most));
          const float inverse = inverse_power(byte);
          if (there && write && slot >= 0 && slot < places) {
            const int64_t entry = (slot / block_size * kv_heads + part - heads) * block_size + slot % block_size;
            code_t* to = k_cache + entry * dim + d;
            store_codes<V>(to, x[u], inverse);
            store_codes<V>(to + half, y[u], inverse);
            if (lane == 0) k_scale[entry] = static_cast<uint8_t>(byte);
          }
        }
      }
    }
    return;
  }
  // ---- 16 tokens of one head of v
  const int stride = dim + V;                                              // bytes of a row of codes in LDS
  int64_t* entries = reinterpret_cast<int64_t*>(lds + V_TOKENS * (MOST_WRITE_DIMS + 8));          // of each token; -1: not written
  const int block = blockIdx.x - shape.qk_blocks, head = block % kv_heads, token0 = block / kv_heads * V_TOKENS;
  for (int first = 0; first < V_TOKENS; first += shape.rows) {
    const int row = first + at_row, token = min(token0 + row, tokens - 1);
    const S* from = qkv + token * row_stride + static_cast<int64_t>(heads + kv_heads + head) * dim + d;
    float x[V], y[V];
    load(from, x);
    load(from + half, y);
    const int64_t slot = slots[token];
    const int byte = power_byte(__float_as_uint(group_max(works ? most_of<V>(x, y) : 0.f, shape.lanes)));
    const float inverse = inverse_power(byte);
    if (row < V_TOKENS) {
      const bool there = token0 + row < tokens && slot >= 0 && slot < places;
      const int64_t page = there ? slot / block_size : 0, at = there ? slot % block_size : 0;
      if (works) {
        store_codes<V>(lds + row * stride + d, x, inverse);
        store_codes<V>(lds + row * stride + half + d, y, inverse);
      }
      if (lane == 0) {
        // where dimension 0 of the token's entry lies
        entries[row] = there ? (page * kv_heads + head) * dim * block_size + at : -1;
        if (there) v_scale[(page * kv_heads + head) * block_size + at] = static_cast<uint8_t>(byte);
      }
    }
  }
  __syncthreads();
  const uint8_t* codes = reinterpret_cast<const uint8_t*>(lds);
  for (int i = threadIdx.x; i < dim * (V_TOKENS / 4); i += WRITE_THREADS) {
    const int four = i % (V_TOKENS / 4) * 4, dimension = i / (V_TOKENS / 4);
    const int64_t first = entries[four];
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) word |= static_cast<uint32_t>(codes[(four + e) * stride + dimension]) << (8 * e);
    // the places of a page are counted from the start of a row of V^T, so neighbours in memory of one row are neighbours in the page
    const bool together = first >= 0 && block_size % 4 == 0 && first % 4 == 0 && entries[four + 1] == first + 1 && entries[four + 2] == first + 2 &&
                          entries[four + 3] == first + 3;
    if (together) {
      *reinterpret_cast<uint32_t*>(v_cache + first + static_cast<int64_t>(dimension) * block_size) = word;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (entries[four + e] >= 0) v_cache[entries[four + e] + static_cast<int64_t>(dimension) * block_size] = static_cast<code_t>(word >> (8 * e));
    }
  }
}

// qkv: `slices` times [tokens, (heads + 2 kv_heads) dim], added up while they are read (rows row_stride apart, slices slice_stride);
// q_out [tokens, heads dim] in `out_dtype`.
extern "C" int distie_rope_kv_write_e4m3(const void* qkv, int dtype, int64_t row_stride, int slices, int64_t slice_stride, void* q_out, int out_dtype,
                                         const int32_t* positions, const int32_t* slots, void* k_cache, void* v_cache, uint8_t* k_scale,
                                         uint8_t* v_scale, const float* inv_freq, int pairs, int tokens, int heads, int kv_heads, int dim,
                                         int block_size, int64_t pages, int write, hipStream_t stream) {
  if (tokens <= 0) return 0;
  if (heads < 1 || kv_heads < 1 || heads + 2 * kv_heads > 65535 || dim < 1 || dim > MOST_DIMS || block_size < 1 || pages < 1 || slices < 1 || pairs < 0 ||
      2 * pairs > dim || (pairs > 0 && inv_freq == nullptr))
    return DISTIE_BAD_ARGUMENT;
  const int values = dim % 16 == 0 ? 8 : 4;                                  // of each half a lane
  const int64_t each = dtype == DISTIE_F32 ? 4 : 2, piece = values * each < 16 ? values * each : 16;          // bytes of a value, of a load
  const bool aligned = (reinterpret_cast<uintptr_t>(qkv) | static_cast<uintptr_t>(row_stride * each) | static_cast<uintptr_t>(slice_stride * each)) % piece == 0 &&
                       reinterpret_cast<uintptr_t>(q_out) % 16 == 0 && reinterpret_cast<uintptr_t>(k_cache) % 8 == 0 && reinterpret_cast<uintptr_t>(v_cache) % 4 == 0;
  if (dim % 8 == 0 && dim >= 32 && dim <= MOST_WRITE_DIMS && (pairs == 0 || 2 * pairs == dim) && aligned) {
    WriteShape shape;
    const int needed = dim / 2 / values;
    shape.lanes = needed <= 4 ? 4 : needed <= 8 ? 8 : needed <= 16 ? 16 : 32;
    shape.rows = WRITE_THREADS / shape.lanes;
    // few tokens: one a block, and so few heads that two passes' rows fill it; many: all heads of several tokens
    const int parts = heads + kv_heads;
    shape.tokens_each = tokens >= 1024 ? 4 : tokens >= 512 ? 2 : 1;
    shape.parts_each = tokens >= 256 ? parts : min(parts, shape.rows);
    shape.part_blocks = (parts + shape.parts_each - 1) / shape.parts_each;
    const int64_t qk = static_cast<int64_t>((tokens + shape.tokens_each - 1) / shape.tokens_each) * shape.part_blocks;
    const int64_t all = qk + (write ? static_cast<int64_t>((tokens + V_TOKENS - 1) / V_TOKENS) * kv_heads : 0);
    if (all <= 0x7fffffff) {
      shape.qk_blocks = static_cast<int>(qk);
      const size_t lds = max(static_cast<size_t>(shape.tokens_each) * dim / 2 * sizeof(float2), static_cast<size_t>(V_TOKENS) * (MOST_WRITE_DIMS + 8 + 8));
#define WRITE(SLICED, V)                                                                                                                  \
  DISTIE_DISPATCH(dtype, S, DISTIE_DISPATCH(out_dtype, T, (rope_kv_write_e4m3_kernel<S, T, SLICED, V><<<static_cast<unsigned>(all), WRITE_THREADS, lds, stream>>>( \
      static_cast<const S*>(qkv), row_stride, slices, slice_stride, static_cast<T*>(q_out), positions, slots, static_cast<code_t*>(k_cache), \
      static_cast<code_t*>(v_cache), k_scale, v_scale, inv_freq, pairs, tokens, heads, kv_heads, dim, block_size, pages * block_size, write, shape))))
      if (slices == 1 && values == 8) WRITE(false, 8);
      else if (slices == 1) WRITE(false, 4);
      else if (values == 8) WRITE(true, 8);
      else WRITE(true, 4);
#undef WRITE
      return launch_status();
    }
  }
  const dim3 grid(tokens, heads + 2 * kv_heads);
  DISTIE_DISPATCH(dtype, S, DISTIE_DISPATCH(out_dtype, T, (rope_kv_write_e4m3_any_kernel<S, T><<<grid, DISTIE_WAVE, 0, stream>>>(
      static_cast<const S*>(qkv), row_stride, slices, slice_stride, static_cast<T*>(q_out), positions, slots, static_cast<code_t*>(k_cache),
      static_cast<code_t*>(v_cache), k_scale, v_scale, inv_freq, pairs, heads, kv_heads, dim, block_size, pages * block_size, write))));
  return launch_status();
}

// Entries read back: for slot n the values of k and v, [count, kv_heads, dim] each. A slot outside the cache gives zeros. A block takes 16
// slots of one kv head; the rows of V^T, 16 entries of a dimension beside each other where the slots are neighbours, turn around in LDS.
constexpr int READ_SLOTS = 16;
constexpr int READ_THREADS = 256;
template <typename T>
__global__ __launch_bounds__(READ_THREADS) void read_kv_e4m3_kernel(const code_t* __restrict__ k_cache, const code_t* __restrict__ v_cache,
                                                                    const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                                                                    const int32_t* __restrict__ slots, T* __restrict__ k_out, T* __restrict__ v_out,
                                                                    int count, int kv_heads, int dim, int block_size, int64_t places) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  int64_t* entry = reinterpret_cast<int64_t*>(lds);                       // [16]: (page, head) * P + place; -1 outside
  int64_t* v_entry = entry + READ_SLOTS;                                   // of dimension 0 in V^T
  float* powers = reinterpret_cast<float*>(v_entry + READ_SLOTS);          // of k, then of v
  uint8_t* codes = reinterpret_cast<uint8_t*>(powers + 2 * READ_SLOTS);     // [16][stride]
  const int stride = (dim + 3) / 4 * 4 + 4;
  const int head = blockIdx.y, first = blockIdx.x * READ_SLOTS, here = min(READ_SLOTS, count - first);
  if (threadIdx.x < READ_SLOTS) {
    const int64_t slot = static_cast<int>(threadIdx.x) < here ? slots[first + threadIdx.x] : -1;
    const bool inside = slot >= 0 && slot < places;
    const int64_t held = (inside ? slot / block_size : 0) * kv_heads + head, at = inside ? slot % block_size : 0;
    entry[threadIdx.x] = inside ? held * block_size + at : -1;
    v_entry[threadIdx.x] = held * dim * block_size + at;
    powers[threadIdx.x] = inside ? power_of(k_scale[held * block_size + at]) : 0.f;
    powers[READ_SLOTS + threadIdx.x] = inside ? power_of(v_scale[held * block_size + at]) : 0.f;
  }
  __syncthreads();
  // four neighbouring entries of a page are one word of a row of V^T
  for (int i = threadIdx.x; i < dim * (READ_SLOTS / 4); i += READ_THREADS) {
    const int four = i % (READ_SLOTS / 4) * 4, d = i / (READ_SLOTS / 4);
    const int64_t begin = v_entry[four];
    const code_t* from = v_cache + static_cast<int64_t>(d) * block_size;
    uint32_t word = 0;
    if (block_size % 4 == 0 && begin % 4 == 0 && v_entry[four + 1] == begin + 1 && v_entry[four + 2] == begin + 2 && v_entry[four + 3] == begin + 3) {
      word = *reinterpret_cast<const uint32_t*>(from + begin);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) word |= static_cast<uint32_t>(from[v_entry[four + e]]) << (8 * e);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) codes[(four + e) * stride + d] = static_cast<uint8_t>(word >> (8 * e));
  }
  if (dim % 4 == 0) {
    const int pieces = dim / 4;
    const auto four = [&](T* to, uint32_t word, float power) {
      const floatx2 low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), false), high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), true);
      const float v[4] = {low[0] * power, low[1] * power, high[0] * power, high[1] * power};
      store_values<4>(to, v);
    };
    for (int i = threadIdx.x; i < here * pieces; i += READ_THREADS) {
      const int n = i / pieces, d = i % pieces * 4;
      const uint32_t word = entry[n] < 0 ? 0u : *reinterpret_cast<const uint32_t*>(k_cache + entry[n] * dim + d);
      four(k_out + (static_cast<int64_t>(first + n) * kv_heads + head) * dim + d, word, powers[n]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < here * pieces; i += READ_THREADS) {
      const int n = i / pieces, d = i % pieces * 4;
      four(v_out + (static_cast<int64_t>(first + n) * kv_heads + head) * dim + d, entry[n] < 0 ? 0u : *reinterpret_cast<const uint32_t*>(codes + n * stride + d),
           powers[READ_SLOTS + n]);
    }
    return;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < here * dim; i += READ_THREADS) {
    const int n = i / dim, d = i % dim;
    const int64_t to = (static_cast<int64_t>(first + n) * kv_heads + head) * dim + d;
    k_out[to] = from_float<T>(entry[n] < 0 ? 0.f : value_of(k_cache[entry[n] * dim + d]) * powers[n]);
    v_out[to] = from_float<T>(entry[n] < 0 ? 0.f : value_of(codes[n * stride + d]) * powers[READ_SLOTS + n]);
  }
}

extern "C" int distie_read_kv_e4m3(const void* k_cache, const void* v_cache, const uint8_t* k_scale, const uint8_t* v_scale,
                                   const int32_t* slots, void* k_out, void* v_out, int dtype, int count, int kv_heads, int dim,
                                   int block_size, int64_t pages, hipStream_t stream) {
  if (count <= 0) return 0;
  if (kv_heads < 1 || kv_heads > 65535 || dim < 1 || dim > MOST_DIMS || block_size < 1 || pages < 1 ||
      reinterpret_cast<uintptr_t>(v_cache) % 4 != 0 ||
      (dim % 4 == 0 && (reinterpret_cast<uintptr_t>(k_cache) % 4 != 0 || (reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16 != 0)))
    return DISTIE_BAD_ARGUMENT;
  const dim3 grid((count + READ_SLOTS - 1) / READ_SLOTS, kv_heads);
  const size_t lds = READ_SLOTS * (2 * sizeof(int64_t) + 2 * sizeof(float) + static_cast<size_t>((dim + 3) / 4 * 4 + 4));
  DISTIE_DISPATCH(dtype, T, (read_kv_e4m3_kernel<T><<<grid, READ_THREADS, lds, stream>>>(
      static_cast<const code_t*>(k_cache), static_cast<const code_t*>(v_cache), k_scale, v_scale, slots, static_cast<T*>(k_out),
      static_cast<T*>(v_out), count, kv_heads, dim, block_size, pages * block_size)));
  return launch_status();
}

// slab [layers, pages, outer, P, inner] of values of sizeof(U) bytes: of request b the entry of position past[b] + path[b, d] goes
// to past[b] + d, for d = 0, 1, ... A path rises, so path[b, d] >= d and what a thread still has to read lies behind what it has written: every
// thread moves its own value of all entries, KEEP_AHEAD of them read in front of the first that is written, and nothing is shared but where
// they lie. The path ends at its first entry that does not rise or is negative, or whose place is outside the request's pages.
constexpr int KEEP_AHEAD = 12;
constexpr int KEEP_MOST = 256;            // entries of a path whose places are worked out at once
template <int N, typename U>
__device__ __forceinline__ void keep_some(U* base, const int64_t* from, const int64_t* to, int first, int end) {
  U held[N];
#pragma unroll
  for (int k = 0; k < N; ++k) held[k] = base[from[min(first + k, end - 1)]];
  loads_first();
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (first + k < end) base[to[first + k]] = held[k];
}
template <typename U>
__global__ __launch_bounds__(256) void keep_drafted_kernel(U* __restrict__ slab, const int32_t* __restrict__ table, int table_width,
                                                           const int32_t* __restrict__ table_rows, const int32_t* __restrict__ past,
                                                           const int32_t* __restrict__ path, int length, int64_t pages, int64_t outer,
                                                           int block_size, int64_t inner, int64_t values) {
  __shared__ int64_t from[KEEP_MOST], to[KEEP_MOST];
  __shared__ int good, still;              // how many entries of the path count, and how many in front of the first that moves
  const int request = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;          // (layer, outer, inner)
  const int64_t in = i % inner, out = i / inner % outer, layer = i / inner / outer;
  const int32_t* row = table + static_cast<int64_t>(table_rows != nullptr ? table_rows[request] : request) * table_width;
  const int32_t* sources = path + static_cast<int64_t>(request) * length;
  const int64_t begin = past[request];
  if (begin < 0) return;
  U* base = slab + layer * pages * outer * block_size * inner + out * block_size * inner + in;
  for (int first = 0; first < length; first += KEEP_MOST) {
    const int count = min(KEEP_MOST, length - first), d = first + threadIdx.x;
    __syncthreads();
    if (threadIdx.x == 0) good = still = count;
    __syncthreads();
    if (static_cast<int>(threadIdx.x) < count) {
      const int source = sources[d], before = d > 0 ? sources[d - 1] : -1;
      const int64_t p = begin + source, q = begin + d;
      // (a path that rises is never behind d; behind its end an entry may be, and the place of d then outside the table)
      bool fine = source > before && source >= d && p / block_size < table_width;
      if (fine) {
        const int64_t p_page = row[p / block_size], q_page = row[q / block_size];
        fine = p_page >= 0 && p_page < pages && q_page >= 0 && q_page < pages;
        from[threadIdx.x] = (p_page * outer * block_size + p % block_size) * inner;
        to[threadIdx.x] = (q_page * outer * block_size + q % block_size) * inner;
      }
      if (!fine) atomicMin(&good, static_cast<int>(threadIdx.x));
      if (source != d) atomicMin(&still, static_cast<int>(threadIdx.x));          // (as long as a path rises, all behind that one move too)
    }
    __syncthreads();
    const int moved = good;
    if (i < values) {
      int e = min(still, moved);
      for (; e + 4 < moved; e += KEEP_AHEAD) keep_some<KEEP_AHEAD>(base, from, to, e, moved);
      if (e < moved) keep_some<4>(base, from, to, e, moved);
    }
    if (moved < count) return;
  }
}

// `unit`: bytes of a value as it is moved (1, 2, 4, 8 or 16); inner counts such values
extern "C" int distie_keep_drafted(void* slab, int unit, const int32_t* table, int table_width, const int32_t* table_rows,
                                   const int32_t* past, const int32_t* path, int requests, int length, int64_t layers, int64_t pages,
                                   int64_t outer, int block_size, int64_t inner, hipStream_t stream) {
  if (requests <= 0 || length <= 0) return 0;
  const int64_t values = layers * outer * inner;
  if (table_width < 1 || layers < 1 || pages < 1 || outer < 1 || block_size < 1 || inner < 1 || requests > 65535 || values > (1LL << 38))
    return DISTIE_BAD_ARGUMENT;
  const dim3 grid(static_cast<unsigned>((values + 255) / 256), requests);
#define KEEP(U)                                                                                                             \
  keep_drafted_kernel<U><<<grid, 256, 0, stream>>>(static_cast<U*>(slab), table, table_width, table_rows, past, path, length, pages, \
                                                   outer, block_size, inner, values)
  switch (unit) {
    case 1: KEEP(uint8_t); break;
    case 2: KEEP(uint16_t); break;
    case 4: KEEP(uint32_t); break;
    case 8: KEEP(uint2); break;
    case 16: KEEP(uint4); break;
    default: return DISTIE_BAD_ARGUMENT;
  }
#undef KEEP
  return launch_status();
}
