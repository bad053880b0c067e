// A cache of keys and values in 8 bits: written behind the rotation, read back, and (for a cache of any type) the entries of an
// accepted path of drafted tokens moved to their places.
//
// A row x of D values (the key or the value of one token and kv head) is kept as codes c (e4m3: 4 significant bits, largest 448)
// and one power of two: e is the smallest with max|x| <= 448 * 2^e (within -126..127), c = e4m3(x * 2^-e) rounded to nearest, ties
// to even, and the byte e + 127. x * 2^-e is exact, so the code's rounding is the only one, and c * 2^e is exact in bfloat16. A
// float scale would fill the code's range better, but a floating-point code gains nothing from that. Values that are not
// finite become the code NaN and are left out of the maximum.
//
// Layout: k [pages, kv_heads, P, D], v [pages, kv_heads, D, P] (one byte a value), powers [pages, kv_heads, P] each.

#include "vector_values.h"

typedef uint8_t code_t;
typedef __attribute__((__vector_size__(2 * sizeof(float)))) float floatx2;

constexpr int MOST_DIMS = 1024;

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
  const dim3 grid(tokens, heads + 2 * kv_heads);
  DISTIE_DISPATCH(dtype, S, DISTIE_DISPATCH(out_dtype, T, (rope_kv_write_e4m3_any_kernel<S, T><<<grid, DISTIE_WAVE, 0, stream>>>(
      static_cast<const S*>(qkv), row_stride, slices, slice_stride, static_cast<T*>(q_out), positions, slots, static_cast<code_t*>(k_cache),
      static_cast<code_t*>(v_cache), k_scale, v_scale, inv_freq, pairs, heads, kv_heads, dim, block_size, pages * block_size, write))));
  return launch_status();
}

// Entries read back: for slot n the values of k and v, [count, kv_heads, dim] each. A slot outside the cache gives zeros.
template <typename T>
__global__ __launch_bounds__(256) void read_kv_e4m3_kernel(const code_t* __restrict__ k_cache, const code_t* __restrict__ v_cache,
                                                           const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale,
                                                           const int32_t* __restrict__ slots, T* __restrict__ k_out, T* __restrict__ v_out,
                                                           int kv_heads, int dim, int block_size, int64_t places) {
  const int64_t n = blockIdx.x, head = blockIdx.y, slot = slots[n];
  const bool inside = slot >= 0 && slot < places;
  const int64_t page = inside ? slot / block_size : 0, at = inside ? slot % block_size : 0, base = page * kv_heads + head;
  const float k_power = power_of(k_scale[base * block_size + at]), v_power = power_of(v_scale[base * block_size + at]);
  for (int d = threadIdx.x; d < dim; d += blockDim.x) {
    const float k = value_of(k_cache[(base * block_size + at) * dim + d]) * k_power;
    const float v = value_of(v_cache[(base * dim + d) * block_size + at]) * v_power;
    k_out[(n * kv_heads + head) * dim + d] = from_float<T>(inside ? k : 0.f);
    v_out[(n * kv_heads + head) * dim + d] = from_float<T>(inside ? v : 0.f);
  }
}

extern "C" int distie_read_kv_e4m3(const void* k_cache, const void* v_cache, const uint8_t* k_scale, const uint8_t* v_scale,
                                   const int32_t* slots, void* k_out, void* v_out, int dtype, int count, int kv_heads, int dim,
                                   int block_size, int64_t pages, hipStream_t stream) {
  if (count <= 0) return 0;
  if (kv_heads < 1 || kv_heads > 65535 || dim < 1 || block_size < 1 || pages < 1) return DISTIE_BAD_ARGUMENT;
  const dim3 grid(count, kv_heads);
  DISTIE_DISPATCH(dtype, T, (read_kv_e4m3_kernel<T><<<grid, dim < 256 ? 128 : 256, 0, stream>>>(
      static_cast<const code_t*>(k_cache), static_cast<const code_t*>(v_cache), k_scale, v_scale, slots, static_cast<T*>(k_out),
      static_cast<T*>(v_out), kv_heads, dim, block_size, pages * block_size)));
  return launch_status();
}

// slab [layers, pages, outer, P, inner] of values of sizeof(U) bytes: of request b the entry of position past[b] + path[b, d] goes
// to past[b] + d, for d = 0, 1, ... A path rises, so path[b, d] >= d and what a thread still has to read lies behind what it has written: every
// thread moves its own value of all entries, one behind the other, and nothing is shared. The path ends at its first entry that
// does not rise or is negative, or whose place is outside the request's pages.
template <typename U>
__global__ __launch_bounds__(256) void keep_drafted_kernel(U* __restrict__ slab, const int32_t* __restrict__ table, int table_width,
                                                           const int32_t* __restrict__ table_rows, const int32_t* __restrict__ past,
                                                           const int32_t* __restrict__ path, int length, int64_t pages, int64_t outer,
                                                           int block_size, int64_t inner, int64_t values) {
  const int request = blockIdx.y;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;          // (layer, outer, inner)
  if (i >= values) return;
  const int64_t in = i % inner, out = i / inner % outer, layer = i / inner / outer;
  const int32_t* row = table + static_cast<int64_t>(table_rows != nullptr ? table_rows[request] : request) * table_width;
  const int64_t begin = past[request];
  if (begin < 0) return;
  U* base = slab + layer * pages * outer * block_size * inner + out * block_size * inner + in;
  int before = -1;
  for (int d = 0; d < length; ++d) {
    const int source = path[static_cast<int64_t>(request) * length + d];
    if (source <= before) return;
    before = source;
    const int64_t from = begin + source, to = begin + d;
    if (from / block_size >= table_width) return;
    const int64_t from_page = row[from / block_size], to_page = row[to / block_size];
    if (from_page < 0 || from_page >= pages || to_page < 0 || to_page >= pages) return;
    if (source != d)
      base[(to_page * outer * block_size + to % block_size) * inner] = base[(from_page * outer * block_size + from % block_size) * inner];
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
