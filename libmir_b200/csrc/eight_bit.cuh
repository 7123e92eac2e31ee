// What the kernels of the 8-bit operators share: e4m3 numbers, scales that are powers of two, and the page of a key.
//
// An e4m3 number has four significant bits (the leading one included), 448 is the largest and 2^-9 the smallest.  It and
// its product with a power of two are exact in float16 or bfloat16 wherever that format's range reaches.
#pragma once
#include <cuda_fp8.h>
#include "common.cuh"

namespace mir {

constexpr int kLeastScaleExponent = -118;    // of a scale that is a power of two: its inverse is a number too
constexpr float kLog2e = 1.4426950408889634f;

// 2^e for a whole e; 0 below the normal numbers.
__device__ __forceinline__ float power_of_two(int e) { return e < -126 ? 0.0f : __int_as_float((e + 127) << 23); }

// The exponent of a scale; kLeastScaleExponent for 0 (a page that was never written).
__device__ __forceinline__ int scale_exponent_of(float scale) {
  return max(((__float_as_int(scale) >> 23) & 0xff) - 127, kLeastScaleExponent);
}

// The least e >= kLeastScaleExponent with largest <= 448 * 2^e; `largest` is finite and not negative.  448 is
// 1.75 * 2^8, so the mantissa decides whether the exponent less 8 is enough.
__device__ __forceinline__ int least_scale_exponent(float largest) {
  const int bits = __float_as_int(largest);
  return max((bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0), kLeastScaleExponent);
}

// Two numbers rounded to nearest even to e4m3, beyond 448 (infinities too) to 448; the first in the low byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float first, float second) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(first, second), __NV_SATFINITE, __NV_E4M3);
}
// Two numbers within 448 as e4m3 and what that leaves as e5m2 (the first in the low bytes).
__device__ __forceinline__ __half2 e4m3_low(uint32_t word);
__device__ __forceinline__ void split_e4m3_e5m2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = to_e4m3x2(a, b);
  const float2 taken = __half22float2(e4m3_low(hi));
  lo = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a - taken.x, b - taken.y), __NV_SATFINITE, __NV_E5M2);
}
// The two e4m3 numbers of the low (high) half of a word as float16, exact.
__device__ __forceinline__ __half2 e4m3_low(uint32_t word) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word & 0xffffu), __NV_E4M3));
}
__device__ __forceinline__ __half2 e4m3_high(uint32_t word) {
  return __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word >> 16), __NV_E4M3));
}
// Two of them times a power of two, as packed bfloat16 (exact).
__device__ __forceinline__ uint32_t scaled_bf16(__half2 pair, float scale) {
  const float2 f = __half22float2(pair);
  const __nv_bfloat162 b = __floats2bfloat162_rn(f.x * scale, f.y * scale);
  return *reinterpret_cast<const uint32_t*>(&b);
}

__device__ __forceinline__ float approximate_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A word of e4m3 numbers: whether one of them is NaN; and with zeros in the places of those that are.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t word) { return ((word & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ uint32_t without_nans(uint32_t word) { return word & ~((nan_bytes(word) >> 7) * 0xffu); }

// Two e4m3 numbers (bytes `selector` of `word`, spread with their signs) as bf16 numbers 2^-120 times as large.
template <uint32_t SELECTOR> __device__ __forceinline__ uint32_t lifted(uint32_t word) {
  uint32_t spread;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(spread) : "r"(word), "n"(SELECTOR));
  return (spread << 4) & 0x87f087f0u;
}
__device__ __forceinline__ uint32_t times(uint32_t pair, uint32_t factor) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(pair), "r"(factor));
  return d;
}
// bf16 pair of 2^e, e from -126 to 127.
__device__ __forceinline__ uint32_t power_pair(int e) { return (uint32_t)(e + 127) << 7 | (uint32_t)(e + 127) << 23; }

// The inverse of a query row's scale 2^e for splitting it: NaN where the row holds an infinity, whose scores are no numbers.
__device__ __forceinline__ float query_inverse(float largest, int e) {
  return largest < INFINITY ? power_of_two(-e) : __int_as_float(0x7fffffff);
}

// The tokens of request r among `tokens` rows; what lies beyond them is cut off.
struct Portion {
  int first, count;
};
__device__ __forceinline__ Portion portion_of(const int* query_starts, int r, int tokens) {
  const int first = min(max(query_starts[r], 0), tokens);
  return {first, max(0, min(query_starts[r + 1], tokens) - first)};
}

// The request that the batch's tile `tile` (ROWS rows of one request each) belongs to, which then is the tile of that request; -1 beyond
// the last.  Called by whole warps: 32 requests at a time are passed over together.
template <int ROWS>
__device__ __forceinline__ int request_of_tile(const int* query_starts, int num_rows, int tokens, int group, int& tile, Portion& portion) {
  int r = 0;
  for (; r + 32 < num_rows; r += 32) {
    const int mine = portion_of(query_starts, r + (int)(threadIdx.x & 31), tokens).count;
    const int tiles = __reduce_add_sync(0xffffffffu, (mine * group + ROWS - 1) / ROWS);
    if (tile < tiles) break;
    tile -= tiles;
  }
  for (; r < num_rows; ++r) {
    portion = portion_of(query_starts, r, tokens);
    const int tiles = (portion.count * group + ROWS - 1) / ROWS;
    if (tile < tiles) return r;
    tile -= tiles;
  }
  return -1;
}

// The paged 8-bit cache of one layer.
struct Cache8 {
  const uint8_t* k;              // [pages * page_size, kv_heads, head_dim]
  const uint8_t* v;
  const float* k_scales;         // [pages, kv_heads], powers of two
  const float* v_scales;
  int pages, page_size, kv_heads;
};

// The page of block `block` of a request: -1 where its table ends, has no page, or names one that the pool does not have.
__device__ __forceinline__ int page_of_block(const int* table, int table_width, int block, int pages) {
  if (block >= table_width) return -1;
  const int page = table[block];
  return page >= 0 && page < pages ? page : -1;
}

}  // namespace mir
