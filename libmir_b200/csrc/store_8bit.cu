// Keys and values of a step into the 8-bit cache: e4m3 with one scale, a power of two, per page and kv head.
//
//   largest = max |x| over a page's new elements of the head (finite ones),  e' = the least e with largest <= 448 * 2^e,
//   e = e' if the page is begun (a token goes to its first place), else max(e', the page's exponent so far);
//   new rows: round(clamp(x * 2^-e, +-448));  where e grew, what the page holds already is taken along: round(code * 2^(old - e)).
//
// A scale that is a power of two costs e4m3 no precision (it only moves the exponent), and a page that is taken to a
// larger scale again and again, as single tokens arrive, loses nothing but what falls below 2^-9 of the scale.
//
// One warp takes one head of k or of v of one page: the step's tokens of a page stand side by side (they are one
// request's), and the first of them finds the others.  A lane owns HEAD_DIM / 32 columns, so that a row is one contiguous
// access and no lane ever reads what another one wrote.  The rows' loads are all on their way before the first is used (16
// rows at a time in registers; a longer run is read a second time, from the L2).
// The kernel is bound by its reads, 2 bytes an element against 1 written.
#include "eight_bit.cuh"

using namespace mir;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kWarps = 16;
constexpr int kHeld = 16;       // rows that a warp holds in registers

// COLUMNS consecutive bf16 elements: 4 (8 bytes) or 2 (4 bytes).
template <int COLUMNS> struct Piece;
template <> struct Piece<4> { typedef uint2 Raw; typedef uint32_t Codes; };
template <> struct Piece<2> { typedef uint32_t Raw; typedef uint16_t Codes; };

__device__ __forceinline__ void unpack(uint2 raw, float (&x)[4]) {
  x[0] = __uint_as_float(raw.x << 16);
  x[1] = __uint_as_float(raw.x & 0xffff0000u);
  x[2] = __uint_as_float(raw.y << 16);
  x[3] = __uint_as_float(raw.y & 0xffff0000u);
}
__device__ __forceinline__ void unpack(uint32_t raw, float (&x)[2]) {
  x[0] = __uint_as_float(raw << 16);
  x[1] = __uint_as_float(raw & 0xffff0000u);
}
__device__ __forceinline__ uint32_t round_all(const float (&x)[4], float inverse) {
  return to_e4m3x2(x[0] * inverse, x[1] * inverse) | (to_e4m3x2(x[2] * inverse, x[3] * inverse) << 16);
}
__device__ __forceinline__ uint16_t round_all(const float (&x)[2], float inverse) {
  return (uint16_t)to_e4m3x2(x[0] * inverse, x[1] * inverse);
}
__device__ __forceinline__ uint32_t rescale(uint32_t codes, float factor) {
  const float2 a = __half22float2(e4m3_low(codes)), b = __half22float2(e4m3_high(codes));
  const float x[4] = {a.x, a.y, b.x, b.y};
  return round_all(x, factor);
}
__device__ __forceinline__ uint16_t rescale(uint16_t codes, float factor) {
  const float2 a = __half22float2(e4m3_low(codes));
  const float x[2] = {a.x, a.y};
  return round_all(x, factor);
}
// The bits of the largest finite magnitude (they order as the numbers do).
template <int COLUMNS> __device__ __forceinline__ uint32_t largest_bits(const float (&x)[COLUMNS], uint32_t so_far) {
#pragma unroll
  for (int i = 0; i < COLUMNS; ++i) {
    const uint32_t bits = __float_as_uint(x[i]) & 0x7fffffffu;
    if (bits < 0x7f800000u) so_far = max(so_far, bits);
  }
  return so_far;
}

template <int HEAD_DIM>
__global__ void __launch_bounds__(kWarps * 32)
store_8bit_kernel(const bf16* __restrict__ qkv, long long stride, const int* __restrict__ slots, uint8_t* __restrict__ k_pages,
                  uint8_t* __restrict__ v_pages, float* __restrict__ k_scales, float* __restrict__ v_scales, int tokens,
                  int tokens_per_block, int page_size, int pages, int heads, int kv_heads) {
  constexpr int kColumns = HEAD_DIM / 32;
  typedef typename Piece<kColumns>::Raw Raw;
  typedef typename Piece<kColumns>::Codes Codes;
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.y * kWarps + warp;                    // k heads, then v heads
  if (unit >= 2 * kv_heads) return;
  const bool is_v = unit >= kv_heads;
  const int head = is_v ? unit - kv_heads : unit;
  const bf16* source = qkv + (size_t)(heads + unit) * HEAD_DIM + lane * kColumns;
  uint8_t* out = (is_v ? v_pages : k_pages) + (size_t)head * HEAD_DIM + lane * kColumns;
  float* scales = is_v ? v_scales : k_scales;
  const size_t row_bytes = (size_t)kv_heads * HEAD_DIM;
  const int limit = pages * page_size;
  auto page_of = [&](int token) {
    const int slot = slots[token];
    return slot >= 0 && slot < limit ? slot / page_size : -1;     // a row without a slot, or with one that is not there
  };
  const int first = blockIdx.x * tokens_per_block, last = min(tokens, first + tokens_per_block);
  for (int token = first; token < last; ++token) {
    const int page = page_of(token);
    if (page < 0 || (token > 0 && page_of(token - 1) == page)) continue;
    // the run of tokens that goes to this page, and whether it begins the page
    int count = 0;
    bool begun = false;
    for (bool more = true; more;) {
      const int mine = token + count + lane;
      const bool same = mine < tokens && page_of(mine) == page;
      const unsigned differ = __ballot_sync(0xffffffffu, !same);
      const int taken = differ == 0u ? 32 : __ffs(differ) - 1;
      begun |= __any_sync(0xffffffffu, lane < taken && slots[min(mine, tokens - 1)] % page_size == 0);
      count += taken;
      more = taken == 32;
    }
    Raw held[kHeld];
    uint32_t bits = 0;
    float x[kColumns];
    for (int base = 0; base < count; base += kHeld) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (base + i < count) held[i] = *reinterpret_cast<const Raw*>(source + (size_t)(token + base + i) * stride);
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (base + i < count) {
          unpack(held[i], x);
          bits = largest_bits<kColumns>(x, bits);
        }
    }
    bits = __reduce_max_sync(0xffffffffu, bits);
    float* scale = scales + (size_t)page * kv_heads + head;
    int exponent = least_scale_exponent(__uint_as_float(bits));
    if (!begun) {
      const int before = scale_exponent_of(*scale);
      if (before < exponent) {
        const float factor = power_of_two(before - exponent);
        uint8_t* row = out + (size_t)page * page_size * row_bytes;
        for (int i = 0; i < page_size; ++i, row += row_bytes) {
          Codes* codes = reinterpret_cast<Codes*>(row);
          *codes = rescale(*codes, factor);
        }
      }
      exponent = max(exponent, before);
    }
    __syncwarp();                                                 // every lane has read the scale
    if (lane == 0) *scale = power_of_two(exponent);
    const float inverse = power_of_two(-exponent);
    for (int base = 0; base < count; base += kHeld) {
      if (count > kHeld) {                                        // (a run of at most kHeld rows is still held)
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
          if (base + i < count) held[i] = *reinterpret_cast<const Raw*>(source + (size_t)(token + base + i) * stride);
      }
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (base + i < count) {
          unpack(held[i], x);
          *reinterpret_cast<Codes*>(out + (size_t)slots[token + base + i] * row_bytes) = round_all(x, inverse);
        }
    }
  }
}

}  // namespace

// Tokens' keys and values (columns behind `heads` query heads of the packed bf16 rows, already normed and rotated) into
// their slots; a slot below 0 is no slot.  k_pages, v_pages: [pages * page_size, kv_heads, head_dim] e4m3; the scales:
// [pages, kv_heads].
MIR_EXPORT int mir_store_8bit(const void* qkv, long long stride, const int* slots, void* k_pages, void* v_pages, float* k_scales,
                              float* v_scales, int tokens, int page_size, int pages, int heads, int kv_heads, int head_dim,
                              cudaStream_t stream) {
  if (tokens == 0) return MIR_OK;
  if (tokens < 0 || page_size <= 0 || pages <= 0 || heads < 0 || kv_heads <= 0 || (head_dim != 64 && head_dim != 128) ||
      stride < (long long)(heads + 2 * kv_heads) * head_dim || (stride % 4) || ((uintptr_t)qkv & 7) || ((uintptr_t)k_pages & 3) ||
      ((uintptr_t)v_pages & 3) || (long long)pages * page_size > 0x7fffffffll) {
    mir_set_error("store_kv_8bit: takes head_dim 64 or 128, rows and pages on 8-byte boundaries (head_dim %d, heads %d, kv heads %d, "
                  "page %d, pages %d, row stride %lld)", head_dim, heads, kv_heads, page_size, pages, stride);
    return MIR_BAD_ARGUMENT;
  }
  // Few tokens: a block for each, so that their pages are worked on side by side.  Many: most tokens are no page's first, and a
  // block looks through 16 of them.
  const int per_block = tokens <= 1024 ? 1 : 16;
  const dim3 grid((tokens + per_block - 1) / per_block, (2 * kv_heads + kWarps - 1) / kWarps);
  auto kernel = head_dim == 128 ? store_8bit_kernel<128> : store_8bit_kernel<64>;
  return mir_launch("store_kv_8bit", kernel, grid, dim3(kWarps * 32), 0, stream, 0, (const bf16*)qkv, stride, slots,
                    (uint8_t*)k_pages, (uint8_t*)v_pages, k_scales, v_scales, tokens, per_block, page_size, pages, heads, kv_heads);
}
