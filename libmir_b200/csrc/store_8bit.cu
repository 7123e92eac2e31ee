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
// Few tokens are bound by the chain of loads (slots, rows, stores: 6 us for 8 tokens with the launch), many by the bytes, 2 an element
// read and 1 written: 5,000 tokens of 8 heads of 128 (31 MB, 4.7 us at the copy rate) take 11 us, 2.8 TB/s: each warp reads all its
// rows before it writes the first.  Where a token's run of its page begins is looked up by a lane for each token at once (one after the
// other, with the divisions by the page size, and 16 warps a block, that took 29 us).
#include "eight_bit.cuh"

using namespace mir;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kWarps = 4;
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

// TEAM: warps that share a run's rows, 1 or the block's.  (Seven blocks an SM: 72 registers cost a spill or two, 86 left five blocks and
// took 37 us for 16,384 tokens instead of 29.)
template <int HEAD_DIM, int TEAM>
__global__ void __launch_bounds__(kWarps * 32, 7)
store_8bit_kernel(const bf16* __restrict__ qkv, long long stride, const int* __restrict__ slots, uint8_t* __restrict__ k_pages,
                  uint8_t* __restrict__ v_pages, float* __restrict__ k_scales, float* __restrict__ v_scales, int tokens,
                  int tokens_per_block, int page_size, int pages, int heads, int kv_heads) {
  constexpr int kColumns = HEAD_DIM / 32;
  typedef typename Piece<kColumns>::Raw Raw;
  typedef typename Piece<kColumns>::Codes Codes;
  __shared__ uint32_t largest[TEAM];
  grid_dependency_wait();
  grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = TEAM == 1 ? (int)blockIdx.y * kWarps + warp : (int)blockIdx.y;      // k heads, then v heads
  const int mine = TEAM == 1 ? 0 : warp * kHeld;                  // this warp's first row of a run (or of a page)
  if (unit >= 2 * kv_heads) return;
  const bool is_v = unit >= kv_heads;
  const int head = is_v ? unit - kv_heads : unit;
  const bf16* source = qkv + (size_t)(heads + unit) * HEAD_DIM + lane * kColumns;
  uint8_t* out = (is_v ? v_pages : k_pages) + (size_t)head * HEAD_DIM + lane * kColumns;
  float* scales = is_v ? v_scales : k_scales;
  const size_t row_bytes = (size_t)kv_heads * HEAD_DIM;
  const int limit = pages * page_size;
  auto page_at = [&](int token, bool& begins) {
    const int slot = token >= 0 && token < tokens ? slots[token] : -1;
    const int page = slot >= 0 && slot < limit ? slot / page_size : -1;     // -1: a row without a slot, or with one that is not there
    begins = page >= 0 && slot == page * page_size;
    return page;
  };
  // Lane l looks at token first - 1 + l; lanes 1 .. tokens_per_block at this warp's tokens, the others at what stands around them.
  const int first = blockIdx.x * tokens_per_block, here = min(tokens, first + tokens_per_block) - first;
  bool begins;
  const int page_here = page_at(first - 1 + lane, begins), page_before = __shfl_up_sync(0xffffffffu, page_here, 1);
  const unsigned begin_bits = __ballot_sync(0xffffffffu, begins), changes = __ballot_sync(0xffffffffu, lane > 0 && page_here != page_before);
  unsigned starts = __ballot_sync(0xffffffffu, lane > 0 && lane <= here && page_here >= 0 && page_here != page_before);
  for (; starts != 0u; starts &= starts - 1u) {
    // the run of tokens that goes to this page, and whether it begins the page
    const int at = __ffs(starts) - 1, token = first - 1 + at, page = __shfl_sync(0xffffffffu, page_here, at);
    const unsigned behind = at == 31 ? 0u : changes & (0xfffffffeu << at);
    const int next = behind == 0u ? 32 : __ffs(behind) - 1;
    int count = next - at;
    bool begun = (begin_bits & (0xffffffffu << at) & (next == 32 ? 0xffffffffu : (1u << next) - 1u)) != 0u;
    for (bool more = next == 32; more;) {
      bool first_place;
      const bool same = page_at(token + count + lane, first_place) == page;
      const unsigned differ = __ballot_sync(0xffffffffu, !same);
      const int taken = differ == 0u ? 32 : __ffs(differ) - 1;
      begun |= __any_sync(0xffffffffu, lane < taken && first_place);
      count += taken;
      more = taken == 32;
    }
    float* scale = scales + (size_t)page * kv_heads + head;
    const float scale_before = begun ? 0.0f : *scale;
    Raw held[kHeld];
    uint32_t bits = 0;
    float x[kColumns];
    for (int base = mine; base < count; base += TEAM * kHeld) {
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
    if (TEAM > 1) {
      if (lane == 0) largest[warp] = bits;
      __syncthreads();                                            // (every warp has read the scale)
#pragma unroll
      for (int i = 0; i < TEAM; ++i) bits = max(bits, largest[i]);
    }
    int exponent = least_scale_exponent(__uint_as_float(bits));
    if (!begun) {
      const int before = scale_exponent_of(scale_before);
      if (before < exponent) {
        const float factor = power_of_two(before - exponent);
        uint8_t* row = out + ((size_t)page * page_size + mine) * row_bytes;
        for (int base = mine; base < page_size; base += TEAM * kHeld, row += TEAM * kHeld * row_bytes) {
          Codes codes[kHeld];
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            if (base + i < page_size) codes[i] = *reinterpret_cast<const Codes*>(row + i * row_bytes);
#pragma unroll
          for (int i = 0; i < kHeld; ++i)
            if (base + i < page_size) *reinterpret_cast<Codes*>(row + i * row_bytes) = rescale(codes[i], factor);
        }
      }
      exponent = max(exponent, before);
    }
    if (TEAM > 1) __syncthreads();                                // the page is at the new scale, `largest` has been read
    else __syncwarp();                                            // every lane has read the scale
    if (lane == 0 && mine == 0) *scale = power_of_two(exponent);
    const float inverse = power_of_two(-exponent);
    for (int base = mine; base < count; base += TEAM * kHeld) {
      if (count > TEAM * kHeld) {                                 // (a run of no more rows than that is still held)
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
  // block looks through 4 or 16 of them (1,024 tokens in pages of 64: 25 us with a block each, 14 with a block for four).
  const int per_block = tokens <= 256 ? 1 : tokens <= 1024 ? 4 : 16;
  // Pages of more rows than a warp holds: a block's warps share them (5,000 tokens, pages of 128: 37 us by one warp each, 25 shared;
  // 1,100 tokens: 33 and 18).
  const bool team = page_size > kHeld;
  const dim3 grid((tokens + per_block - 1) / per_block, team ? 2 * kv_heads : (2 * kv_heads + kWarps - 1) / kWarps);
  auto kernel = head_dim == 128 ? (team ? store_8bit_kernel<128, kWarps> : store_8bit_kernel<128, 1>)
                                : (team ? store_8bit_kernel<64, kWarps> : store_8bit_kernel<64, 1>);
  return mir_launch("store_kv_8bit", kernel, grid, dim3(kWarps * 32), 0, stream, 0, (const bf16*)qkv, stride, slots,
                    (uint8_t*)k_pages, (uint8_t*)v_pages, k_scales, v_scales, tokens, per_block, page_size, pages, heads, kv_heads);
}
