// Attention over the 8-bit cache on mma.sync, for every size the operators take (head_dim 64 and 128, any page size), portions and single
// tokens, and the entry points:
//
//   out = sum_j p_j S_v[page of j] V_j / sum_j p_j,   p_j = exp(scale q . (S_k[page of j] K_j) - max)
//
// over the keys j <= position (inside the window, if any) whose page the block table has.  K and V are e4m3, S_k and S_v
// one power of two per page and kv head: a number times its scale is exact in bf16, so a tile of keys and values is
// scaled on its way into shared memory and everything behind that is bf16 attention with 32-bit scores, maxima,
// exponentials and sums (the weights p are rounded to bf16 for the product with V, as in the kernels over bf16 pages).
//
// Portions: a CTA takes 64 rows of one request and one kv head, and one partition of the keys.  A row is a (token, query head of the
// group) pair: all heads of the group share the tile's keys, so that the cache is read once per group.  Four warps of 16
// rows; the next tile's bytes are on their way in registers while this one is worked on.  Partitions' results are joined by
// a second kernel (merge_8bit_kernel), a warp for each token and head.
#include <algorithm>
#include "eight_bit.cuh"
#include "eight_bit.h"

using namespace mir;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kRows = 64, kKeys = 64, kThreads = 128;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float low, float high) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

// Where a partition's keys end: at the last that is seen, the partition's or the block table's.
__device__ __forceinline__ int end_of_keys(long long seen, long long partition_end, int table_width, int page_size) {
  return (int)min(min(seen, partition_end), min((long long)table_width * page_size, 0x7fffff00ll));
}
// Two elements of a query; NaN for an infinity, whose scores are no numbers.
__device__ __forceinline__ uint32_t query_pair(const bf16* from) {
  uint32_t pair = *reinterpret_cast<const uint32_t*>(from);
  if ((pair & 0x7fffu) == 0x7f80u) pair |= 0x7fffu;
  if ((pair & 0x7fff0000u) == 0x7f800000u) pair |= 0x7fff0000u;
  return pair;
}

template <int DIM>
__global__ void __launch_bounds__(kThreads)
attention_8bit_kernel(const bf16* __restrict__ q, long long q_stride, bf16* __restrict__ out, Cache8 cache,
                      const int* __restrict__ block_table, int table_width, const int* __restrict__ query_starts,
                      const int* __restrict__ context_lens, int num_rows, int group,
                      float scale_log2, int window, int partition, int num_partitions, float* __restrict__ partial_o,
                      float* __restrict__ partial_ml, const float* __restrict__ sinks, int all_tokens) {
  constexpr int kStride = DIM + 8;              // bf16 elements of a shared row: an odd number of 16-byte pieces
  constexpr int kPieces = DIM / 16;             // 16-byte pieces of a cached row
  constexpr int kRounds = kKeys * kPieces / kThreads;
  __shared__ __align__(16) bf16 k_tile[kKeys * kStride];
  __shared__ __align__(16) bf16 v_tile[kKeys * kStride];
  __shared__ unsigned long long there_bits[2];  // [tile parity]: keys of the tile whose page the table has
  __shared__ int hidden_nans;                   // whether NaN values were left out that some of the rows see
  grid_dependency_wait();
  grid_launch_dependents();
  const int part = blockIdx.x % num_partitions, tile = blockIdx.x / num_partitions, kv_head = blockIdx.y;
  // the request and its rows
  int remaining = tile;
  Portion portion{0, 0};
  const int request = request_of_tile<kRows>(query_starts, num_rows, all_tokens, group, remaining, portion);
  if (request < 0) return;
  const int first_row = remaining * kRows, first_token = portion.first, count = portion.count, first_position = context_lens[request] - count;
  const int rows = min(kRows, count * group - first_row);
  const int lowest = first_position + first_row / group, highest = first_position + (first_row + rows - 1) / group;
  const int* table = block_table + (size_t)request * table_width;
  const int heads = group * cache.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // this thread's two rows of the accumulators: their tokens and heads
  int token[2], head[2], position[2];
  bool valid[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int local = warp * 16 + lane / 4 + 8 * i;
    valid[i] = local < rows;
    const int row = first_row + min(local, rows - 1);
    token[i] = first_token + row / group;
    head[i] = kv_head * group + row % group;
    position[i] = first_position + row / group;
  }
  uint32_t query[DIM / 16][4];
#pragma unroll
  for (int kk = 0; kk < DIM / 16; ++kk)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      query[kk][i] = query_pair(q + (size_t)token[i & 1] * q_stride + (size_t)head[i & 1] * DIM + kk * 16 + (i >> 1) * 8 + (lane & 3) * 2);

  const int from = (int)min(max((long long)part * partition, (long long)((window > 0 ? max(0, lowest - window + 1) : 0) / kKeys * kKeys)), 0x7fffff00ll);
  const int end = end_of_keys((long long)highest + 1, (long long)(part + 1) * partition, table_width, cache.page_size);
  float o[DIM / 8][4];
#pragma unroll
  for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

  uint4 k_raw[kRounds], v_raw[kRounds];
  float k_scale[kRounds], v_scale[kRounds];
  unsigned there = 0;                                              // which of this thread's pieces are of keys that are there
  auto fetch = [&](int key0) {
    there = 0;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int piece = threadIdx.x + i * kThreads;
      const int key = key0 + piece / kPieces;
      k_raw[i] = v_raw[i] = make_uint4(0u, 0u, 0u, 0u);
      k_scale[i] = v_scale[i] = 0.0f;
      if (key < end) {
        const int block = key / cache.page_size;
        const int page = page_of_block(table, table_width, block, cache.pages);
        if (page >= 0) {
          const size_t row = (size_t)page * cache.page_size + (key - block * cache.page_size);
          const size_t at = (row * cache.kv_heads + kv_head) * DIM + piece % kPieces * 16;
          k_raw[i] = *reinterpret_cast<const uint4*>(cache.k + at);
          v_raw[i] = *reinterpret_cast<const uint4*>(cache.v + at);
          k_scale[i] = cache.k_scales[(size_t)page * cache.kv_heads + kv_head];
          v_scale[i] = cache.v_scales[(size_t)page * cache.kv_heads + kv_head];
          there |= 1u << i;
        }
      }
    }
  };
  auto put = [&](bf16* tile_rows, const uint4& raw, float scale, int piece) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t packed[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      packed[2 * w] = scaled_bf16(e4m3_low(words[w]), scale);
      packed[2 * w + 1] = scaled_bf16(e4m3_high(words[w]), scale);
    }
    uint4* to = reinterpret_cast<uint4*>(tile_rows + piece / kPieces * kStride + piece % kPieces * 16);
    to[0] = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    to[1] = make_uint4(packed[4], packed[5], packed[6], packed[7]);
  };

  if (threadIdx.x == 0) {
    there_bits[0] = 0ull;
    hidden_nans = 0;
  }
  if (from < end) fetch(from);
  int parity = 0;
  for (int key0 = from; key0 < end; key0 += kKeys, parity ^= 1) {
    __syncthreads();                                               // (the last tile has been read)
    unsigned long long mine = 0ull;
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int piece = threadIdx.x + i * kThreads;
      put(k_tile, k_raw[i], k_scale[i], piece);
      if (nan_bytes(v_raw[i].x) | nan_bytes(v_raw[i].y) | nan_bytes(v_raw[i].z) | nan_bytes(v_raw[i].w)) {
        // a weight of 0 times NaN would be NaN for the rows that do not see the key: it is left out here and put in at the end
        const int key = key0 + piece / kPieces;
        if (key > lowest || (window > 0 && key <= highest - window)) {
          v_raw[i] = make_uint4(without_nans(v_raw[i].x), without_nans(v_raw[i].y), without_nans(v_raw[i].z), without_nans(v_raw[i].w));
          hidden_nans = 1;
        }
      }
      put(v_tile, v_raw[i], v_scale[i], piece);
      if ((there >> i & 1u) && piece % kPieces == 0) mine |= 1ull << (piece / kPieces);
    }
    if (mine) atomicOr(&there_bits[parity], mine);
    __syncthreads();
    const unsigned long long seen = there_bits[parity];
    if (threadIdx.x == 0) there_bits[parity ^ 1] = 0ull;           // (the tile before's: every thread has read it)
    if (key0 + kKeys < end) fetch(key0 + kKeys);

    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < DIM / 16; kk += 2) {
        uint32_t b[4];
        ldmatrix_x4(b, smem_u32(k_tile + (n * 8 + (lane & 7)) * kStride + kk * 16 + (lane >> 3) * 8));
        mma_bf16(s[n], query[kk], b[0], b[1]);
        mma_bf16(s[n], query[kk + 1], b[2], b[3]);
      }
    }
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int column = n * 8 + (lane & 3) * 2 + (i & 1), key = key0 + column, at = position[i >> 1];
        const bool visible = key <= at && (window == 0 || key > at - window) && (seen >> column & 1ull) && key < end;
        s[n][i] = visible ? s[n][i] * scale_log2 : -INFINITY;
        best[i >> 1] = fmaxf(best[i >> 1], s[n][i]);
      }
    float shift[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float now = fmaxf(top[i], quad_max(best[i]));
      const float factor = now == top[i] ? 1.0f : approximate_exp2(top[i] - now);    // 0 where nothing was seen before
      top[i] = now;
      sum[i] *= factor;
#pragma unroll
      for (int n = 0; n < DIM / 8; ++n) {
        o[n][2 * i] *= factor;
        o[n][2 * i + 1] *= factor;
      }
      shift[i] = now == -INFINITY ? 0.0f : now;
    }
    uint32_t weights[kKeys / 16][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[n][i] = approximate_exp2(s[n][i] - shift[i >> 1]);
        sum[i >> 1] += s[n][i];
      }
      weights[n / 2][(n & 1) * 2] = pack(s[n][0], s[n][1]);
      weights[n / 2][(n & 1) * 2 + 1] = pack(s[n][2], s[n][3]);
    }
#pragma unroll
    for (int kk = 0; kk < kKeys / 16; ++kk)
#pragma unroll
      for (int n = 0; n < DIM / 8; n += 2) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, smem_u32(v_tile + (kk * 16 + (lane & 15)) * kStride + n * 8 + (lane >> 4) * 8));
        mma_bf16(o[n], weights[kk], b[0], b[1]);
        mma_bf16(o[n + 1], weights[kk], b[2], b[3]);
      }
  }

  if (from < end && hidden_nans) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      for (int key = max(from, window > 0 ? position[i] - window + 1 : 0); key < end && key <= position[i]; ++key) {
        if (key <= lowest && (window == 0 || key > highest - window)) continue;         // (every row sees it: left in)
        const int block = key / cache.page_size, page = page_of_block(table, table_width, block, cache.pages);
        if (page < 0) continue;
        const uint8_t* codes = cache.v + (((size_t)page * cache.page_size + (key - block * cache.page_size)) * cache.kv_heads + kv_head) * DIM;
#pragma unroll
        for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if ((codes[n * 8 + (lane & 3) * 2 + j] & 0x7f) == 0x7f) o[n][2 * i + j] = __int_as_float(0x7fffffff);
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float total = quad_sum(sum[i]);
    if (!valid[i]) continue;
    const size_t row = (size_t)token[i] * heads + head[i];
    if (num_partitions == 1) {
      if (total != 0.0f && sinks != nullptr) total += exp2f(sinks[head[i]] * kLog2e - top[i]);
      const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
      for (int n = 0; n < DIM / 8; ++n)
        *reinterpret_cast<uint32_t*>(out + row * DIM + n * 8 + (lane & 3) * 2) = pack(o[n][2 * i] * inverse, o[n][2 * i + 1] * inverse);
    } else {
      const size_t at = row * num_partitions + part;
      if ((lane & 3) == 0) *reinterpret_cast<float2*>(partial_ml + at * 2) = make_float2(top[i], total);
      if (total != 0.0f) {
#pragma unroll
        for (int n = 0; n < DIM / 8; ++n)
          *reinterpret_cast<float2*>(partial_o + at * DIM + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
      }
    }
  }
}

// Single tokens of any size: a warp by itself takes chunks of keys, up to 16 query heads of the group as the rows of the products, and needs
// neither shared memory nor a barrier until the end.  The fragments come from the cache as they are: which element of a head is which
// index of a product is free as long as queries and keys (values and results) agree, so a thread takes DIM / 4 neighbouring bytes of a key
// for the scores, and DIM / 8 of each of four keys for the result.  The next chunk's bytes are on their way while this one is worked on, the
// table's entries a chunk ahead of those.  A hidden key's values are zeros.  64 contexts of 2,048 keys, 16 heads of 64 over 4 (67 MB): 70 us (150
// by tiles of 64 rows in shared memory, of which a group of four fills four); heads of 128 in pages of 24, 32 over 8 (268 MB): 204 us, 324
// before.  Bound by the chain of a chunk (shuffles, widening, two products, a rescaled sum), not by the CTAs an SM: three to six were the same.
template <int DIM>
__global__ void __launch_bounds__(128)
single_8bit_kernel(const bf16* __restrict__ q, long long q_stride, bf16* __restrict__ out, Cache8 cache, const int* __restrict__ block_table,
                   int table_width, const int* __restrict__ positions, int group, float scale_log2, int window, int partition,
                   int num_partitions, float* __restrict__ partial_o, float* __restrict__ partial_ml, const float* __restrict__ sinks) {
  constexpr int kHeads = 16, kWarps = 4, kChunk = DIM == 64 ? 32 : 16, kSteps = kChunk / 16;      // steps of 16 keys
  constexpr int kWords = DIM / 16;              // 32-bit words of a thread's piece of a key, which are also steps of 16 elements
  constexpr int kValueWords = DIM / 32;         // of its piece of a row of values
  __shared__ float o_shared[kWarps][kHeads][DIM];
  __shared__ float ml_shared[kWarps][kHeads][2];
  grid_dependency_wait();
  grid_launch_dependents();
  const int part = blockIdx.x % num_partitions, tile = blockIdx.x / num_partitions, kv_head = blockIdx.y;
  const int tiles = (group + kHeads - 1) / kHeads, request = tile / tiles, first_row = tile % tiles * kHeads;
  const int position = positions[request];
  if (position < 0) return;                                        // a padding row: left as it is
  const int rows = min(kHeads, group - first_row), heads = group * cache.kv_heads, first_head = kv_head * group + first_row;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int* table = block_table + (size_t)request * table_width;
  const int first_key = (window > 0 && position >= window) ? position + 1 - window : 0;
  const int end = end_of_keys((long long)position + 1, (long long)(part + 1) * partition, table_width, cache.page_size);
  const int from = (int)min(max((long long)part * partition, (long long)first_key), (long long)end);

  uint32_t query[kWords][4];
#pragma unroll
  for (int s = 0; s < kWords; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      query[s][i] = query_pair(q + (size_t)request * q_stride + (size_t)(first_head + min(g + 8 * (i & 1), rows - 1)) * DIM + t * (DIM / 4) +
                               4 * s + 2 * (i >> 1));
  struct Chunk {
    uint32_t k[kSteps][2][kWords], v[kSteps][4][kValueWords];
    int row;                                                       // by lane: a key's row in the cache, below 0: hidden
    float k_scale, v_scale;                                        // its page's
  };
  // (What is loaded is looked at only where it is used, an iteration later: a comparison or a product here would wait for it.)
  // The table's entry for this lane's key of a chunk, -1 where the key is hidden or behind the table.
  auto look_up = [&](int key0) {
    const int key = key0 + lane;
    return lane < kChunk && key < end ? table[key / cache.page_size] : -1;            // (end is no further than the table)
  };
  auto fetch = [&](int key0, int page, Chunk& c) {
    const int key = key0 + lane;
    const bool there = page >= 0 && page < cache.pages;
    c.row = there ? page * cache.page_size + key % cache.page_size : -1;
    c.k_scale = c.v_scale = 1.0f;
    if (there) {
      c.k_scale = cache.k_scales[(size_t)page * cache.kv_heads + kv_head];
      c.v_scale = cache.v_scales[(size_t)page * cache.kv_heads + kv_head];
    }
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = __shfl_sync(0xffffffffu, c.row, step * 16 + 8 * i + g);
        const uint4* at = reinterpret_cast<const uint4*>(cache.k + ((size_t)max(row, 0) * cache.kv_heads + kv_head) * DIM + t * (DIM / 4));
#pragma unroll
        for (int w = 0; w < kWords / 4; ++w) {
          const uint4 raw = row >= 0 ? at[w] : make_uint4(0u, 0u, 0u, 0u);
          c.k[step][i][4 * w] = raw.x; c.k[step][i][4 * w + 1] = raw.y; c.k[step][i][4 * w + 2] = raw.z; c.k[step][i][4 * w + 3] = raw.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {                                // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the step
        const int row = __shfl_sync(0xffffffffu, c.row, step * 16 + 2 * t + (i & 1) + 8 * (i >> 1));
        const uint2* at = reinterpret_cast<const uint2*>(cache.v + ((size_t)max(row, 0) * cache.kv_heads + kv_head) * DIM + g * (DIM / 8));
#pragma unroll
        for (int w = 0; w < kValueWords / 2; ++w) {
          const uint2 raw = row >= 0 ? at[w] : make_uint2(0u, 0u);
          c.v[step][i][2 * w] = raw.x; c.v[step][i][2 * w + 1] = raw.y;
        }
      }
    }
  };
  // The four numbers of a word as two pairs of bf16 times a power of two.
  auto widen = [&](uint32_t word, uint32_t factor, uint32_t rest, uint32_t (&pair)[2]) {
    pair[0] = times(times(lifted<0x9180>(word), factor), rest);
    pair[1] = times(times(lifted<0xb3a2>(word), factor), rest);
    const uint32_t nans = nan_bytes(word);
    if (nans != 0u) {                                              // (the lifted number of a NaN is 480)
      if (nans & 0x80u) pair[0] |= 0x7fffu;
      if (nans & 0x8000u) pair[0] |= 0x7fff0000u;
      if (nans & 0x800000u) pair[1] |= 0x7fffu;
      if (nans & 0x80000000u) pair[1] |= 0x7fff0000u;
    }
  };
  float o[DIM / 8][4];
#pragma unroll
  for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
  float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  constexpr int kStride = kWarps * kChunk;
  const uint32_t lift = power_pair(120), one = 0x3f803f80u;
  int key0 = from + warp * kChunk;
  Chunk now, next;
  fetch(key0, look_up(key0), now);
  int page = look_up(key0 + kStride);
  for (; key0 < end; key0 += kStride) {
    fetch(key0 + kStride, page, next);
    page = look_up(min(key0 + kStride, 0x7fffff00) + kStride);
    const float k_factor = now.k_scale * scale_log2;
    const int v_exponent = ((__float_as_int(now.v_scale) >> 23) & 0xff) - 127;
    const uint32_t v_factor = power_pair(min(v_exponent, 7) + 120), v_rest = power_pair(max(v_exponent - 7, 0));
    float s[2 * kSteps][4], best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < 2 * kSteps; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        uint32_t pair[2];
        widen(now.k[j / 2][j & 1][w], lift, one, pair);
        mma_bf16(s[j], query[w], pair[0], pair[1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {                                // key 8j + 2t + i, of both rows
        const int from_lane = 8 * j + 2 * t + i;
        const bool visible = __shfl_sync(0xffffffffu, now.row, from_lane) >= 0;
        const float factor = __shfl_sync(0xffffffffu, k_factor, from_lane);
        s[j][i] = visible ? s[j][i] * factor : -INFINITY;
        s[j][i + 2] = visible ? s[j][i + 2] * factor : -INFINITY;
        best[0] = fmaxf(best[0], s[j][i]);
        best[1] = fmaxf(best[1], s[j][i + 2]);
      }
    }
    float shift[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float highest = fmaxf(top[i], quad_max(best[i]));
      const float factor = highest == top[i] ? 1.0f : approximate_exp2(top[i] - highest);      // 0 where nothing was seen before
      top[i] = highest;
      sum[i] *= factor;
      shift[i] = highest == -INFINITY ? 0.0f : highest;
      if (__any_sync(0xffffffffu, factor != 1.0f)) {
#pragma unroll
        for (int n = 0; n < DIM / 8; ++n) {
          o[n][2 * i] *= factor;
          o[n][2 * i + 1] *= factor;
        }
      }
    }
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      uint32_t weights[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float(&p)[4] = s[2 * step + h];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = approximate_exp2(p[i] - shift[i >> 1]);
          sum[i >> 1] += p[i];
        }
        weights[2 * h] = pack(p[0], p[1]);
        weights[2 * h + 1] = pack(p[2], p[3]);
      }
      uint32_t factor[4], rest[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int from_lane = step * 16 + 2 * t + (i & 1) + 8 * (i >> 1);
        factor[i] = __shfl_sync(0xffffffffu, v_factor, from_lane);
        rest[i] = __shfl_sync(0xffffffffu, v_rest, from_lane);
      }
#pragma unroll
      for (int w = 0; w < kValueWords; ++w) {
        uint32_t wide[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) widen(now.v[step][i][w], factor[i], rest[i], wide[i]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {                              // element 4w + n of this thread's piece: of two keys side by side
          const uint32_t pick = n & 1 ? 0x7632u : 0x5410u;
          mma_bf16(o[4 * w + n], weights, __byte_perm(wide[0][n >> 1], wide[1][n >> 1], pick), __byte_perm(wide[2][n >> 1], wide[3][n >> 1], pick));
        }
      }
    }
    now = next;
  }

#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float total = quad_sum(sum[i]);
    if (t == 0) {
      ml_shared[warp][g + 8 * i][0] = top[i];
      ml_shared[warp][g + 8 * i][1] = total;
    }
#pragma unroll
    for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) o_shared[warp][g + 8 * i][(2 * t + j) * (DIM / 8) + n] = o[n][2 * i + j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * DIM; i += 128) {
    const int row = i / DIM, element = i % DIM;
    float highest = -INFINITY, total = 0.0f, value = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (ml_shared[w][row][1] != 0.0f) highest = fmaxf(highest, ml_shared[w][row][0]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (ml_shared[w][row][1] == 0.0f) continue;                  // (no key of this warp was visible)
      const float factor = exp2f(ml_shared[w][row][0] - highest);
      total += ml_shared[w][row][1] * factor;
      value += o_shared[w][row][element] * factor;
    }
    const size_t at = (size_t)request * heads + first_head + row;
    if (num_partitions == 1) {
      if (total != 0.0f && sinks != nullptr) total += exp2f(sinks[first_head + row] * kLog2e - highest);
      out[at * DIM + element] = __float2bfloat16_rn(total == 0.0f ? 0.0f : value / total);
    } else {
      partial_o[(at * num_partitions + part) * DIM + element] = value;
      if (element == 0) *reinterpret_cast<float2*>(partial_ml + (at * num_partitions + part) * 2) = make_float2(highest, total);
    }
  }
}

// A warp for each token and head: the partitions' parts, each relative to a maximum of its own, to one result.  A part
// whose denominator is 0 holds nothing (no key of it was visible) and is not read.
template <int DIM>
__global__ void __launch_bounds__(256)
merge_8bit_kernel(const float* __restrict__ partial_o, const float* __restrict__ partial_ml, bf16* __restrict__ out,
                  const int* __restrict__ positions, const int* __restrict__ query_starts, int num_rows, int tokens, int heads,
                  int num_partitions, const float* __restrict__ sinks, const int* __restrict__ error) {
  grid_dependency_wait();
  grid_launch_dependents();
  if (error != nullptr && *reinterpret_cast<const volatile int*>(error) != 0) return;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= (long long)tokens * heads) return;
  const int token = (int)(row / heads), head = (int)(row % heads);
  if (query_starts == nullptr ? positions[token] < 0 : (token < query_starts[0] || token >= query_starts[num_rows])) return;
  const float2* ml = reinterpret_cast<const float2*>(partial_ml) + row * num_partitions;
  float top = -INFINITY;
  for (int p = lane; p < num_partitions; p += 32)
    if (ml[p].y != 0.0f) top = fmaxf(top, ml[p].x);
  top = warp_max(top);
  constexpr int kColumns = DIM / 32;
  float o[kColumns], total = 0.0f;
#pragma unroll
  for (int c = 0; c < kColumns; ++c) o[c] = 0.0f;
  const float* part = partial_o + (size_t)row * num_partitions * DIM + lane * kColumns;
  for (int p = 0; p < num_partitions; ++p, part += DIM) {
    const float2 mine = ml[p];
    if (mine.y == 0.0f) continue;
    const float factor = exp2f(mine.x - top);
    total += mine.y * factor;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) o[c] += part[c] * factor;
  }
  if (total != 0.0f && sinks != nullptr) total += exp2f(sinks[head] * kLog2e - top);
  const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
  uint32_t* to = reinterpret_cast<uint32_t*>(out + (size_t)row * DIM + lane * kColumns);
#pragma unroll
  for (int c = 0; c < kColumns; c += 2) to[c / 2] = pack(o[c] * inverse, o[c + 1] * inverse);
}

}  // namespace

int mir_merge_8bit(const Attention8& a, int tokens) {
  const long long blocks = ((long long)tokens * a.heads + 7) / 8;
  return mir_launch("merge_8bit", a.head_dim == 128 ? merge_8bit_kernel<128> : merge_8bit_kernel<64>, dim3((unsigned)blocks),
                    dim3(256), 0, a.stream, 0, a.partial_o(tokens), a.partial_ml(tokens), (bf16*)a.out, a.positions, a.query_starts,
                    a.num_rows, tokens, a.heads, a.num_partitions, a.sinks, a.error);
}

int mir_attention_8bit_general(const Attention8& a, int tokens) {
  const int group = a.heads / a.cache.kv_heads;
  if (a.query_starts == nullptr) {
    const long long blocks = (long long)a.num_rows * ((group + 15) / 16) * a.num_partitions;
    if (blocks > 0x7fffffffll || a.cache.kv_heads > 65535) {
      mir_set_error("%s: %d tokens are more than one launch takes", a.what, tokens);
      return MIR_BAD_ARGUMENT;
    }
    const int status = mir_launch("single_8bit", a.head_dim == 128 ? single_8bit_kernel<128> : single_8bit_kernel<64>,
                                  dim3((unsigned)blocks, a.cache.kv_heads), dim3(128), 0, a.stream, 0, (const bf16*)a.q, a.q_stride, (bf16*)a.out,
                                  a.cache, a.block_table, a.table_width, a.positions, group, a.scale * kLog2e, a.window, a.partition,
                                  a.num_partitions, a.partial_o(tokens), a.partial_ml(tokens), a.sinks);
    if (status != MIR_OK || a.num_partitions == 1) return status;
    return mir_merge_8bit(a, tokens);
  }
  // tiles of 64 rows; of portions an upper bound (spare ones find no request and end)
  const long long tiles = ((long long)tokens * group + kRows - 1) / kRows + a.num_rows;
  if (tiles * a.num_partitions > 0x7fffffffll || a.cache.kv_heads > 65535) {
    mir_set_error("%s: %d tokens are more than one launch takes", a.what, tokens);
    return MIR_BAD_ARGUMENT;
  }
  const dim3 grid((unsigned)(tiles * a.num_partitions), a.cache.kv_heads);
  const int status = mir_launch("attention_8bit", a.head_dim == 128 ? attention_8bit_kernel<128> : attention_8bit_kernel<64>, grid,
                                dim3(kThreads), 0, a.stream, 0, (const bf16*)a.q, a.q_stride, (bf16*)a.out, a.cache, a.block_table,
                                a.table_width, a.query_starts, a.context_lens, a.num_rows, group,
                                a.scale * kLog2e, a.window, a.partition, a.num_partitions, a.partial_o(tokens), a.partial_ml(tokens),
                                a.sinks, tokens);
  if (status != MIR_OK || a.num_partitions == 1) return status;
  return mir_merge_8bit(a, tokens);
}

static bool attention_8bit_refused(const Attention8& a, int tokens, bool shared_out) {
  const bool bad =
      (a.head_dim != 64 && a.head_dim != 128) || a.heads <= 0 || a.cache.kv_heads <= 0 || a.heads % a.cache.kv_heads ||
      a.cache.page_size <= 0 || a.cache.pages <= 0 || (long long)a.cache.pages * a.cache.page_size > 0x7fffffffll || a.table_width < 0 || (a.table_width == 0 && a.num_rows > 0) ||
      !(a.scale > 0.0f) || a.window < 0 || (a.q_stride % 8) || a.q_stride < (long long)a.heads * a.head_dim || ((uintptr_t)a.q & 15) ||
      ((uintptr_t)a.out & 15) || ((uintptr_t)a.cache.k & 15) || ((uintptr_t)a.cache.v & 15) ||
      (shared_out ? a.partition != 0 : a.partition <= 0 || a.partition % 128 != 0) || a.num_partitions <= 0 || a.num_partitions > 65535 || a.num_rows < 0 || tokens < 0;
  if (bad) {
    mir_set_error("%s: takes head_dim 64 or 128, a positive scale, a plan's partitions and 16-byte aligned tensors (head_dim "
                  "%d, heads %d, kv heads %d, page %d, pages %d, partition %d x %d, row stride %lld)", a.what, a.head_dim, a.heads,
                  a.cache.kv_heads, a.cache.page_size, a.cache.pages, a.partition, a.num_partitions, a.q_stride);
    return true;
  }
  const long long need = shared_out ? mir_decode_8bit_floats(a.num_partitions, a.heads / a.cache.kv_heads) : a.num_partitions == 1 ? 0 : (long long)tokens * a.heads * a.num_partitions * (a.head_dim + 2);
  if (need > 0 && (a.scratch == nullptr || a.scratch_floats < need || ((uintptr_t)a.scratch & 15))) {      // (read 16 bytes at a time)
    mir_set_error("%s: scratch of %lld floats on a 16-byte boundary is needed, got %lld", a.what, need, a.scratch_floats);
    return true;
  }
  return false;
}

// How single tokens are split over the keys: partitions of `keys`, `count` of them, and the floats of scratch.  keys 0: shared out
// evenly over `count` CTAs.
MIR_EXPORT int mir_decode_attention_8bit_plan(int rows, int heads, int kv_heads, int head_dim, int page_size, int max_context,
                                              int* keys, int* count, long long* floats) {
  if (rows < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_context < 0 || page_size <= 0) {
    mir_set_error("decode_attention_8bit_plan: bad sizes (rows %d, heads %d, kv heads %d, context %d)", rows, heads, kv_heads, max_context);
    return MIR_BAD_ARGUMENT;
  }
  const int group = heads / kv_heads;
  if (mir_decode_8bit_takes(head_dim, page_size)) {
    // the tcgen05 kernel shares all requests' keys out over its CTAs by the positions that it finds
    *keys = 0;
    *count = mir_decode_8bit_ctas(rows * std::max(1ll, (max_context + 127ll) / 128), heads, kv_heads);
    *floats = mir_decode_8bit_floats(*count, group);
    return MIR_OK;
  }
  const long long ctas = std::max(1ll, (long long)rows * kv_heads * ((group + 15) / 16));
  const long long wanted = std::max(1ll, (long long)mir_sm_count() * 4 / ctas);
  const long long tiles = std::max(1ll, (max_context + 127ll) / 128);
  const long long each = std::max(1ll, (tiles + wanted - 1) / wanted);
  *keys = (int)(each * 128);
  *count = (int)((tiles + each - 1) / each);
  *floats = *count == 1 ? 0 : (long long)rows * heads * *count * (head_dim + 2);
  return MIR_OK;
}

// One token per request: row r of q at positions[r] (below 0: a padding row, whose result is left as it is).
MIR_EXPORT int mir_decode_attention_8bit(const void* q, long long q_stride, void* out, const void* k_pages, const void* v_pages,
                                         const float* k_scales, const float* v_scales, int pages, const int* block_table,
                                         int table_width, const int* positions, int rows, int page_size, int heads, int kv_heads,
                                         int head_dim, float scale, int window, int partition, int num_partitions, float* scratch,
                                         long long scratch_floats, const float* sinks, cudaStream_t stream) {
  Attention8 a;
  a.what = "decode_attention_8bit";
  a.q = q; a.q_stride = q_stride; a.out = out;
  a.cache = Cache8{(const uint8_t*)k_pages, (const uint8_t*)v_pages, k_scales, v_scales, pages, page_size, kv_heads};
  a.block_table = block_table; a.table_width = table_width; a.positions = positions;
  a.num_rows = rows; a.heads = heads; a.head_dim = head_dim; a.scale = scale; a.window = window;
  a.partition = partition; a.num_partitions = num_partitions; a.scratch = scratch; a.scratch_floats = scratch_floats;
  a.sinks = sinks; a.stream = stream;
  const bool shared_out = mir_decode_8bit_takes(head_dim, page_size);
  if (attention_8bit_refused(a, rows, shared_out)) return MIR_BAD_ARGUMENT;
  if (rows == 0) return MIR_OK;
  return shared_out ? mir_attention_8bit_decode(a) : mir_attention_8bit_general(a, rows);
}

// How portions are split over the keys: a few tokens behind a long context are fewer items (tiles of rows and kv heads) than CTAs that run
// at once, and each would walk over all of it (16 tokens at 16,384, 32 heads over 8: 8 items).  The cut is the one with the least
// time in tiles of keys: as many rounds as the items take, each a partition's tiles and the start of an item, which is worth some four
// tiles of the tcgen05 kernel and one of the other, and the joining; a sixth has to be gained.  Heads of 128: 16 tokens at 16,384 take 165 us
// in one part, 34 in 17 (one round), 51 in 26 (two); 300 tokens 180 and in 3 parts 135; 512 tokens, 128 items, 171 and in 2 parts 187.  Heads of
// 64, 16 over 4: 16 tokens at 1,000 65 and in 2 parts 37, 400 at 16,384 in 2 parts 573 and in 5 472.
MIR_EXPORT int mir_prefill_attention_8bit_plan(int rows, int tokens, int heads, int kv_heads, int head_dim, int page_size, int max_context,
                                               int* keys, int* count, long long* floats) {
  if (rows < 0 || tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || max_context < 0 || page_size <= 0) {
    mir_set_error("prefill_attention_8bit: bad sizes (%d requests, %d tokens, heads %d, kv heads %d, context %d)", rows, tokens, heads,
                  kv_heads, max_context);
    return MIR_BAD_ARGUMENT;
  }
  const long long group = heads / kv_heads, tile = mir_decode_8bit_takes(head_dim, page_size) ? 128 : kRows;
  const long long items = std::max(1ll, (tokens * group + tile - 1) / tile) * kv_heads;       // (at least as many as that)
  const long long tiles = std::max(1ll, (max_context + 127ll) / 128);
  // one CTA an SM of the tcgen05 kernel, two of the other
  const bool tensor_memory = mir_decode_8bit_takes(head_dim, page_size);
  const long long at_once = mir_sm_count() * (tensor_memory ? 1ll : 2ll), start = tensor_memory ? 4 : 1, join = tensor_memory ? 2 : 1;
  long long each = tiles, parts = 1, least = (items + at_once - 1) / at_once * (tiles + start) * 5 / 6 + 1;
  // as many partitions as one or two rounds take, at least four tiles of keys each
  for (long long rounds = 1; rounds <= 2; ++rounds) {
    const long long wanted = std::min(rounds * at_once / items, tiles / 4);
    if (wanted < 2) continue;
    const long long keys_each = (tiles + wanted - 1) / wanted, there = (tiles + keys_each - 1) / keys_each;
    const long long time = (items * there + at_once - 1) / at_once * (keys_each + start) + join;
    if (time < least) {
      least = time;
      each = keys_each;
      parts = there;
    }
  }
  *keys = (int)(each * 128);
  *count = (int)parts;
  *floats = *count == 1 ? 0 : (long long)tokens * heads * *count * (head_dim + 2);
  return MIR_OK;
}

// Portions: request r has tokens query_starts[r] .. query_starts[r + 1] - 1 of the packed rows, and its context_lens[r]
// cached tokens include them.  Rows that no request has are left as they are.
MIR_EXPORT int mir_prefill_attention_8bit(const void* q, long long q_stride, void* out, const void* k_pages, const void* v_pages,
                                          const float* k_scales, const float* v_scales, int pages, const int* block_table,
                                          int table_width, const int* query_starts, const int* context_lens, int num_rows, int tokens,
                                          int page_size, int heads, int kv_heads, int head_dim, float scale, int window, int partition,
                                          int num_partitions, float* scratch, long long scratch_floats, const float* sinks,
                                          cudaStream_t stream) {
  Attention8 a;
  a.what = "prefill_attention_8bit";
  a.q = q; a.q_stride = q_stride; a.out = out;
  a.cache = Cache8{(const uint8_t*)k_pages, (const uint8_t*)v_pages, k_scales, v_scales, pages, page_size, kv_heads};
  a.block_table = block_table; a.table_width = table_width; a.query_starts = query_starts; a.context_lens = context_lens;
  a.num_rows = num_rows; a.heads = heads; a.head_dim = head_dim; a.scale = scale; a.window = window;
  a.partition = partition; a.num_partitions = num_partitions; a.scratch = scratch; a.scratch_floats = scratch_floats;
  a.sinks = sinks; a.stream = stream;
  if (attention_8bit_refused(a, tokens, false)) return MIR_BAD_ARGUMENT;
  if (num_rows == 0 || tokens == 0) return MIR_OK;
  return mir_decode_8bit_takes(head_dim, page_size) ? mir_attention_8bit_prefill(a, tokens) : mir_attention_8bit_general(a, tokens);
}
