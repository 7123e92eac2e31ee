// Attention of single tokens over the 8-bit cache on the 5th-generation tensor cores, head_dim 128, pages of 8 to 128 keys:
// the bytes of the cache go from memory into the products as they are, nothing is widened.
//
// A CTA takes one request, one kv head (up to 16 query heads of its group) and one partition of the keys, and walks over it in
// tiles of 128 keys.  The products are transposed, so that the keys (then the elements of the head) are the 128 rows of the tensor
// cores and the query heads the 16 columns:
//
//   S^T = K Q^T    kind::f8f6f4, A = the key tile as the cache holds it (a key is a row of 128 bytes), B = the queries in two parts:
//                  q = hi + lo, hi = e4m3(q 2^-e), lo = e5m2 of what hi leaves.  A bf16 number has eight significant bits, hi takes
//                  four and lo the signed rest, so the two are exact down to 2^-14 of the head's largest element (e puts that
//                  below 448) and off by at most 2^-25 of it below;
//   O^T += V^T P   A = the value tile as the cache holds it (MN-major: nothing is transposed), B = the softmax's weights in the same
//                  two parts: 2^-4 from hi, 2^-3 of that from lo, so a weight is off by at most 2^-7 of itself.
//
// The scales: a score is multiplied by its key's page's scale on its way out of tensor memory, in 32 bits.  A value's scale 2^f goes
// into the weight, exp2(s + f - M) with a reference M of its own (the running maximum of s + f), so that the weights of loud pages
// stay below 448 and those of quiet ones are no smaller than their share of the result; the denominator sums exp2(s - m) in 32
// bits.  Both references rise only when a tile's maximum exceeds them by 2^8.
//
// Four warps of softmax (a thread is a key, then an element of the head), a loader (TMA, one box for each page, or one for the tile
// where its pages lie one behind the other), an issuer.  Two stages of keys and values, 72 KB a CTA, three CTAs an SM.  A hidden key's
// score becomes -inf by selection, and its row of values is zeroed in shared memory (0 times what lies behind a context could
// be NaN).  The kernel is bound by the cache's bytes.
#include <algorithm>
#include "eight_bit_tc.cuh"

using namespace mir;
using namespace mir::tc;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kKeys = 128, kDim = 128, kHeads = 16, kStages = 2;
constexpr int kTile = kKeys * kDim;                    // bytes of a tile of keys or of values
constexpr int kPart = kHeads * 128;                    // bytes of 16 rows of one part of Q or P
constexpr int kOffK = 0, kOffV = kStages * kTile, kOffQ = 2 * kStages * kTile, kOffP = kOffQ + 2 * kPart;
constexpr int kSmemBytes = kOffP + 2 * kPart + 1024;
constexpr int kSoftmaxThreads = 128, kThreads = kSoftmaxThreads + 64;
constexpr uint32_t kTmemColumns = 32;                  // S^T at 0, O^T at 16
constexpr float kRises = 8.0f, kHeadroom = 4.0f;       // log2: a reference rises when it is exceeded by kRises; M to kHeadroom below the maximum
static_assert(kSmemBytes >= kLeastSharedBeside, "never beside a kernel that takes all tensor memory");

enum { K_FULL = 0, K_FREE = K_FULL + kStages, V_FULL = K_FREE + kStages, V_FREE = V_FULL + kStages, S_FULL = V_FREE + kStages, P_READY,
       Q_READY, O_DONE, BARRIERS };

__device__ int g_error = 0;

__device__ __forceinline__ float warp_largest(float v) {
  float top;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v));
  return top;
}

// N consecutive accumulator columns of this thread's lane.
template <int N> __device__ __forceinline__ void tmem_load(uint32_t address, float (&v)[N]);
template <> __device__ __forceinline__ void tmem_load<4>(uint32_t address, float (&v)[4]) {
  uint32_t r[4];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[i]);
}
template <> __device__ __forceinline__ void tmem_load<8>(uint32_t address, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(address) : "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
template <> __device__ __forceinline__ void tmem_load<16>(uint32_t address, float (&v)[16]) { tmem_load_16(address, v); }

template <int N> __device__ __forceinline__ void tmem_store(uint32_t address, const float (&v)[N]) {
#pragma unroll
  for (int c = 0; c < N; c += 4)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(address + (uint32_t)c), "r"(__float_as_uint(v[c])),
                 "r"(__float_as_uint(v[c + 1])), "r"(__float_as_uint(v[c + 2])), "r"(__float_as_uint(v[c + 3]))
                 : "memory");
}

// Byte offset of element (row, column) of 16 rows of 128 bytes with the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int column) {
  return (uint32_t)(row * 128 + (((column >> 4) ^ (row & 7)) << 4) + (column & 15));
}
// Two numbers within 448 as e4m3 and what that leaves as e5m2 (the first in the low bytes).
__device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = to_e4m3x2(a, b);
  const float2 taken = __half22float2(e4m3_low(hi));
  lo = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a - taken.x, b - taken.y), __NV_SATFINITE, __NV_E5M2);
}

// G: heads that the softmax threads handle (the CTA's heads rounded up to 4, 8 or 16).
template <int G>
__global__ void __launch_bounds__(kThreads)
decode_8bit_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                   const __grid_constant__ CUtensorMap k_tile_map, const __grid_constant__ CUtensorMap v_tile_map,
                   const bf16* __restrict__ q, long long q_stride, Cache8 cache, const int* __restrict__ block_table, int table_width,
                   const int* __restrict__ positions, int heads, float scale_log2, int window, int partition, int num_partitions,
                   int part_slow, float* __restrict__ partial_o, float* __restrict__ partial_ml, bf16* __restrict__ out,
                   const float* __restrict__ sinks) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long barriers[BARRIERS];
  __shared__ uint32_t tmem_slot;
  __shared__ float exchange[2][4][2 * G];              // [tile parity][warp]: the warps' maxima of s, then of s + f
  __shared__ float sums[4][G];
  __shared__ float factors[G];                         // of a head's scores: scale, log2 e, and the power of two taken out of its queries
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem), bar0 = smem_u32(&barriers[0]);
  auto bar = [&](int index) { return bar0 + 8u * (uint32_t)index; };
  if (threadIdx.x == kSoftmaxThreads) {
    for (int i = 0; i < BARRIERS; ++i) barrier_init(bar(i), (i == P_READY || i == Q_READY) ? (uint32_t)kSoftmaxThreads : 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // the rows of Q and P that no head has stay zeros
  for (int i = threadIdx.x; i < 4 * kPart / 16; i += kThreads) *reinterpret_cast<uint4*>(smem + kOffQ + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tensor_fence_before_sync();
  __syncthreads();
  tensor_fence_after_sync();
  const uint32_t tmem_s = tmem_slot, tmem_o = tmem_slot + 16u;
  grid_dependency_wait();                              // the cache, the queries and the positions may come from the kernel in front
  grid_launch_dependents();

  const int part = part_slow ? blockIdx.z : blockIdx.x, row = part_slow ? blockIdx.x : blockIdx.z;
  const int group = heads / cache.kv_heads, group_tiles = (group + kHeads - 1) / kHeads;
  const int kv_head = blockIdx.y / group_tiles;
  const int head0 = kv_head * group + (blockIdx.y % group_tiles) * kHeads;
  const int valid_heads = min(kHeads, kv_head * group + group - head0);
  const int position = positions[row];
  const int first_key = (window > 0 && position >= window) ? position + 1 - window : 0;
  const int part_end = (int)min((long long)position + 1, (long long)(part + 1) * partition);
  const int begin = max(part * partition, first_key / kKeys * kKeys);
  const int tiles = position >= 0 && begin < part_end ? (part_end - begin + kKeys - 1) / kKeys : 0;
  const bool go = *reinterpret_cast<volatile int*>(&g_error) == 0;
  const int* table = block_table + (size_t)row * table_width;
  const int shift = 31 - __clz(cache.page_size);       // pages are powers of two
  if (tiles == 0 || !go) {
    // a padding row, or a partition without keys: the merge reads a denominator of 0; without a merge the row is zeros
    if (position >= 0 && threadIdx.x < kDim) {
      for (int g = 0; g < valid_heads; ++g) {
        const size_t head = (size_t)row * heads + head0 + g;
        if (num_partitions == 1) out[head * kDim + threadIdx.x] = __float2bfloat16_rn(0.0f);
        else if (threadIdx.x == 0) {
          partial_ml[(head * num_partitions + part) * 2] = -INFINITY;
          partial_ml[(head * num_partitions + part) * 2 + 1] = 0.0f;
        }
      }
    }
  } else if (warp == 4) {
    // ------------------------------------------------------------------ loader: lane l has page slot l of the tile
    const int pages_per_tile = kKeys >> shift, page_size = cache.page_size;
    const uint32_t box_bytes = (uint32_t)page_size * kDim;
    const bool loads = lane < pages_per_tile;
    auto row_of = [&](int t) {
      const int key = begin + t * kKeys + lane * page_size;
      int page = -1;
      if (loads && t < tiles && key < part_end && key + page_size > first_key) page = page_of_block(table, table_width, key >> shift, cache.pages);
      return page >= 0 ? page << shift : -page_size;   // a negative row lies outside the tensor: zeros
    };
    int cache_row = row_of(0);
    bool alive = true;
    for (int t = 0; t < tiles && alive; ++t) {
      const uint32_t stage = (uint32_t)t % kStages, parity = (uint32_t)(t / kStages) & 1u;
      const int next_row = row_of(t + 1);              // on its way while this tile's stage is awaited
      const int first_row = __shfl_sync(0xffffffffu, cache_row, 0);
      const bool in_a_row = first_row >= 0 && __all_sync(0xffffffffu, !loads || cache_row == first_row + (lane << shift));
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const uint32_t full = bar((which ? V_FULL : K_FULL) + (int)stage);
        if (!wait_barrier(bar((which ? V_FREE : K_FREE) + (int)stage), parity ^ 1u)) { g_error = 1; alive = false; }
        alive = __all_sync(0xffffffffu, alive);
        if (!alive) break;
        const uint32_t to = smem_base + (uint32_t)(which ? kOffV : kOffK) + stage * (uint32_t)kTile;
        if (lane == 0) barrier_expect_bytes(full, (uint32_t)kTile);
        __syncwarp();
        if (in_a_row) {
          if (lane == 0) tma_load_2d(to, which ? &v_tile_map : &k_tile_map, full, kv_head * kDim, first_row);
        } else if (loads) {
          tma_load_2d(to + (uint32_t)lane * box_bytes, which ? &v_map : &k_map, full, kv_head * kDim, cache_row);
        }
      }
      cache_row = next_row;
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------------ issuer (tcgen05.cuh: from a whole warp)
    constexpr uint32_t scores_hi = instruction_descriptor_8bit(kKeys, kHeads, E4M3, E4M3);
    constexpr uint32_t scores_lo = instruction_descriptor_8bit(kKeys, kHeads, E4M3, E5M2);
    constexpr uint32_t values_hi = instruction_descriptor_8bit(kDim, kHeads, E4M3, E4M3, true);
    constexpr uint32_t values_lo = instruction_descriptor_8bit(kDim, kHeads, E4M3, E5M2, true);
    const uint32_t elected = elect_one();
    const uint32_t k_low = operand_low(smem_base + kOffK), q_low = operand_low(smem_base + kOffQ);
    const uint32_t v_low = operand_low_mn_major(smem_base + kOffV, kTile), p_low = operand_low(smem_base + kOffP);
    constexpr uint32_t kPartStep = kPart >> 4, kTileStep = kTile >> 4;
    bool alive = true;
    auto check = [&](int index, uint32_t parity) {
      if (alive && !wait_barrier(bar(index), parity)) { g_error = 2; alive = false; }
    };
    auto issue_scores = [&](int t) {
      const uint32_t stage = (uint32_t)t % kStages;
      check(K_FULL + (int)stage, (uint32_t)(t / kStages) & 1u);
      tensor_fence_after_sync();
      const uint32_t a = k_low + stage * kTileStep;
#pragma unroll
      for (int kk = 0; kk < kDim / 32; ++kk) mma_8bit_ss_halves(tmem_s, a + 2u * kk, q_low + 2u * kk, scores_hi, kk > 0 ? 1u : 0u, elected);
#pragma unroll
      for (int kk = 0; kk < kDim / 32; ++kk) mma_8bit_ss_halves(tmem_s, a + 2u * kk, q_low + kPartStep + 2u * kk, scores_lo, 1u, elected);
      mma_commit_elected(bar(S_FULL), elected);
      mma_commit_elected(bar(K_FREE + (int)stage), elected);
    };
    check(Q_READY, 0u);
    issue_scores(0);
    for (int t = 0; t < tiles; ++t) {
      const uint32_t stage = (uint32_t)t % kStages;
      check(V_FULL + (int)stage, (uint32_t)(t / kStages) & 1u);
      check(P_READY, (uint32_t)t & 1u);
      tensor_fence_after_sync();
      const uint32_t a = v_low + stage * kTileStep;
      // 32 keys are 32 rows of 128 bytes further down the values, 32 bytes further along the weights
#pragma unroll
      for (int kk = 0; kk < kKeys / 32; ++kk)
        mma_8bit_ss_halves(tmem_o, a + (uint32_t)kk * (4096u >> 4), p_low + 2u * kk, values_hi, t > 0 || kk > 0 ? 1u : 0u, elected);
#pragma unroll
      for (int kk = 0; kk < kKeys / 32; ++kk)
        mma_8bit_ss_halves(tmem_o, a + (uint32_t)kk * (4096u >> 4), p_low + kPartStep + 2u * kk, values_lo, 1u, elected);
      mma_commit_elected(bar(V_FREE + (int)stage), elected);
      // the next scores are issued behind this product, so that their barrier also says that O^T may be rescaled
      if (t + 1 < tiles) issue_scores(t + 1);
      else mma_commit_elected(bar(O_DONE), elected);
    }
  } else {
    // ------------------------------------------------------------------ softmax: thread = key of the tile, then element
    const int r = threadIdx.x;
    const uint32_t lane_bits = (uint32_t)(warp * 32) << 16;
    bool alive = true;
    // the group's queries in their two parts: a warp takes a head at a time, a lane four elements
    for (int h = warp; h < valid_heads; h += 4) {
      const uint2 raw = *reinterpret_cast<const uint2*>(q + (size_t)row * q_stride + (size_t)(head0 + h) * kDim + lane * 4);
      float x[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                    __uint_as_float(raw.y & 0xffff0000u)};
      const float largest = warp_largest(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
      const int e = least_scale_exponent(fminf(largest, 3.38953139e38f));
      const float inverse = power_of_two(-e);
      uint32_t hi[2], lo[2];
      split(x[0] * inverse, x[1] * inverse, hi[0], lo[0]);
      split(x[2] * inverse, x[3] * inverse, hi[1], lo[1]);
      unsigned char* to = smem + kOffQ + swizzled(h, lane * 4);
      *reinterpret_cast<uint32_t*>(to) = hi[0] | (hi[1] << 16);
      *reinterpret_cast<uint32_t*>(to + kPart) = lo[0] | (lo[1] << 16);
      if (lane == 0 && h < G) factors[h] = power_of_two(e) * scale_log2;
    }
    if (r < G && r >= valid_heads) factors[r] = 0.0f;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    barrier_arrive(bar(Q_READY));
    asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
    float factor_of[G], top[G], top_weight[G], denominator[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      factor_of[g] = factors[g];
      top[g] = top_weight[g] = -INFINITY;
      denominator[g] = 0.0f;
    }
    unsigned char* p_smem = smem + kOffP;
    // a key's page two tiles ahead of its use, its page's scales one
    auto page_at = [&](int t) {
      const int key = begin + t * kKeys + r;
      return t < tiles && key <= position && key >= first_key ? page_of_block(table, table_width, key >> shift, cache.pages) : -1;
    };
    auto scale_at = [&](const float* scales, int page) { return page >= 0 ? scales[(size_t)page * cache.kv_heads + kv_head] : 1.0f; };
    int page = page_at(0), page_next = page_at(1);
    float k_scale = scale_at(cache.k_scales, page), v_scale = scale_at(cache.v_scales, page);
    for (int t = 0; t < tiles; ++t) {
      const uint32_t stage = (uint32_t)t % kStages;
      const int page_after = page_at(t + 2);
      const float k_next = scale_at(cache.k_scales, page_next), v_next = scale_at(cache.v_scales, page_next);
      const bool visible = page >= 0 && begin + t * kKeys + r < part_end;
      const float shift_v = (float)(((__float_as_int(v_scale) >> 23) & 0xff) - 127);      // the exponent of a power of two
      if (!visible) {
        // what the product with this key's weight of 0 reads is zeros, not whatever lies there
        if (alive && !wait_barrier(bar(V_FULL + (int)stage), (uint32_t)(t / kStages) & 1u)) { g_error = 3; alive = false; }
        uint4* mine = reinterpret_cast<uint4*>(smem + kOffV + stage * kTile + r * kDim);
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[i] = make_uint4(0u, 0u, 0u, 0u);
      }
      __syncwarp();
      if (alive && !wait_barrier(bar(S_FULL), (uint32_t)t & 1u)) { g_error = 3; alive = false; }
      __syncwarp();
      tensor_fence_after_sync();
      float s[G];
      tmem_load<G>(tmem_s + lane_bits, s);
      float* mine = &exchange[t & 1][warp][0];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        s[g] = visible ? s[g] * (k_scale * factor_of[g]) : -INFINITY;
        const float a = warp_largest(s[g]), b = warp_largest(s[g] + shift_v);
        if (lane == 0) { mine[g] = a; mine[G + g] = b; }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
      float rescale[G];
      bool grow = false;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float a = fmaxf(fmaxf(exchange[t & 1][0][g], exchange[t & 1][1][g]), fmaxf(exchange[t & 1][2][g], exchange[t & 1][3][g]));
        const float b = fmaxf(fmaxf(exchange[t & 1][0][G + g], exchange[t & 1][1][G + g]),
                              fmaxf(exchange[t & 1][2][G + g], exchange[t & 1][3][G + g]));
        if (a > top[g] + kRises) {
          denominator[g] *= approximate_exp2(top[g] - a);      // 0 when nothing was seen before
          top[g] = a;
        }
        const bool rises = b > top_weight[g] + kRises;
        rescale[g] = rises ? approximate_exp2(top_weight[g] - (b - kHeadroom)) : 1.0f;
        top_weight[g] = rises ? b - kHeadroom : top_weight[g];
        grow = grow || rises;
      }
      // The product with the last tile's weights is over (these scores were issued behind it), so O^T may be rescaled: this thread's
      // lane is an element of the head, its columns are the heads.
      if (t > 0 && grow) {
        float o[G];
        tmem_load<G>(tmem_o + lane_bits, o);
#pragma unroll
        for (int g = 0; g < G; ++g) o[g] *= rescale[g];
        tmem_store<G>(tmem_o + lane_bits, o);
        tmem_store_wait();
      }
#pragma unroll
      for (int g = 0; g < G; g += 2) {
        float w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          denominator[g + i] += visible ? approximate_exp2(s[g + i] - top[g + i]) : 0.0f;
          w[i] = visible ? approximate_exp2(s[g + i] + shift_v - top_weight[g + i]) : 0.0f;
        }
        uint32_t hi, lo;
        split(w[0], w[1], hi, lo);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          unsigned char* to = p_smem + swizzled(g + i, r);
          to[0] = (unsigned char)(hi >> (8 * i));
          to[kPart] = (unsigned char)(lo >> (8 * i));
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tensor_fence_before_sync();
      barrier_arrive(bar(P_READY));
      page = page_next;
      page_next = page_after;
      k_scale = k_next;
      v_scale = v_next;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float total = warp_sum(denominator[g]);    // every thread holds its keys' share
      if (lane == 0) sums[warp][g] = total;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
    if (alive && !wait_barrier(bar(O_DONE), 0u)) { g_error = 3; alive = false; }
    __syncwarp();
    tensor_fence_after_sync();
    float o[G];
    tmem_load<G>(tmem_o + lane_bits, o);
    if (alive) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        if (g >= valid_heads) break;
        float total = (sums[0][g] + sums[1][g]) + (sums[2][g] + sums[3][g]);
        const size_t head = (size_t)row * heads + head0 + g;
        // the products are relative to 2^top_weight, the sum to 2^top
        const float value = total == 0.0f ? 0.0f : o[g] * exp2f(top_weight[g] - top[g]);    // (NaN stays NaN)
        if (num_partitions == 1) {
          if (total != 0.0f && sinks != nullptr) total += exp2f(sinks[head0 + g] * kLog2e - top[g]);
          out[head * kDim + r] = __float2bfloat16_rn(total == 0.0f ? 0.0f : value / total);
        } else {
          partial_o[(head * num_partitions + part) * kDim + r] = value;
          if (r == 0) {
            partial_ml[(head * num_partitions + part) * 2] = top[g];
            partial_ml[(head * num_partitions + part) * 2 + 1] = total;
          }
        }
      }
    }
    tensor_fence_before_sync();
  }
  __syncthreads();
  if (warp == 5) {
    tensor_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(kTmemColumns) : "memory");
  }
}

template <int G>
int launch(const Attention8& a, const CUtensorMap (&maps)[4]) {
  const cudaError_t err = cudaFuncSetAttribute(decode_8bit_kernel<G>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  if (err != cudaSuccess) {
    mir_set_error("%s: cannot reserve %d bytes of shared memory: %s", a.what, kSmemBytes, cudaGetErrorString(err));
    return MIR_CUDA_ERROR;
  }
  const int group = a.heads / a.cache.kv_heads, units = a.cache.kv_heads * ((group + kHeads - 1) / kHeads);
  // a request's CTAs start together; with a handful of rows partitions beyond the contexts come last
  const dim3 grid = a.num_rows <= 4 ? dim3(a.num_rows, units, a.num_partitions) : dim3(a.num_partitions, units, a.num_rows);
  return mir_launch("decode_attention_8bit", decode_8bit_kernel<G>, grid, dim3(kThreads), (size_t)kSmemBytes, a.stream, 0, maps[0], maps[1],
                    maps[2], maps[3], (const bf16*)a.q, a.q_stride, a.cache, a.block_table, a.table_width, a.positions, a.heads,
                    a.scale * kLog2e, a.window, a.partition, a.num_partitions, a.num_rows <= 4 ? 1 : 0, a.partial_o(a.num_rows),
                    a.partial_ml(a.num_rows), (bf16*)a.out, a.sinks);
}

}  // namespace

// 0 if no bounded wait of the kernel ever ran out; else which role gave up last (1 loader, 2 issuer, 3 softmax).  Synchronises the device.
MIR_EXPORT int mir_decode_attention_8bit_error() {
  int flag = 0;
  if (cudaMemcpyFromSymbol(&flag, g_error, sizeof(int)) != cudaSuccess) return -1;
  return flag;
}

// Whether the kernel takes these sizes: head_dim 128, pages of 8 to 128 keys that divide 128.
bool mir_decode_8bit_takes(int head_dim, int page_size) {
  return head_dim == kDim && page_size >= 8 && page_size <= kKeys && kKeys % page_size == 0;
}

int mir_attention_8bit_decode(const Attention8& a) {
  if (a.num_rows > 65535) {
    mir_set_error("%s: %d rows are more than one launch takes", a.what, a.num_rows);
    return MIR_BAD_ARGUMENT;
  }
  const long long rows = (long long)a.cache.pages * a.cache.page_size, width = (long long)a.cache.kv_heads * kDim;
  CUtensorMap maps[4];
  const void* tensors[2] = {a.cache.k, a.cache.v};
  for (int i = 0; i < 4; ++i) {
    const int status = tensor_map_of_bytes(tensors[i & 1], rows, width, width, i < 2 ? a.cache.page_size : kKeys, &maps[i]);
    if (status != MIR_OK) return status;
  }
  const int columns = std::min(a.heads / a.cache.kv_heads, kHeads);
  const int status = columns <= 4 ? launch<4>(a, maps) : (columns <= 8 ? launch<8>(a, maps) : launch<16>(a, maps));
  if (status != MIR_OK || a.num_partitions == 1) return status;
  return mir_merge_8bit(a, a.num_rows);
}
