// Products of few rows (1 to 128) with an 8-bit weight: the weight's bytes are what takes the time.
//
//   out[m, n] = sum over blocks b of 128 columns of  sx[b, m] sw[n / 128, b] (xq[m, b] . wq[n, b])
//
// A tile of 128 weight rows is the A operand of tcgen05.mma kind::f8f6f4 (a block of it is 128 rows of 128 bytes, one TMA box),
// the rows of x are the B operand (N = 16, 32, 64 or 128 columns), so a block's sums are [128 weight rows, N rows of x] in tensor
// memory: four warps read them, a weight row per thread, scale them (the weight's scale is the same for the whole tile and
// block) and add them up in registers, while the tensor cores fill the next accumulator.
//
// K is cut over a cluster of up to eight CTAs, so that enough CTAs have loads on their way whatever the shape; the ranks' sums are
// added in rank order by way of distributed shared memory.  Up to 16 rows are rounded to e4m3 by the CTAs themselves (each its
// share of K, while the first weights are on their way); more come rounded from a kernel in front, a box of them beside each block
// of weights.
//
// Measured: 8 rows x 2,560 x 19,456 (50 MB): 14.9 us, 3.4 TB/s; 1 x 2,560 x 152,064 (389 MB): 60.0 us, 6.5 TB/s, the copy rate; 1 x 2,560 x
// 2,560: 5.9 us on the GPU, latency alone.
#include <algorithm>
#include "eight_bit_tc.cuh"

using namespace mir;
using namespace mir::tc;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kRows = 128, kBlock = 128;
constexpr int kWorkers = 128, kThreads = kWorkers + 64;     // four warps that round, scale and add; loader; issuer
constexpr int kLoader = 4, kIssuer = 5;                     // warps
constexpr int kMostStages = 6, kMostBlocks = 40;
constexpr int kOwnRows = 16;                                // rows that the CTAs round themselves, a quarter of their blocks after the other
constexpr int kQuarters = 4;

enum { FULL = 0, EMPTY = FULL + kMostStages, SUM_FULL = EMPTY + kMostStages, SUM_FREE = SUM_FULL + 4, X_READY = SUM_FREE + 4, BARRIERS = X_READY + kQuarters };

__device__ int g_error = 0;

// N: columns of the products (rows of x, filled up).  OWN: x is bf16 and rounded here (N is 16 then), else it comes rounded.
template <int N, bool OWN>
__global__ void __launch_bounds__(kThreads)
linear_8bit_few_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const bf16* __restrict__ x,
                       long long x_stride, const float* __restrict__ x_scales, int scale_stride, const float* __restrict__ w_scales,
                       const void* __restrict__ bias, void* __restrict__ out, long long out_stride, int m, int n, int k, int splits,
                       int per_split, int stages, int ring_bytes, int x_block_bytes, bool out_float, bool accumulate) {
  constexpr int kBuffers = N <= 32 ? 4 : 2;
  constexpr uint32_t kColumns = (uint32_t)(kBuffers * N);
  constexpr int kChunk = 16;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long barriers[BARRIERS];
  __shared__ uint32_t tmem_slot;
  __shared__ bool go_slot;
  __shared__ int gave_up_slot;                                // a wait of this CTA ran out, or nothing was begun: no result comes of it
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // without a cluster the CTAs walk over the tiles of 128 weight rows
  const int first_tile = blockIdx.x / splits, tile_step = gridDim.x / splits, rank = blockIdx.x % splits;
  const int tiles = (n + kRows - 1) / kRows, blocks = (k + kBlock - 1) / kBlock, first = rank * per_split;
  const int mine = max(0, min(blocks, first + per_split) - first);      // blocks of this CTA
  // shared memory: the ring (a block of weights, and of x where it comes rounded; in its place, when the products are over, the sums for
  // the other ranks, [row of x][128]), x's own blocks (8 or 16 rows of 128 bytes; with 8 the products read what follows as the
  // other columns, which nobody looks at), the rows' scales [block][N]
  const int stage_bytes = kRows * kBlock + (OWN ? 0 : N * kBlock);
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* own_x = smem + ring_bytes;
  float* scales = reinterpret_cast<float*>(own_x + (OWN ? (size_t)per_split * x_block_bytes + 1024 : 0));
  float* sums = reinterpret_cast<float*>(smem);
  const uint32_t smem_base = smem_u32(smem), bar0 = smem_u32(&barriers[0]);
  auto bar = [&](int index) { return bar0 + 8u * (uint32_t)index; };
  if (threadIdx.x == 0) {
    go_slot = *reinterpret_cast<volatile int*>(&g_error) == 0;             // an earlier wait ran out: nothing is begun
    gave_up_slot = go_slot ? 0 : 1;
    for (int i = 0; i < BARRIERS; ++i)
      barrier_init(bar(i), i >= SUM_FREE && i < SUM_FREE + 4 ? 4u : (i >= X_READY ? (uint32_t)kWorkers : 1u));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tensor_fence_before_sync();
  __syncthreads();
  tensor_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  grid_dependency_wait();
  grid_launch_dependents();
  const bool go = go_slot;
  volatile int* gave_up = &gave_up_slot;
  auto give_up = [&](int role) {
    g_error = role;
    *gave_up = 1;
    __threadfence_block();                                    // (before whatever this thread lets the others go on with)
  };

  if (warp == kLoader) {
    if (lane == 0 && go) {
      uint32_t stage = 0, parity = 0;
      bool alive = true;
      for (int tile = first_tile; tile < tiles && alive; tile += tile_step)
      for (int b = 0; b < mine; ++b) {
        if (!wait_barrier(bar(EMPTY + (int)stage), parity ^ 1u)) { give_up(1); alive = false; break; }
        const uint32_t full = bar(FULL + (int)stage), to = smem_base + stage * (uint32_t)stage_bytes;
        barrier_expect_bytes(full, (uint32_t)stage_bytes);
        tma_load_2d(to, &w_map, full, (first + b) * kBlock, tile * kRows);
        if (!OWN) tma_load_2d(to + kRows * kBlock, &x_map, full, (first + b) * kBlock, 0);
        if (++stage == (uint32_t)stages) { stage = 0; parity ^= 1u; }
      }
      wait_for_copies(bar(FULL), (uint32_t)stages, stage, parity);
    }
  } else if (warp == kIssuer) {
    if (go) {
      constexpr uint32_t idesc = instruction_descriptor_8bit(kRows, N, E4M3, E4M3);
      const uint32_t elected = elect_one();
      const uint32_t a0 = operand_low(smem_base), x0 = operand_low(smem_u32(own_x));
      bool alive = true;
      auto check = [&](int index, uint32_t phase) {
        if (alive && !wait_barrier(bar(index), phase)) { give_up(2); alive = false; }
      };
      uint32_t stage = 0, parity = 0, buffer = 0, buffer_parity = 0;
      const int quarter = (mine + kQuarters - 1) / kQuarters;
      for (int tile = first_tile; tile < tiles; tile += tile_step)
      for (int b = 0; b < mine; ++b) {
        if (OWN && tile == first_tile && b % quarter == 0) check(X_READY + b / quarter, 0u);
        check(SUM_FREE + (int)buffer, buffer_parity ^ 1u);
        check(FULL + (int)stage, parity);
        __syncwarp();
        tensor_fence_after_sync();
        const uint32_t a = a0 + stage * (uint32_t)(stage_bytes >> 4);
        const uint32_t c = OWN ? x0 + (uint32_t)b * (uint32_t)(x_block_bytes >> 4) : a + (uint32_t)(kRows * kBlock >> 4);
#pragma unroll
        for (int kk = 0; kk < kBlock / 32; ++kk)
          mma_8bit_ss_halves(tmem + buffer * (uint32_t)N, a + 2u * kk, c + 2u * kk, idesc, kk > 0 ? 1u : 0u, elected);
        mma_commit_elected(bar(EMPTY + (int)stage), elected);
        mma_commit_elected(bar(SUM_FULL + (int)buffer), elected);
        if (++stage == (uint32_t)stages) { stage = 0; parity ^= 1u; }
        if (++buffer == (uint32_t)kBuffers) { buffer = 0; buffer_parity ^= 1u; }
      }
    }
  } else {
    // ------------------------------------------------------------------ workers
    if (OWN) {
      // a warp rounds a row's block at a time, a lane four columns of it
      constexpr int kAhead = 8;
      const int quarter = (mine + kQuarters - 1) / kQuarters;
      for (int q = 0; q < kQuarters; ++q) {
        const int begin = min(mine, q * quarter) * m, end = min(mine, (q + 1) * quarter) * m;      // units: (block, row)
        for (int u0 = begin + warp; u0 < end; u0 += 4 * kAhead) {
          uint2 raw[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int unit = u0 + 4 * i, block = unit / m, row = unit - block * m, column = (first + block) * kBlock + lane * 4;
            raw[i] = make_uint2(0u, 0u);
            if (unit < end && column < k) raw[i] = *reinterpret_cast<const uint2*>(x + (size_t)row * x_stride + column);
          }
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            const int unit = u0 + 4 * i, block = unit / m, row = unit - block * m;
            if (unit >= end) break;
            const float v[4] = {__uint_as_float(raw[i].x << 16), __uint_as_float(raw[i].x & 0xffff0000u), __uint_as_float(raw[i].y << 16),
                                __uint_as_float(raw[i].y & 0xffff0000u)};
            uint32_t bits = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t magnitude = __float_as_uint(v[j]) & 0x7fffffffu;
              if (magnitude < 0x7f800000u) bits = max(bits, magnitude);
            }
            bits = __reduce_max_sync(0xffffffffu, bits);
            const int exponent = least_scale_exponent(__uint_as_float(bits));
            const float inverse = power_of_two(-exponent);
            *reinterpret_cast<uint32_t*>(own_x + (size_t)block * x_block_bytes + row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) =
                to_e4m3x2(v[0] * inverse, v[1] * inverse) | (to_e4m3x2(v[2] * inverse, v[3] * inverse) << 16);
            if (lane == 0) scales[block * N + row] = power_of_two(exponent);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        barrier_arrive(bar(X_READY + q));
      }
    } else {
      for (int i = threadIdx.x; i < mine * N; i += kWorkers) {
        const int block = i / N, row = i % N;
        scales[i] = row < m ? x_scales[(size_t)(first + block) * scale_stride + row] : 0.0f;
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory");
    // a tile's scales, a block to a lane (40 at most), the next tile's ahead of their use
    auto weight_scales = [&](int tile, float (&held)[2]) {
      const float* theirs = w_scales + (size_t)min(tile, tiles - 1) * blocks;
      held[0] = theirs[min(first + lane, blocks - 1)];
      held[1] = theirs[min(first + 32 + lane, blocks - 1)];
    };
    float held[2], next[2];
    weight_scales(first_tile, held);
    bool alive = go;
    uint32_t buffer = 0, buffer_parity = 0;
    const uint32_t lane_bits = (uint32_t)(warp * 32) << 16;
    for (int tile = first_tile; tile < tiles; tile += tile_step) {
      weight_scales(tile + tile_step, next);
      float total[N];
#pragma unroll
      for (int i = 0; i < N; ++i) total[i] = 0.0f;
      for (int b = 0; b < mine; ++b) {
        const float w_scale = __shfl_sync(0xffffffffu, b < 32 ? held[0] : held[1], b & 31);
        if (alive && !wait_barrier(bar(SUM_FULL + (int)buffer), buffer_parity)) { give_up(3); alive = false; }
        __syncwarp();
        tensor_fence_after_sync();
        const uint32_t from = tmem + buffer * (uint32_t)N + lane_bits;
#pragma unroll
        for (int c = 0; c < N; c += kChunk) {
          float v[kChunk];
          tmem_load_16(from + (uint32_t)c, v);
          if (c + kChunk == N) {                              // all of this warp's columns are in registers
            tensor_fence_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(bar(SUM_FREE + (int)buffer));
          }
#pragma unroll
          for (int i = 0; i < kChunk; i += 4) {
            // the two scales first: sums times a row's scale alone may lie beyond the 32-bit numbers where the results do not (a row's
            // scale is a power of two, so only the addition rounds)
            const float4 x_scale = *reinterpret_cast<const float4*>(scales + b * N + c + i);
            total[c + i] = fmaf(v[i], x_scale.x * w_scale, total[c + i]);
            total[c + i + 1] = fmaf(v[i + 1], x_scale.y * w_scale, total[c + i + 1]);
            total[c + i + 2] = fmaf(v[i + 2], x_scale.z * w_scale, total[c + i + 2]);
            total[c + i + 3] = fmaf(v[i + 3], x_scale.w * w_scale, total[c + i + 3]);
          }
        }
        if (++buffer == (uint32_t)kBuffers) { buffer = 0; buffer_parity ^= 1u; }
      }
      held[0] = next[0];
      held[1] = next[1];
      const int column = tile * kRows + threadIdx.x;
      if (splits > 1) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i < m) sums[i * kRows + threadIdx.x] = total[i];
      } else if (column < n && alive && *gave_up == 0) {
        const float extra = bias == nullptr ? 0.0f : (out_float ? static_cast<const float*>(bias)[column]
                                                                : __bfloat162float(static_cast<const bf16*>(bias)[column]));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i >= m) continue;
          const size_t at = (size_t)i * out_stride + column;
          if (out_float) {
            float* to = static_cast<float*>(out) + at;
            *to = accumulate ? *to + (total[i] + extra) : total[i] + extra;
          } else {
            static_cast<bf16*>(out)[at] = __float2bfloat16_rn(total[i] + extra);
          }
        }
      }
    }
    tensor_fence_before_sync();
  }
  if (splits > 1) {
    // the ranks' sums, added in rank order: rank r finishes the rows r, r + splits, ...
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int column = first_tile * kRows + threadIdx.x;
    // a rank that gave up has no sums: then nothing is stored, whichever rank's rows they are (a lane asks a rank)
    int missing = 0;
    if (warp < kWorkers / 32 && lane < splits) {
      uint32_t there;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(&gave_up_slot)), "r"(lane));
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(missing) : "r"(there) : "memory");
    }
    missing = __any_sync(0xffffffffu, missing != 0);
    if (threadIdx.x < kWorkers && column < n && missing == 0) {
      const float extra = bias == nullptr ? 0.0f : (out_float ? static_cast<const float*>(bias)[column]
                                                              : __bfloat162float(static_cast<const bf16*>(bias)[column]));
      for (int row = rank; row < m; row += splits) {
        const uint32_t here = smem_u32(sums + row * kRows + threadIdx.x);
        float value = 0.0f;
        for (int r = 0; r < splits; ++r) {
          uint32_t there;
          float part;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(r));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(there) : "memory");
          value += part;
        }
        value += extra;
        const size_t at = (size_t)row * out_stride + column;
        if (out_float) {
          float* to = static_cast<float*>(out) + at;
          *to = accumulate ? *to + value : value;
        } else {
          static_cast<bf16*>(out)[at] = __float2bfloat16_rn(value);
        }
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncthreads();
  if (warp == kIssuer) {
    tensor_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
  }
}

// How a call is cut: K over `splits` CTAs of a cluster, and `ctas` of them on an SM.
struct Cut {
  int splits, per_split, stages, ring_bytes, x_block_bytes, bytes, ctas;
};
Cut cut_for(int m, int n_columns, bool own, int blocks, int splits) {
  Cut c;
  c.splits = splits;
  c.per_split = (blocks + splits - 1) / splits;
  c.x_block_bytes = own ? (m <= 8 ? 8 : 16) * kBlock : 0;
  const int stage_bytes = kRows * kBlock + (own ? 0 : n_columns * kBlock);
  const int sums = splits > 1 ? (m * kRows * 4 + 1023) / 1024 * 1024 : 0;
  const int rest = 1024 + (own ? c.per_split * c.x_block_bytes + 1024 : 0) + c.per_split * n_columns * 4;
  // three CTAs an SM where that leaves each a ring of three stages, else two
  for (c.ctas = n_columns <= 32 ? 3 : 2; c.ctas >= 1; --c.ctas) {          // (registers: two with more columns)
    const int budget = kSharedOfSm / c.ctas - 1024 - 512;
    c.stages = std::min({c.per_split, kMostStages, (budget - rest) / stage_bytes});
    if (rest + sums <= budget && (c.stages >= std::min(3, c.per_split) || c.ctas == 1)) break;
  }
  c.ring_bytes = std::max(c.stages * stage_bytes, sums);
  c.bytes = std::max(rest + c.ring_bytes, kLeastSharedBeside);      // (no less than keeps it off an SM whose tensor memory is all taken)
  return c;
}

template <int N, bool OWN>
int launch(const uint8_t* codes, const float* scales, int scale_stride, const void* x, long long x_stride, const uint8_t* weight,
           const float* w_scales, const void* bias, void* out, long long out_stride, int m, int n, int k, bool out_float, bool accumulate,
           int forced, cudaStream_t stream) {
  const int blocks = (k + kBlock - 1) / kBlock, tiles = (n + kRows - 1) / kRows;
  CUtensorMap w_map, x_map;
  int status = tensor_map_of_bytes(weight, n, k, k, kRows, &w_map);
  if (status != MIR_OK) return status;
  x_map = w_map;
  if (!OWN) {
    status = tensor_map_of_bytes(codes, m, k, k, N, &x_map);
    if (status != MIR_OK) return status;
  }
  // the most CTAs that are all there at once, two blocks each at least; with more tiles than that they walk over the tiles
  Cut cut = cut_for(m, N, OWN, blocks, 1);
  for (int splits = forced > 0 ? forced : 8; splits >= 1; splits /= 2) {
    while ((blocks + splits - 1) / splits > kMostBlocks) splits *= 2;          // (no more than 8: mir_linear_8bit_few_takes)
    cut = cut_for(m, N, OWN, blocks, splits);
    if (splits == 1 || forced > 0 || (blocks + splits / 2 - 1) / (splits / 2) > kMostBlocks || ((long long)tiles * splits <= (long long)cut.ctas * mir_sm_count() && blocks >= 2 * splits)) break;
  }
  status = reserve_shared(linear_8bit_few_kernel<N, OWN>, cut.bytes, "linear_8bit");
  if (status != MIR_OK) return status;
  const int walkers = cut.splits > 1 ? tiles : std::min(tiles, cut.ctas * mir_sm_count());
  return mir_launch_cluster(mir_pdl_enabled(), "linear_8bit_few", linear_8bit_few_kernel<N, OWN>, dim3((unsigned)walkers * cut.splits),
                            dim3(kThreads), (size_t)cut.bytes, stream, dim3(cut.splits, 1, 1), w_map, x_map, (const bf16*)x, x_stride, scales,
                            scale_stride, w_scales, bias, out, out_stride, m, n, k, cut.splits, cut.per_split, cut.stages, cut.ring_bytes,
                            cut.x_block_bytes, out_float, accumulate);
}

int g_forced_splits = 0;          // for measurements (0: the launcher chooses)

}  // namespace

// 0 if no bounded wait of the kernel ever ran out; else which role gave up last (1 loader, 2 issuer, 3 workers).  Synchronises the device.  `next`: exchange_flag.
MIR_EXPORT int mir_linear_8bit_few_error(int next) {
  return exchange_flag(g_error, next);
}

// Whether the kernel takes the sizes: a CTA keeps its share of K as rounded rows and scales, 40 blocks at most of it; and whether it
// then rounds the rows itself.
bool mir_linear_8bit_few_takes(int m, int k) { return m <= 128 && (k + kBlock - 1) / kBlock <= 8 * kMostBlocks; }
bool mir_linear_8bit_few_rounds(int m) { return m <= kOwnRows; }

int mir_linear_8bit_few(const uint8_t* codes, const float* scales, int scale_stride, const void* x, long long x_stride,
                        const uint8_t* weight, const float* w_scales, const void* bias, void* out, long long out_stride, int m, int n, int k,
                        bool out_float, bool accumulate, cudaStream_t stream) {
#define MIR_FEW(N, OWN) \
  launch<N, OWN>(codes, scales, scale_stride, x, x_stride, weight, w_scales, bias, out, out_stride, m, n, k, out_float, accumulate, g_forced_splits, stream)
  if (m <= kOwnRows) return MIR_FEW(16, true);
  if (m <= 32) return MIR_FEW(32, false);
  if (m <= 64) return MIR_FEW(64, false);
  return MIR_FEW(128, false);
#undef MIR_FEW
}

// For measurements: over how many CTAs K is cut (1, 2, 4 or 8; 0: the launcher's rule).
MIR_EXPORT int mir_linear_8bit_few_set_splits(int splits) {
  if (splits != 0 && splits != 1 && splits != 2 && splits != 4 && splits != 8) return MIR_BAD_ARGUMENT;
  g_forced_splits = splits;
  return MIR_OK;
}
