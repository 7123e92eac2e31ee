// Products of many rounded rows with an 8-bit weight on the 5th-generation tensor cores:
//
//   out[m, n] = sum over blocks b of 128 columns of  sx[b, m] sw[n / 128, b] (xq[m, b] . wq[n, b])
//
// One CTA per SM walks over tiles of 128 rows x 256 columns.  A block of 128 columns is one stage of the ring (16 KB of xq,
// 32 KB of wq: rows of 128 bytes, TMA with the 128-byte swizzle) and four tcgen05.mma kind::f8f6f4 (K = 32 each) into one of
// two accumulators in tensor memory.  The blocks' scales differ, so a block's sums cannot stay there: eight warps read them
// (tcgen05.ld), multiply them with the block's scale and add them to 32-bit sums in registers, 128 columns of one row per thread
// (a weight's scale is the same for 128 columns: one factor per thread and block), while the tensor cores fill the other
// accumulator.  The tensor cores need 512 cycles at their nominal rate for a block of a tile and 750 were measured without the adding; a
// warp reads 4 x 32 columns and adds them with 64 two-wide FMAs, two warps a scheduler, 930 cycles a block with its waits, which sets
// the pace.  4,096 x 5,120 x 25,600: 496 us, 2,160 TFLOP/s (411 us with zeros, so the power limit is part of it); 2,048 x 4,096 x 6,144:
// 60 us, 384 tiles on 148 SMs.  A wait of its own for the rows' scales cost 8%; the first sums of a block asked for only when the block
// before was added, 2%.
#include <algorithm>
#include "eight_bit_tc.cuh"

using namespace mir;
using namespace mir::tc;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kRows = 128, kColumns = 256, kBlock = 128;
constexpr int kStages = 4, kStageBytes = (kRows + kColumns) * kBlock;
// Loader, issuer and two warps that only make up the first warpgroup, then the adders: registers are handed out to four warps at a
// time.  Launched with 168 a thread (3 * 168 = 504); the first four warps give theirs up, 40 + 2 * 232 = 504.
constexpr int kAddingWarps = 8, kThreads = (4 + kAddingWarps) * 32;
constexpr int kFewRegisters = 40, kManyRegisters = 232;
static_assert(kFewRegisters + 2 * kManyRegisters <= 3 * 168, "no more registers than the launch holds");
constexpr uint32_t kTmemColumns = 512;
constexpr int kBox = 32 * 64;               // bytes of a warp's box of results: 32 rows of 64 bytes
constexpr int kSmemBytes = kStages * kStageBytes + kAddingWarps * kBox + 1024;
static_assert(kSmemBytes + kLeastSharedBeside > kSharedOfSm, "no other kernel with tensor memory beside this one");

// Rows' scales of a block, 512 bytes a slot.  The slot of block b is written again for block b + kScaleSlots, which the loader asks for
// when the products of block b + kScaleSlots - kStages = b + 2 are over; those were issued when every adder had read the sums (and the
// scales) of block b.
constexpr int kScaleSlots = kStages + 2;

enum { FULL = 0, EMPTY = FULL + kStages, SUM_FULL = EMPTY + kStages, SUM_FREE = SUM_FULL + 2, BARRIERS = SUM_FREE + 2 };

__device__ int g_error = 0;

// A box of results out of shared memory (in the swizzled layout), stored or, ADD, added in 32 bits.
template <bool ADD>
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  if (ADD)
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                     reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(src), "r"(x), "r"(y) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

template <bool OUT_FLOAT>
__global__ void __launch_bounds__(kThreads, 1)
linear_8bit_tiles_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
                         const __grid_constant__ CUtensorMap out_map, bool boxes, const float* __restrict__ x_scales, const float* __restrict__ w_scales, const void* __restrict__ bias,
                         void* __restrict__ out, long long out_stride, int m, int n, int k, int scale_stride, int row_tiles, int all_tiles, bool accumulate) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long barriers[BARRIERS];
  __shared__ __align__(16) float scales_here[kScaleSlots * kRows];
  __shared__ uint32_t tmem_slot;
  __shared__ int tiles_slot, gave_up_slot;                    // (gave_up: a wait of this CTA ran out, no tile from then on is stored)
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem), bar0 = smem_u32(&barriers[0]);
  auto bar = [&](int index) { return bar0 + 8u * (uint32_t)index; };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int blocks = (k + kBlock - 1) / kBlock;
  if (threadIdx.x == 0) {
    gave_up_slot = 0;
    tiles_slot = *reinterpret_cast<volatile int*>(&g_error) != 0 ? 0 : all_tiles;       // an earlier wait ran out: nothing is begun
    for (int i = 0; i < BARRIERS; ++i) barrier_init(bar(i), i >= SUM_FREE ? (uint32_t)kAddingWarps : (i >= SUM_FULL ? 2u : 1u));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tensor_fence_before_sync();
  __syncthreads();
  tensor_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const int tiles = tiles_slot;
  volatile int* gave_up = &gave_up_slot;
  auto give_up = [&](int role) {
    g_error = role;
    *gave_up = 1;
    __threadfence_block();                                    // (before whatever this thread lets the others go on with)
  };
  grid_dependency_wait();
  grid_launch_dependents();

  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewRegisters));
  if (warp == 0) {
    // ------------------------------------------------------------------ loader
    if (lane == 0) {
      uint32_t stage = 0, parity = 0, slot = 0;
      bool alive = true;
      for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
        const int row0 = tile % row_tiles * kRows, column0 = tile / row_tiles * kColumns;
        for (int b = 0; b < blocks; ++b) {
          if (!wait_barrier(bar(EMPTY + stage), parity ^ 1u)) { give_up(1); alive = false; break; }
          const uint32_t full = bar(FULL + stage), to = smem_base + stage * (uint32_t)kStageBytes;
          barrier_expect_bytes(full, (uint32_t)(kStageBytes + kRows * sizeof(float)));
          tma_load_2d(to, &x_map, full, b * kBlock, row0);
          tma_load_2d(to + kRows * kBlock, &w_map, full, b * kBlock, column0);
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                           smem_u32(scales_here + slot * kRows)), "l"(x_scales + (size_t)b * scale_stride + row0),
                       "r"((uint32_t)(kRows * sizeof(float))), "r"(full)
                       : "memory");
          if (++slot == (uint32_t)kScaleSlots) slot = 0;
          if (++stage == (uint32_t)kStages) { stage = 0; parity ^= 1u; }
        }
      }
      wait_for_copies(bar(FULL), kStages, stage, parity);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ issuer (tcgen05.cuh: from a whole warp)
    constexpr uint32_t idesc = instruction_descriptor_8bit(kRows, kColumns, E4M3, E4M3);
    const uint32_t elected = elect_one();
    const uint32_t a0 = operand_low(smem_base), b0 = operand_low(smem_base + kRows * kBlock);
    uint32_t stage = 0, parity = 0, sum = 0, sum_parity = 0;
    bool alive = true;
    auto check = [&](int index, uint32_t phase) {
      if (alive && !wait_barrier(bar(index), phase)) { give_up(2); alive = false; }
    };
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x)
      for (int b = 0; b < blocks; ++b) {
        check(SUM_FREE + (int)sum, sum_parity ^ 1u);
        check(FULL + (int)stage, parity);
        tensor_fence_after_sync();
        const uint32_t offset = stage * (uint32_t)(kStageBytes >> 4), d = tmem + sum * (uint32_t)kColumns;
#pragma unroll
        for (int kk = 0; kk < kBlock / 32; ++kk)
          mma_8bit_ss_halves(d, a0 + offset + 2u * kk, b0 + offset + 2u * kk, idesc, kk > 0 ? 1u : 0u, elected);
        mma_commit_elected(bar(EMPTY + (int)stage), elected);
        mma_commit_elected(bar(SUM_FULL + (int)sum), elected);
        if (lane == 0) barrier_arrive(bar(SUM_FULL + (int)sum));          // (the rows' scales came with the operands)
        if (++stage == (uint32_t)kStages) { stage = 0; parity ^= 1u; }
        if (++sum == 2u) { sum = 0; sum_parity ^= 1u; }
      }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kManyRegisters));
    // ------------------------------------------------------------------ adders: 128 columns of a row per thread
    const int quarter = warp & 3, half = (warp - 4) >> 2;      // a warp may read the accumulator lanes 32 quarter .. + 31
    const uint32_t lane_bits = (uint32_t)(quarter * 32) << 16;
    uint32_t sum = 0, sum_parity = 0, slot = 0;
    bool alive = true;
    for (int tile = blockIdx.x; tile < tiles && alive; tile += gridDim.x) {
      const int row = tile % row_tiles * kRows + quarter * 32 + lane, column0 = tile / row_tiles * kColumns + half * 128;
      // A weight's scales come 32 blocks at a time, a block to a lane, the next 32 ahead of their use.
      const float* theirs = w_scales + (size_t)min(column0 / kBlock, (n - 1) / kBlock) * blocks;
      float w_held = theirs[min(lane, blocks - 1)], w_next = theirs[min(32 + lane, blocks - 1)];
      float2 total[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) total[i] = make_float2(0.0f, 0.0f);
      // The first columns of a block are asked for before the last ones of the block in front are added.
      uint32_t v[2][32];
      uint32_t from = 0;
      float next_factor = 0.0f;
      auto begin_block = [&](int b) {
        if (b > 0 && (b & 31) == 0) {
          w_held = w_next;
          w_next = theirs[min(b + 32 + lane, blocks - 1)];
        }
        if (alive && !wait_barrier(bar(SUM_FULL + (int)sum), sum_parity)) { give_up(3); alive = false; }
        __syncwarp();
        tensor_fence_after_sync();
        from = tmem + sum * (uint32_t)kColumns + (uint32_t)(half * 128) + lane_bits;
        tmem_load_32_ahead(from, v[0]);
        next_factor = scales_here[slot * kRows + quarter * 32 + lane] * __shfl_sync(0xffffffffu, w_held, b & 31);
        if (++slot == (uint32_t)kScaleSlots) slot = 0;
      };
      begin_block(0);
      for (int b = 0; b < blocks; ++b) {
        const float2 both = make_float2(next_factor, next_factor);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tmem_load_done(v[c & 1]);
          if (c < 3) tmem_load_32_ahead(from + 32u * (c + 1), v[(c + 1) & 1]);
          if (c == 3) {                                        // all of this warp's columns are in registers
            tensor_fence_before_sync();
            __syncwarp();
            if (lane == 0) barrier_arrive(bar(SUM_FREE + (int)sum));
            if (++sum == 2u) { sum = 0; sum_parity ^= 1u; }
            if (b + 1 < blocks) begin_block(b + 1);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i)
            total[c * 16 + i] = fma_two(make_float2(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])), both,
                                        total[c * 16 + i]);
        }
      }
      alive = __all_sync(0xffffffffu, alive && *gave_up == 0);
      if (boxes) {
        // Results by way of shared memory, a box of 32 rows of 64 bytes a warp: the stores are whole sectors, and the next tile's
        // sums are waited for while they are on their way (a thread that stores its own row, 16 bytes of a line at a time, took
        // a tenth of the kernel's time).
        constexpr int kPart = OUT_FLOAT ? 16 : 32;             // columns of a box
        const int row_first = tile % row_tiles * kRows + quarter * 32;
        const uint32_t box = smem_base + (uint32_t)(kStages * kStageBytes + (warp - 4) * kBox);
#pragma unroll
        for (int part = 0; part < 128 / kPart; ++part) {
          const int column = column0 + part * kPart;
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");          // the box before has been read
          __syncwarp();
#pragma unroll
          for (int chunk = 0; chunk < 4; ++chunk) {            // 16 bytes of this thread's row
            uint32_t words[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (OUT_FLOAT) {
                const float2 pair = total[part * 8 + chunk * 2 + i / 2];
                float value = i % 2 ? pair.y : pair.x;
                if (bias != nullptr && column + chunk * 4 + i < n) value += static_cast<const float*>(bias)[column + chunk * 4 + i];
                words[i] = __float_as_uint(value);
              } else {
                float2 pair = total[part * 16 + chunk * 4 + i];
                const int at = column + chunk * 8 + 2 * i;
                if (bias != nullptr && at < n) pair.x += __bfloat162float(static_cast<const bf16*>(bias)[at]);
                if (bias != nullptr && at + 1 < n) pair.y += __bfloat162float(static_cast<const bf16*>(bias)[at + 1]);
                const __nv_bfloat162 both = __floats2bfloat162_rn(pair.x, pair.y);
                words[i] = *reinterpret_cast<const uint32_t*>(&both);
              }
            }
            const uint32_t to = box + (uint32_t)(lane * 64 + ((chunk ^ (lane >> 1 & 3)) << 4));      // (64-byte swizzle)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(words[0]), "r"(words[1]), "r"(words[2]), "r"(words[3])
                         : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0 && alive && row_first < m && column < n) {
            if (OUT_FLOAT && accumulate) tma_store_2d<true>(&out_map, box, column, row_first);
            else tma_store_2d<false>(&out_map, box, column, row_first);
          }
        }
        continue;
      }
      if (!alive || row >= m || column0 >= n) continue;
      const int columns = min(128, n - column0);
      const size_t at = (size_t)row * out_stride + column0;
      if (OUT_FLOAT) {
        float* to = static_cast<float*>(out) + at;
        const float* extra = static_cast<const float*>(bias);
        const bool wide = columns == 128 && (reinterpret_cast<uintptr_t>(to) & 15) == 0;
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          float4 value = make_float4(total[i].x, total[i].y, total[i + 1].x, total[i + 1].y);
          float* part = reinterpret_cast<float*>(&value);
          if (extra != nullptr)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (2 * i + j < columns) part[j] += extra[column0 + 2 * i + j];
          if (wide) {
            if (accumulate) {
              const float4 old = *reinterpret_cast<const float4*>(to + 2 * i);
              value.x += old.x; value.y += old.y; value.z += old.z; value.w += old.w;
            }
            *reinterpret_cast<float4*>(to + 2 * i) = value;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (2 * i + j < columns) to[2 * i + j] = accumulate ? to[2 * i + j] + part[j] : part[j];
          }
        }
      } else {
        bf16* to = static_cast<bf16*>(out) + at;
        const bf16* extra = static_cast<const bf16*>(bias);
        const bool wide = columns == 128 && (reinterpret_cast<uintptr_t>(to) & 15) == 0;
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          if (extra != nullptr)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (2 * (i + j) < columns) total[i + j].x += __bfloat162float(extra[column0 + 2 * (i + j)]);
              if (2 * (i + j) + 1 < columns) total[i + j].y += __bfloat162float(extra[column0 + 2 * (i + j) + 1]);
            }
          if (wide) {
            uint4 packed;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
            for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(total[i + j].x, total[i + j].y);
            *reinterpret_cast<uint4*>(to + 2 * i) = packed;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (2 * (i + j) < columns) to[2 * (i + j)] = __float2bfloat16_rn(total[i + j].x);
              if (2 * (i + j) + 1 < columns) to[2 * (i + j) + 1] = __float2bfloat16_rn(total[i + j].y);
            }
          }
        }
      }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    tensor_fence_before_sync();
  }
  __syncthreads();
  if (warp == 1) {
    tensor_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
  }
}

}  // namespace

// 0 if no bounded wait of the kernel ever ran out; else which role gave up last (1 loader, 2 issuer, 3 adders).
// Synchronises the device.  `next`: exchange_flag.
MIR_EXPORT int mir_linear_8bit_tiles_error(int next) {
  return exchange_flag(g_error, next);
}

int mir_linear_8bit_tiles(const uint8_t* codes, const float* scales, int scale_stride, const uint8_t* weight, const float* w_scales, const void* bias,
                          void* out, long long out_stride, int m, int n, int k, bool out_float, bool accumulate, cudaStream_t stream) {
  CUtensorMap x_map, w_map;
  int status = tensor_map_of_bytes(codes, m, k, k, kRows, &x_map);
  if (status != MIR_OK) return status;
  status = tensor_map_of_bytes(weight, n, k, k, kColumns, &w_map);
  if (status != MIR_OK) return status;
  const int row_tiles = (m + kRows - 1) / kRows;
  const long long tiles = (long long)row_tiles * ((n + kColumns - 1) / kColumns);
  if (tiles > 0x7fffffffll) {
    mir_set_error("linear_8bit: %d rows of %d columns are more than one launch takes", m, n);
    return MIR_BAD_ARGUMENT;
  }
  auto kernel = out_float ? linear_8bit_tiles_kernel<true> : linear_8bit_tiles_kernel<false>;
  status = reserve_shared(kernel, kSmemBytes, "linear_8bit");
  if (status != MIR_OK) return status;
  // results by way of shared memory where their rows begin and lie on 16-byte boundaries
  const int width = out_float ? 4 : 2;
  const bool boxes = ((uintptr_t)out & 15) == 0 && (out_stride * width) % 16 == 0;
  CUtensorMap out_map = x_map;
  if (boxes) {
    status = tensor_map_of_results(out, out_float, m, n, out_stride * width, &out_map);
    if (status != MIR_OK) return status;
  }
  const int ctas = (int)std::min<long long>(tiles, mir_sm_count());
  return mir_launch("linear_8bit_tiles", kernel, dim3(ctas), dim3(kThreads), (size_t)kSmemBytes, stream, 0, x_map, w_map, out_map, boxes,
                    scales, w_scales, bias, out, out_stride, m, n, k, scale_stride, row_tiles, (int)tiles, accumulate);
}
