// Causal attention of portions over the 8-bit cache on the 5th-generation tensor cores, head_dim 128, pages of 8 to 128 keys:
//
//   out = sum_j p_j S_v[page of j] V_j / sum_j p_j,   p_j = exp(scale q . (S_k[page of j] K_j) - reference)
//
// A row is a (token, query head of the kv head's group) pair, a work item 128 rows of one request and kv head (and one partition of
// the keys, where few items are split): the heads of a group share the tiles of keys, and a short portion still fills a tile.
// A CTA per SM walks over items, heaviest first; every ring and barrier runs on across them.  Per tile of 128 keys:
//
//   S = Q K^T     kind::f8f6f4, K as the cache holds it, Q in two parts q = hi + lo, hi = e4m3(q 2^-e), lo = e5m2 of what hi leaves (a
//                 bf16 number's eight significant bits fit into the two; off by at most 2^-21.8 of the row's largest element);
//   P = exp2(S S_k scale log2 e - reference), rounded to bf16, over the scores in tensor memory;
//   O += P V      kind::f16, V as bf16: an e4m3 number times a power of two is exact in bf16, so the page's scale is in it.
//
// K needs no conversion, V four instructions for two elements: a byte's sign is spread over 16 bits (prmt), shifted by 4 and masked,
// which is the bf16 number of the same exponent field, 2^-120 times the e4m3 one (subnormals too); a product in bf16 with 2^120
// times the page's scale puts that right.  Both products take as long as they would in bf16.
//
// Measured: 512 tokens at 16,384 (32 heads over 8, pages of 16; 128 items): 171 us, 800 TFLOP/s; three prompts of up to 2,048: 159 us.
// The tensor cores are busy for two fifths of the time; the schedulers' slots (seven tenths are taken) and the chain of hand-overs of a tile, of which the widening is the longest, bound the kernel, and it is close to the instruction caches: writing a
// loop out that is short now (the widening's, twice as long) takes 25% more.  Every wait left out was worth 1 to 3%.
//
// Roles: a scout reads block table and scales ahead and leaves them in shared memory; two loaders (TMA) for keys and values; an
// issuer; eight warps that split queries and widen values; two streams of eight softmax warps that take the tiles in turn, with a
// running reference that they hand to each other (raised when a tile's maximum exceeds it by 2^8), three score accumulators and
// one for the output, which a stream that raises the reference rescales when the product of the tile before is over.
// A hidden key's score becomes -inf by selection; rows of values that no query of the item sees are written as zeros, and so are NaN
// values that only some of its queries see (0 times NaN is NaN): those queries get them when the item is over.
#include <algorithm>
#include "eight_bit_tc.cuh"

using namespace mir;
using namespace mir::tc;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kRows = 128, kKeys = 128, kDim = 128;
constexpr int kTile8 = kKeys * kDim;                        // bytes of a tile of keys, values or query parts as they are
constexpr int kHalf = 128 * 128, kTile16 = 2 * kHalf;       // bytes of a tile of bf16 values: two halves of 64 elements
constexpr int kKeyStages = 3, kRawStages = 3, kValueStages = 2, kInfos = 8, kSlots = 16;
constexpr int kOffQ = 0, kOffK = 2 * kTile8, kOffRaw = kOffK + kKeyStages * kTile8, kOffV = kOffRaw + kRawStages * kTile8;
constexpr int kSmemBytes = kOffV + kValueStages * kTile16 + 1024;
static_assert(kSmemBytes + kLeastSharedBeside > kSharedOfSm, "no other kernel with tensor memory beside this one");
constexpr int kParts = 2, kCols = kKeys / kParts;           // softmax threads of a row and stream; columns of each
constexpr int kStreams = 2, kStreamThreads = kRows * kParts;
enum { kKeyLoader = 0, kIssuer = 1, kValueLoader = 2, kScout = 3, kFirstConverter = 4, kFirstSoftmax = 12 };     // warps
// (Eight converting warps: four had a quarter of their schedulers' slots each, took 3,100 cycles for a tile's values and set the pace.)
constexpr int kConverters = 256, kThreads = (kFirstSoftmax + 8 * kStreams) * 32;
// launched with 72 registers a thread (7 * 72 = 504); the first twelve warps give some up: 40 + 2 * 40 + 4 * 96 = 504
constexpr int kRoleRegisters = 40, kConverterRegisters = 40, kSoftmaxRegisters = 96;
static_assert(kRoleRegisters + 2 * kConverterRegisters + 4 * kSoftmaxRegisters <= 7 * 72, "no more registers than the launch holds");
constexpr uint32_t kTmemColumns = 512;                      // S at 0, 128, 256; O at 384
constexpr float kRises = 8.0f;

// Tiles are counted over a CTA's items (g), items with tiles too (n).  Three stages: g % 3, phase g / 3; two: g & 1, g >> 1.
// Q_FULL goes by n & 3: the softmax may begin item n when the queries of the items behind it are there already.
enum { Q_FULL = 0, Q_FREE = Q_FULL + 4, K_FULL, K_FREE = K_FULL + 3, RAW_FULL = K_FREE + 3, RAW_FREE = RAW_FULL + 3, V_FULL = RAW_FREE + 3,
       V_FREE = V_FULL + 2, S_FULL = V_FREE + 2, P_READY = S_FULL + 3, REF_READY = P_READY + 3, PV_DONE = REF_READY + 2,
       ITEM_DONE = PV_DONE + 2, O_FREE, INFO_FULL, INFO_FREE = INFO_FULL + kInfos, BARRIERS = INFO_FREE + kInfos };

__device__ int g_error = 0;

__device__ __forceinline__ float warp_largest(float v) {
  float top;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(v));
  return top;
}

// What the scout leaves of a tile: each page's first row of the cache (below 0: not there, or no query of the item sees it), its scales.
struct Info {
  int row[kSlots];
  float k_scale[kSlots];
  uint32_t v_factor[kSlots], v_rest[kSlots];               // what a lifted value is multiplied by: 2^120 times its scale, as one or two bf16 pairs
  int whole, one_factor;                                   // all pages are there; v_rest is 1 throughout
};

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994), (n + n m / 2^32) >> s: s the bits of d - 1, m = floor(2^32 (2^s - d) / d) + 1 (a division takes some 25
// instructions, and every role works out its items by itself).
struct Divider {
  uint32_t factor;
  int bits, by;
  explicit Divider(int d) : bits(0), by(d) {
    while ((1ll << bits) < d) ++bits;
    factor = (uint32_t)((((1ull << bits) - (unsigned long long)d) << 32) / (unsigned long long)d + 1ull);
  }
  __device__ __forceinline__ int operator()(int n) const { return (int)((__umulhi((uint32_t)n, factor) + (uint32_t)n) >> bits); }
};

struct Work {
  int request, kv_head, part, first_row, rows, first_token, first_position, last_position, first_key, begin, end, tiles;
};

struct Items {
  const int* query_starts;
  const int* context_lens;
  int num_rows, tokens, window, partition, row_tiles, count;
  const Divider &kv_heads, &num_partitions, &group;
  // Item `index`: the kv head is the fast index, then the partition, then the batch's tiles of rows from the last one of the last request
  // backwards (late tiles see the most keys and come first).  False beyond the last item.
  __device__ __forceinline__ bool at(int index, Work& w) const {
    if (index < 0 || index >= count) return false;
    const int rest = kv_heads(index), from_last = num_partitions(rest);
    w.kv_head = index - rest * kv_heads.by;
    w.part = rest - from_last * num_partitions.by;
    int remaining = row_tiles - 1 - from_last;
    Portion portion{0, 0};
    w.request = request_of_tile<kRows>(query_starts, num_rows, tokens, group.by, remaining, portion);
    if (w.request < 0) return false;
    w.first_row = remaining * kRows;
    w.rows = min(kRows, portion.count * group.by - w.first_row);
    w.first_token = portion.first;
    const int start = context_lens[w.request] - portion.count;
    w.first_position = start + group(w.first_row);
    w.last_position = start + group(w.first_row + w.rows - 1);
    w.first_key = (window > 0 && w.first_position >= window) ? w.first_position + 1 - window : 0;
    w.begin = max(w.first_key / kKeys * kKeys, w.part * partition);
    w.end = (int)min((long long)w.last_position + 1, (long long)(w.part + 1) * partition);
    w.tiles = w.end > w.begin ? (w.end - w.begin + kKeys - 1) / kKeys : 0;
    return true;
  }
};

// The k-th item of CTA `cta`: rounds are dealt out back and forth, so that the CTA with a round's heaviest item gets the next one's lightest.
__device__ __forceinline__ int item_of(int k, int cta, int ctas) { return k * ctas + ((k & 1) ? ctas - 1 - cta : cta); }

struct Counter {                                            // stage and phase of a ring
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void step(uint32_t stages) {
    if (++stage == stages) { stage = 0; phase ^= 1u; }
  }
};

__device__ __forceinline__ float max_of_three(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

struct Handoff {
  bool has_from;
  uint32_t from_barrier, from_phase, to_barrier;
  const float* from;
  float* to;
};

// One tile of the softmax for this thread's kCols columns of its row, from column `first` on: the scores, times their pages' scales; the hidden
// ones (outside low .. high, or of pages that are not there) -inf; the row's maximum with the thread that has the other columns; the
// reference, which comes from the tile before and goes to the next; the weights, packed to bf16.  Returns their sum.
template <bool MASKED>
__device__ __forceinline__ float softmax_tile(uint32_t scores, int first, int low, int high, float scale, const Info& info, int shift,
                                              float& reference, float& factor, bool& grow, float& own_factor, uint32_t (&packed)[kCols / 2],
                                              float* shared_max, int part, int team, const Handoff& handoff, bool& alive) {
  uint32_t raw[2][32];
  tmem_load_32_ahead(scores + (uint32_t)first, raw[0]);
  tmem_load_32_ahead(scores + (uint32_t)first + 32u, raw[1]);
  // Eight columns are of one page (a page has eight keys or more): their scores share a factor, which is positive, so that the maximum is
  // taken first and the multiplication is part of the exponent's.  (Where two least scales meet the factor would be 0, and a hidden
  // key's -inf times that no number.)
  float factors[kCols / 8];
  uint32_t seen[kCols / 32];
  if (MASKED) {
#pragma unroll
    for (int i = 0; i < kCols / 32; ++i) {
      const int from = min(max(low - first - 32 * i, 0), 32), to = min(max(high - first - 32 * i + 1, 0), 32);
      seen[i] = __funnelshift_lc(0xffffffffu, 0u, to) & ~__funnelshift_lc(0xffffffffu, 0u, from);
    }
  }
#pragma unroll
  for (int i = 0; i < kCols / 8; ++i) {
    const int slot = (first + 8 * i) >> shift;
    factors[i] = info.k_scale[slot] * scale;
    if (MASKED) {
      factors[i] = fmaxf(factors[i], 1e-37f);
      if (info.row[slot] < 0) seen[i / 4] &= ~(0xffu << (8 * (i & 3)));
    }
  }
  tmem_load_done(raw[0]);
  tmem_load_done(raw[1]);
  float v[kCols];
  float maximum = -INFINITY;
#pragma unroll
  for (int c8 = 0; c8 < kCols; c8 += 8) {
    float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const int c = c8 + i;
      v[c] = __uint_as_float(raw[c / 32][c % 32]);
      v[c + 1] = __uint_as_float(raw[c / 32][c % 32 + 1]);
      if (MASKED) {
        v[c] = (seen[c / 32] & (1u << (c % 32))) != 0u ? v[c] : -INFINITY;
        v[c + 1] = (seen[c / 32] & (2u << (c % 32))) != 0u ? v[c + 1] : -INFINITY;
      }
      best[i >> 1 & 1] = max_of_three(best[i >> 1 & 1], v[c], v[c + 1]);
    }
    maximum = fmaxf(maximum, fmaxf(best[0], best[1]) * factors[c8 / 8]);
  }
  shared_max[part * kRows] = maximum;
  asm volatile("bar.sync %0, %1;" ::"r"(team), "n"(32 * kParts) : "memory");
#pragma unroll
  for (int other = 0; other < kParts; ++other) maximum = fmaxf(maximum, shared_max[other * kRows]);
  float before = -INFINITY;
  if (handoff.has_from) {
    if (alive && !wait_barrier(handoff.from_barrier, handoff.from_phase)) { g_error = 3; alive = false; }
    before = *handoff.from;
  }
  const float now = maximum > before + kRises ? maximum : before;
  if (part == 0) *handoff.to = now;
  barrier_arrive(handoff.to_barrier);
  grow = now != before;
  factor = grow ? approximate_exp2(before - now) : 1.0f;                  // 0 when nothing was seen before
  own_factor = reference == now ? 1.0f : approximate_exp2(reference - now);
  reference = now;
  const float down = reference == -INFINITY ? 0.0f : -reference;       // (a row that has seen nothing yet, or scores of -inf alone)
  const float2 downs = make_float2(down, down);
  float2 sums[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int c = 0; c < kCols; c += 2) {
    const float2 both = make_float2(factors[c / 8], factors[c / 8]);
    float2 weight = fma_two(make_float2(v[c], v[c + 1]), both, downs);
    weight = make_float2(approximate_exp2(weight.x), approximate_exp2(weight.y));
    sums[(c >> 1) & 1] = add_two(sums[(c >> 1) & 1], weight);
    const __nv_bfloat162 rounded = __floats2bfloat162_rn(weight.x, weight.y);
    packed[c >> 1] = *reinterpret_cast<const uint32_t*>(&rounded);
  }
  return (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
}

__global__ void __launch_bounds__(kThreads, 1)
prefill_8bit_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                    const __grid_constant__ CUtensorMap k_tile_map, const __grid_constant__ CUtensorMap v_tile_map, const bf16* __restrict__ q,
                    long long q_stride, Cache8 cache, const int* __restrict__ block_table, int table_width,
                    const int* __restrict__ query_starts, const int* __restrict__ context_lens, int num_rows, int tokens,
                    const __grid_constant__ Divider kv_heads, const __grid_constant__ Divider group, const __grid_constant__ Divider parts,
                    float scale_log2, int window, int partition, float* __restrict__ partial_o, float* __restrict__ partial_ml,
                    bf16* __restrict__ out, const float* __restrict__ sinks) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long barriers[BARRIERS];
  __shared__ uint32_t tmem_slot;
  __shared__ int row_tiles_slot;
  __shared__ Info infos[kInfos];
  __shared__ float row_scales[4][kRows];                    // by n & 3: a row's scale, log2 e and the power of two taken out of its queries
  __shared__ float exchange[kStreams][2][kParts][kRows];    // [stream][its tile's parity][part]: a row's maxima
  __shared__ float denominators[2][kStreams][kParts][kRows];
  __shared__ float references[2][kStreams][kRows];
  __shared__ float handed[2][kRows];                        // a row's reference after tile g, by g & 1
  __shared__ int hidden_nans[4];                            // by n & 3: n + 1 if NaN values were left out that some rows of item n see
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem), bar0 = smem_u32(&barriers[0]);
  auto bar = [&](int index) { return bar0 + 8u * (uint32_t)index; };
  const int heads = group.by * kv_heads.by, num_partitions = parts.by;
  if (threadIdx.x == 0) {
    for (int i = 0; i < BARRIERS; ++i) {
      uint32_t count = 1u;
      if ((i >= Q_FULL && i < Q_FULL + 4) || (i >= V_FULL && i < V_FULL + 2) || (i >= RAW_FREE && i < RAW_FREE + 3)) count = kConverters;
      if ((i >= P_READY && i < P_READY + 3) || i == REF_READY || i == REF_READY + 1) count = kStreamThreads;
      if (i >= S_FULL && i < S_FULL + 3) count = 2u;
      if (i == O_FREE) count = kStreamThreads * kStreams;
      barrier_init(bar(i), count);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();
  if (warp == 0) {
    int total = 0;
    for (int r = lane; r < num_rows; r += 32) total += (portion_of(query_starts, r, tokens).count * group.by + kRows - 1) / kRows;
    total = __reduce_add_sync(0xffffffffu, total);
    if (lane == 0) {
      if (*reinterpret_cast<volatile int*>(&g_error) != 0) total = 0;     // an earlier wait ran out: nothing is begun
      row_tiles_slot = total;
      for (int i = 0; i < 4; ++i) hidden_nans[i] = 0;
    }
  }
  tensor_fence_before_sync();
  __syncthreads();
  tensor_fence_after_sync();
  grid_launch_dependents();
  const uint32_t tmem = tmem_slot, tmem_o = tmem + 384u;
  const int shift = 31 - __clz(cache.page_size);            // pages are powers of two
  const Items items{query_starts, context_lens, num_rows, tokens, window, partition, row_tiles_slot,
                    row_tiles_slot * kv_heads.by * num_partitions, kv_heads, parts, group};
  const int cta = blockIdx.x, ctas = gridDim.x;
  // whether all queries of an item see all keys of its tile t (that are there)
  auto seen_by_all = [&](const Work& of, int t) {
    const int key0 = of.begin + t * kKeys;
    return key0 + kKeys - 1 <= of.first_position && (window == 0 || of.last_position - window + 1 <= key0);
  };
  auto more = [&](int k) { return (long long)k * ctas < items.count; };
  Work w;

  if (warp < kFirstConverter) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRoleRegisters));
    if (warp == kScout) {
      // ---------------------------------------------------------------- scout: two tiles at a time, half a warp each
      const int half = lane >> 4, slot = lane & 15, slots = kKeys >> shift;
      bool alive = true;
      int g = 0;
      for (int k = 0; more(k); ++k) {
        if (!items.at(item_of(k, cta, ctas), w)) continue;
        const int* table = block_table + (size_t)w.request * table_width;
        for (int t = 0; t < w.tiles; t += 2) {
          const int tile = t + half, key = w.begin + tile * kKeys + (slot << shift);
          int page = -1;
          if (slot < slots && tile < w.tiles && key < w.end && key + cache.page_size > w.first_key)
            page = page_of_block(table, table_width, key >> shift, cache.pages);
          float k_scale = 1.0f, v_scale = 1.0f;
          if (page >= 0) {
            k_scale = cache.k_scales[(size_t)page * cache.kv_heads + w.kv_head];
            v_scale = cache.v_scales[(size_t)page * cache.kv_heads + w.kv_head];
          }
          const int v_exponent = ((__float_as_int(v_scale) >> 23) & 0xff) - 127;
          const unsigned there = __ballot_sync(0xffffffffu, page >= 0), loud = __ballot_sync(0xffffffffu, v_exponent > 7);
          for (int i = 0; i < 2 && t + i < w.tiles; ++i) {
            const int info = (g + i) % kInfos;
            if (alive && !wait_barrier(bar(INFO_FREE + info), (uint32_t)((g + i) / kInfos & 1) ^ 1u)) { g_error = 1; alive = false; }
            __syncwarp();
            if (half == i) {
              infos[info].row[slot] = page >= 0 ? page << shift : -cache.page_size;
              infos[info].k_scale[slot] = k_scale;
              infos[info].v_factor[slot] = power_pair(min(v_exponent, 7) + 120);
              infos[info].v_rest[slot] = power_pair(max(v_exponent - 7, 0));
            }
            if (lane == 0) {
              infos[info].whole = __popc((there >> (16 * i)) & 0xffffu) == slots;
              infos[info].one_factor = ((loud >> (16 * i)) & 0xffffu) == 0u;
            }
            __syncwarp();
            if (lane == 0) barrier_arrive(bar(INFO_FULL + info));
          }
          g += min(2, w.tiles - t);
        }
      }
    } else if (warp == kKeyLoader || warp == kValueLoader) {
      // ---------------------------------------------------------------- loaders: lane l has page slot l
      const bool values = warp == kValueLoader;
      const bool loads = lane < (kKeys >> shift);
      const uint32_t box_bytes = (uint32_t)cache.page_size * kDim;
      const uint32_t base = smem_base + (uint32_t)(values ? kOffRaw : kOffK);
      const int full0 = values ? RAW_FULL : K_FULL, free0 = values ? RAW_FREE : K_FREE;
      bool alive = true;
      Counter ring;
      int g = 0;
      for (int k = 0; more(k) && alive; ++k) {
        if (!items.at(item_of(k, cta, ctas), w)) continue;
        for (int t = 0; t < w.tiles; ++t, ++g) {
          const int info = g % kInfos;
          if (!wait_barrier(bar(INFO_FULL + info), (uint32_t)(g / kInfos & 1))) { g_error = 1; alive = false; }
          const int cache_row = loads ? infos[info].row[lane] : 0;
          if (alive && !wait_barrier(bar(free0 + (int)ring.stage), ring.phase ^ 1u)) { g_error = 1; alive = false; }
          alive = __all_sync(0xffffffffu, alive);
          if (!alive) break;
          const int first_row = __shfl_sync(0xffffffffu, cache_row, 0);
          const bool in_a_row = first_row >= 0 && __all_sync(0xffffffffu, !loads || cache_row == first_row + (lane << shift));
          const uint32_t full = bar(full0 + (int)ring.stage), to = base + ring.stage * (uint32_t)kTile8;
          if (lane == 0) barrier_expect_bytes(full, (uint32_t)kTile8);
          __syncwarp();
          if (in_a_row) {
            if (lane == 0) tma_load_2d(to, values ? &v_tile_map : &k_tile_map, full, w.kv_head * kDim, first_row);
          } else if (loads) {                               // (a negative row lies outside the tensor: zeros)
            tma_load_2d(to + (uint32_t)lane * box_bytes, values ? &v_map : &k_map, full, w.kv_head * kDim, cache_row);
          }
          ring.step(3);
        }
      }
      wait_for_copies(bar(full0), 3u, ring.stage, ring.phase);
    } else {
      // ---------------------------------------------------------------- issuer (tcgen05.cuh: from a whole warp)
      constexpr uint32_t scores_hi = instruction_descriptor_8bit(kRows, kKeys, E4M3, E4M3);
      constexpr uint32_t scores_lo = instruction_descriptor_8bit(kRows, kKeys, E5M2, E4M3);
      constexpr uint32_t values_of = instruction_descriptor(kRows, kDim, true);
      const uint32_t elected = elect_one();
      const uint32_t q_low = operand_low(smem_base + kOffQ), k_low = operand_low(smem_base + kOffK);
      const uint32_t v_low = operand_low_mn_major(smem_base + kOffV, kHalf);
      bool alive = true;
      auto check = [&](int index, uint32_t phase) {
        if (alive && !wait_barrier(bar(index), phase)) { g_error = 2; alive = false; }
      };
      int g0 = 0, n = 0;
      Counter keys, scores, weights, values;
      for (int k = 0; more(k); ++k) {
        if (!items.at(item_of(k, cta, ctas), w)) continue;
        const int tiles = __shfl_sync(0xffffffffu, w.tiles, 0);
        if (tiles == 0) continue;
        check(Q_FULL + (n & 3), (uint32_t)(n >> 2 & 1));
        auto issue_scores = [&](int t) {
          check(K_FULL + (int)keys.stage, keys.phase);
          __syncwarp();
          tensor_fence_after_sync();
          const uint32_t b = k_low + keys.stage * (uint32_t)(kTile8 >> 4), d = tmem + scores.stage * 128u;
#pragma unroll
          for (int kk = 0; kk < kDim / 32; ++kk) mma_8bit_ss_halves(d, q_low + 2u * kk, b + 2u * kk, scores_hi, kk > 0 ? 1u : 0u, elected);
#pragma unroll
          for (int kk = 0; kk < kDim / 32; ++kk)
            mma_8bit_ss_halves(d, q_low + (uint32_t)(kTile8 >> 4) + 2u * kk, b + 2u * kk, scores_lo, 1u, elected);
          mma_commit_elected(bar(S_FULL + (int)scores.stage), elected);
          if (lane == 0) barrier_arrive(bar(S_FULL + (int)scores.stage));     // (what the scout left of the tile came before its keys)
          mma_commit_elected(bar(K_FREE + (int)keys.stage), elected);
          if (t == tiles - 1) mma_commit_elected(bar(Q_FREE), elected);
          keys.step(3);
          scores.step(3);
        };
        // S(t + 3) takes the accumulator that holds P(t): behind the product with it
        for (int t = 0; t < min(3, tiles); ++t) issue_scores(t);
        for (int t = 0; t < tiles; ++t) {
          const int g = g0 + t;
          check(V_FULL + (int)values.stage, values.phase);
          check(P_READY + (int)weights.stage, weights.phase);
          if (t == 0 && n > 0) check(O_FREE, (uint32_t)(n - 1) & 1u);       // the last item's result has been read out
          __syncwarp();
          tensor_fence_after_sync();
          const uint32_t p = tmem + weights.stage * 128u, b = v_low + values.stage * (uint32_t)(kTile16 >> 4);
          mma_bf16_ts_halves(tmem_o, p, b, values_of, t > 0 ? 1u : 0u, elected);
#pragma unroll
          for (int kk = 1; kk < kKeys / 16; ++kk)
            mma_bf16_ts_halves(tmem_o, p + (uint32_t)kk * 8u, b + (uint32_t)kk * (2048u >> 4), values_of, 1u, elected);
          mma_commit_elected(bar(V_FREE + (int)values.stage), elected);
          mma_commit_elected(bar(PV_DONE + (g & 1)), elected);
          mma_commit_elected(bar(INFO_FREE + g % kInfos), elected);          // everybody is done with the tile
          if (t == tiles - 1) mma_commit_elected(bar(ITEM_DONE), elected);
          values.step(2);
          weights.step(3);
          if (t + 3 < tiles) issue_scores(t + 3);
        }
        g0 += tiles;
        ++n;
      }
    }
  } else if (warp < kFirstSoftmax) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConverterRegisters));
    // ------------------------------------------------------------------ converters: an item's queries, then its tiles' values
    const int thread = threadIdx.x - kFirstConverter * 32, my_warp = warp - kFirstConverter;
    bool alive = true;
    Counter raw, values;
    int g = 0, n = 0;
    for (int k = 0; more(k); ++k) {
      if (!items.at(item_of(k, cta, ctas), w) || w.tiles == 0) continue;
      // a warp takes 16 rows, eight at a time, a lane four elements of each; rows that are not there repeat the last.  Where a row's
      // queries lie a lane each works out once (a division a row in every lane took longer than the rounding).
      constexpr int kHeld = 8, kWarpRows = kRows / (kConverters / 32);
      long long offset;
      {
        const int row = w.first_row + min(my_warp * kWarpRows + (lane & (kWarpRows - 1)), w.rows - 1), token = group(row);
        offset = (long long)(w.first_token + token) * q_stride + (long long)(w.kv_head * group.by + row - token * group.by) * kDim;
      }
#pragma unroll 1
      for (int half = 0; half < kWarpRows; half += kHeld) {
        uint2 held[kHeld];
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
          held[i] = *reinterpret_cast<const uint2*>(q + __shfl_sync(0xffffffffu, offset, half + i) + lane * 4);
        // (asked for while the products with the last item's queries may still run)
        if (half == 0 && n > 0) {
          if (alive && !wait_barrier(bar(Q_FREE), (uint32_t)(n - 1) & 1u)) { g_error = 4; alive = false; }
          __syncwarp();
        }
        const int r0 = my_warp * kWarpRows + half;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
          const float x[4] = {__uint_as_float(held[i].x << 16), __uint_as_float(held[i].x & 0xffff0000u), __uint_as_float(held[i].y << 16),
                              __uint_as_float(held[i].y & 0xffff0000u)};
          const float largest = warp_largest(max_of_three(fmaxf(fabsf(x[0]), fabsf(x[1])), fabsf(x[2]), fabsf(x[3])));
          const int e = least_scale_exponent(fminf(largest, 3.38953139e38f));
          const float inverse = query_inverse(largest, e);
          uint32_t hi[2], lo[2];
          split_e4m3_e5m2(x[0] * inverse, x[1] * inverse, hi[0], lo[0]);
          split_e4m3_e5m2(x[2] * inverse, x[3] * inverse, hi[1], lo[1]);
          const int r = r0 + i;
          unsigned char* to = smem + kOffQ + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4;
          *reinterpret_cast<uint32_t*>(to) = hi[0] | (hi[1] << 16);
          *reinterpret_cast<uint32_t*>(to + kTile8) = lo[0] | (lo[1] << 16);
          if (lane == 0) row_scales[n & 3][r] = power_of_two(e) * scale_log2;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      barrier_arrive(bar(Q_FULL + (n & 3)));
      ++n;
      for (int t = 0; t < w.tiles; ++t, ++g) {
        const int info = g % kInfos;
        if (alive && !wait_barrier(bar(RAW_FULL + (int)raw.stage), raw.phase)) { g_error = 4; alive = false; }
        if (alive && !wait_barrier(bar(V_FREE + (int)values.stage), values.phase ^ 1u)) { g_error = 4; alive = false; }
        const unsigned char* from = smem + kOffRaw + raw.stage * kTile8;
        unsigned char* to = smem + kOffV + values.stage * kTile16;
        // thread: two pieces of 8 bytes, j and j + 8, of every 32nd row (whose place in the swizzle is the same), two rows at a time; a piece
        // becomes 16 bytes, so that eight threads write a whole row of 128 bytes, and of two rows that are read together one begins with the
        // first eight pieces and the other with the last, so that no two threads meet in a bank
        const int j = thread & 7, r0 = thread >> 3, swap = r0 & 1;
        const bool all_seen = infos[info].whole && w.begin + t * kKeys >= w.first_key && w.begin + (t + 1) * kKeys <= w.end;
        const bool one_factor = infos[info].one_factor, hides = !seen_by_all(w, t);
        from += r0 * 128;
        const unsigned char* piece[2] = {from + ((((j >> 1) + 4 * swap) ^ (r0 & 7)) << 4) + (j & 1) * 8,
                                         from + ((((j >> 1) + 4 - 4 * swap) ^ (r0 & 7)) << 4) + (j & 1) * 8};
        to += r0 * 128 + ((j ^ (r0 & 7)) << 4);
        unsigned char* wide_piece[2] = {to + swap * kHalf, to + (1 - swap) * kHalf};
        constexpr int kStep = kConverters / 8, kTogether = 2;
#pragma unroll 1
        for (int base = 0; base < kKeys; base += kStep * kTogether) {
          uint2 word[kTogether][2];
          uint32_t factor[kTogether];
#pragma unroll
          for (int i = 0; i < kTogether; ++i) {
            factor[i] = infos[info].v_factor[(base + i * kStep + r0) >> shift];
#pragma unroll
            for (int h = 0; h < 2; ++h) word[i][h] = *reinterpret_cast<const uint2*>(piece[h] + (base + i * kStep) * 128);
          }
#pragma unroll
          for (int i = 0; i < kTogether; ++i) {
            const int r = base + i * kStep + r0;
            if (!all_seen) {
              const int key = w.begin + t * kKeys + r;
              if (key >= w.end || key < w.first_key || infos[info].row[r >> shift] < 0) word[i][0] = word[i][1] = make_uint2(0u, 0u);
            }
            uint32_t wide[8];
            const uint32_t words[4] = {word[i][0].x, word[i][0].y, word[i][1].x, word[i][1].y};
            uint32_t last = 0u;                              // a byte's upper bit: its magnitude is e4m3's last code, NaN
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              wide[2 * c] = times(lifted<0x9180>(words[c]), factor[i]);
              wide[2 * c + 1] = times(lifted<0xb3a2>(words[c]), factor[i]);
              last |= (words[c] & 0x7f7f7f7fu) + 0x01010101u;
            }
            if ((last & 0x80808080u) != 0u || !one_factor) {       // (rare: the lifted number of a NaN is 480; a scale beyond one bf16 factor)
              const uint32_t rest = infos[info].v_rest[r >> shift];
              // a weight of 0 times NaN would be NaN for the rows that do not see the key: it is left out here and put in at the end
              if (hides && (last & 0x80808080u) != 0u) hidden_nans[(n - 1) & 3] = n;
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                wide[c] = times(wide[c], rest);
                const uint32_t pair = words[c / 2] >> (16 * (c & 1));
                if ((pair & 0x7fu) == 0x7fu) wide[c] = hides ? wide[c] & 0xffff0000u : wide[c] | 0x7fffu;
                if ((pair & 0x7f00u) == 0x7f00u) wide[c] = hides ? wide[c] & 0xffffu : wide[c] | 0x7fff0000u;
              }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
              *reinterpret_cast<uint4*>(wide_piece[h] + (base + i * kStep) * 128) =
                  make_uint4(wide[4 * h], wide[4 * h + 1], wide[4 * h + 2], wide[4 * h + 3]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        barrier_arrive(bar(V_FULL + (int)values.stage));
        barrier_arrive(bar(RAW_FREE + (int)raw.stage));
        raw.step(3);
        values.step(2);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    // ------------------------------------------------------------------ softmax
    const int stream = (warp - kFirstSoftmax) >> 3;          // takes the tiles t = stream, stream + 2, ...
    const int quarter = warp & 3;                            // the accumulator lanes this warp may touch
    const int part = ((warp - kFirstSoftmax) >> 2) & 1;      // which kCols columns of the row
    const int r = quarter * 32 + lane, first = part * kCols;
    const uint32_t lane_bits = (uint32_t)(quarter * 32) << 16;
    const int team = 1 + stream * 4 + quarter;
    bool alive = true;
    int g0 = 0, n = 0;
    for (int k = 0; more(k); ++k) {
      if (!items.at(item_of(k, cta, ctas), w)) continue;
      const int row = w.first_row + min(r, w.rows - 1), token = group(row), head = w.kv_head * group.by + row - token * group.by;
      const size_t out_row = (size_t)(w.first_token + token) * heads + head;
      if (w.tiles == 0) {                                    // a partition without keys, or rows that see none
        if (stream == 0 && part == 0 && r < w.rows) {
          if (num_partitions > 1) {
            *reinterpret_cast<float2*>(partial_ml + (out_row * num_partitions + w.part) * 2) = make_float2(-INFINITY, 0.0f);
          } else {
            uint4* to = reinterpret_cast<uint4*>(out + out_row * kDim);
#pragma unroll
            for (int i = 0; i < kDim / 8; ++i) to[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        continue;
      }
      const int position = w.first_position + token - group(w.first_row);
      float reference = -INFINITY, denominator = 0.0f, scale = 0.0f;
      if (stream < w.tiles) {
        if (alive && !wait_barrier(bar(Q_FULL + (n & 3)), (uint32_t)(n >> 2 & 1))) { g_error = 3; alive = false; }
        scale = row_scales[n & 3][r];
      }
      for (int t = stream; t < w.tiles; t += kStreams) {
        const int g = g0 + t, stage = g % 3, info = g % kInfos, key0 = w.begin + t * kKeys;
        if (alive && !wait_barrier(bar(S_FULL + stage), (uint32_t)(g / 3 & 1))) { g_error = 3; alive = false; }
        __syncwarp();
        tensor_fence_after_sync();
        const uint32_t scores = tmem + (uint32_t)stage * 128u + lane_bits;
        const int high = min(position, w.end - 1) - key0, low = window > 0 ? position - window + 1 - key0 : -1;
        const bool every = infos[info].whole && key0 + kKeys <= w.end && seen_by_all(w, t);
        uint32_t packed[kCols / 2];
        bool grow;
        float factor, own_factor;
        Handoff handoff;
        handoff.has_from = t > 0;
        handoff.from_barrier = bar(REF_READY + ((g - 1) & 1));
        handoff.from_phase = (uint32_t)((g - 1) >> 1) & 1u;
        handoff.from = &handed[(g - 1) & 1][r];
        handoff.to_barrier = bar(REF_READY + (g & 1));
        handoff.to = &handed[g & 1][r];
        float* shared_max = &exchange[stream][(t / kStreams) & 1][0][r];
        const float sum = every ? softmax_tile<false>(scores, first, low, high, scale, infos[info], shift, reference, factor, grow, own_factor,
                                                      packed, shared_max, part, team, handoff, alive)
                                : softmax_tile<true>(scores, first, low, high, scale, infos[info], shift, reference, factor, grow, own_factor,
                                                     packed, shared_max, part, team, handoff, alive);
        denominator = denominator * own_factor + sum;
        // the accumulator holds the products up to tile t - 1, whose end is waited for; the product with this tile's weights is not
        // issued before this stream arrives, so nothing else touches it meanwhile
        if (t > 0 && __any_sync(0xffffffffu, grow)) {
          if (alive && !wait_barrier(bar(PV_DONE + ((g - 1) & 1)), (uint32_t)((g - 1) >> 1) & 1u)) { g_error = 3; alive = false; }
          __syncwarp();
          tensor_fence_after_sync();
#pragma unroll 1
          for (int c0 = 0; c0 < kDim / kParts; c0 += 32) {
            float o[32];
            tmem_load_32(tmem_o + lane_bits + (uint32_t)(part * (kDim / kParts) + c0), o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] *= factor;
            tmem_store_32(tmem_o + lane_bits + (uint32_t)(part * (kDim / kParts) + c0), o);
          }
        }
        tmem_store_32_bits(scores + (uint32_t)(first / 2), packed);
        tmem_store_wait();
        tensor_fence_before_sync();
        barrier_arrive(bar(P_READY + stage));
      }
      // every softmax thread learns every stream's reference and denominator
      const int slot = n & 1;
      denominators[slot][stream][part][r] = denominator;
      if (part == 0) references[slot][stream][r] = reference;
      asm volatile("bar.sync 9, %0;" ::"n"(kStreamThreads * kStreams) : "memory");
      const float top = fmaxf(references[slot][0][r], references[slot][1][r]);
      float total = 0.0f;
#pragma unroll
      for (int other = 0; other < kStreams; ++other) {
        // (0: that stream saw no key of this row; NaN beside a reference of -inf: nothing else)
        const float theirs = references[slot][other][r], sum = denominators[slot][other][0][r] + denominators[slot][other][1][r];
        if (sum != 0.0f) total += sum * approximate_exp2(theirs - top);
      }
      if (alive && !wait_barrier(bar(ITEM_DONE), (uint32_t)n & 1u)) { g_error = 3; alive = false; }
      __syncwarp();
      tensor_fence_after_sync();
      constexpr int kOut = kDim / (kParts * kStreams);       // 32 columns of the row for each of its threads
      const int column = (stream * kParts + part) * kOut;
      float o[kOut];
      tmem_load_32(tmem_o + lane_bits + (uint32_t)column, o);
      tensor_fence_before_sync();
      barrier_arrive(bar(O_FREE));                           // (the next item's products may overwrite it)
      if (r < w.rows && alive) {
        if (num_partitions == 1) {
          if (total != 0.0f && sinks != nullptr) total += exp2f(sinks[head] * kLog2e - top);
          const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
          uint4* to = reinterpret_cast<uint4*>(out + out_row * kDim + column);
#pragma unroll
          for (int i = 0; i < kOut; i += 8) {
            uint4 packed_out;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&packed_out);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              h[c] = __floats2bfloat162_rn(total == 0.0f ? 0.0f : o[i + 2 * c] * inverse, total == 0.0f ? 0.0f : o[i + 2 * c + 1] * inverse);
            to[i / 8] = packed_out;
          }
        } else {
          const size_t at = out_row * num_partitions + w.part;
          if (column == 0) *reinterpret_cast<float2*>(partial_ml + at * 2) = make_float2(top, total);
          if (total != 0.0f) {
            float4* to = reinterpret_cast<float4*>(partial_o + at * kDim + column);
#pragma unroll
            for (int i = 0; i < kOut; i += 4) to[i / 4] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      }
      if (hidden_nans[n & 3] == n + 1 && r < w.rows && total != 0.0f) {
        // the NaN values that were left out, for the rows that see their keys (over what was stored in larger words)
        asm volatile("" ::: "memory");
        const int* table = block_table + (size_t)w.request * table_width;
#pragma unroll 1
        for (int key = max(w.begin, window > 0 ? position - window + 1 : 0); key <= min(position, w.end - 1); ++key) {
          if (seen_by_all(w, (key - w.begin) / kKeys)) continue;                                // (left in)
          const int page = page_of_block(table, table_width, key >> shift, cache.pages);
          const uint8_t* codes = cache.v + ((((size_t)max(page, 0) << shift) + (key & (cache.page_size - 1))) * cache.kv_heads + w.kv_head) * kDim;
#pragma unroll 1
          for (int i = column; page >= 0 && i < column + kOut; ++i) {
            if ((codes[i] & 0x7f) != 0x7f) continue;
            if (num_partitions == 1) out[out_row * kDim + i] = __float2bfloat16_rn(__int_as_float(0x7fffffff));
            else partial_o[(out_row * num_partitions + w.part) * kDim + i] = __int_as_float(0x7fffffff);
          }
        }
      }
      g0 += w.tiles;
      ++n;
    }
    tensor_fence_before_sync();
  }
  __syncthreads();
  if (warp == kIssuer) {
    tensor_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
  }
}

}  // namespace

// 0 if no bounded wait of the kernel ever ran out; else which role gave up last (1 scout or loader, 2 issuer, 3 softmax, 4 converters).
// Synchronises the device.  `next`: exchange_flag.
MIR_EXPORT int mir_prefill_attention_8bit_error(int next) {
  return exchange_flag(g_error, next);
}

int mir_attention_8bit_prefill(const Attention8& a, int tokens) {
  const int group = a.heads / a.cache.kv_heads;
  // an upper bound of the items (the kernel counts them); as many CTAs as there can be work for
  const long long items = (((long long)tokens * group + kRows - 1) / kRows + a.num_rows) * a.cache.kv_heads * a.num_partitions;
  if (items > 0x7fffffffll || (long long)tokens * group > 0x7fffffffll - kRows) {
    mir_set_error("%s: %d tokens in %d rows are more than one launch takes", a.what, tokens, a.num_rows);
    return MIR_BAD_ARGUMENT;
  }
  const long long rows = (long long)a.cache.pages * a.cache.page_size, width = (long long)a.cache.kv_heads * kDim;
  CUtensorMap maps[4];
  const void* tensors[2] = {a.cache.k, a.cache.v};
  for (int i = 0; i < 4; ++i) {
    const int status = tensor_map_of_bytes(tensors[i & 1], rows, width, width, i < 2 ? a.cache.page_size : kKeys, &maps[i]);
    if (status != MIR_OK) return status;
  }
  int status = reserve_shared(prefill_8bit_kernel, kSmemBytes, a.what);
  if (status != MIR_OK) return status;
  status = mir_launch("prefill_attention_8bit", prefill_8bit_kernel, dim3((unsigned)std::min<long long>(items, mir_sm_count())), dim3(kThreads),
                      (size_t)kSmemBytes, a.stream, 0, maps[0], maps[1], maps[2], maps[3], (const bf16*)a.q, a.q_stride, a.cache, a.block_table,
                      a.table_width, a.query_starts, a.context_lens, a.num_rows, tokens, Divider(a.cache.kv_heads), Divider(group),
                      Divider(a.num_partitions), a.scale * kLog2e, a.window, a.partition, a.partial_o(tokens), a.partial_ml(tokens), (bf16*)a.out, a.sinks);
  if (status != MIR_OK || a.num_partitions == 1) return status;
  Attention8 parts = a;
  void* error = nullptr;
  const cudaError_t found = cudaGetSymbolAddress(&error, g_error);
  if (found != cudaSuccess) {
    mir_set_error("%s: %s", a.what, cudaGetErrorString(found));
    return MIR_CUDA_ERROR;
  }
  parts.error = static_cast<const int*>(error);
  return mir_merge_8bit(parts, tokens);
}
