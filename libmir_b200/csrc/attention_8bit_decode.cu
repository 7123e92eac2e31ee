// Attention of single tokens over the 8-bit cache on the 5th-generation tensor cores, head_dim 128, pages of 8 to 128 keys:
// the bytes of the cache go from memory into the products as they are, nothing is widened.
//
// The work is all requests' tiles of 128 keys, one behind the other, for every unit (a kv head and up to 16 query heads of its
// group).  It is shared out evenly over teams of CTAs, a CTA for each unit, by the positions alone and on the device, so that requests
// of any lengths load all SMs alike and a captured launch fits contexts that have grown.  The CTAs of a team read the same rows of the
// cache at the same time, 128 bytes beside each other: a CTA that took one unit's tiles after another's read those pieces by
// themselves and got 4.5 TB/s.  Stretches of a request that lie within a team are finished there; the parts of one that is cut
// are joined by a second kernel.
// The products are transposed, so that the keys (then the elements of the head) are the 128 rows of the tensor
// cores and the query heads the 16 columns:
//
//   S^T = K Q^T    kind::f8f6f4, A = the key tile as the cache holds it (a key is a row of 128 bytes), B = the queries in two parts:
//                  q = hi + lo, hi = e4m3(q 2^-e), lo = e5m2 of what hi leaves.  A bf16 number has eight significant bits, hi takes
//                  four and lo the signed rest, so the two are exact down to 2^-13 of the head's largest element (e puts that
//                  below 448) and off by at most 2^-21.8 of it below (2^-14 of a largest one of 224);
//   O^T = V^T P    A = the value tile as the cache holds it (MN-major: nothing is transposed), B = the softmax's weights in two parts
//                  again.
//
// The scales: a score is multiplied by its key's page's scale on its way out of tensor memory, in 32 bits.  A value's scale 2^f goes
// into the weight, exp2(s + f - M), M the tile's own maximum of s + f less 8, so that the largest weight is 256.  The two parts hold
// a weight of 2^-6 or more up to 2^-8 of itself (2^-4 from hi, 2^-4 of that from lo); smaller ones run into the formats' least numbers.
// So the weights lie in four bands of 14 binades, band b multiplied by 2^(14 b), each with columns of its own (with up to four heads
// the product has them anyway): whatever is 2^-56 of the tile's largest or more, 38 nats, is off by at most 2^-8 of itself, and what is
// less by at most 2^-67 of the largest.  One reference for a whole stretch and one band lost what lay 14 nats below the largest weight,
// or was 2^20 less loud, from the result and not from the denominator: where the keys that are ahead hold small values, or a page is
// loud for one channel's sake, the others are all there is.
// A tile's products start from zero; the softmax threads, one for each element of the head, add them up in 32-bit registers, relative
// to the running maximum m of s, as the denominator is, the sum of exp2(s - m).
//
// Roles: four warps of softmax (a thread is a key of the tile, then an element of the head); a scout, which reads block table, scales
// and queries ahead of everyone and leaves them in shared memory (read where they are used, those dependent loads cost every
// tile 2,000 to 3,400 of its 4,000 cycles); a loader each for keys and values (TMA, one box for each page, or one for the tile
// where its pages lie one behind the other); an issuer.  Two score accumulators, so that the scores of the next tile
// are formed while the softmax works on this one, across the borders of requests and heads too.  Three stages of keys and
// values, two CTAs an SM.  A hidden key's score becomes -inf by selection, and its row of values is zeroed in shared memory (0
// times what lies behind a context could be NaN).  The kernel is bound by the cache's bytes: 64 contexts of 1,000 to 2,048 keys (204 MB)
// take 50 us, 4.0 TB/s, four of up to 32,768 with 64 heads (219 MB) 57 us; a page of 16 rows is 16 pieces of 128 bytes for a head.
// (The bands and the sums in registers are 2 and 4 us of that.  Going over a tile again for what lies below two bands, instead of four
// bands at once, took 67 and 108 us.)
#include <algorithm>
#include "eight_bit_tc.cuh"

using namespace mir;
using namespace mir::tc;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kKeys = 128, kDim = 128, kHeads = 16;
constexpr int kTile = kKeys * kDim;                    // bytes of a tile of keys or of values
constexpr int kSoftmaxThreads = 128, kThreads = kSoftmaxThreads + 4 * 32;
constexpr int kKeyLoader = 4, kValueLoader = 5, kIssuer = 6, kScout = 7;      // warps
constexpr int kBands = 4;
constexpr float kTop = 8.0f, kBand = 14.0f;            // log2 of a tile's largest weight; binades of a band
constexpr int kChunk = 4, kSlots = 16;                 // tiles that the scout looks up together, pages of a tile at most

// Shared memory for G heads.  A part (hi or lo) of Q is 16 rows of 128 bytes, the columns of the products; up to 8 heads need only
// 8 of them, and the product then reads the next part's (or what follows) as the other columns, which nobody looks at.  A part of P is
// G rows for each band.
template <int G> struct Layout {
  static constexpr int kStages = G <= 8 ? 3 : 2;
  static constexpr int kPart = (G <= 8 ? 8 : 16) * 128, kWeightPart = kBands * G * 128;
  static constexpr int kOffK = 0, kOffV = kStages * kTile, kOffQ = 2 * kStages * kTile, kOffP = kOffQ + 4 * kPart;
  static constexpr int kSmemBytes = kOffP + 2 * kWeightPart + 1024 /* alignment */;
  static constexpr int kHeldRows = G == 8 ? 256 : 512;       // positions that a CTA keeps there (8 heads leave no room for more, with two CTAs)
  // S^T of even and odd tiles at 0 and 16, O^T at 32
  static constexpr int kValueColumns = kBands * G;
  static constexpr uint32_t kTmemColumns = 32 + kValueColumns <= 64 ? 64 : 128;
};
static_assert(Layout<16>::kSmemBytes >= kLeastSharedBeside, "never beside a kernel that takes all tensor memory");

enum { K_FULL = 0, K_FREE = K_FULL + 3, V_FULL = K_FREE + 3, V_FREE = V_FULL + 3, S_FULL = V_FREE + 3, P_READY = S_FULL + 2,
       Q_READY = P_READY + 2, Q_FREE = Q_READY + 4, CHUNK_FULL = Q_FREE + 2, CHUNK_FREE = CHUNK_FULL + 2, ROWS_FULL = CHUNK_FREE + 2,
       PV_DONE = ROWS_FULL + 2, BARRIERS = PV_DONE + 2 };
// Tiles are counted over the CTA's whole stretch (g): stage g % kStages of the rings, g & 1 of S_FULL, P_READY and PV_DONE (who waits for
// tile g of one of them knows that tile g - 2 is over, so the parity says which), chunk g / kChunk.
// Parts are counted too (n): the queries' buffers and Q_FREE go by n & 1, Q_READY by n & 3: the softmax may begin part n when the
// queries of part n + 2 are there already, but never those of part n + 4 (see `factors`).

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

// Byte offset of element (row, column) of rows of 128 bytes with the 128-byte swizzle.
__device__ __forceinline__ uint32_t swizzled(int row, int column) {
  return (uint32_t)(row * 128 + (((column >> 4) ^ (row & 7)) << 4) + (column & 15));
}
// A row's share of the work: its tiles of keys, from the tile that holds its first visible key to the last that the table can have
// (one at least: a row that sees nothing gets zeros).  All rows' tiles together are below 2^31: the launcher checks.
struct Row {
  int position, first_key, begin, tiles;
};
__device__ __forceinline__ Row row_at(const int* __restrict__ positions, int row, int window, int table_keys) {
  Row r;
  r.position = positions[row];
  r.first_key = (window > 0 && r.position >= window) ? r.position + 1 - window : 0;
  r.begin = r.first_key / kKeys * kKeys;
  r.tiles = r.position < 0 ? 0 : max(1, (min(r.position, table_keys - 1) - r.begin) / kKeys + 1);       // (a padding row: none)
  return r;
}

// The least share with which `teams` of them hold `total`.
__device__ __forceinline__ unsigned shares_of(unsigned total, int teams) { return (total + (unsigned)teams - 1u) / (unsigned)teams; }

// Where a team's stretch of tiles begins, and how long it is.
struct Stretch {
  int row, tile, count;
};

// One part of a stretch: tiles [first, last) of a row.
struct Part {
  int row, first, last;
  Row of;
  __device__ __forceinline__ bool whole() const { return first == 0 && last == of.tiles; }
};

// The parts of a stretch, one after the other.
struct Walk {
  Stretch at;
  const int* positions;
  int num_rows, window, table_keys;
  __device__ __forceinline__ bool next(Part& part) {
    if (at.count <= 0) return false;
    Row r = row_at(positions, at.row, window, table_keys);
    while (at.tile >= r.tiles) {                         // the next row that has tiles
      at.tile = 0;
      if (++at.row >= num_rows) return false;
      r = row_at(positions, at.row, window, table_keys);
    }
    part.row = at.row;
    part.first = at.tile;
    part.last = min(r.tiles, at.tile + at.count);
    part.of = r;
    at.count -= part.last - part.first;
    at.tile = part.last;
    return true;
  }
};

// What the scout leaves of a chunk of tiles.
struct Chunk {
  int row[kChunk][kSlots];                             // a page's first row of the cache; below 0 where it is not there or not wanted
  float2 scale[kChunk][kSlots];                        // its scales, of keys and of values
  int first[kChunk], last[kChunk];                     // whether the tile is its part's first, its last
};

// G: heads that the softmax threads handle (a unit's heads rounded up to 4, 8 or 16).
template <int G>
__global__ void __launch_bounds__(kThreads, 2)
decode_8bit_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                   const __grid_constant__ CUtensorMap k_tile_map, const __grid_constant__ CUtensorMap v_tile_map,
                   const bf16* __restrict__ q, long long q_stride, Cache8 cache, const int* __restrict__ block_table, int table_width,
                   const int* __restrict__ all_positions, int num_rows, int heads, float scale_log2, int window,
                   float* __restrict__ parts, bf16* __restrict__ out, const float* __restrict__ sinks) {
  using L = Layout<G>;
  constexpr int kStages = L::kStages, kPart = L::kPart;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) unsigned long long barriers[BARRIERS];
  __shared__ uint32_t tmem_slot;
  __shared__ Stretch stretch;
  __shared__ Chunk chunks[2];
  __shared__ int held_positions[L::kHeldRows];
  __shared__ __align__(16) float exchange[2][2 * G][4];        // [tile parity][maxima of s, then of s + f][warp]
  __shared__ float sums[4][G];
  // Of a head's scores: scale, log2 e, and the power of two taken out of its queries, by n & 3: part n + 4's are written when the scores
  // of part n + 2 are over, which were formed when the softmax was past every tile but the last two, so past part n.
  __shared__ float factors[4][G];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t smem_base = smem_u32(smem), bar0 = smem_u32(&barriers[0]);
  auto bar = [&](int index) { return bar0 + 8u * (uint32_t)index; };
  const int group = heads / cache.kv_heads, group_tiles = (group + kHeads - 1) / kHeads, units = cache.kv_heads * group_tiles;
  const int unit = blockIdx.x % units, team = blockIdx.x / units, teams = gridDim.x / units;
  const int kv_head = unit / group_tiles, head0 = kv_head * group + unit % group_tiles * kHeads;
  const int valid_heads = min(kHeads, kv_head * group + group - head0);
  const int table_keys = (int)min(0x7fffffffll, (long long)table_width * cache.page_size);
  if (threadIdx.x == 0) {
    for (int i = 0; i < BARRIERS; ++i) {
      const bool softmax = i == P_READY || i == P_READY + 1, chunk = i == CHUNK_FREE || i == CHUNK_FREE + 1;
      barrier_init(bar(i), softmax ? (uint32_t)kSoftmaxThreads : (chunk ? 7u : 1u));      // (a chunk: both loaders, issuer, four warps)
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(L::kTmemColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  grid_dependency_wait();                              // the cache, the queries and the positions may come from the kernel in front
  for (int r = threadIdx.x; r < min(num_rows, L::kHeldRows); r += kThreads) held_positions[r] = all_positions[r];
  __syncthreads();
  const int* positions = num_rows <= L::kHeldRows ? held_positions : all_positions;
  if (warp == 0) {
    // this team's stretch: all tiles over the teams, then the row that the first one lies in
    unsigned total = 0;
    for (int r = lane; r < num_rows; r += 32) total += (unsigned)row_at(positions, r, window, table_keys).tiles;
    total = __reduce_add_sync(0xffffffffu, total);
    const unsigned each = shares_of(total, teams), first = min(total, each * (unsigned)team);
    Stretch mine;
    mine.row = mine.tile = 0;
    mine.count = (int)min(each, total - first);
    unsigned before = 0;
    for (int r0 = 0; r0 < num_rows && mine.count > 0; r0 += 32) {
      const unsigned tiles = r0 + lane < num_rows ? (unsigned)row_at(positions, r0 + lane, window, table_keys).tiles : 0u;
      const unsigned all = __reduce_add_sync(0xffffffffu, tiles);
      if (before + all > first) {
        unsigned through = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned left = __shfl_up_sync(0xffffffffu, through, o);
          if (lane >= o) through += left;
        }
        through += before;
        const int in = __ffs(__ballot_sync(0xffffffffu, through > first)) - 1;
        mine.row = r0 + in;
        mine.tile = (int)(first - __shfl_sync(0xffffffffu, through - tiles, in));
        break;
      }
      before += all;
    }
    if (lane == 0) {
      if (*reinterpret_cast<volatile int*>(&g_error) != 0) mine.count = 0;       // an earlier wait ran out: nothing is begun
      stretch = mine;
    }
  }
  tensor_fence_before_sync();
  __syncthreads();
  tensor_fence_after_sync();
  grid_launch_dependents();
  const uint32_t tmem_s = tmem_slot, tmem_o = tmem_slot + 32u;
  const int shift = 31 - __clz(cache.page_size);       // pages are powers of two
  const int count = stretch.count;                     // tiles of this CTA
  Walk walk{stretch, positions, num_rows, window, table_keys};
  Part part;

  if (warp == kScout) {
    // ------------------------------------------------------------------ scout: the table's entries are on their way a chunk ahead of
    // the scales that they lead to (the memory is busy: a load takes 2 us and more)
    const int slot_shift = 7 - shift, page_size = cache.page_size;     // (128 >> shift pages a tile)
    const int entries = kChunk << slot_shift, slot = lane & ((1 << slot_shift) - 1);
    bool alive = true;
    // this lane's two entries (tile, page slot) of the next chunk of `ahead`: the raw numbers of the table, -1 where none is wanted
    Walk ahead = walk;
    Part ahead_part;
    ahead_part.last = 0;
    int ahead_tile = 0;
    auto look_up = [&](int tiles, int (&page)[2]) {
      const int* from[2] = {block_table, block_table};
      bool wanted[2] = {false, false};
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        if (j >= tiles) break;
        if (ahead_tile >= ahead_part.last) {
          ahead.next(ahead_part);
          ahead_tile = ahead_part.first;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int entry = lane + 32 * i;
          if (entry >> slot_shift == j) {
            const int key = ahead_part.of.begin + ahead_tile * kKeys + (slot << shift);
            from[i] = block_table + (size_t)ahead_part.row * table_width + (key >> shift);
            wanted[i] = key <= ahead_part.of.position && key + page_size > ahead_part.of.first_key && (key >> shift) < table_width;
          }
        }
        ++ahead_tile;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        page[i] = -1;
        if (wanted[i]) page[i] = *from[i];
      }
    };
    auto load_queries = [&](const Part& of, uint2 (&raw)[G]) {
      const bf16* from = q + (size_t)of.row * q_stride + (size_t)head0 * kDim + lane * 4;
#pragma unroll
      for (int h = 0; h < G; ++h) raw[h] = *reinterpret_cast<const uint2*>(from + min(h, valid_heads - 1) * kDim);
    };
    int tile = 0, parts_begun = 0;                     // the walk's next tile of `part`
    part.last = 0;
    int page[2], page_next[2] = {-1, -1};
    look_up(min(kChunk, count), page);
    for (int g0 = 0; g0 < count; g0 += kChunk) {
      const int buffer = g0 / kChunk & 1, tiles = min(kChunk, count - g0);
      if (g0 + kChunk < count) look_up(min(kChunk, count - g0 - kChunk), page_next);
      Part begun[kChunk];                              // the parts that begin in this chunk
      int beginning = 0, last_tiles = 0;
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        if (j < tiles) {
          if (tile >= part.last) {
            walk.next(part);
            tile = part.first;
          }
          if (tile == part.first) begun[j] = part;     // (an index known at compile time: registers)
          beginning |= (tile == part.first ? 1 : 0) << j;
          last_tiles |= (tile == part.last - 1 ? 1 : 0) << j;
          ++tile;
        }
      }
      uint2 raw[G];                                    // of the CTA's first part: beside the first table entries
      if (g0 == 0) load_queries(begun[0], raw);
      float2 scale[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (page[i] >= cache.pages) page[i] = -1;
        const size_t at = (size_t)max(page[i], 0) * cache.kv_heads + kv_head;
        scale[i] = make_float2(1.0f, 1.0f);
        if (page[i] >= 0) scale[i] = make_float2(cache.k_scales[at], cache.v_scales[at]);
      }
      if (alive && !wait_barrier(bar(CHUNK_FREE + buffer), (uint32_t)(g0 / kChunk >> 1 & 1) ^ 1u)) { g_error = 1; alive = false; }
      __syncwarp();
      Chunk& chunk = chunks[buffer];
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        if (lane == j) {
          chunk.first[j] = beginning >> j & 1;
          chunk.last[j] = last_tiles >> j & 1;
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int entry = lane + 32 * i;
        if (entry < entries) chunk.row[entry >> slot_shift][slot] = page[i] >= 0 ? page[i] << shift : -page_size;
      }
      __syncwarp();
      if (lane == 0) barrier_arrive(bar(ROWS_FULL + buffer));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int entry = lane + 32 * i;
        if (entry < entries) chunk.scale[entry >> slot_shift][slot] = scale[i];
      }
      __syncwarp();
      if (lane == 0) barrier_arrive(bar(CHUNK_FULL + buffer));
      // the queries of the parts that begin here, in their two parts, as operands: a lane has four elements of a head
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        if ((beginning >> j & 1) == 0) continue;
        const int parity = parts_begun & 1;
        if (g0 + j > 0) load_queries(begun[j], raw);
        if (alive && !wait_barrier(bar(Q_FREE + parity), (uint32_t)(parts_begun >> 1 & 1) ^ 1u)) { g_error = 1; alive = false; }
        __syncwarp();
#pragma unroll
        for (int h = 0; h < G; ++h) {
          float x[4] = {__uint_as_float(raw[h].x << 16), __uint_as_float(raw[h].x & 0xffff0000u), __uint_as_float(raw[h].y << 16),
                        __uint_as_float(raw[h].y & 0xffff0000u)};
          const float largest = warp_largest(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
          const int e = least_scale_exponent(fminf(largest, 3.38953139e38f));
          const float inverse = query_inverse(largest, e);
          uint32_t hi[2], lo[2];
          split_e4m3_e5m2(x[0] * inverse, x[1] * inverse, hi[0], lo[0]);
          split_e4m3_e5m2(x[2] * inverse, x[3] * inverse, hi[1], lo[1]);
          unsigned char* to = smem + L::kOffQ + parity * 2 * kPart + swizzled(h, lane * 4);
          *reinterpret_cast<uint32_t*>(to) = hi[0] | (hi[1] << 16);
          *reinterpret_cast<uint32_t*>(to + kPart) = lo[0] | (lo[1] << 16);
          if (lane == 0) factors[parts_begun & 3][h] = power_of_two(e) * scale_log2;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(bar(Q_READY + (parts_begun & 3)));
        ++parts_begun;
      }
      page[0] = page_next[0];
      page[1] = page_next[1];
    }
  } else if (warp == kKeyLoader || warp == kValueLoader) {
    // ------------------------------------------------------------------ loaders: lane l has page slot l of the tile
    const bool values = warp == kValueLoader;
    const uint32_t box_bytes = (uint32_t)cache.page_size * kDim;
    const bool loads = lane < (kKeys >> shift);
    const uint32_t full0 = bar(values ? V_FULL : K_FULL), free0 = bar(values ? V_FREE : K_FREE);
    const uint32_t base = smem_base + (uint32_t)(values ? L::kOffV : L::kOffK);
    bool alive = true;
    uint32_t stage = 0, parity = 0;
    for (int g = 0; g < count; ++g) {
      const int buffer = g / kChunk & 1;
      if (g % kChunk == 0 && alive && !wait_barrier(bar(ROWS_FULL + buffer), (uint32_t)(g / kChunk >> 1 & 1))) { g_error = 1; alive = false; }
      alive = __all_sync(0xffffffffu, alive);
      const int cache_row = loads ? chunks[buffer].row[g % kChunk][lane] : 0;
      __syncwarp();
      if (g % kChunk == kChunk - 1 && lane == 0) barrier_arrive(bar(CHUNK_FREE + buffer));
      if (alive && !wait_barrier(free0 + 8u * stage, parity ^ 1u)) { g_error = 1; alive = false; }
      alive = __all_sync(0xffffffffu, alive);
      if (!alive) break;
      // Where the tile's pages lie one behind the other in the pool one box takes them all (a copy instruction costs the warp about 75
      // cycles for every lane that takes part).
      const int first_row = __shfl_sync(0xffffffffu, cache_row, 0);
      const bool in_a_row = first_row >= 0 && __all_sync(0xffffffffu, !loads || cache_row == first_row + (lane << shift));
      const uint32_t full = full0 + 8u * stage, to = base + stage * (uint32_t)kTile;
      if (lane == 0) barrier_expect_bytes(full, (uint32_t)kTile);
      __syncwarp();
      if (in_a_row) {
        if (lane == 0) tma_load_2d(to, values ? &v_tile_map : &k_tile_map, full, kv_head * kDim, first_row);
      } else if (loads) {                              // (a negative row lies outside the tensor: zeros)
        tma_load_2d(to + (uint32_t)lane * box_bytes, values ? &v_map : &k_map, full, kv_head * kDim, cache_row);
      }
      if (++stage == (uint32_t)kStages) { stage = 0; parity ^= 1u; }
    }
    wait_for_copies(full0, (uint32_t)kStages, stage, parity);
  } else if (warp == kIssuer) {
    // ------------------------------------------------------------------ issuer (tcgen05.cuh: from a whole warp)
    constexpr uint32_t scores_hi = instruction_descriptor_8bit(kKeys, kHeads, E4M3, E4M3);
    constexpr uint32_t scores_lo = instruction_descriptor_8bit(kKeys, kHeads, E4M3, E5M2);
    constexpr uint32_t values_hi = instruction_descriptor_8bit(kDim, L::kValueColumns, E4M3, E4M3, true);
    constexpr uint32_t values_lo = instruction_descriptor_8bit(kDim, L::kValueColumns, E4M3, E5M2, true);
    const uint32_t elected = elect_one();
    const uint32_t k_low = operand_low(smem_base + L::kOffK), q_low = operand_low(smem_base + L::kOffQ);
    const uint32_t v_low = operand_low_mn_major(smem_base + L::kOffV, kTile), p_low = operand_low(smem_base + L::kOffP);
    constexpr uint32_t kPartStep = kPart >> 4, kWeightStep = L::kWeightPart >> 4, kTileStep = kTile >> 4;
    bool alive = true;
    auto check = [&](int index, uint32_t parity) {
      if (alive && !wait_barrier(bar(index), parity)) { g_error = 2; alive = false; }
    };
    uint32_t k_stage = 0, k_parity = 0, v_stage = 0, v_parity = 0;
    int n = 0;                                         // parts whose scores are under way
    auto issue_scores = [&](int g) {
      const int buffer = g / kChunk & 1;
      if (g % kChunk == 0) check(ROWS_FULL + buffer, (uint32_t)(g / kChunk >> 1 & 1));
      __syncwarp();
      const bool first = __shfl_sync(0xffffffffu, chunks[buffer].first[g % kChunk], 0) != 0;
      const bool last = __shfl_sync(0xffffffffu, chunks[buffer].last[g % kChunk], 0) != 0;
      __syncwarp();
      if (g % kChunk == kChunk - 1 && lane == 0) barrier_arrive(bar(CHUNK_FREE + buffer));
      if (first) check(Q_READY + (n & 3), (uint32_t)(n >> 2 & 1));
      check(K_FULL + (int)k_stage, k_parity);
      __syncwarp();
      tensor_fence_after_sync();
      const uint32_t a = k_low + k_stage * kTileStep, b = q_low + (uint32_t)(n & 1) * 2u * kPartStep, d = tmem_s + (uint32_t)(g & 1) * 16u;
#pragma unroll
      for (int kk = 0; kk < kDim / 32; ++kk) mma_8bit_ss_halves(d, a + 2u * kk, b + 2u * kk, scores_hi, kk > 0 ? 1u : 0u, elected);
#pragma unroll
      for (int kk = 0; kk < kDim / 32; ++kk) mma_8bit_ss_halves(d, a + 2u * kk, b + kPartStep + 2u * kk, scores_lo, 1u, elected);
      mma_commit_elected(bar(S_FULL + (g & 1)), elected);
      mma_commit_elected(bar(K_FREE + (int)k_stage), elected);
      if (last) {
        mma_commit_elected(bar(Q_FREE + (n & 1)), elected);
        ++n;
      }
      if (++k_stage == (uint32_t)kStages) { k_stage = 0; k_parity ^= 1u; }
    };
    // Whether all lanes see the phase with this parity complete, without waiting for it.
    auto complete = [&](int index, uint32_t parity) {
      uint32_t done;
      asm volatile("{\n\t.reg .pred P1;\n\tmbarrier.test_wait.parity.shared::cta.b64 P1, [%1], %2;\n\tselp.b32 %0, 1, 0, P1;\n\t}"
                   : "=r"(done) : "r"(bar(index)), "r"(parity) : "memory");
      return __all_sync(0xffffffffu, done != 0u) != 0;
    };
    // Scores are issued up to two tiles ahead of the product with the values, but a product whose values and weights are there does
    // not wait behind scores whose keys are not.
    int issued = 0;
    for (int g = 0; g < count; ++g) {
      unsigned long long start = 0;
      for (unsigned poll = 1; alive; ++poll) {
        if (issued < min(count, g + 2) && (issued == 0 || complete(K_FULL + (int)k_stage, k_parity))) issue_scores(issued++);
        else if (complete(V_FULL + (int)v_stage, v_parity) && complete(P_READY + (g & 1), (uint32_t)(g >> 1 & 1))) break;
        if ((poll & 63u) == 0u) {
          const unsigned long long now = global_nanoseconds();
          if (start == 0) start = now;
          else if (__any_sync(0xffffffffu, now - start > kWaitNanoseconds)) { g_error = 2; alive = false; }
        }
      }
      __syncwarp();
      tensor_fence_after_sync();
      const uint32_t a = v_low + v_stage * kTileStep;
      // 32 keys are 32 rows of 128 bytes further down the values, 32 bytes further along the weights
#pragma unroll
      for (int kk = 0; kk < kKeys / 32; ++kk)
        mma_8bit_ss_halves(tmem_o, a + (uint32_t)kk * (4096u >> 4), p_low + 2u * kk, values_hi, kk > 0 ? 1u : 0u, elected);
#pragma unroll
      for (int kk = 0; kk < kKeys / 32; ++kk)
        mma_8bit_ss_halves(tmem_o, a + (uint32_t)kk * (4096u >> 4), p_low + kWeightStep + 2u * kk, values_lo, 1u, elected);
      mma_commit_elected(bar(V_FREE + (int)v_stage), elected);
      mma_commit_elected(bar(PV_DONE + (g & 1)), elected);
      if (++v_stage == (uint32_t)kStages) { v_stage = 0; v_parity ^= 1u; }
      // (The scores of the tile after next take the accumulator that the softmax has read: P_READY says so.)
    }
  } else {
    // ------------------------------------------------------------------ softmax: thread = key of the tile, then element
    const int r = threadIdx.x, slot = r >> shift;
    const uint32_t lane_bits = (uint32_t)(warp * 32) << 16;
    bool alive = true;
    uint32_t stage = 0, stage_parity = 0;
    // The products of a tile are added while the next one's maxima are on their way; with 16 heads before that, their scores and sums do not
    // fit the registers together (32 contexts of 2,048 to 4,096 keys, 32 heads over 2: 42 us, 47 the other way; with 4 heads 52 and 50).
    constexpr bool kAddsFirst = G > 8;
    // The weights' bytes of this thread's key, zeros but for one band of each head; which it is (two bits a head).
    unsigned char* p_smem = smem + L::kOffP;
    uint32_t bands = 0u;
#pragma unroll
    for (int row = 0; row < kBands * G; ++row) p_smem[swizzled(row, r)] = p_smem[L::kWeightPart + swizzled(row, r)] = 0;
    int g = 0;
    for (int n = 0; walk.next(part); ++n) {
      const Row& of = part.of;
      float top[G], denominator[G], sum[G];              // of s; of exp2(s - top); this thread's element of the head, relative to top
#pragma unroll
      for (int h = 0; h < G; ++h) {
        top[h] = -INFINITY;
        denominator[h] = sum[h] = 0.0f;
      }
      float reference[G];
      // Adds the products of tile `of_tile`, whose references are still there.
      auto add = [&](int of_tile) {
        if (alive && !wait_barrier(bar(PV_DONE + (of_tile & 1)), (uint32_t)(of_tile >> 1 & 1))) { g_error = 3; alive = false; }
        __syncwarp();
        tensor_fence_after_sync();
        float value[G];
        constexpr int kAtOnce = 16 / G;                      // bands, the last ones first
#pragma unroll
        for (int b = kBands - kAtOnce; b >= 0; b -= kAtOnce) {
          float o[16];
          tmem_load_16(tmem_o + (uint32_t)(b * G) + lane_bits, o);
#pragma unroll
          for (int i = kAtOnce - 1; i >= 0; --i)
#pragma unroll
            for (int h = 0; h < G; ++h) value[h] = b + i == kBands - 1 ? o[i * G + h] : fmaf(value[h], 6.103515625e-5f, o[i * G + h]);      // 2^-14
        }
        tensor_fence_before_sync();                          // (the next product writes there behind P_READY)
#pragma unroll
        for (int h = 0; h < G; ++h) {
          // (2^e may lie below the 32-bit numbers where what it is multiplied with does not.  Without a visible key the products are
          // zeros, or NaN where the only visible scores are.)
          const float e = reference[h] > -INFINITY ? reference[h] - top[h] : 0.0f;
          value[h] *= approximate_exp2(fmaxf(e, -100.0f));
          if (e < -100.0f) value[h] *= approximate_exp2(e + 100.0f);
          sum[h] += value[h];
        }
      };
      const float* factor_of = factors[n & 3];
      if (alive && !wait_barrier(bar(Q_READY + (n & 3)), (uint32_t)(n >> 2 & 1))) { g_error = 3; alive = false; }
      for (int t = part.first; t < part.last; ++t, ++g) {
        if (kAddsFirst && t > part.first) add(g - 1);
        const int buffer = g / kChunk & 1, key = of.begin + t * kKeys + r;
        if (g % kChunk == 0 && alive && !wait_barrier(bar(CHUNK_FULL + buffer), (uint32_t)(g / kChunk >> 1 & 1))) { g_error = 3; alive = false; }
        const bool visible = chunks[buffer].row[g % kChunk][slot] >= 0 && key <= of.position && key >= of.first_key;
        const float2 scale = chunks[buffer].scale[g % kChunk][slot];
        __syncwarp();
        if (g % kChunk == kChunk - 1 && lane == 0) barrier_arrive(bar(CHUNK_FREE + buffer));
        const float shift_v = (float)(((__float_as_int(scale.y) >> 23) & 0xff) - 127);    // the exponent of a power of two
        if (!visible) {
          // what the product with this key's weight of 0 reads is zeros, not whatever lies there
          if (alive && !wait_barrier(bar(V_FULL + (int)stage), stage_parity)) { g_error = 3; alive = false; }
          uint4* mine = reinterpret_cast<uint4*>(smem + L::kOffV + stage * kTile + r * kDim);
#pragma unroll
          for (int i = 0; i < 8; ++i) mine[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
        if (alive && !wait_barrier(bar(S_FULL + (g & 1)), (uint32_t)(g >> 1 & 1))) { g_error = 3; alive = false; }
        __syncwarp();
        tensor_fence_after_sync();
        float s[G];
        tmem_load<G>(tmem_s + (uint32_t)(g & 1) * 16u + lane_bits, s);
        float(*seen)[4] = exchange[g & 1];
        float mine = -INFINITY;
#pragma unroll
        for (int h = 0; h < G; ++h) {
          s[h] = visible ? s[h] * (scale.x * factor_of[h]) : -INFINITY;
          const float a = warp_largest(s[h]), b = warp_largest(s[h] + shift_v);
          mine = lane == h ? a : (lane == G + h ? b : mine);
        }
        if (lane < 2 * G) seen[lane][warp] = mine;
        asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
        if (!kAddsFirst && t > part.first) add(g - 1);         // (its weights' places are free then)
#pragma unroll
        for (int h = 0; h < G; ++h) {
          const float4 four = *reinterpret_cast<const float4*>(seen[h]), more = *reinterpret_cast<const float4*>(seen[G + h]);
          const float a = fmaxf(fmaxf(four.x, four.y), fmaxf(four.z, four.w));
          reference[h] = fmaxf(fmaxf(more.x, more.y), fmaxf(more.z, more.w)) - kTop;
          if (a > top[h]) {
            const float factor = approximate_exp2(top[h] - a);                          // 0 when nothing was seen before
            denominator[h] *= factor;
            sum[h] *= factor;
            top[h] = a;
          }
          // (scores of -inf weigh nothing, also where there is no other yet)
          denominator[h] += visible ? approximate_exp2(s[h] - (top[h] > -INFINITY ? top[h] : 0.0f)) : 0.0f;
        }
#pragma unroll
        for (int h = 0; h < G; h += 2) {
          float w[2];
          int band[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            // the band is the whole number next to (kTop - x) / kBand - 1/2, from 0 (a NaN's too) to the last one's
            const float x = s[h + i] + shift_v - (reference[h + i] > -INFINITY ? reference[h + i] : 0.0f);
            const float whole = fminf(fmaxf(fmaf(x, -1.0f / kBand, kTop / kBand - 0.5f), 0.0f), (float)(kBands - 1)) + 12582912.0f;      // 1.5 * 2^23
            band[i] = __float_as_int(whole) & (kBands - 1);
            w[i] = visible ? approximate_exp2(fmaf(whole - 12582912.0f, kBand, x)) : 0.0f;
          }
          uint32_t hi, lo;
          split_e4m3_e5m2(w[0], w[1], hi, lo);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int before = (int)(bands >> (2 * (h + i)) & 3u);
            unsigned char *to = p_smem + swizzled(band[i] * G + h + i, r), *old = p_smem + swizzled(before * G + h + i, r);
            if (before != band[i]) old[0] = old[L::kWeightPart] = 0;
            to[0] = (unsigned char)(hi >> (8 * i));
            to[L::kWeightPart] = (unsigned char)(lo >> (8 * i));
            bands ^= (uint32_t)(before ^ band[i]) << (2 * (h + i));
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        tensor_fence_before_sync();
        barrier_arrive(bar(P_READY + (g & 1)));
        if (++stage == (uint32_t)kStages) { stage = 0; stage_parity ^= 1u; }
      }
#pragma unroll
      for (int h = 0; h < G; ++h) {
        const float total = warp_sum(denominator[h]);  // every thread holds its keys' share
        if (lane == 0) sums[warp][h] = total;
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");
      add(g - 1);
      if (alive) {
        // a part that is not the whole: in its CTA's second place if it begins here, in the first if it goes on from the team before
        const int heads_of_unit = min(group, kHeads);
        float* to = parts + ((size_t)blockIdx.x * 2 + (part.first == 0 ? 1 : 0)) * heads_of_unit * (kDim + 2);
#pragma unroll
        for (int h = 0; h < G; ++h) {
          if (h >= valid_heads) break;
          float total = (sums[0][h] + sums[1][h]) + (sums[2][h] + sums[3][h]);
          const float value = sum[h];
          if (part.whole()) {
            if (total != 0.0f && sinks != nullptr) total += exp2f(sinks[head0 + h] * kLog2e - top[h]);
            out[((size_t)part.row * heads + head0 + h) * kDim + r] = __float2bfloat16_rn(total == 0.0f ? 0.0f : value / total);
          } else {
            to[h * (kDim + 2) + r] = value;
            if (r == 0) {
              to[h * (kDim + 2) + kDim] = top[h];
              to[h * (kDim + 2) + kDim + 1] = total;
            }
          }
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kSoftmaxThreads) : "memory");     // (the sums have been read)
    }
    tensor_fence_before_sync();
  }
  __syncthreads();
  if (warp == kIssuer) {
    tensor_fence_after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_s), "r"(L::kTmemColumns) : "memory");
  }
}

// Joins the parts of what was cut: a block for each row and head, whose warps take the parts in turn.
constexpr int kJoinWarps = 4;
__global__ void __launch_bounds__(kJoinWarps * 32)
join_8bit_kernel(const float* __restrict__ parts, const int* __restrict__ positions, int num_rows, int heads, int kv_heads, int window,
                 int table_keys, int teams, bf16* __restrict__ out, const float* __restrict__ sinks) {
  grid_dependency_wait();
  grid_launch_dependents();
  if (*reinterpret_cast<volatile int*>(&g_error) != 0) return;               // parts are missing
  __shared__ float4 sums_of[kJoinWarps][32];
  __shared__ float denominators[kJoinWarps];
  const int row = blockIdx.y, head = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // all tiles, and those of the rows before this one
  unsigned total = 0, before = 0;
  for (int r = lane; r < num_rows; r += 32) {
    const unsigned tiles = (unsigned)row_at(positions, r, window, table_keys).tiles;
    total += tiles;
    before += r < row ? tiles : 0u;
  }
  total = __reduce_add_sync(0xffffffffu, total);
  before = __reduce_add_sync(0xffffffffu, before);
  const int group = heads / kv_heads, group_tiles = (group + kHeads - 1) / kHeads, units = kv_heads * group_tiles;
  const unsigned tiles = (unsigned)row_at(positions, row, window, table_keys).tiles;
  if (tiles == 0u) return;
  const unsigned each = shares_of(total, teams);
  const int heads_of_unit = min(group, kHeads);
  const int in_group = head % group, unit = head / group * group_tiles + in_group / kHeads, h = in_group % kHeads;
  const int from = (int)(before / each), to = (int)((before + tiles - 1u) / each);
  if (from == to) return;                              // one team had all of it
  auto place = [&](int team) { return parts + ((((size_t)team * units + unit) * 2 + (team == from ? 1 : 0)) * heads_of_unit + h) * (kDim + 2); };
  float top = -INFINITY;
  for (int c = from + lane; c <= to; c += 32) {
    const float2 ml = *reinterpret_cast<const float2*>(place(c) + kDim);
    if (ml.y != 0.0f) top = fmaxf(top, ml.x);
  }
  top = warp_max(top);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
#pragma unroll 4
  for (int c = from + warp; c <= to; c += kJoinWarps) {
    const float* p = place(c);
    const float2 ml = *reinterpret_cast<const float2*>(p + kDim);
    const float2 a = *reinterpret_cast<const float2*>(p + lane * 4), b = *reinterpret_cast<const float2*>(p + lane * 4 + 2);
    const float factor = ml.y == 0.0f ? 0.0f : exp2f(ml.x - top);            // 0: no visible key (its values are zeros)
    sum += ml.y * factor;
    o.x += a.x * factor; o.y += a.y * factor; o.z += b.x * factor; o.w += b.y * factor;
  }
  sums_of[warp][lane] = o;
  if (lane == 0) denominators[warp] = sum;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    const float4 theirs = sums_of[w][lane];
    o.x += theirs.x; o.y += theirs.y; o.z += theirs.z; o.w += theirs.w;
    sum += denominators[w];
  }
  if (sum != 0.0f && sinks != nullptr) sum += exp2f(sinks[head] * kLog2e - top);
  const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
  __nv_bfloat162 both[2] = {__floats2bfloat162_rn(o.x * inverse, o.y * inverse), __floats2bfloat162_rn(o.z * inverse, o.w * inverse)};
  *reinterpret_cast<uint2*>(out + ((size_t)row * heads + head) * kDim + lane * 4) = *reinterpret_cast<const uint2*>(both);
}

template <int G>
int launch(const Attention8& a, const CUtensorMap (&maps)[4]) {
  const int status = reserve_shared(decode_8bit_kernel<G>, Layout<G>::kSmemBytes, a.what);
  if (status != MIR_OK) return status;
  return mir_launch("decode_attention_8bit", decode_8bit_kernel<G>, dim3(a.num_partitions), dim3(kThreads), (size_t)Layout<G>::kSmemBytes, a.stream, 0,
                    maps[0], maps[1], maps[2], maps[3], (const bf16*)a.q, a.q_stride, a.cache, a.block_table, a.table_width, a.positions,
                    a.num_rows, a.heads, a.scale * kLog2e, a.window, a.scratch, (bf16*)a.out, a.sinks);
}

}  // namespace

// 0 if no bounded wait of the kernel ever ran out; else which role gave up last (1 loader, 2 issuer, 3 softmax).  Synchronises the device.  `next`: exchange_flag.
MIR_EXPORT int mir_decode_attention_8bit_error(int next) {
  return exchange_flag(g_error, next);
}

// Whether the kernel takes these sizes: head_dim 128, pages of 8 to 128 keys that divide 128.
bool mir_decode_8bit_takes(int head_dim, int page_size) {
  return head_dim == kDim && page_size >= 8 && page_size <= kKeys && kKeys % page_size == 0;
}

// The CTAs of a call whose rows have at most `most_tiles` tiles together, and the floats of scratch for two parts of each.
int mir_decode_8bit_ctas(long long most_tiles, int heads, int kv_heads) {
  const long long units = (long long)kv_heads * ((heads / kv_heads + kHeads - 1) / kHeads);
  return (int)(units * std::max(1ll, std::min(most_tiles, 2ll * mir_sm_count() / units)));
}
long long mir_decode_8bit_floats(int ctas, int group) { return 2ll * ctas * std::min(group, kHeads) * (kDim + 2); }

int mir_attention_8bit_decode(const Attention8& a) {
  if (a.num_rows > 65535) {
    mir_set_error("%s: %d rows are more than one launch takes", a.what, a.num_rows);
    return MIR_BAD_ARGUMENT;
  }
  const int group = a.heads / a.cache.kv_heads, units = a.cache.kv_heads * ((group + kHeads - 1) / kHeads);
  if (a.num_partitions % units != 0) {
    mir_set_error("%s: %d partitions are not a plan's for %d heads and %d kv heads", a.what, a.num_partitions, a.heads, a.cache.kv_heads);
    return MIR_BAD_ARGUMENT;
  }
  const long long table_keys = std::min(0x7fffffffll, (long long)a.table_width * a.cache.page_size);
  if ((long long)a.num_rows * (table_keys / kKeys + 1) > 0x7fffffffll) {
    mir_set_error("%s: %d rows of up to %lld keys are more than one launch takes", a.what, a.num_rows, table_keys);
    return MIR_BAD_ARGUMENT;
  }
  const long long rows = (long long)a.cache.pages * a.cache.page_size, width = (long long)a.cache.kv_heads * kDim;
  CUtensorMap maps[4];
  const void* tensors[2] = {a.cache.k, a.cache.v};
  for (int i = 0; i < 4; ++i) {
    const int status = tensor_map_of_bytes(tensors[i & 1], rows, width, width, i < 2 ? a.cache.page_size : kKeys, &maps[i]);
    if (status != MIR_OK) return status;
  }
  const int columns = std::min(group, kHeads);
  const int status = columns <= 4 ? launch<4>(a, maps) : (columns <= 8 ? launch<8>(a, maps) : launch<16>(a, maps));
  if (status != MIR_OK || a.num_partitions == units) return status;          // (one team cuts nothing)
  return mir_launch("join_8bit", join_8bit_kernel, dim3(a.heads, a.num_rows), dim3(kJoinWarps * 32), 0, a.stream, 0, (const float*)a.scratch, a.positions,
                    a.num_rows, a.heads, a.cache.kv_heads, a.window, (int)table_keys, a.num_partitions / units, (bf16*)a.out, a.sinks);
}
