// What the 8-bit kernels on the 5th-generation tensor cores share: products of 8-bit operands, tensor maps of bytes.
//
// tcgen05.mma kind::f8f6f4 takes K = 32 elements an instruction, A and B each e4m3 or e5m2, 32-bit accumulators.  An operand
// row of 128 elements is 128 bytes: one row of the 128-byte swizzle, so the descriptors of tcgen05.cuh apply as they are,
// 32 elements are 32 bytes further along a K-major row, and 4 KB (32 rows) further down an MN-major tile.
#pragma once
#include "eight_bit.h"
#include "tcgen05.cuh"

namespace mir {
namespace tc {

enum Format8 : uint32_t { E4M3 = 0, E5M2 = 1 };

__host__ __device__ constexpr uint32_t instruction_descriptor_8bit(int m, int n, Format8 a, Format8 b, bool a_mn_major = false,
                                                                   bool b_mn_major = false) {
  return (1u << 4) | ((uint32_t)a << 7) | ((uint32_t)b << 10) | ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// As mma_bf16_ss_halves (issued by the elected lane of a converged warp, descriptors as their lower halves).
__device__ __forceinline__ void mma_8bit_ss_halves(uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate,
                                                   uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, {%6, %6, %6, %6}, p;\n\t}"
      :
      : "r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kOperandHigh), "r"(0u), "r"(elected)
      : "memory");
}

// Tensor map of a row-major matrix [rows, columns] of bytes, bf16 or float32 with row stride `ld` bytes (a multiple of 16): boxes of
// box_rows rows x box_bytes (64 or 128) with the swizzle of that width, out-of-range elements read as zero and not written.
inline int tensor_map_of(const void* base, CUtensorMapDataType type, int width, long long rows, long long columns, long long ld,
                         int box_rows, int box_bytes, CUtensorMap* map) {
  static std::mutex g_mutex;
  static EncodeTiled g_encode = nullptr;
  std::unique_lock<std::mutex> lock(g_mutex);
  if (g_encode == nullptr) {
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess || entry == nullptr) {
      mir_set_error("tensor map: the driver has no cuTensorMapEncodeTiled");
      return MIR_LIBRARY_ERROR;
    }
    g_encode = reinterpret_cast<EncodeTiled>(entry);
  }
  const EncodeTiled encode = g_encode;
  lock.unlock();
  const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld};
  const cuuint32_t box[2] = {(cuuint32_t)(box_bytes / width), (cuuint32_t)box_rows};
  const cuuint32_t element_strides[2] = {1, 1};
  const CUresult status = encode(map, type, 2, const_cast<void*>(base), dims, strides, box, element_strides,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, box_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (status != CUDA_SUCCESS) {
    mir_set_error("tensor map: cuTensorMapEncodeTiled refused %lld rows of %lld columns with row stride %lld (status %d)", rows, columns,
                  ld, (int)status);
    return MIR_LIBRARY_ERROR;
  }
  return MIR_OK;
}
inline int tensor_map_of_bytes(const void* base, long long rows, long long bytes, long long ld, int box_rows, CUtensorMap* map) {
  return tensor_map_of(base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, bytes, ld, box_rows, 128, map);
}
inline int tensor_map_of_results(const void* base, bool is_float, long long rows, long long columns, long long ld, CUtensorMap* map) {
  return tensor_map_of(base, is_float ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, is_float ? 4 : 2, rows, columns,
                       ld, 32, 64, map);
}

// Lets a kernel have this much shared memory, once for each device.
template <typename Kernel>
inline int reserve_shared(Kernel kernel, int bytes, const char* what) {
  static std::mutex g_mutex;
  static std::map<std::pair<const void*, int>, int> g_done;
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err == cudaSuccess) {
    std::lock_guard<std::mutex> lock(g_mutex);
    int& done = g_done[std::make_pair(reinterpret_cast<const void*>(kernel), device)];
    if (done >= bytes) return MIR_OK;
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess) done = bytes;
  }
  if (err != cudaSuccess) {
    mir_set_error("%s: cannot reserve %d bytes of shared memory: %s", what, bytes, cudaGetErrorString(err));
    return MIR_CUDA_ERROR;
  }
  return MIR_OK;
}

// A kernel's error flag, once everything on the device is done: a copy alone waits for the default stream, and not for streams that do
// not wait for that one.  `next`: what it is from then on (0: the kernel works again), below 0: what it was.  -1: it could not be read.
inline int exchange_flag(const int& flag, int next) {
  int value = 0;
  if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&value, flag, sizeof(int)) != cudaSuccess) return -1;
  if (next >= 0 && (cudaMemcpyToSymbol(flag, &next, sizeof(int)) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess)) return -1;
  return value;
}

// The end of a loader whose next copy would go to `stage` of a ring in `phase`: the last copies into every stage are waited for (their
// readers did already, unless one gave up), so that none is on its way when the CTA ends.
__device__ __forceinline__ void wait_for_copies(uint32_t full0, uint32_t stages, uint32_t stage, uint32_t phase) {
  for (uint32_t s = 0; s < stages; ++s) (void)wait_barrier(full0 + 8u * s, s < stage ? phase : phase ^ 1u);
}

// a * b + c of two numbers side by side.
__device__ __forceinline__ float2 fma_two(float2 a, float2 b, float2 c) {
  unsigned long long x, y, z, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "f"(c.x), "f"(c.y));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}

// a + b of two numbers side by side.
__device__ __forceinline__ float2 add_two(float2 a, float2 b) {
  unsigned long long x, y, d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(y) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(d));
  return r;
}

// 32 consecutive accumulator columns of this thread's lane, without waiting for them (tmem_load_done).
__device__ __forceinline__ void tmem_load_32_ahead(uint32_t address, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(address)
      : "memory");
}
// Waits for the loads above; no use of `r` moves ahead of it.
__device__ __forceinline__ void tmem_load_done(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

}  // namespace tc
}  // namespace mir
