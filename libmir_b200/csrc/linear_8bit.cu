// Products with 8-bit weights:  out = x . w^T (+ bias) (+ out)  where
//
//   w[n, k] = wq[n, k] * sw[n / 128, k / 128]      wq e4m3, sw any 32-bit number (as checkpoints bring them),
//   x[m, k] is rounded to xq[m, k] * sx[m, k / 128]  on its way in: sx the least power of two with |x| <= 448 sx over the 128
//   columns, xq = x / sx rounded to nearest even to e4m3,
//
// so out[m, n] = sum over blocks b of 128 columns of  sx[m, b] sw[n / 128, b] (sum over k in b of xq[m, k] wq[n, k]), the inner
// sums and the outer one in 32 bits.
#include <algorithm>
#include "eight_bit.h"

using namespace mir;
typedef __nv_bfloat16 bf16;

namespace {

constexpr int kBlock = 128;             // columns (and rows of a weight) that share a scale

// A warp rounds 128 columns of one row: a lane four of them.  scales: [blocks, scale_stride], rows side by side.
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const bf16* __restrict__ x, long long stride, uint8_t* __restrict__ codes, float* __restrict__ scales, int rows,
                     int columns, int blocks, int scale_stride) {
  grid_dependency_wait();
  grid_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (unit >= (long long)rows * blocks) return;
  const int row = (int)(unit / blocks), block = (int)(unit % blocks);
  const int column = block * kBlock + lane * 4;
  const bool there = column < columns;                        // columns is a multiple of 16
  uint2 raw = make_uint2(0u, 0u);
  if (there) raw = *reinterpret_cast<const uint2*>(x + (size_t)row * stride + column);
  const float v[4] = {__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xffff0000u), __uint_as_float(raw.y << 16),
                      __uint_as_float(raw.y & 0xffff0000u)};
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    if (b < 0x7f800000u) bits = max(bits, b);
  }
  bits = __reduce_max_sync(0xffffffffu, bits);
  const int exponent = least_scale_exponent(__uint_as_float(bits));
  const float inverse = power_of_two(-exponent);
  if (there)
    *reinterpret_cast<uint32_t*>(codes + (size_t)row * columns + column) =
        to_e4m3x2(v[0] * inverse, v[1] * inverse) | (to_e4m3x2(v[2] * inverse, v[3] * inverse) << 16);
  if (lane == 0) scales[(size_t)block * scale_stride + row] = power_of_two(exponent);
}

// A weight's blocks of 128 x 128 to e4m3 with scale largest / 448: what a checkpoint would hold.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_weight_kernel(const T* __restrict__ weight, uint8_t* __restrict__ codes, float* __restrict__ scales, int rows, int columns) {
  __shared__ float largest[8];
  grid_dependency_wait();
  grid_launch_dependents();
  const int row0 = blockIdx.y * kBlock, column0 = blockIdx.x * kBlock;
  const int row_end = min(rows, row0 + kBlock), columns_here = min(kBlock, columns - column0);
  float top = 0.0f;
  for (int i = threadIdx.x; i < kBlock * kBlock; i += blockDim.x) {
    const int row = row0 + i / kBlock, column = i % kBlock;
    if (row < row_end && column < columns_here) {
      const float v = fabsf(to_float<T>(weight[(size_t)row * columns + column0 + column]));
      if (v < INFINITY) top = fmaxf(top, v);
    }
  }
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) largest[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, largest[i]);
  const float scale = top > 0.0f ? fmaxf(top / 448.0f, 1.17549435e-38f) : 1.0f;
  for (int i = threadIdx.x; i < kBlock * kBlock; i += blockDim.x) {
    const int row = row0 + i / kBlock, column = i % kBlock;
    if (row < row_end && column < columns_here) {
      const size_t at = (size_t)row * columns + column0 + column;
      codes[at] = (uint8_t)to_e4m3x2(to_float<T>(weight[at]) / scale, 0.0f);
    }
  }
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = scale;
}

}  // namespace

// Scales of a block: one for each row, filled up to whole tiles of 128 rows.
static int scale_stride_of(int m) { return (m + kBlock - 1) / kBlock * kBlock; }

// Bytes of workspace for m rows of k columns: the rounded rows, then their scales (none where the product rounds the rows itself).
MIR_EXPORT long long mir_linear_8bit_workspace(int m, int k) {
  if (m <= 0 || k <= 0 || (mir_linear_8bit_few_takes(m, k) && mir_linear_8bit_few_rounds(m))) return 0;
  const long long codes = ((long long)m * k + 255) / 256 * 256;
  return codes + (long long)scale_stride_of(m) * ((k + kBlock - 1) / kBlock) * (long long)sizeof(float);
}

MIR_EXPORT int mir_quantize_weight_8bit(int is_bf16, const void* weight, void* codes, float* scales, int rows, int columns,
                                        cudaStream_t stream) {
  if (rows <= 0 || columns <= 0 || (rows + kBlock - 1) / kBlock > 65535) {
    mir_set_error("quantize_weight_8bit: a weight of %d x %d is not one it takes", rows, columns);
    return MIR_BAD_ARGUMENT;
  }
  const dim3 grid((columns + kBlock - 1) / kBlock, (rows + kBlock - 1) / kBlock);
  if (is_bf16)
    return mir_launch("quantize_weight_8bit", quantize_weight_kernel<bf16>, grid, dim3(256), 0, stream, 0, (const bf16*)weight,
                      (uint8_t*)codes, scales, rows, columns);
  return mir_launch("quantize_weight_8bit", quantize_weight_kernel<float>, grid, dim3(256), 0, stream, 0, (const float*)weight,
                    (uint8_t*)codes, scales, rows, columns);
}

MIR_EXPORT int mir_linear_8bit(const void* x, long long x_stride, const void* weight, const float* w_scales, const void* bias, void* out,
                               long long out_stride, int out_float, int accumulate, int m, int n, int k, void* workspace,
                               long long workspace_bytes, cudaStream_t stream) {
  if (m == 0 || n == 0) return MIR_OK;
  if (m < 0 || n < 0 || k <= 0 || (k % 16) || x_stride < k || (x_stride % 4) || out_stride < n || ((uintptr_t)x & 7) ||
      ((uintptr_t)weight & 15) || (accumulate && !out_float)) {
    mir_set_error("linear_8bit: takes columns in multiples of 16, rows of x on 8-byte boundaries and weights on 16-byte ones, "
                  "and accumulates into float32 (m %d, n %d, k %d, row strides %lld and %lld)", m, n, k, x_stride, out_stride);
    return MIR_BAD_ARGUMENT;
  }
  const long long need = mir_linear_8bit_workspace(m, k);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    mir_set_error("linear_8bit: %lld bytes of 16-byte aligned workspace are needed, got %lld", need, workspace_bytes);
    return MIR_BAD_ARGUMENT;
  }
  const int blocks = (k + kBlock - 1) / kBlock;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  float* scales = reinterpret_cast<float*>(codes + ((size_t)m * k + 255) / 256 * 256);
  // Up to 128 rows the weight's bytes are what takes the time, from there on the products.
  const bool few = mir_linear_8bit_few_takes(m, k);
  if (!few || !mir_linear_8bit_few_rounds(m)) {
    const long long units = (long long)m * blocks;
    if ((units + 7) / 8 > 0x7fffffffll) {
      mir_set_error("linear_8bit: %d rows of %d columns are more than one launch takes", m, k);
      return MIR_BAD_ARGUMENT;
    }
    const int status = mir_launch("quantize_rows_8bit", quantize_rows_kernel, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, stream, 0,
                                  (const bf16*)x, x_stride, codes, scales, m, k, blocks, scale_stride_of(m));
    if (status != MIR_OK) return status;
  }
  if (few)
    return mir_linear_8bit_few(codes, scales, scale_stride_of(m), x, x_stride, static_cast<const uint8_t*>(weight), w_scales, bias, out,
                               out_stride, m, n, k, out_float != 0, accumulate != 0, stream);
  return mir_linear_8bit_tiles(codes, scales, scale_stride_of(m), static_cast<const uint8_t*>(weight), w_scales, bias, out, out_stride, m, n,
                               k, out_float != 0, accumulate != 0, stream);
}
