// The norms after a block and before the next with what lies between them, one kernel: RMS norm of
// the block's output, gate, residual scale, residual sum, RMS norm.  In the reference these are
// separate nodes around its products; here a row is read once, its two sums of squares are taken
// over values that stay in registers, and the next product's Q8_1 rows (q8_1.cu) can come with it.
//
//   u = block * rsqrt(mean(block^2) + eps) * (offset + post)   (post NULL: u = block)
//   r = residual + scale * gate * u                            (NULL: no residual, no gate)
//   h = r * rsqrt(mean(r^2) + eps) * (offset + pre)
//
// All in F32; r and h are rounded once, when they are stored (h is of the unrounded r).
#include <algorithm>

#include "q8_1.cuh"
#include "w4.cuh"

namespace llmp_b200 {
namespace {

using w4::LoadValue;
using w4::StoreValue;

constexpr int kMaxWidth = 32768;

__device__ __forceinline__ float BlockSum(float v, float* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int warps = static_cast<int>(blockDim.x) >> 5;
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  v = lane < warps ? shared[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A CTA a row, a thread the values tid, tid + blockDim, ...
__global__ void __launch_bounds__(1024)
BlockNormKernel(const llmp_b200_block_norm_desc a) {
  extern __shared__ __align__(16) float row_values[];  // with q8: the row's h
  __shared__ float sums[2][32];
  GridLaunchDependents();
  GridDependencyWait();
  const std::int64_t row = blockIdx.x;
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x);
  constexpr int kValues = 32;
  float v[kValues];
  float square = 0.0f;
#pragma unroll
  for (int i = 0; i < kValues; ++i) {
    const int c = tid + (i * threads);
    v[i] = c < a.width ? LoadValue(a.block, (row * a.block_stride) + c, a.type) : 0.0f;
    square = fmaf(v[i], v[i], square);
  }
  float inverse = 1.0f;
  if (a.post != nullptr) inverse = rsqrtf((BlockSum(square, sums[0]) / static_cast<float>(a.width)) + a.eps);
  square = 0.0f;
#pragma unroll
  for (int i = 0; i < kValues; ++i) {
    const int c = tid + (i * threads);
    if (c >= a.width) continue;
    float u = v[i];
    if (a.post != nullptr) u = u * inverse * (LoadValue(a.post, c, a.weight_type) + a.offset);
    if (a.gate != nullptr) u *= LoadValue(a.gate, (row * a.gate_stride) + c, a.type);
    u *= a.scale;
    if (a.residual != nullptr) u += LoadValue(a.residual, (row * a.residual_stride) + c, a.type);
    v[i] = u;
    square = fmaf(u, u, square);
    if (a.out_residual != nullptr) StoreValue(a.out_residual, (row * a.out_residual_stride) + c, a.type, u);
  }
  if (a.pre == nullptr) return;
  inverse = rsqrtf((BlockSum(square, sums[1]) / static_cast<float>(a.width)) + a.eps);
#pragma unroll
  for (int i = 0; i < kValues; ++i) {
    const int c = tid + (i * threads);
    if (c >= a.width) continue;
    const float h = v[i] * inverse * (LoadValue(a.pre, c, a.weight_type) + a.offset);
    if (a.out != nullptr) StoreValue(a.out, (row * a.out_stride) + c, a.type, h);
    if (a.q8 != nullptr) row_values[c] = h;
  }
  if (a.q8 == nullptr) return;
  __syncthreads();
  const int blocks = (a.width + 511) / 512 * 16;
  auto* out = static_cast<std::uint8_t*>(a.q8) + (row * blocks * 36);
  for (int first = 0; first < blocks * 8; first += threads) {
    const int i = first + tid;
    float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if ((i * 4) + c < a.width) q[c] = row_values[(i * 4) + c];
    }
    QuantizeQ8_1Lane(q, i & 7, i < blocks * 8, out + ((i >> 3) * 36));
  }
}

}  // namespace
}  // namespace llmp_b200

extern "C" int llmp_b200_block_norm(const llmp_b200_block_norm_desc* desc, void* stream) {
  using namespace llmp_b200;
  if (desc == nullptr) return Reject("block_norm: null descriptor");
  const llmp_b200_block_norm_desc& a = *desc;
  if (a.width < 1 || a.width > kMaxWidth) return Reject("block_norm: rows of 1 to 32768 values");
  if (!w4::FloatType(a.type) || (a.weight_type != w4::kF32 && a.weight_type != a.type)) {
    return Reject("block_norm: F32, F16 or BF16 rows, weights of that type or F32");
  }
  if (a.rows < 0 || a.rows > 0x7fffffffLL) return Reject("block_norm: 0 to 2^31 - 1 rows");
  if (a.rows == 0) return 0;
  if (a.block == nullptr) return Reject("block_norm: the block's output");
  if (a.out_residual == nullptr && a.out == nullptr && a.q8 == nullptr) return Reject("block_norm: an output");
  if ((a.out != nullptr || a.q8 != nullptr) != (a.pre != nullptr)) {
    return Reject("block_norm: a second norm's weight with its output, and only then");
  }
  if (a.q8 != nullptr && a.type != w4::kF32) return Reject("block_norm: Q8_1 rows of F32 ones");
  const int b = w4::TypeBytes(a.type), wb = w4::TypeBytes(a.weight_type);
  if (!Aligned(a.block, b) || !Aligned(a.residual, b) || !Aligned(a.gate, b) || !Aligned(a.out_residual, b) ||
      !Aligned(a.out, b) || !Aligned(a.q8, 4) || !Aligned(a.post, wb) || !Aligned(a.pre, wb)) {
    return Reject("block_norm: operands aligned to their elements, Q8_1 rows to 4 bytes");
  }
  if (a.rows > 1 && (a.block_stride < 0 || a.residual_stride < 0 || a.gate_stride < 0 ||
                     (a.out_residual != nullptr && a.out_residual_stride < a.width) ||
                     (a.out != nullptr && a.out_stride < a.width))) {
    return Reject("block_norm: output rows at least a row apart, no negative strides");
  }
  if (const int status = DeviceStatus(); status != 0) return status;
  const int smem = a.q8 != nullptr ? a.width * 4 : 0;
  static thread_local int configured_device = -1;
  int device = -1;
  cudaGetDevice(&device);
  if (configured_device != device) {
    const cudaError_t set = cudaFuncSetAttribute(BlockNormKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxWidth * 4);
    if (set != cudaSuccess) return Failed(set, "block_norm attribute");
    configured_device = device;
  }
  const cudaError_t e = LaunchPdl(BlockNormKernel, dim3(static_cast<unsigned>(a.rows)), dim3(1024),
                                  static_cast<std::size_t>(smem), static_cast<cudaStream_t>(stream), a);
  return e == cudaSuccess ? 0 : Failed(e, "block_norm launch");
}
