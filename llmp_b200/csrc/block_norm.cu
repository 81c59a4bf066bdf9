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

// A CTA a row.  A thread holds kUnits units of eight values from the first load to the
// last store, every row operand's loads in flight together, so a row is read once and the kernel is bound by
// memory where there are many rows (4096 rows of 4096 bf16 values with a gate a token: 32 to 34 us, 5.0 to 5.3 TB/s, 76 to
// 81 % of the copy rate; of F32 values 58 us, 5.8 TB/s, 88 %) and by two reductions and three trips to memory where there is
// one (2560 F32 values: 2.6 us).  One unit, and two of 16-bit values, stay in registers.  Four do not: 1024 threads leave 64
// registers each, 112 to 252 bytes a thread go to local memory (two units of F32 vectors: 16), and rows above 8192 values take
// more of the copy rate's time: 1024 rows of 16384 bf16 values with a gate a token 47 us, 3.6 TB/s, 54 %, of F32 values 96.
// A thread a value 1024 threads apart, unpacked as it comes, took 395 and 9.2 us.  kVec: 16-byte loads (whole rows of eight
// values, aligned); otherwise unit u's value i is column (8 u + i) threads + tid, so that a warp's
// loads are still neighbours.
template <int kType>
struct Raw8 {
  uint4 q[kType == w4::kF32 ? 2 : 1];
};

template <int kType>
__device__ __forceinline__ void Unpack8(const Raw8<kType>& raw, float (&v)[8]) {
  if constexpr (kType == w4::kF32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[4 * i] = __uint_as_float(raw.q[i].x), v[(4 * i) + 1] = __uint_as_float(raw.q[i].y);
      v[(4 * i) + 2] = __uint_as_float(raw.q[i].z), v[(4 * i) + 3] = __uint_as_float(raw.q[i].w);
    }
  } else {
    const std::uint32_t w[4] = {raw.q[0].x, raw.q[0].y, raw.q[0].z, raw.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kType == w4::kBF16) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[(2 * i) + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[2 * i] = HalfBitsToFloat(w[i] & 0xffffu);
        v[(2 * i) + 1] = HalfBitsToFloat(w[i] >> 16);
      }
    }
  }
}
template <int kType>
__device__ __forceinline__ Raw8<kType> Pack8(const float (&v)[8]) {
  Raw8<kType> raw;
  if constexpr (kType == w4::kF32) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      raw.q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[(4 * i) + 1]), __float_as_uint(v[(4 * i) + 2]),
                            __float_as_uint(v[(4 * i) + 3]));
    }
  } else {
    std::uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kType == w4::kBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[(2 * i) + 1]);
        w[i] = *reinterpret_cast<const std::uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * i], v[(2 * i) + 1]);
        w[i] = *reinterpret_cast<const std::uint32_t*>(&h);
      }
    }
    raw.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return raw;
}

template <int kType, bool kVec>
__device__ __forceinline__ Raw8<kType> LoadUnit(const void* row, int unit, int threads, int tid, int width) {
  Raw8<kType> raw;
  if constexpr (kVec) {
    const int c = ((unit * threads) + tid) * 8;
    constexpr int kQuads = kType == w4::kF32 ? 2 : 1;
    const auto* p = reinterpret_cast<const uint4*>(static_cast<const std::uint8_t*>(row) + (static_cast<std::int64_t>(c) * w4::TypeBytes(kType)));
#pragma unroll
    for (int i = 0; i < kQuads; ++i) raw.q[i] = c < width ? p[i] : make_uint4(0, 0, 0, 0);
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (((unit * 8) + i) * threads) + tid;
      v[i] = c < width ? LoadValue(row, c, kType) : 0.0f;
    }
    raw = Pack8<kType>(v);  // exact: they came from the type
  }
  return raw;
}
template <int kType, bool kVec>
__device__ __forceinline__ void StoreUnit(void* row, int unit, int threads, int tid, int width, const float (&v)[8]) {
  if constexpr (kVec) {
    const int c = ((unit * threads) + tid) * 8;
    if (c >= width) return;
    const Raw8<kType> raw = Pack8<kType>(v);
    auto* p = reinterpret_cast<uint4*>(static_cast<std::uint8_t*>(row) + (static_cast<std::int64_t>(c) * w4::TypeBytes(kType)));
    p[0] = raw.q[0];
    if constexpr (kType == w4::kF32) p[1] = raw.q[1];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = (((unit * 8) + i) * threads) + tid;
      if (c < width) StoreValue(row, c, kType, v[i]);
    }
  }
}

template <int kType, int kUnits, bool kVec>
__global__ void __launch_bounds__(kUnits == 4 ? 1024 : 512)
BlockNormKernel(const llmp_b200_block_norm_desc a) {
  extern __shared__ __align__(16) float row_values[];  // with q8: the row's h
  __shared__ float sums[2][32];
  constexpr int kBytes = w4::TypeBytes(kType);
  GridLaunchDependents();
  const std::int64_t row = blockIdx.x;
  const int tid = static_cast<int>(threadIdx.x), threads = static_cast<int>(blockDim.x), width = a.width;
  auto at = [&](const void* base, std::int64_t stride) { return static_cast<const std::uint8_t*>(base) + (row * stride * kBytes); };
  auto out_at = [&](void* base, std::int64_t stride) { return static_cast<std::uint8_t*>(base) + (row * stride * kBytes); };
  // weights: of the rows' type, or F32
  auto weight = [&](const void* w, int unit, float (&v)[8]) {
    if (a.weight_type == kType) {
      Unpack8<kType>(LoadUnit<kType, kVec>(w, unit, threads, tid, width), v);
    } else {
      Unpack8<w4::kF32>(LoadUnit<w4::kF32, kVec>(w, unit, threads, tid, width), v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += a.offset;
  };
  GridDependencyWait();
  Raw8<kType> block[kUnits], residual[kUnits], gate[kUnits];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) block[u] = LoadUnit<kType, kVec>(at(a.block, a.block_stride), u, threads, tid, width);
  if (a.residual != nullptr) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) residual[u] = LoadUnit<kType, kVec>(at(a.residual, a.residual_stride), u, threads, tid, width);
  }
  if (a.gate != nullptr) {
#pragma unroll
    for (int u = 0; u < kUnits; ++u) gate[u] = LoadUnit<kType, kVec>(at(a.gate, a.gate_stride), u, threads, tid, width);
  }
  float r[kUnits][8];
  float square = 0.0f;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    Unpack8<kType>(block[u], r[u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) square = fmaf(r[u][i], r[u][i], square);
  }
  if (a.post != nullptr) {
    const float inverse = rsqrtf((BlockSum(square, sums[0]) / static_cast<float>(width)) + a.eps);
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      float w[8];
      weight(a.post, u, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[u][i] = r[u][i] * inverse * w[i];
    }
  }
  square = 0.0f;
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    if (a.gate != nullptr) {
      float v[8];
      Unpack8<kType>(gate[u], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[u][i] *= v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) r[u][i] *= a.scale;
    if (a.residual != nullptr) {
      float v[8];
      Unpack8<kType>(residual[u], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) r[u][i] += v[i];
    }
    // (columns past the row hold zero unless a zero met an infinity: they must not reach the sum)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = kVec ? ((u * threads) + tid) * 8 : (((u * 8) + i) * threads) + tid;
      if (c < width) square = fmaf(r[u][i], r[u][i], square);
    }
    if (a.out_residual != nullptr) {
      StoreUnit<kType, kVec>(out_at(a.out_residual, a.out_residual_stride), u, threads, tid, width, r[u]);
    }
  }
  if (a.pre == nullptr) return;
  const float inverse = rsqrtf((BlockSum(square, sums[1]) / static_cast<float>(width)) + a.eps);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    float w[8];
    weight(a.pre, u, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[u][i] = r[u][i] * inverse * w[i];
    if (a.out != nullptr) StoreUnit<kType, kVec>(out_at(a.out, a.out_stride), u, threads, tid, width, r[u]);
    if constexpr (kType == w4::kF32) {
      if (a.q8 != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = kVec ? (((u * threads) + tid) * 8) + i : (((u * 8) + i) * threads) + tid;
          if (c < width) row_values[c] = r[u][i];
        }
      }
    }
  }
  if constexpr (kType == w4::kF32) {
    if (a.q8 == nullptr) return;
    __syncthreads();
    const int blocks = (width + 511) / 512 * 16;
    auto* out = static_cast<std::uint8_t*>(a.q8) + (row * blocks * 36);
    for (int first = 0; first < blocks * 8; first += threads) {
      const int i = first + tid;
      float q[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if ((i * 4) + c < width) q[c] = row_values[(i * 4) + c];
      }
      QuantizeQ8_1Lane(q, i & 7, i < blocks * 8, out + ((i >> 3) * 36));
    }
  }
}

template <int kType, int kUnits, bool kVec>
int LaunchNorm(const llmp_b200_block_norm_desc& a, int threads, cudaStream_t stream) {
  static thread_local int configured_device = -1;
  int device = -1;
  cudaGetDevice(&device);
  if (configured_device != device) {
    const cudaError_t set = cudaFuncSetAttribute(BlockNormKernel<kType, kUnits, kVec>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxWidth * 4);
    if (set != cudaSuccess) return Failed(set, "block_norm attribute");
    configured_device = device;
  }
  const cudaError_t e = LaunchPdl(BlockNormKernel<kType, kUnits, kVec>, dim3(static_cast<unsigned>(a.rows)),
                                  dim3(static_cast<unsigned>(threads)), static_cast<std::size_t>(a.q8 != nullptr ? a.width * 4 : 0), stream, a);
  return e == cudaSuccess ? 0 : Failed(e, "block_norm launch");
}

template <int kType, bool kVec>
int LaunchUnits(const llmp_b200_block_norm_desc& a, cudaStream_t stream) {
  // One unit a thread up to 512 threads, two up to 1024, then four.  Many rows of single-element loads take two from 256
  // threads on, or a row's CTA is too large for its work.  (Vectors, one unit and two: 600 rows of 4096 bf16 values 8.6 and
  // 10.2 us, 4096 rows 33.6 and 33.5, of F32 values 58 and 65; one bf16 row of 2048 2.2 and 2.7.  Elements of bf16: 128 rows
  // of 4095 values 6.3 and 7.7, 320 rows 10.6 and 8.1, 2048 rows 38.8 and 34.4.)
  const int units = (a.width + 7) / 8;
  auto threads = [&](int each) { return std::max(32, (((units + each - 1) / each) + 31) / 32 * 32); };
  if (units <= 256 || ((kVec || a.rows < 2 * SmCount()) && units <= 512)) return LaunchNorm<kType, 1, kVec>(a, threads(1), stream);
  if (units <= 1024) return LaunchNorm<kType, 2, kVec>(a, threads(2), stream);
  return LaunchNorm<kType, 4, kVec>(a, threads(4), stream);
}

template <int kType>
int LaunchType(const llmp_b200_block_norm_desc& a, cudaStream_t stream) {
  const int b = w4::TypeBytes(kType);
  auto vec = [&](const void* p, std::int64_t stride, int bytes) {
    return p == nullptr || (Aligned(p, 16) && (a.rows == 1 || (stride * bytes) % 16 == 0));
  };
  const bool all = a.width % 8 == 0 && vec(a.block, a.block_stride, b) && vec(a.residual, a.residual_stride, b) &&
                   vec(a.gate, a.gate_stride, b) && vec(a.out_residual, a.out_residual_stride, b) &&
                   vec(a.out, a.out_stride, b) && vec(a.post, 0, b) && vec(a.pre, 0, b);
  return all ? LaunchUnits<kType, true>(a, stream) : LaunchUnits<kType, false>(a, stream);
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
  const auto s = static_cast<cudaStream_t>(stream);
  if (a.type == w4::kF32) return LaunchType<w4::kF32>(a, s);
  if (a.type == w4::kF16) return LaunchType<w4::kF16>(a, s);
  return LaunchType<w4::kBF16>(a, s);
}
