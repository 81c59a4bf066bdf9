// 4-bit weights with group scales: the load-time relayout into the slab of w4.cuh, and the
// matrix-vector products of 1 to 16 activation rows, plain or as the GLU of a gate and an up
// product.  No counterpart in the reference's templates (its affine decoders,
// src/kernels/decode, are the nearest); stands beside decode_vector.cu and mxfp8_gemv.cu.
#include "w4.cuh"

#include <algorithm>

namespace llmp_b200 {
namespace w4 {

int CheckMatrix(const llmp_b200_w4_matrix& m, const char* what) {
  if (m.slab == nullptr || !Aligned(m.slab, 256)) return Reject("%s: a 256-byte aligned slab", what);
  if (m.group != 32 && m.group != 64 && m.group != 128) return Reject("%s: groups of 32, 64 or 128", what);
  if (m.n < 1 || m.k < m.group || m.k % m.group != 0 || m.experts < 1) {
    return Reject("%s: at least one row and expert, k a multiple of the group", what);
  }
  if (m.n > (1 << 28) || m.k > (1 << 24)) return Reject("%s: at most 2^28 rows of 2^24 values", what);
  if (m.scale_type != kF16 && m.scale_type != kBF16) return Reject("%s: F16 or BF16 scales", what);
  if (m.glu != 0 && (m.glu != 1 || m.n % 2 != 0)) return Reject("%s: a GLU slab has as many gate as up rows", what);
  return 0;
}

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct Source {
  llmp_b200_w4_source s;
  int n, k, group, glu, tiles, steps, block_bytes;
  bool words;  // codes may be read as 32-bit words
  std::int64_t blocks;
};

// A block of threads a (expert, tile, step): 64 threads write a 16-byte piece of codes each, the
// others the words.
__global__ void __launch_bounds__(128)
RelayoutKernel(const Source a, std::uint8_t* __restrict__ slab) {
  const int groups = kStep / a.group;
  for (std::int64_t block = blockIdx.x; block < a.blocks; block += gridDim.x) {
    const std::int64_t tile_index = block / a.steps;
    const int step = static_cast<int>(block % a.steps);
    const std::int64_t expert = tile_index / a.tiles;
    const int tile = static_cast<int>(tile_index % a.tiles);
    std::uint8_t* out = slab + (block * a.block_bytes);
    const int half = a.n / 2;
    auto source_row = [&](int r) -> std::int64_t {  // -1: a padding row
      if (a.glu == 0) {
        const std::int64_t row = (static_cast<std::int64_t>(tile) * 16) + r;
        return row < a.n ? row : -1;
      }
      const std::int64_t row = (static_cast<std::int64_t>(tile) * 8) + (r & 7);
      return row < half ? row + (r < 8 ? 0 : half) : -1;
    };
    const int tid = static_cast<int>(threadIdx.x);
    if (tid < 64) {
      const int lane = tid & 31;
      const std::int64_t row = source_row((tid < 32 ? 0 : 8) + (lane >> 2));
      std::uint32_t piece[4] = {0, 0, 0, 0};
      if (row >= 0) {
        const std::uint8_t* src = a.s.codes + (expert * a.s.code_expert) + (row * a.s.code_row) +
                                  (static_cast<std::int64_t>(step) * 64) + ((lane & 3) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((step * kStep) + (32 * i) >= a.k) break;  // k is a multiple of 32
          std::uint32_t w;
          if (a.words) {
            w = *reinterpret_cast<const std::uint32_t*>(src + (16 * i));
          } else {
            const std::uint8_t* b = src + (16 * i);
            w = b[0] | (static_cast<std::uint32_t>(b[1]) << 8) | (static_cast<std::uint32_t>(b[2]) << 16) |
                (static_cast<std::uint32_t>(b[3]) << 24);
          }
          std::uint32_t even = 0, odd = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            even |= ((w >> (8 * j)) & 15u) << (4 * j);
            odd |= ((w >> ((8 * j) + 4)) & 15u) << (4 * j);
          }
          piece[i] = even | (odd << 16);
        }
      }
      *reinterpret_cast<uint4*>(out + (tid * 16)) = make_uint4(piece[0], piece[1], piece[2], piece[3]);
    } else if (tid - 64 < 16 * groups) {
      const int r = (tid - 64) / groups, gi = (tid - 64) % groups;
      const std::int64_t row = source_row(r);
      const int group = (step * groups) + gi;
      std::uint32_t word = 0x43000000u;  // scale 0, zero 0
      if (row >= 0 && group < a.k / a.group) {
        const std::uint32_t scale = static_cast<const unsigned short*>(
            a.s.scales)[(expert * a.s.scale_expert) + (row * a.s.scale_row) + group];
        std::uint32_t zero = 8;
        if (a.s.zeros != nullptr) {
          zero = a.s.zeros[(expert * a.s.zero_expert) + (row * a.s.zero_row) + (group / 2)];
          zero = (group & 1) != 0 ? zero >> 4 : zero & 15u;
        }
        word = scale | ((0x4300u + zero) << 16);  // 128 + zero, exact in bf16
      }
      *reinterpret_cast<std::uint32_t*>(out + 1024 + ((tid - 64) * 4)) = word;
    }
  }
}

struct VectorArgs {
  const std::uint8_t* slab;
  int tiles, steps, k, outputs, rows;
  const void* x;
  std::int64_t x_stride;
  bool x_vec;
  void* y;
  std::int64_t y_stride;
  int y_type;
  bool bf16_scales;
  int glu;
  float limit;
};

// Staged activations: kChunk values a column at a pitch of 64 more bytes, so the two columns that a
// quarter warp reads (64 bytes each) lie in different halves of the banks.
constexpr int kChunk = 1024;
constexpr int kPitch = (kChunk * 2) + 64;

// A warp a tile of 16 rows over all of k; the activations staged a chunk at a time.
template <int kTiles, int kType, int kGroups>
__global__ void __launch_bounds__(kThreads)
VectorKernel(const VectorArgs a) {
  constexpr int kPieces = Pieces(kType);
  extern __shared__ __align__(128) std::uint8_t smem[];
  const int lane = static_cast<int>(threadIdx.x) & 31, warp = static_cast<int>(threadIdx.x) >> 5;
  const int g = lane >> 2, t = lane & 3;
  GridLaunchDependents();
  GridDependencyWait();
  const int tile = (static_cast<int>(blockIdx.x) * kWarps) + warp;
  const bool live = tile < a.tiles;
  constexpr int kBlock = BlockBytes(kStep / kGroups);
  const std::uint8_t* block = a.slab + (static_cast<std::size_t>(live ? tile : 0) * a.steps * kBlock);
  float total[kTiles][4];
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) total[nt][0] = total[nt][1] = total[nt][2] = total[nt][3] = 0.0f;
  // this lane's column of each column tile: the token and piece it stands for
  const int piece = g % Cols(kPieces);
  std::uint32_t column_at[kTiles];
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) {
    const int token = (nt * TokensATile(kPieces)) + (g / Cols(kPieces));
    const bool real = token < a.rows && piece < kPieces;
    column_at[nt] = real ? static_cast<std::uint32_t>(((token * kPieces) + piece) * kPitch + (t * 16)) : 0xffffffffu;
  }
  for (int first = 0; first < a.k; first += kChunk) {
    __syncthreads();
    const int values = min(kChunk, a.k - first);
    const int padded = (values + kStep - 1) / kStep * kStep;
    for (int i = static_cast<int>(threadIdx.x); i < a.rows * (padded / 8); i += kThreads) {
      const int token = i / (padded / 8), at = (i % (padded / 8)) * 8;
      uint4 quads[kPieces];
      const auto* row = static_cast<const std::uint8_t*>(a.x) + (token * a.x_stride * TypeBytes(kType));
      LoadSplit8<kType>(row, first + at, values - at, a.x_vec, quads);
#pragma unroll
      for (int s = 0; s < kPieces; ++s) {
        *reinterpret_cast<uint4*>(smem + (((token * kPieces) + s) * kPitch) + (at * 2)) = quads[s];
      }
    }
    __syncthreads();
    if (!live) continue;
    for (int step = 0; step < padded / kStep; ++step, block += kBlock) {
      StepWeights<kGroups> w;
      w.Load(block, lane);
      MultiplyStep<kGroups, kTiles>(w, a.bf16_scales, kTiles, total, [&](int nt, int i) {
        if (column_at[nt] == 0xffffffffu) return make_uint4(0, 0, 0, 0);
        return *reinterpret_cast<const uint4*>(smem + column_at[nt] + (step * 256) + (i * 64));
      });
    }
  }
  if (!live) return;
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) {
    float v[2][2];
    FoldColumns<kPieces>(total[nt], v);
#pragma unroll
    for (int j = 0; j < (kPieces == 1 ? 2 : 1); ++j) {
      const int token = (nt * TokensATile(kPieces)) + TokenOf<kPieces>(t, j);
      if (token >= a.rows) continue;
      if (a.glu != LLMP_B200_GLU_NONE) {
        const int row = (tile * 8) + g;
        if (row < a.outputs) {
          StoreValue(a.y, (token * a.y_stride) + row, a.y_type,
                     Glu(a.glu, v[0][j] * Up(kType), v[1][j] * Up(kType), a.limit));
        }
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = (tile * 16) + g + (8 * r);
          if (row < a.outputs) StoreValue(a.y, (token * a.y_stride) + row, a.y_type, v[r][j] * Up(kType));
        }
      }
    }
  }
}

template <int kTiles, int kType, int kGroups>
int LaunchVector(const VectorArgs& a, cudaStream_t stream) {
  const int smem = a.rows * Pieces(kType) * kPitch;
  static thread_local int configured_device = -1;
  int device = -1;
  cudaGetDevice(&device);
  if (configured_device != device) {
    const cudaError_t set = cudaFuncSetAttribute(VectorKernel<kTiles, kType, kGroups>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, 16 * Pieces(kType) * kPitch);
    if (set != cudaSuccess) return Failed(set, "w4_vector attribute");
    configured_device = device;
  }
  const dim3 grid(static_cast<unsigned>((a.tiles + kWarps - 1) / kWarps));
  const cudaError_t e = LaunchPdl(VectorKernel<kTiles, kType, kGroups>, grid, dim3(kThreads),
                                  static_cast<std::size_t>(smem), stream, a);
  return e == cudaSuccess ? 0 : Failed(e, "w4_vector launch");
}

template <int kTiles, int kType>
int LaunchGroups(int group, const VectorArgs& a, cudaStream_t stream) {
  if (group == 128) return LaunchVector<kTiles, kType, 1>(a, stream);
  if (group == 64) return LaunchVector<kTiles, kType, 2>(a, stream);
  return LaunchVector<kTiles, kType, 4>(a, stream);
}

template <int kType>
int LaunchTiles(int group, const VectorArgs& a, cudaStream_t stream) {
  constexpr int kTokens = TokensATile(Pieces(kType));
  if (a.rows <= kTokens) return LaunchGroups<1, kType>(group, a, stream);
  if (a.rows <= 2 * kTokens) return LaunchGroups<2, kType>(group, a, stream);
  if constexpr (kTokens <= 4) {
    if (a.rows <= 4 * kTokens) return LaunchGroups<4, kType>(group, a, stream);
  }
  if constexpr (kTokens <= 2) return LaunchGroups<8, kType>(group, a, stream);
  return Reject("w4_vector: too many rows");
}

}  // namespace
}  // namespace w4
}  // namespace llmp_b200

extern "C" {

size_t llmp_b200_w4_slab_bytes(int n, int k, int group, int experts, int glu) {
  using namespace llmp_b200;
  if (n < 1 || k < 1 || n > (1 << 28) || k > (1 << 24) || experts < 1 || (group != 32 && group != 64 && group != 128)) {
    return 0;
  }
  return static_cast<size_t>(experts) * w4::Tiles(n, glu) * w4::Steps(k) * w4::BlockBytes(group);
}

int llmp_b200_w4_relayout(const llmp_b200_w4_source* source, const llmp_b200_w4_matrix* matrix, void* stream) {
  using namespace llmp_b200;
  if (source == nullptr || matrix == nullptr) return Reject("w4_relayout: null descriptor");
  if (const int status = w4::CheckMatrix(*matrix, "w4_relayout"); status != 0) return status;
  const llmp_b200_w4_source& s = *source;
  if (s.codes == nullptr || s.scales == nullptr || !Aligned(s.scales, 2)) {
    return Reject("w4_relayout: codes and 2-byte aligned scales");
  }
  const int groups = matrix->k / matrix->group;
  if (s.code_row < matrix->k / 2 || s.scale_row < groups || (s.zeros != nullptr && s.zero_row < (groups + 1) / 2) ||
      s.code_expert < 0 || s.scale_expert < 0 || s.zero_expert < 0) {
    return Reject("w4_relayout: rows at least k / 2 code bytes, k / group scales and (k / group + 1) / 2 zero bytes apart");
  }
  if (const int status = DeviceStatus(); status != 0) return status;
  w4::Source a{};
  a.s = s;
  a.n = matrix->n, a.k = matrix->k, a.group = matrix->group, a.glu = matrix->glu;
  a.tiles = w4::Tiles(a.n, a.glu), a.steps = w4::Steps(a.k), a.block_bytes = w4::BlockBytes(a.group);
  a.words = Aligned(s.codes, 4) && s.code_row % 4 == 0 && s.code_expert % 4 == 0;
  a.blocks = static_cast<std::int64_t>(matrix->experts) * a.tiles * a.steps;
  const unsigned grid = static_cast<unsigned>(std::min<std::int64_t>(a.blocks, 1 << 20));
  // an ordinary launch: a product after it on the stream starts when all of the slab is written
  w4::RelayoutKernel<<<dim3(grid), dim3(128), 0, static_cast<cudaStream_t>(stream)>>>(
      a, static_cast<std::uint8_t*>(const_cast<void*>(matrix->slab)));
  return Launched("w4_relayout launch");
}

int llmp_b200_w4_vector(const llmp_b200_w4_product* product, void* stream) {
  using namespace llmp_b200;
  if (product == nullptr) return Reject("w4_vector: null descriptor");
  const llmp_b200_w4_product& p = *product;
  if (const int status = w4::CheckMatrix(p.w, "w4_vector"); status != 0) return status;
  if (p.w.experts != 1) return Reject("w4_vector: one matrix");
  if (p.rows == 0) return 0;
  if (p.x == nullptr || p.y == nullptr) return Reject("w4_vector: activations and an output");
  if (p.rows < 1 || p.rows > 16) return Reject("w4_vector: 1 to 16 rows");
  if (!w4::FloatType(p.x_type) || !w4::FloatType(p.y_type)) return Reject("w4_vector: F32, F16 or BF16 activations and output");
  if ((p.w.glu != 0) != (p.glu != LLMP_B200_GLU_NONE)) {
    return Reject("w4_vector: a GLU and a slab of gate and up rows, or neither");
  }
  if (p.glu < LLMP_B200_GLU_NONE || p.glu > LLMP_B200_GLU_GEGLU) return Reject("w4_vector: GLU %d", p.glu);
  const int outputs = p.w.glu ? p.w.n / 2 : p.w.n;
  const int xb = w4::TypeBytes(p.x_type);
  if (!Aligned(p.x, xb) || !Aligned(p.y, w4::TypeBytes(p.y_type)) || p.x_stride < (p.rows > 1 ? p.w.k : 0) ||
      p.y_stride < (p.rows > 1 ? outputs : 0)) {
    return Reject("w4_vector: aligned rows at least k activations and n outputs apart");
  }
  if (const int status = DeviceStatus(); status != 0) return status;
  w4::VectorArgs a{};
  a.slab = static_cast<const std::uint8_t*>(p.w.slab);
  a.tiles = w4::Tiles(p.w.n, p.w.glu), a.steps = w4::Steps(p.w.k), a.k = p.w.k, a.outputs = outputs, a.rows = p.rows;
  a.x = p.x, a.x_stride = p.x_stride;
  a.x_vec = Aligned(p.x, 16) && (p.rows == 1 || (p.x_stride * xb) % 16 == 0);
  a.y = p.y, a.y_stride = p.y_stride, a.y_type = p.y_type;
  a.bf16_scales = p.w.scale_type == w4::kBF16;
  a.glu = p.glu, a.limit = p.limit;
  const auto s = static_cast<cudaStream_t>(stream);
  if (p.x_type == w4::kF32) return w4::LaunchTiles<w4::kF32>(p.w.group, a, s);
  if (p.x_type == w4::kF16) return w4::LaunchTiles<w4::kF16>(p.w.group, a, s);
  return w4::LaunchTiles<w4::kBF16>(p.w.group, a, s);
}

}  // extern "C"
