// 4-bit weights with group scales: the load-time relayout into the slab of w4.cuh, and the
// matrix-vector products of 1 to 16 activation rows, plain or as the GLU of a gate and an up
// product.  No counterpart in the reference's templates (its affine decoders,
// src/kernels/decode, are the nearest); stands beside decode_vector.cu and mxfp8_gemv.cu.
#include <cooperative_groups.h>

#include <algorithm>

#include "w4.cuh"

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

namespace cg = cooperative_groups;


struct Source {
  llmp_b200_w4_source s;
  int n, k, group, glu, tiles, steps, block_bytes;
  bool bf16;   // the scales' type
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
      std::uint32_t word = 0;
      if (row >= 0 && group < a.k / a.group) {
        const std::uint32_t scale = static_cast<const unsigned short*>(
            a.s.scales)[(expert * a.s.scale_expert) + (row * a.s.scale_row) + group];
        std::uint32_t zero = 8;
        if (a.s.zeros != nullptr) {
          zero = a.s.zeros[(expert * a.s.zero_expert) + (row * a.s.zero_row) + (group / 2)];
          zero = (group & 1) != 0 ? zero >> 4 : zero & 15u;
        }
        // exact in F32, with at least 13 last bits of zero (but for a NaN's)
        word = a.bf16 ? scale << 16 : __float_as_uint(HalfBitsToFloat(scale));
        word = (word & 0xffffff00u) | zero;
      }
      *reinterpret_cast<std::uint32_t*>(out + 1024 + ((tid - 64) * 4)) = word;
    }
  }
}

struct VectorArgs {
  const std::uint8_t* slab;
  int tiles, steps, k, outputs, rows;
  int parts;          // warps that divide a tile's steps
  int rounds;         // of warps / parts tiles each
  int meet_floats;    // one buffer of partial sums
  bool zero_column;   // behind the staged columns, for the MMA's columns that stand for no token: any values would
                      // do, but zeros are faster (4096 -> 20480, one f16 row: 13.5 us against 17.3)
  const void* x;
  std::int64_t x_stride;
  bool x_vec;
  void* y;
  std::int64_t y_stride;
  int y_type;
  int glu;
  float limit;
};

// Persistent CTAs.  A round is a few tiles of 16 weight rows, each tile's steps divided among `parts`
// warps, whose sums meet in shared memory: with one token a matrix of 4096 x 4096 is 8.7 MB in 256 tiles,
// too few for a warp each.  The activations are staged (scaled, split) once a CTA.  Weights come
// through a ring of kSlots steps a warp (cp.async, its own lanes' copies: no CTA barrier, any depth of
// requests without registers) that runs on from one round's tile to the next.  Warps of their own
// add the parts up and store the results: those that multiply only arrive at the barrier and go on to the
// next round's other buffer of sums.  Where the activations of all of k do not fit, the CTAs of a
// cluster divide k as well and read each other's sums.
//
// What bounds it: the weights' way through the rings with the rounds' meetings, and on top of it the instructions of a step
// (about 120 to 200 a warp for 1.1 to 1.3 KB: taking the codes apart on the logic and half-precision pipes, the MMAs) and the
// staging, which all of a CTA's warps wait for.  Measured, weights from HBM, in brackets without the products, without the
// staging, without both: 4096 x 4096, one bf16 row 5.1 us (3.4, 5.0, 3.2); 4096 -> 14336 11.0 us, 2.8 TB/s (7.4, 11.0, 7.1: 3.03
// rounds a CTA, the busiest does four); 4096 -> 20480 14.0 us, 3.1 TB/s (9.4, 13.9, 9.1); gate | up 2560 -> 10240, eight F16
// rows 11.1 us (8.5, 9.9, 7.3), four F32 rows 15.6 us (12.8, 9.7, 7.1: rows read twice behind two barriers);
// 4096 -> 32003 in groups of 32, sixteen F16 rows 28.1 us, 2.7 TB/s (18.9, 26.4, 17: issue slots 56 % full, tensor pipe 24 %,
// rings of three steps beside 131 KB of activations); 8192 -> 4096, sixteen F32 rows 36.4 us (29.5, 19.6, 12.8).  (Clusters of
// eight dividing k in every call, so that each CTA stages an eighth of the activations: 31 and 83 us for the four F32 rows and
// the sixteen F16 ones, the clusters leave SMs idle and their barrier waits for the copies in flight.)
constexpr int kMaxRows = 16;

template <int kTiles, int kType, int kGroups, bool kWide>
__global__ void __launch_bounds__(Threads(kWide), kWide ? 1 : 2)
VectorKernel(const VectorArgs a) {
  constexpr int kWarps = Warps(kWide), kSlots = Slots(kWide), threads = Threads(kWide);
  constexpr int kPieces = HalfPieces(kType);
  constexpr int kBlock = BlockBytes(kStep / kGroups);
  extern __shared__ __align__(128) std::uint8_t smem[];
  __shared__ std::uint32_t magnitude[kMaxRows];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int clusters = static_cast<int>(gridDim.x) / ranks, first_round = static_cast<int>(blockIdx.x) / ranks;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int step0 = a.steps * rank / ranks, steps = (a.steps * (rank + 1) / ranks) - step0;  // this CTA's
  const int tiles_a_round = kWarps / a.parts;
  const int my_tile = warp / a.parts, part = warp % a.parts;
  const int begin = steps * part / a.parts, count = (steps * (part + 1) / a.parts) - begin;  // this warp's
  const int pitch = Pitch(steps);
  const bool multiplies = warp < kWarps;
  const std::uint32_t ring = SharedAddress(smem) + (warp * kSlots * kBlock) + (lane * 16);  // + this lane's piece
  float* meet = reinterpret_cast<float*>(smem + (kWarps * kSlots * kBlock));  // [2][warps][rows][16]
  const std::uint32_t staged_at = StagedAt(kWide, a.rows, kBlock);
  std::uint8_t* staged = smem + staged_at;

  // this warp's steps, round after round: where the next request reads
  const int first_tile = (first_round * tiles_a_round) + my_tile;
  const std::uint8_t* src =
      a.slab + ((static_cast<std::size_t>(first_tile) * a.steps) + step0 + begin) * kBlock + (lane * 16);
  const std::size_t to_next_round = ((static_cast<std::size_t>(clusters) * tiles_a_round * a.steps) - count) * kBlock;
  const int rounds_mine = first_tile < a.tiles && multiplies
                              ? ((a.tiles - 1 - first_tile) / (clusters * tiles_a_round)) + 1 : 0;
  int left = rounds_mine * count, left_of_round = count;
  auto request = [&](int slot) {  // one commit a call, so that the waits can count
    if (left > 0) {
      const std::uint32_t dst = ring + (slot * kBlock);
      CopyAsync16<0>(dst, src);
      CopyAsync16<512>(dst, src);
      if (lane < 4 * kGroups) CopyAsync16<1024>(dst, src);
      --left;
      src += kBlock;
      if (--left_of_round == 0) src += to_next_round, left_of_round = count;
    }
    CopyAsyncCommit();
  };
  GridLaunchDependents();
  if (rounds_mine > 0) {  // into L2 only: what a kernel before may still write is not read yet
    const std::size_t bytes = static_cast<std::size_t>(count) * kBlock;
    for (std::size_t at = 0; at < bytes; at += 32 * 128) {
      if (at + (lane * 128) < bytes) asm volatile("prefetch.global.L2 [%0];" ::"l"(src + at + (lane * 112)));
    }
  }
  GridDependencyWait();
#pragma unroll
  for (int i = 0; i < kSlots - 1; ++i) request(i);

  const int octets = steps * (kStep / 8), x0 = step0 * kStep;
  auto row_of = [&](int token) { return static_cast<const std::uint8_t*>(a.x) + (token * a.x_stride * TypeBytes(kType)); };
  if (a.zero_column) {
    for (int i = tid; i < octets; i += threads) {
      *reinterpret_cast<uint4*>(staged + (a.rows * kPieces * pitch) + (i * 16)) = make_uint4(0, 0, 0, 0);
    }
  }
  if constexpr (kType == kF32) {
    // twice over the rows, four octets of a thread in flight at once: the largest magnitudes, then the pieces
    if (tid < kMaxRows) magnitude[tid] = 0;
    __syncthreads();
    constexpr int kBatch = 4;
    const int all = a.rows * octets;  // octets are whole half warps
    for (int first = tid; first - tid < all; first += kBatch * threads) {
      std::uint32_t most[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int i = first + (q * threads), token = i / octets, at = x0 + ((i - (token * octets)) * 8);
        most[q] = i < all ? Magnitude8(row_of(token), at, a.k - at, a.x_vec) : 0;
      }
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int i = first + (q * threads);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most[q] = max(most[q], __shfl_xor_sync(0xffffffffu, most[q], o));
        if ((lane & 15) == 0 && i < all) atomicMax(&magnitude[i / octets], most[q]);
      }
    }
    __syncthreads();
    for (int first = tid; first < all; first += kBatch * threads) {
#pragma unroll
      for (int q = 0; q < kBatch; ++q) {
        const int i = first + (q * threads), token = i / octets, octet = i - (token * octets), at = x0 + (octet * 8);
        if (i >= all) break;
        uint4 quads[2];
        LoadHalf8(row_of(token), at, a.k - at, a.x_vec, PowerOfTwo(ScaleExponent(magnitude[token])), quads);
        std::uint8_t* out = staged + ((token * 2) * pitch) + (octet * 16);
        *reinterpret_cast<uint4*>(out) = quads[0];
        *reinterpret_cast<uint4*>(out + pitch) = quads[1];
      }
    }
  } else {
    for (int token = 0; token < a.rows; ++token) {
      for (int i = tid; i < octets; i += threads) {
        Stage8(staged + (token * pitch) + (i * 16), row_of(token), x0 + (i * 8), a.k - x0 - (i * 8), a.x_vec);
      }
    }
    CopyAsyncCommit();
    CopyAsyncWait<0>();
  }
  __syncthreads();

  // barriers 1, 2: buffer 0, 1 holds a round's sums; 3, 4: it may be written again
  if (multiplies) {
    // this lane's column of each column tile: the token and piece it stands for, or the zeros
    const int piece = g % Cols(kPieces);
    std::uint32_t column[kTiles];
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const int token = (nt * TokensATile(kPieces)) + (g / Cols(kPieces));
      column[nt] = staged_at + (StagedColumn(token, piece, a.rows, kPieces) * pitch) + (t * 16) + (begin * 256);
    }
    int slot = 0, buffer = 0;
    for (int round = first_round, n = 0; round < a.rounds; round += clusters, buffer ^= 1, ++n) {
      Sums total[kTiles];
      if (n < rounds_mine) {
        for (int step = 0; step < count; ++step) {
          CopyAsyncWait<kSlots - 2>();
          __syncwarp();  // all lanes' copies of this step are in, and the slot before it has been read
          request(slot == 0 ? kSlots - 1 : slot - 1);
          StepWeights<kGroups> w;
          w.LoadShared(smem + (((warp * kSlots) + slot) * kBlock), lane);
          MultiplyStep<kType != kBF16, kGroups, kTiles>(w, kTiles, total, [&](int nt, int i) {
            return *reinterpret_cast<const uint4*>(smem + column[nt] + (step * 256) + (i * 64));
          });
          slot = slot == kSlots - 1 ? 0 : slot + 1;
        }
      }
      if (ranks == 1 && n >= 2) BarrierSync(3 + buffer, threads);
      float* mine = meet + (buffer * a.meet_floats) + (warp * kTileRows * a.rows);
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
        float v[2][2];
        FoldColumns<kType != kBF16, kPieces>(total[nt], v);
#pragma unroll
        for (int j = 0; j < (kPieces == 1 ? 2 : 1); ++j) {
          const int token = (nt * TokensATile(kPieces)) + TokenOf<kPieces>(t, j);
          if (token < a.rows) {
            mine[(token * kTileRows) + g] = v[0][j];
            mine[(token * kTileRows) + g + 8] = v[1][j];
          }
        }
      }
      // of a cluster all threads meet: no buffer is written again before every rank has met once more
      if (ranks > 1) cluster.sync(); else BarrierArrive(1 + buffer, threads);
    }
  } else {
    // a lane adds up four rows of a token (with a GLU two, of gate and of up), a tile's tokens side by side
    const bool glu = a.glu != LLMP_B200_GLU_NONE;
    const int lane_row = glu ? (lane & 3) * 2 : (lane & 3) * 4;
    int buffer = 0;
    for (int round = first_round; round < a.rounds; round += clusters, buffer ^= 1) {
      if (ranks > 1) cluster.sync(); else BarrierSync(1 + buffer, threads);
      for (int o = rank; o < tiles_a_round; o += ranks) {
        const int tile = (round * tiles_a_round) + o;
        if (tile >= a.tiles) break;
        for (int token = ((warp - kWarps) * 8) + (lane >> 2); token < a.rows; token += Reducers(kWide) * 8) {
          float4 first = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // four rows, or two gate rows and two up rows
          for (int q = 0; q < ranks; ++q) {
            const float* p = (ranks > 1 ? cluster.map_shared_rank(meet, q) : meet) + (buffer * a.meet_floats) +
                             (((o * a.parts * a.rows) + token) * kTileRows) + lane_row;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (glu) {
#pragma unroll 4
              for (int s = 0; s < a.parts; ++s, p += kTileRows * a.rows) {
                const float2 v = *reinterpret_cast<const float2*>(p), u = *reinterpret_cast<const float2*>(p + 8);
                sum.x += v.x, sum.y += v.y, sum.z += u.x, sum.w += u.y;
              }
            } else {
#pragma unroll 8
              for (int s = 0; s < a.parts; ++s, p += kTileRows * a.rows) {
                const float4 v = *reinterpret_cast<const float4*>(p);
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
              }
            }
            float up = Up(kType != kBF16);  // (each rank's F32 activations have their own scale)
            if constexpr (kType == kF32) {
              up = PowerOfTwo(-ScaleExponent(ranks > 1 ? *cluster.map_shared_rank(&magnitude[token], q) : magnitude[token]));
            }
            first.x = fmaf(sum.x, up, first.x), first.y = fmaf(sum.y, up, first.y);
            first.z = fmaf(sum.z, up, first.z), first.w = fmaf(sum.w, up, first.w);
          }
          float out[4] = {first.x, first.y, first.z, first.w};
          if (glu) out[0] = GluOf(a.glu, first.x, first.z, a.limit), out[1] = GluOf(a.glu, first.y, first.w, a.limit);
          const int row = (tile * (glu ? 8 : 16)) + lane_row;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (row + r >= a.outputs || (glu && r >= 2)) break;
            StoreValue(a.y, (token * a.y_stride) + row + r, a.y_type, out[r]);
          }
        }
      }
      if (ranks == 1) BarrierArrive(3 + buffer, threads);
    }
  }
  if (ranks > 1) cluster.sync();  // nobody leaves while another reads its sums
}

constexpr int kSmemLimit = 226 * 1024, kSmemOfTwo = 112 * 1024;
constexpr int kMaxRanks = 8;

template <int kTiles, int kType, int kGroups, bool kWide>
int LaunchVector(VectorArgs a, int ranks, std::int64_t smem, cudaStream_t stream) {
  constexpr int kWarps = Warps(kWide);
  static thread_local int configured_device = -1;
  int device = -1;
  cudaGetDevice(&device);
  if (configured_device != device) {
    const cudaError_t set = cudaFuncSetAttribute(VectorKernel<kTiles, kType, kGroups, kWide>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    if (set != cudaSuccess) return Failed(set, "w4_vector attribute");
    configured_device = device;
  }
  const int ctas = std::max(1, SmCount() * (smem <= kSmemOfTwo ? 2 : 1) / ranks);
  // The busiest CTA's rounds times a warp's steps in one, a round costing about 0.7 of a step besides: many parts balance
  // the CTAs where tiles are few, few parts make long runs where they are many, two rounds a CTA and more.  (4096 -> 32003,
  // sixteen F16 rows: 28.1 us; with a round at nothing 31.4, at two steps 30.8.  2560 -> 2 x 10240, four F32 rows: 15.6,
  // 16.3, 15.6.)  In a cluster
  // every round ends in a barrier of all its CTAs, worth a dozen steps: as few rounds as keep the clusters busy
  // (16 rows of 16384 F16 values -> 4096: 56 us by the other rule, 25 by this; of 8192 F32 values 44 and 36).
  const double round_cost = ranks > 1 ? 12.0 : 0.7;
  const int steps = a.steps / ranks;
  double best = 0.0;
  for (int parts = kWarps; parts >= 1; parts /= 2) {
    if (parts > steps && parts > 1) continue;
    const int rounds = (a.tiles + (kWarps / parts) - 1) / (kWarps / parts);
    if (best != 0.0 && rounds < (ranks > 1 ? ctas : 2 * ctas)) break;
    const double cost = ((rounds + ctas - 1) / ctas) * (((steps + parts - 1) / parts) + round_cost);
    if (best == 0.0 || cost < best) best = cost, a.parts = parts;
  }
  a.rounds = (a.tiles + (kWarps / a.parts) - 1) / (kWarps / a.parts);
  a.meet_floats = kWarps * kTileRows * a.rows;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(std::min(a.rounds, ctas) * ranks));
  config.blockDim = dim3(static_cast<unsigned>(Threads(kWide)));
  config.dynamicSmemBytes = static_cast<std::size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = static_cast<unsigned>(ranks);
  attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, VectorKernel<kTiles, kType, kGroups, kWide>, a);
  return e == cudaSuccess ? 0 : Failed(e, "w4_vector launch");
}

template <int kTiles, int kType, int kGroups>
int LaunchPlanned(VectorArgs a, cudaStream_t stream) {
  auto bytes = [&](bool wide, int ranks) {
    return SmemBytes(wide, ranks, a.rows, a.steps, HalfPieces(kType), BlockBytes(kStep / kGroups));
  };
  a.zero_column = ZeroColumn(a.rows, HalfPieces(kType));
  // Two CTAs of eight warps where an SM's shared memory takes them; else one of sixteen, over as few CTAs of a cluster as hold the
  // activations; else (the rings of sixteen not fitting) one of eight.  (One of sixteen and of eight: sixteen F16 rows 4096 -> 32003 28.1
  // and 31.2 us, sixteen bf16 4096 -> 4096 7.5 and 8.8, sixteen F32 8192 -> 4096 36 and 51.)
  if (const std::int64_t smem = bytes(false, 1); smem <= kSmemOfTwo) {
    return LaunchVector<kTiles, kType, kGroups, false>(a, 1, smem, stream);
  }
  int ranks = 1;
  while (ranks < kMaxRanks && bytes(false, ranks) > kSmemLimit) ranks *= 2;
  if (const std::int64_t smem = bytes(true, ranks); smem <= kSmemLimit) {
    return LaunchVector<kTiles, kType, kGroups, true>(a, ranks, smem, stream);
  }
  return LaunchVector<kTiles, kType, kGroups, false>(a, ranks, bytes(false, ranks), stream);
}

template <int kTiles, int kType>
int LaunchGroups(int group, const VectorArgs& a, cudaStream_t stream) {
  if (group == 128) return LaunchPlanned<kTiles, kType, 1>(a, stream);
  if (group == 64) return LaunchPlanned<kTiles, kType, 2>(a, stream);
  return LaunchPlanned<kTiles, kType, 4>(a, stream);
}

template <int kType>
int LaunchTiles(int group, const VectorArgs& a, cudaStream_t stream) {
  constexpr int kPieces = HalfPieces(kType);
  const int tiles = ColumnTiles(a.rows, kPieces);
  if (tiles == 1) return LaunchGroups<1, kType>(group, a, stream);
  if (tiles == 2) return LaunchGroups<2, kType>(group, a, stream);
  if constexpr (TokensATile(kPieces) <= 4) return LaunchGroups<4, kType>(group, a, stream);
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
  a.bf16 = matrix->scale_type == w4::kBF16;
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
  if (p.w.k > 131072) return Reject("w4_vector: k up to 131072");
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
  a.glu = p.glu, a.limit = p.limit;
  const auto s = static_cast<cudaStream_t>(stream);
  // as many rows a launch as a cluster's shared memory takes: all of them but for very long ones
  const int block_bytes = w4::BlockBytes(p.w.group);
  int most = p.rows;
  while (most > 1 && w4::SmemBytes(false, w4::kMaxRanks, most, a.steps, w4::HalfPieces(p.x_type), block_bytes) > w4::kSmemLimit) most = (most + 1) / 2;
  for (int first = 0; first < p.rows; first += most) {
    a.rows = std::min(most, p.rows - first);
    a.x = static_cast<const std::uint8_t*>(p.x) + (first * p.x_stride * xb);
    a.y = static_cast<std::uint8_t*>(p.y) + (first * p.y_stride * w4::TypeBytes(p.y_type));
    const int status = p.x_type == w4::kF32   ? w4::LaunchTiles<w4::kF32>(p.w.group, a, s)
                       : p.x_type == w4::kF16 ? w4::LaunchTiles<w4::kF16>(p.w.group, a, s)
                                              : w4::LaunchTiles<w4::kBF16>(p.w.group, a, s);
    if (status != 0) return status;
  }
  return 0;
}

}  // extern "C"
