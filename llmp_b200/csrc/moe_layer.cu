// A whole mixture-of-experts layer for 1 to 16 tokens in two kernels: the router's product, the
// scores, each token's choice of experts and their weights, every named expert's gate | up product
// with the GLU over 4-bit weights (w4.cuh), the down product, and the weighted sum.  Beside
// moe_decode.cu, which takes the choice from elsewhere and Q4_K experts.
//
// Everything before the experts' products depends on all of the router's output, a meeting of the
// whole grid; here every cluster of eight CTAs works the router's product out for itself, a CTA an
// eighth of the experts, and meets through its own hardware barrier: 0.5 MB of router weights from
// L2 a cluster instead of a kernel of its own or a grid barrier, and no counter that two calls
// could share.  Then every CTA knows the choice and takes its share of (expert, tile) units.
// What bounds it, 128 experts, top 8, 2048 x 768: one bf16 token 22 us, of which the first kernel's way to the choice is 8
// (staging, the router's rows through one SM's share of L2, two cluster barriers, the picks one after the other),
// its products 5 and the second kernel 7; sixteen tokens 102 us for 211 MB, issue slots 56 and 70 % full, 250 and 330
// instructions a warp and step of 1.1 KB where the product's own are about 120: the rest is a round's or item's share of
// addresses and meetings, as a warp's run is four steps and three.  The MMAs' columns that stand for no token read the
// first one's values (sixteen bf16 tokens 106.5 us; zeros of their own 107.4, eight F16 tokens 77.8 and 79.8).
// The second kernel's CTA owns 16 output rows and adds a token's experts up in slot order, so a
// token's sums do not depend on the other tokens of the call.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "w4.cuh"

namespace llmp_b200 {
namespace {

namespace cg = cooperative_groups;
using namespace w4;

constexpr int kWarps = 16, kReducers = 2;          // of the first kernel: that multiply, that add up
constexpr int kThreads = (kWarps + kReducers) * 32;
constexpr int kSlots = 4, kSecondSlots = 6;        // steps a warp's ring of the first and the second kernel holds (six in the
                                                   // first: sixteen bf16 tokens 106 us, not 104)
// CTAs of a cluster of the first kernel.  (Of four, more SMs hold one, but each CTA works twice as much of the router out: five F32
// tokens of 60 experts 38.7 us, not 31.1; sixteen bf16 tokens of 128 experts 104 and 104.)
constexpr int kCluster = 8;
constexpr int kMaxTokens = 16, kMaxUsed = 16, kMaxExperts = 512;
constexpr int kMaxPairs = kMaxTokens * kMaxUsed;
constexpr int kFirstSmemLimit = 211 * 1024;        // dynamic; the choice's lists are static (one token of 16384 F32
                                                   // values, 16 x 512 logits and rings of groups of 32 fit)

// The choice as the first kernel leaves it for the second: groups of tokens that name one expert, experts in ascending
// order, a group's (token, slot) pairs (t * used + j, in token order) being pairs[first[i]] .. pairs[first[i + 1] - 1].
// A group holds no more tokens than GroupTokens: an expert that more name has several, whose weights come from L2 again.
struct Choice {
  std::int32_t groups;
  std::int32_t expert[kMaxPairs], first[kMaxPairs + 1], pairs[kMaxPairs];
};

struct LayerArgs {
  const void* x;
  std::int64_t x_stride;
  bool x_vec, router_vec;
  const void* router;
  std::int64_t router_stride;
  int router_type;
  const float* bias;
  int score, renormalize;
  float scale;
  const std::uint8_t* gate_up;
  const std::uint8_t* down;
  int experts, used, tokens, hidden, inter;
  int tiles_up, steps_up, tiles_down, steps_down;
  int glu;
  float limit;
  void* y;
  std::int64_t y_stride;
  int y_type;
  std::int32_t* ids;
  float* weights;
  Choice* choice;
  unsigned short* h;  // bf16 pieces of the GLU rows: [pair][piece][inter]
  int glu_pieces;     // of them, 2 or 3
  int cap;            // tokens staged at a time
  int group_cap;      // tokens of a group
  int x_pitch;        // bytes of a staged piece of a token
  int router_rows;    // experts of a router tile: 16, or 8 of an F32 router where 16 would leave CTAs of the cluster without one
  int parts;          // warps that divide a tile's steps of hidden
  int round_tiles;    // tiles that a round's warps work on
};

// Tokens of a group, and the column tiles that they take in the products, in registers: one or two (four in the second kernel
// where 16-bit activations have an F32 output).
__host__ __device__ constexpr int GroupTokens(int type) { return type == kF32 ? 4 : 8; }
__host__ __device__ constexpr int GroupTiles(int tokens, int pieces) { return (tokens + TokensATile(pieces) - 1) / TokensATile(pieces); }
// bf16 pieces that a GLU value travels in between the kernels.  Three hold all 24 bits of its F32 form: where activations or
// output are F32.  Two, each rounded to nearest, are within 2^-17 of it, which a 16-bit output rounds away (half its
// step is 2^-9 or 2^-12): four tokens instead of two fill an MMA's columns (sixteen bf16 tokens, 128 experts, top 8,
// 2048 x 768: 106 us, with three pieces 120; one token 22.8 and 24.0).
constexpr int GluPieces(int x_type, int y_type) { return x_type == kF32 || y_type == kF32 ? 3 : 2; }
// The two: a first that would round to infinity is cut off, the second then holds the rest.
__device__ __forceinline__ void SplitNearest(float x, std::uint32_t (&bits)[2]) {
  const std::uint32_t b = __float_as_uint(x), magnitude = b & 0x7fffffffu;
  if (magnitude >= 0x7f800000u) {
    Split<2>(x, bits);
    return;
  }
  std::uint32_t first = magnitude + 0x7fffu + ((magnitude >> 16) & 1u);
  if (first >= 0x7f800000u) first = magnitude;
  first = (first | (b & 0x80000000u)) & 0xffff0000u;
  bits[0] = first >> 16;
  bits[1] = __bfloat16_as_ushort(__float2bfloat16_rn(x - __uint_as_float(first)));
}

// Unsigned order of floats: NaN below everything, the two zeros alike; 0 is no float's.
__device__ __forceinline__ std::uint32_t OrderKey(float v) {
  if (v != v) return 1u;
  const std::uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

struct FirstShared {
  std::int32_t ids[kMaxPairs];
  float weights[kMaxPairs];
  std::uint32_t mask[kMaxExperts];  // tokens that name the expert
  std::int32_t start[kMaxExperts];
  std::int32_t token[kMaxPairs];    // of choice.pairs
  std::int32_t chunk[kMaxExperts / 32];
  Choice choice;
};

// Dynamic shared memory of the first kernel: the rings (before the products: the router's partial sums), two buffers of partial sums, the staged tokens, logits.
struct FirstLayout {
  int ring, meet, staged, logits, bytes;
  __host__ __device__ FirstLayout(int block_bytes, int cap, int group_cap, int pieces, int x_pitch, int tokens, int experts) {
    ring = kWarps * kSlots * block_bytes;
    const int before = kWarps * kTileRows * kMaxTokens * 8;
    if (ring < before) ring = (before + 255) / 256 * 256;
    meet = ring;
    staged = meet + (2 * kWarps * kTileRows * group_cap * 4);
    logits = staged + (cap * pieces * x_pitch);
    bytes = logits + (tokens * experts * 4);
  }
};

// 16 experts' logits for the staged tokens over this warp's share of hidden.  Products of two bf16 pieces are
// exact; kBatch blocks of 32 values are in flight together and added in F32, the batches in 64 bits, because the choice
// compares values that may lie next to each other.
template <int kType, int kRouter, int kTiles>
__device__ __forceinline__ void RouterTile(const LayerArgs& a, const std::uint8_t* smem, int staged, int first_expert,
                                           int first_tile, int tokens, int warp, int lane,
                                           double (&partial)[kTileRows][kMaxTokens]) {
  constexpr int kPieces = BfloatPieces(kType), kRouterPieces = BfloatPieces(kRouter);
  constexpr int kBatch = kRouter == kF16 ? 2 : 4;
  const int g = lane >> 2, t = lane & 3;
  const int piece = g % Cols(kPieces);
  double total[kTiles][4];
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) total[nt][0] = total[nt][1] = total[nt][2] = total[nt][3] = 0.0;
  int column[kTiles];
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) {
    const int token = ((first_tile + nt) * TokensATile(kPieces)) + (g / Cols(kPieces));
    const int c = token < tokens && piece < kPieces ? (token * kPieces) + piece : 0;  // (a column that nobody reads)
    column[nt] = staged + (c * a.x_pitch) + (t * 16);
  }
  const int row_a = first_expert + g, row_b = a.router_rows == 16 ? row_a + 8 : a.experts;
  const auto* base = static_cast<const std::uint8_t*>(a.router);
  const std::int64_t row_bytes = a.router_stride * TypeBytes(kRouter);
  const int blocks = a.hidden / 32, end = (warp + 1) * blocks / kWarps;
  auto load = [&](int row, int block, uint4 (&quads)[kRouterPieces]) {
    const int at = (32 * block) + (8 * t), valid = block < end && row < a.experts ? 8 : 0;
    const std::uint8_t* p = base + (row * row_bytes);
    if (kRouter == kBF16 && a.router_vec && valid == 8) {
      quads[0] = *reinterpret_cast<const uint4*>(p + (at * 2));
    } else {
      LoadBfloat8<kRouter>(p, at, valid, a.router_vec, quads);
    }
  };
  for (int first = warp * blocks / kWarps; first < end; first += kBatch) {
    uint4 qa[kBatch][kRouterPieces], qb[kBatch][kRouterPieces];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      load(row_a, first + q, qa[q]);  // (zero from the share's end on)
      load(row_b, first + q, qb[q]);
    }
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
#pragma unroll
      for (int r = 0; r < kRouterPieces; ++r) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          const uint4 x = first + q < end ? *reinterpret_cast<const uint4*>(smem + column[nt] + ((first + q) * 64))
                                          : make_uint4(0, 0, 0, 0);
          Mma<false, false>(sum, qa[q][r].x, qb[q][r].x, qa[q][r].y, qb[q][r].y, x.x, x.y);
          Mma<false, false>(sum, qa[q][r].z, qb[q][r].z, qa[q][r].w, qb[q][r].w, x.z, x.w);
        }
        // an infinity is its first piece alone: zeros times it in the sums of other pieces are no part of the product
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const bool first_pieces = r == 0 && ((2 * t) + (c & 1)) % Cols(kPieces) == 0;
          if (first_pieces || isfinite(sum[c])) total[nt][c] += sum[c];
        }
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) {
    double v[2][2];
    if (kPieces == 3 && (t & 1) != 0) total[nt][1] = total[nt][3] = 0.0;  // the fourth column stands for nothing
    if constexpr (kPieces == 1) {
      v[0][0] = total[nt][0], v[0][1] = total[nt][1], v[1][0] = total[nt][2], v[1][1] = total[nt][3];
    } else {
      v[0][0] = total[nt][0] + total[nt][1];
      v[1][0] = total[nt][2] + total[nt][3];
      v[0][1] = v[1][1] = 0.0;
      if constexpr (kPieces == 3) {
#pragma unroll
        for (int r = 0; r < 2; ++r) v[r][0] += __shfl_xor_sync(0xffffffffu, v[r][0], 1);
      }
    }
#pragma unroll
    for (int j = 0; j < (kPieces == 1 ? 2 : 1); ++j) {
      const int token = ((first_tile + nt) * TokensATile(kPieces)) + TokenOf<kPieces>(t, j);
      if (token < tokens) {
        partial[g][token] = v[0][j];
        partial[g + 8][token] = v[1][j];
      }
    }
  }
}

// The same of an F32 router for kFew tokens at a time on the multiply-add pipes (the staged
// tokens c_first ..., x's first + c_first ...): a 16-bit value's pieces are joined again, a lane's 8 products are added in F32, those sums in 64 bits.  (On the tensor core the router would have to be split in
// three; that alone took 4 K cycles, the whole of this 5 K with one token.)
constexpr int kFew = 8;
template <int kType>
__device__ __forceinline__ void RouterFew(const LayerArgs& a, const std::uint8_t* smem, int staged, int first_expert,
                                          int first, int c_first, int tokens, int warp, int lane, double (&partial)[kTileRows][kMaxTokens]) {
  constexpr int kPieces = BfloatPieces(kType), kRouter = kF32;
  constexpr int kBatch = 2;
  const int g = lane >> 2, t = lane & 3;
  double total[2][kFew];
#pragma unroll
  for (int c = 0; c < kFew; ++c) total[0][c] = total[1][c] = 0.0;
  const int row_a = first_expert + g, row_b = a.router_rows == 16 ? row_a + 8 : a.experts;
  const auto* base = static_cast<const std::uint8_t*>(a.router);
  const std::int64_t row_bytes = a.router_stride * TypeBytes(kRouter);
  const int blocks = a.hidden / 32, end = (warp + 1) * blocks / kWarps;
  for (int block = warp * blocks / kWarps; block < end; block += kBatch) {
    float va[kBatch][8], vb[kBatch][8];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      const int at = (32 * (block + q)) + (8 * t);
      Load8<kRouter>(base + (row_a * row_bytes), at, block + q < end && row_a < a.experts ? 8 : 0, a.router_vec, va[q]);
      Load8<kRouter>(base + (row_b * row_bytes), at, block + q < end && row_b < a.experts ? 8 : 0, a.router_vec, vb[q]);
    }
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      if (block + q >= end) break;
      auto multiply = [&](const float (&v)[8], int c) {
        float sum_a = 0.0f, sum_b = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum_a = fmaf(va[q][i], v[i], sum_a);
          sum_b = fmaf(vb[q][i], v[i], sum_b);
        }
        total[0][c] += sum_a;
        total[1][c] += sum_b;
      };
      if constexpr (kType == kF32) {
        // from L1, where staging left them, four tokens' loads in flight: cheaper than joining three pieces
#pragma unroll
        for (int c4 = 0; c4 < kFew; c4 += 4) {
          if (c_first + c4 >= tokens) break;
          float v[4][8];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const std::int64_t token = first + min(c_first + c4 + c, tokens - 1);
            Load8<kF32>(static_cast<const float*>(a.x) + (token * a.x_stride), (32 * (block + q)) + (8 * t), 8, a.x_vec, v[c]);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) multiply(v[c], c4 + c);
        }
      } else {
#pragma unroll
        for (int c = 0; c < kFew; ++c) {
          if (c_first + c >= tokens) break;
          uint4 x[kPieces];
#pragma unroll
          for (int s = 0; s < kPieces; ++s) {
            x[s] = *reinterpret_cast<const uint4*>(smem + staged + ((((c_first + c) * kPieces) + s) * a.x_pitch) + ((block + q) * 64) + (t * 16));
          }
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (int s = kPieces - 1; s >= 0; --s) {
              const std::uint32_t w = i < 2 ? x[s].x : i < 4 ? x[s].y : i < 6 ? x[s].z : x[s].w;
              v[i] += __uint_as_float((i & 1) != 0 ? w & 0xffff0000u : w << 16);
            }
          }
          multiply(v, c);
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < kFew; ++c) {
    if (c_first + c >= tokens) break;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      double v = total[r][c];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (t == 0) partial[g + (8 * r)][c_first + c] = v;
    }
  }
}

// Tokens token_of(0 .. count - 1) of x as pieces in shared memory, by threads tid, tid + threads, ...
template <int kType, typename Token>
__device__ __forceinline__ void StageTokens(const LayerArgs& a, std::uint8_t* staged, int count, int tid, int threads,
                                            Token token_of) {
  constexpr int kPieces = BfloatPieces(kType);
  const int octets = a.steps_up * (kStep / 8);
  for (int n = tid; n < count * octets; n += threads) {
    const int c = n / octets, i = n - (c * octets);
    const auto* row = static_cast<const std::uint8_t*>(a.x) + (token_of(c) * a.x_stride * TypeBytes(kType));
    std::uint8_t* out = staged + ((c * kPieces) * a.x_pitch) + (i * 16);
    if constexpr (kType == kBF16) {
      Stage8(out, row, i * 8, a.hidden - (i * 8), a.x_vec);
    } else {
      uint4 quads[kPieces];
      LoadBfloat8<kType>(row, i * 8, a.hidden - (i * 8), a.x_vec, quads);
#pragma unroll
      for (int s = 0; s < kPieces; ++s) *reinterpret_cast<uint4*>(out + (s * a.x_pitch)) = quads[s];
    }
  }
  CopyAsyncCommit();
}

// A warp: token t's experts, best first, and their weights from its logits.  A lane holds the order keys of experts
// lane, lane + 32, ...: each round the warp's largest key, then its lowest index, is taken and struck out.
template <int kPer>
__device__ __forceinline__ void Choose(const LayerArgs& a, const float* row, int t, int lane, FirstShared& s) {
  const bool softmax = a.score == LLMP_B200_SCORE_SOFTMAX;
  const float kMinusInf = __uint_as_float(0xff800000u);
  float logit[kPer];
  float top = kMinusInf, total = 1.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + (32 * i);
    logit[i] = e < a.experts ? row[e] : kMinusInf;
    top = fmaxf(top, logit[i]);
  }
  if (softmax) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (lane + (32 * i) < a.experts) total += expf(logit[i] - top);  // a NaN makes it one
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  auto score = [&](float l) { return softmax ? expf(l - top) / total : 1.0f / (1.0f + expf(-l)); };
  std::uint32_t keys[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int e = lane + (32 * i);
    keys[i] = e < a.experts ? OrderKey(a.bias == nullptr ? logit[i] : score(logit[i]) + a.bias[e]) : 0u;
  }
  int mine = 0;
  for (int j = 0; j < a.used; ++j) {
    std::uint32_t best = 0;
    int at_i = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (keys[i] > best) best = keys[i], at_i = i;
    }
    const std::uint32_t most = __reduce_max_sync(0xffffffffu, best);
    const unsigned int taken = __reduce_min_sync(0xffffffffu, best == most ? static_cast<unsigned>(lane + (32 * at_i)) : 0x7fffffffu);
    if (lane == j) mine = static_cast<int>(taken);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (taken == static_cast<unsigned>(lane + (32 * i))) keys[i] = 0;
    }
  }
  const float p = lane < a.used ? score(row[mine]) : 0.0f;
  float sum = p;
  if (a.renormalize != 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if (lane < a.used) {
    s.ids[(t * a.used) + lane] = mine;
    s.weights[(t * a.used) + lane] = (a.renormalize != 0 ? p / sum : p) * a.scale;
    atomicOr(&s.mask[mine], 1u << t);
  }
}

template <int kType, int kGroups>
__global__ void __launch_bounds__(kThreads, 1)
FirstKernel(const LayerArgs a) {
  constexpr int kPieces = BfloatPieces(kType);
  constexpr int kTiles = GroupTiles(GroupTokens(kType), kPieces);
  constexpr int kBlock = BlockBytes(kStep / kGroups);
  extern __shared__ __align__(128) std::uint8_t smem[];
  __shared__ FirstShared s;
  const FirstLayout at(kBlock, a.cap, a.group_cap, kPieces, a.x_pitch, a.tokens, a.experts);
  std::uint8_t* staged = smem + at.staged;
  float* logits = reinterpret_cast<float*>(smem + at.logits);
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank()), ranks = static_cast<int>(cluster.num_blocks());
  GridLaunchDependents();
  const int round_tiles = a.round_tiles, tile_warps = kWarps / round_tiles;
  const int rounds_a_group = (a.tiles_up + round_tiles - 1) / round_tiles;
  const int my_tile = warp / tile_warps, part = warp % tile_warps;
  const int begin = part < a.parts ? a.steps_up * part / a.parts : 0;
  const int steps = part < a.parts ? (a.steps_up * (part + 1) / a.parts) - begin : 0;
  const int router_rows = a.router_rows, expert_tiles = (a.experts + router_rows - 1) / router_rows;
  {  // this CTA's router rows into L2 while the kernel before ends
    const std::size_t row_bytes = static_cast<std::size_t>(a.hidden) * TypeBytes(a.router_type);
    const int lines = static_cast<int>((row_bytes + 127) / 128);
    for (int m = rank; m < expert_tiles; m += ranks) {
      for (int i = tid; i < router_rows * lines; i += kThreads) {
        const int e = (m * router_rows) + (i / lines);
        if (e < a.experts) {
          asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const std::uint8_t*>(a.router) +
                                                       (e * a.router_stride * TypeBytes(a.router_type)) + ((i % lines) * 128)));
        }
      }
    }
  }
  for (int e = tid; e < a.experts; e += kThreads) s.mask[e] = 0;
  GridDependencyWait();

  // ---- the router's product: a tile of 8 or 16 experts at a time, CTA rank r the tiles r, r + 8, ...
  auto* partial = reinterpret_cast<double(*)[kTileRows][kMaxTokens]>(smem);
  bool met = false;
  for (int first = 0; first < a.tokens; first += a.cap) {
    const int count = min(a.cap, a.tokens - first);
    if (first > 0) __syncthreads();
    StageTokens<kType>(a, staged, count, tid, kThreads, [&](int c) { return static_cast<std::int64_t>(first + c); });
    CopyAsyncWait<0>();
    __syncthreads();
    for (int m = rank; m < expert_tiles; m += ranks) {
      if (warp < kWarps) {
        auto multiply = [&](auto router) {
          constexpr int kRouter = decltype(router)::value;
          if constexpr (kRouter == kF32) {  // by its type alone: a token's logits stay the same whatever its company
            for (int c = 0; c < count; c += kFew) {
              RouterFew<kType>(a, smem, at.staged, m * router_rows, first, c, count, warp, lane, partial[warp]);
            }
          } else {
          constexpr int kAtOnce = kTiles < 2 ? kTiles : 2;
          const int tiles = (count + TokensATile(kPieces) - 1) / TokensATile(kPieces);
          for (int nt = 0; nt < tiles; nt += kAtOnce) {
            RouterTile<kType, kRouter, kAtOnce>(a, smem, at.staged, m * router_rows, nt, count, warp, lane, partial[warp]);
          }
          }
        };
        if (a.router_type == kF32) {
          multiply(std::integral_constant<int, kF32>{});
        } else if (a.router_type == kF16) {
          multiply(std::integral_constant<int, kF16>{});
        } else {
          multiply(std::integral_constant<int, kBF16>{});
        }
      }
      __syncthreads();
      if (!met) cluster.sync();  // every CTA of the cluster has begun: its shared memory may be written
      met = true;
      // eight threads a logit: each adds two warps' sums, all of them up in a fixed order, each stores to a rank
      for (int first_i = 0; first_i < 16 * count * 8; first_i += kThreads) {
        const int i = first_i + tid, q = i % 8, row = (i / 8) % 16, c = (i / 8) / 16, e = (m * router_rows) + row;
        double sum = 0.0;
        if (c < count) sum = partial[2 * q][row][c] + partial[(2 * q) + 1][row][c];
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (c < count && q < ranks && row < router_rows && e < a.experts) {
          cluster.map_shared_rank(logits, q)[((first + c) * a.experts) + e] = static_cast<float>(sum);
        }
      }
      __syncthreads();
    }
  }
  if (!met) cluster.sync();
  cluster.sync();  // the cluster's logits are in every CTA

  // ---- the choice, the same in every CTA
  if (warp < a.tokens) {
    const float* row = logits + (warp * a.experts);
    if (a.experts <= 128) {
      Choose<4>(a, row, warp, lane, s);
    } else {
      Choose<kMaxExperts / 32>(a, row, warp, lane, s);
    }
  }
  __syncthreads();
  const int pairs = a.tokens * a.used;
  // warp w looks at experts 32 w .. + 31: how many pairs and groups come before each
  {
    const int e = tid;
    const int count = warp < kMaxExperts / 32 && e < a.experts ? __popc(s.mask[e]) : 0;
    const int pieces = (count + a.group_cap - 1) / a.group_cap;
    int packed = count | (pieces << 16);  // each at most 256 in all
    const int own = packed;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int below = __shfl_up_sync(0xffffffffu, packed, o);
      if (lane >= o) packed += below;
    }
    if (lane == 31 && warp < kMaxExperts / 32) s.chunk[warp] = packed;
    __syncthreads();
    int before = packed - own;
    for (int w = 0; w < warp && w < kMaxExperts / 32; ++w) before += s.chunk[w];
    if (count > 0) {
      const int begin = before & 0xffff, group = before >> 16;
      s.start[e] = begin;
      for (int q = 0; q < pieces; ++q) {
        s.choice.expert[group + q] = e;
        s.choice.first[group + q] = begin + (q * a.group_cap);
      }
    }
    if (tid == kMaxExperts - 1) {
      const int all = before + own;
      s.choice.groups = all >> 16;
      s.choice.first[all >> 16] = all & 0xffff;
    }
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kThreads) {
    const int e = s.ids[p], t = p / a.used;
    const int place = s.start[e] + __popc(s.mask[e] & ((1u << t) - 1u));
    s.choice.pairs[place] = p;
    s.token[place] = t;
  }
  __syncthreads();

  // ---- this CTA's rounds: a group's next tiles of 8 gate and 8 up rows, each divided among a few warps
  // (a division is some 150 cycles of everyone's latency here: these two, the rest before the dependency wait)
  const unsigned int rounds = static_cast<unsigned int>(s.choice.groups * rounds_a_group);
  const unsigned int quota = rounds / gridDim.x, extra = rounds - (quota * gridDim.x);
  const int first_round = static_cast<int>((quota * blockIdx.x) + min(blockIdx.x, extra));
  const int end_round = first_round + static_cast<int>(quota + (blockIdx.x < extra ? 1u : 0u));
  const int first_group = static_cast<int>(static_cast<unsigned int>(first_round) / static_cast<unsigned int>(rounds_a_group));
  const int first_pair = first_round - (first_group * rounds_a_group);
  const bool all_staged = a.tokens <= a.cap;
  float* meet = reinterpret_cast<float*>(smem + at.meet);
  const int meet_floats = kWarps * kTileRows * a.group_cap;
  if (warp < kWarps) {
    std::uint8_t* ring = smem + (warp * kSlots * kBlock);
    // where the next request reads
    int load_group = first_group, load_pair = first_pair;
    int load_rounds = steps > 0 ? end_round - first_round : 0, load_left = 0;
    const std::uint8_t* src = nullptr;
    const std::size_t tile_bytes = static_cast<std::size_t>(a.steps_up) * kBlock;
    auto next_load_round = [&]() {  // the next round in which this warp has a tile
      while (load_left == 0 && load_rounds > 0) {
        const int tile = (load_pair * round_tiles) + my_tile;
        if (load_pair == 0 || src == nullptr) {
          src = a.gate_up + ((static_cast<std::size_t>(s.choice.expert[load_group]) * a.tiles_up) + tile) * tile_bytes +
                (static_cast<std::size_t>(begin) * kBlock) + (lane * 16);
        } else {
          src += (round_tiles * tile_bytes) - (static_cast<std::size_t>(steps) * kBlock);
        }
        if (tile < a.tiles_up) load_left = steps;
        --load_rounds;
        if (++load_pair == rounds_a_group) load_pair = 0, ++load_group;
      }
    };
    auto request = [&](int slot) {  // one commit a call, so that the waits can count
      if (load_left == 0) next_load_round();
      if (load_left > 0) {
        const std::uint32_t dst = SharedAddress(ring) + (slot * kBlock) + (lane * 16);
        CopyAsync16<0>(dst, src);
        CopyAsync16<512>(dst, src);
        if (lane < 4 * kGroups) CopyAsync16<1024>(dst, src);
        --load_left;
        src += kBlock;
      }
      CopyAsyncCommit();
    };
#pragma unroll
    for (int i = 0; i < kSlots - 1; ++i) request(i);
    const int piece = g % Cols(kPieces);
    int group = first_group, pair = first_pair;
    int slot = 0, buffer = 0, staged_group = -1, column_group = -1, tiles = 1;
    std::uint32_t column[kTiles];
    for (int round = first_round; round < end_round; ++round, buffer ^= 1) {
      const int first = s.choice.first[group], count = s.choice.first[group + 1] - first;
      if (!all_staged && staged_group != group) {
        if (staged_group >= 0) BarrierSync(5, kWarps * 32);
        StageTokens<kType>(a, staged, count, tid, kWarps * 32, [&](int c) { return static_cast<std::int64_t>(s.token[first + c]); });
        CopyAsyncWait<0>();
        BarrierSync(5, kWarps * 32);
        staged_group = group;
      }
      if (column_group != group) {
        column_group = group;
        tiles = (count + TokensATile(kPieces) - 1) / TokensATile(kPieces);
#pragma unroll
        for (int nt = 0; nt < kTiles; ++nt) {
          const int c = (nt * TokensATile(kPieces)) + (g / Cols(kPieces));
          int row = 0;  // (a column that nobody reads)
          if (c < count && piece < kPieces) row = ((all_staged ? s.token[first + c] : c) * kPieces) + piece;
          column[nt] = at.staged + (row * a.x_pitch) + (t4 * 16) + (begin * 256);
        }
      }
      Sums total[kTiles];
      if ((pair * round_tiles) + my_tile < a.tiles_up) {
        for (int step = 0; step < steps; ++step) {
          CopyAsyncWait<kSlots - 2>();
          __syncwarp();  // all lanes' copies of this step are in, and the slot before it has been read
          request(slot == 0 ? kSlots - 1 : slot - 1);
          StepWeights<kGroups> w;
          w.LoadShared(smem + (((warp * kSlots) + slot) * kBlock), lane);
          MultiplyStep<false, kGroups, kTiles>(w, tiles, total, [&](int nt, int i) {
            return *reinterpret_cast<const uint4*>(smem + column[nt] + (step * 256) + (i * 64));
          });
          slot = slot == kSlots - 1 ? 0 : slot + 1;
        }
      }
      // barriers 1, 2: buffer 0, 1 holds a round's sums; 3, 4: it may be written again
      if (round - first_round >= 2) BarrierSync(3 + buffer, kThreads);
      float* mine = meet + (buffer * meet_floats) + (warp * kTileRows * a.group_cap);
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
        if (nt >= tiles) break;
        float v[2][2];
        FoldColumns<false, kPieces>(total[nt], v);
#pragma unroll
        for (int j = 0; j < (kPieces == 1 ? 2 : 1); ++j) {
          const int c = (nt * TokensATile(kPieces)) + TokenOf<kPieces>(t4, j);
          if (c < count) {
            mine[(c * kTileRows) + g] = v[0][j];
            mine[(c * kTileRows) + g + 8] = v[1][j];
          }
        }
      }
      BarrierArrive(1 + buffer, kThreads);
      if (++pair == rounds_a_group) pair = 0, ++group;
    }
  } else {
    if (blockIdx.x == 0) {  // the choice for the caller and the second kernel
      for (int p = tid - (kWarps * 32); p < pairs; p += kReducers * 32) {
        a.ids[p] = s.ids[p];
        a.weights[p] = s.weights[p];
        a.choice->pairs[p] = s.choice.pairs[p];
      }
      for (int i = tid - (kWarps * 32); i < s.choice.groups; i += kReducers * 32) a.choice->expert[i] = s.choice.expert[i];
      for (int i = tid - (kWarps * 32); i <= s.choice.groups; i += kReducers * 32) a.choice->first[i] = s.choice.first[i];
      if (tid == kWarps * 32) a.choice->groups = s.choice.groups;
    }
    // a warp every other tile of the round; a lane a row of every fourth token
    const int row = lane & 7;
    int group = first_group, pair = first_pair, buffer = 0;
    for (int round = first_round; round < end_round; ++round, buffer ^= 1) {
      BarrierSync(1 + buffer, kThreads);
      const int first = s.choice.first[group], count = s.choice.first[group + 1] - first;
      for (int tile = warp - kWarps; tile < round_tiles; tile += kReducers) {
        const int out = (((pair * round_tiles) + tile) * 8) + row;
        const float* p = meet + (buffer * meet_floats) + (tile * tile_warps * kTileRows * a.group_cap) + row;
        for (int c = lane >> 3; c < count && out < a.inter; c += 4) {
          float gate = 0.0f, up = 0.0f;
#pragma unroll 4
          for (int q = 0; q < a.parts; ++q) {
            gate += p[((q * a.group_cap) + c) * kTileRows];
            up += p[(((q * a.group_cap) + c) * kTileRows) + 8];
          }
          const float value = GluOf(a.glu, gate * Up(false), up * Up(false), a.limit);
          const int glu_pieces = kType == kF32 ? 3 : a.glu_pieces;
          unsigned short* h = a.h + (static_cast<std::size_t>(s.choice.pairs[first + c]) * glu_pieces * a.inter) + out;
          auto store = [&](auto& bits) {
#pragma unroll
            for (std::uint32_t b : bits) *h = static_cast<unsigned short>(b), h += a.inter;
          };
          if (glu_pieces == 3) {
            std::uint32_t bits[3];
            Split<3>(value, bits);
            store(bits);
          } else {
            std::uint32_t bits[2];
            SplitNearest(value, bits);
            store(bits);
          }
        }
      }
      BarrierArrive(3 + buffer, kThreads);
      if (++pair == rounds_a_group) pair = 0, ++group;
    }
  }
}

// A CTA's 16 rows of the output: its warps take (group, half of inter) items in turn, their weights through rings as
// in the first kernel, the GLU rows straight from L2 a step ahead; each pair's sums meet in shared memory and
// a token's slots are added in order.
constexpr int kParts = 2;
constexpr int kSecondWarps = 16;

template <int kTokens, int kGlu, int kGroups>
__global__ void __launch_bounds__(kSecondWarps * 32, 1)
SecondKernel(const LayerArgs a) {
  constexpr int kTiles = GroupTiles(kTokens, kGlu);
  constexpr int kBlock = BlockBytes(kStep / kGroups);
  extern __shared__ __align__(128) std::uint8_t smem[];
  __shared__ Choice choice;
  const int threads = static_cast<int>(blockDim.x), warps = threads >> 5;
  auto* sums = reinterpret_cast<float*>(smem + (warps * kSecondSlots * kBlock));  // [pair][part][16 rows]
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  GridLaunchDependents();
  GridDependencyWait();
  const int tile = static_cast<int>(blockIdx.x), pairs = a.tokens * a.used;
  for (int i = tid; i < pairs; i += threads) {
    choice.expert[i] = __ldcg(&a.choice->expert[i]);   // (what is past the groups is not used)
    choice.pairs[i] = __ldcg(&a.choice->pairs[i]);
    choice.first[i] = __ldcg(&a.choice->first[i]);
  }
  if (tid == 0) choice.first[pairs] = __ldcg(&a.choice->first[pairs]);
  if (tid == threads - 1) choice.groups = __ldcg(&a.choice->groups);
  __syncthreads();
  const int items = choice.groups * kParts;
  const int piece = g % Cols(kGlu);
  auto step0_of = [&](int item) { return (item % kParts) * a.steps_down / kParts; };
  auto steps_of = [&](int item) { return (((item % kParts) + 1) * a.steps_down / kParts) - step0_of(item); };
  std::uint8_t* ring = smem + (warp * kSecondSlots * kBlock);
  int load_item = warp - warps, load_left = 0;
  const std::uint8_t* src = nullptr;
  auto request = [&](int slot) {
    while (load_left == 0 && load_item < items) {
      load_item += warps;
      if (load_item >= items) break;
      load_left = steps_of(load_item);
      src = a.down + ((((static_cast<std::size_t>(choice.expert[load_item / kParts]) * a.tiles_down) + tile) * a.steps_down) +
                      step0_of(load_item)) * kBlock + (lane * 16);
    }
    if (load_left > 0) {
      const std::uint32_t dst = SharedAddress(ring) + (slot * kBlock) + (lane * 16);
      CopyAsync16<0>(dst, src);
      CopyAsync16<512>(dst, src);
      if (lane < 4 * kGroups) CopyAsync16<1024>(dst, src);
      --load_left;
      src += kBlock;
    }
    CopyAsyncCommit();
  };
#pragma unroll
  for (int i = 0; i < kSecondSlots - 1; ++i) request(i);
  // the columns of an item's pairs: this lane's in each column tile
  struct Columns {
    const unsigned short* at[kTiles];
  };
  auto columns_of = [&](int item) {
    Columns columns;
    const int begin = choice.first[item / kParts], count = choice.first[(item / kParts) + 1] - begin;
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const int c = (nt * TokensATile(kGlu)) + (g / Cols(kGlu));
      const bool real = c < count && piece < kGlu;  // (a column that nobody reads is the first pair's)
      columns.at[nt] = a.h + (((static_cast<std::size_t>(choice.pairs[real ? begin + c : begin]) * kGlu) + (real ? piece : 0)) * a.inter) + (t4 * 8);
    }
    return columns;
  };
  auto fetch = [&](const unsigned short* column, int step, int b) {
    const int at = (step * kStep) + (32 * b);  // inter is whole 32-value blocks
    if (at >= a.inter) return make_uint4(0, 0, 0, 0);
    return __ldcg(reinterpret_cast<const uint4*>(column + at));
  };
  auto next_item = [&](int item) {  // with a step to it
    do {
      item += warps;
    } while (item < items && steps_of(item) == 0);
    return item;
  };
  int slot = 0, item = next_item(warp - warps);
  Columns columns = {};
  uint4 ahead[4];
  if (item < items) {
    columns = columns_of(item);
#pragma unroll
    for (int b = 0; b < 4; ++b) ahead[b] = fetch(columns.at[0], step0_of(item), b);
  }
  while (item < items) {
    const int begin = choice.first[item / kParts], count = choice.first[(item / kParts) + 1] - begin;
    const int step0 = step0_of(item), end = step0 + steps_of(item), after = next_item(item);
    const int tiles = (count + TokensATile(kGlu) - 1) / TokensATile(kGlu);
    Columns next = columns;
    Sums total[kTiles];
    for (int step = step0; step < end; ++step) {
      uint4 now[4];
#pragma unroll
      for (int b = 0; b < 4; ++b) now[b] = ahead[b];
      int ahead_step = step + 1;
      if (ahead_step == end && after < items) next = columns_of(after), ahead_step = step0_of(after);
      if (step + 1 < end || after < items) {
#pragma unroll
        for (int b = 0; b < 4; ++b) ahead[b] = fetch(next.at[0], ahead_step, b);
      }
      CopyAsyncWait<kSecondSlots - 2>();
      __syncwarp();
      request(slot == 0 ? kSecondSlots - 1 : slot - 1);
      StepWeights<kGroups> w;
      w.LoadShared(smem + (((warp * kSecondSlots) + slot) * kBlock), lane);
      MultiplyStep<false, kGroups, kTiles>(w, tiles, total, [&](int nt, int b) {
        return nt == 0 ? now[b] : fetch(columns.at[nt], step, b);
      });
      slot = slot == kSecondSlots - 1 ? 0 : slot + 1;
    }
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      if (nt >= tiles) break;
      float v[2][2];
      FoldColumns<false, kGlu>(total[nt], v);
      const int c = (nt * TokensATile(kGlu)) + TokenOf<kGlu>(t4, 0);
      if (c < count) {
        float* out = sums + (((choice.pairs[begin + c] * kParts) + (item % kParts)) * kTileRows);
        out[g] = v[0][0];
        out[g + 8] = v[1][0];
      }
    }
    item = after;
    columns = next;
  }
  if (a.steps_down < kParts) {  // the first part of a single step has none
    __syncthreads();
    for (int i = tid; i < pairs * kTileRows; i += threads) sums[((i / kTileRows) * kParts * kTileRows) + (i % kTileRows)] = 0.0f;
  }
  __syncthreads();
  for (int i = tid; i < a.tokens * kTileRows; i += threads) {
    const int t = i / kTileRows, r = i % kTileRows, row = (tile * kTileRows) + r;
    if (row >= a.hidden) continue;
    float y = 0.0f;
    for (int j = 0; j < a.used; ++j) {
      const float* p = sums + (((t * a.used) + j) * kParts * kTileRows) + r;
      y = fmaf(__ldcg(&a.weights[(t * a.used) + j]), (p[0] + p[kTileRows]) * Up(false), y);
    }
    StoreValue(a.y, (t * a.y_stride) + row, a.y_type, y);
  }
}

template <typename Kernel>
cudaError_t Configure(Kernel kernel, int& configured_device, int smem) {
  int device = -1;
  cudaGetDevice(&device);
  if (configured_device == device) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) configured_device = device;
  return e;
}

// Clusters of one first kernel that the device holds at once (a GPC holds whole clusters: more would be a second wave).
template <auto kKernel>
int ResidentClusters(int smem) {
  static thread_local int known_device = -1, known_smem = -1, known = 1;
  int device = -1;
  cudaGetDevice(&device);
  if (known_device == device && known_smem == smem) return known;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(SmCount() / kCluster * kCluster));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = static_cast<std::size_t>(smem);
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = kCluster;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  int clusters = 0;
  if (cudaOccupancyMaxActiveClusters(&clusters, kKernel, &config) != cudaSuccess || clusters < 1) {
    cudaGetLastError();
    clusters = std::max(1, SmCount() / (2 * kCluster));
  }
  known_device = device, known_smem = smem, known = clusters;
  return clusters;
}

template <int kType, int kGroups>
int LaunchFirst(const LayerArgs& a, cudaStream_t stream) {
  static thread_local int configured_device = -1;
  if (const cudaError_t e = Configure(FirstKernel<kType, kGroups>, configured_device, kFirstSmemLimit); e != cudaSuccess) {
    return Failed(e, "moe_layer attribute");
  }
  const int smem = FirstLayout(BlockBytes(kStep / kGroups), a.cap, a.group_cap, BfloatPieces(kType), a.x_pitch, a.tokens, a.experts).bytes;
  if (smem > kFirstSmemLimit) return Reject("moe_layer: %d bytes of shared memory", smem);
  const std::int64_t rounds = static_cast<std::int64_t>(std::min(a.experts, a.tokens * a.used)) *
                              ((a.tiles_up + a.round_tiles - 1) / a.round_tiles);
  const std::int64_t most = ResidentClusters<FirstKernel<kType, kGroups>>(smem);
  const std::int64_t clusters = std::max<std::int64_t>(1, std::min(most, (rounds + kCluster - 1) / kCluster));
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(clusters * kCluster));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = static_cast<std::size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = kCluster;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, FirstKernel<kType, kGroups>, a);
  return e == cudaSuccess ? 0 : Failed(e, "moe_layer launch");
}

template <int kTokens, int kGlu, int kGroups>
int LaunchSecond(const LayerArgs& a, cudaStream_t stream) {
  static thread_local int configured_device = -1;
  if (const cudaError_t e = Configure(SecondKernel<kTokens, kGlu, kGroups>, configured_device, 160 * 1024); e != cudaSuccess) {
    return Failed(e, "moe_layer attribute");
  }
  // Sixteen warps a tile while there are no more tiles than SMs, else eight, two CTAs an SM.  (Sixteen and eight, bf16: 128 tiles,
  // one token 21.3 and 23.1 us, sixteen 102 and 132; 256 tiles, one 26.7 and 22.4, sixteen 72 and 68.)
  const int warps = a.tiles_down <= SmCount() ? kSecondWarps : kSecondWarps / 2;
  const int smem = (warps * kSecondSlots * BlockBytes(kStep / kGroups)) + (a.tokens * a.used * kParts * kTileRows * 4);
  const cudaError_t e = LaunchPdl(SecondKernel<kTokens, kGlu, kGroups>, dim3(static_cast<unsigned>(a.tiles_down)),
                                  dim3(static_cast<unsigned>(warps * 32)), static_cast<std::size_t>(smem), stream, a);
  return e == cudaSuccess ? 0 : Failed(e, "moe_layer down launch");
}

template <int kType>
int LaunchLayer(int group_up, int group_down, const LayerArgs& a, cudaStream_t stream) {
  int status = group_up == 128  ? LaunchFirst<kType, 1>(a, stream)
               : group_up == 64 ? LaunchFirst<kType, 2>(a, stream)
                                : LaunchFirst<kType, 4>(a, stream);
  if (status != 0) return status;
  auto second = [&](auto pieces) {
    constexpr int kTokens = GroupTokens(kType), kGlu = decltype(pieces)::value;
    return group_down == 128  ? LaunchSecond<kTokens, kGlu, 1>(a, stream)
           : group_down == 64 ? LaunchSecond<kTokens, kGlu, 2>(a, stream)
                              : LaunchSecond<kTokens, kGlu, 4>(a, stream);
  };
  if constexpr (kType == kF32) {
    status = second(std::integral_constant<int, 3>{});
  } else {
    status = a.glu_pieces == 3 ? second(std::integral_constant<int, 3>{}) : second(std::integral_constant<int, 2>{});
  }
  return status > 0 ? -1 : status;  // the first kernel is queued
}

std::size_t ChoiceBytes() { return (sizeof(Choice) + 255) / 256 * 256; }

}  // namespace
}  // namespace llmp_b200

extern "C" {

size_t llmp_b200_moe_layer_scratch(int used, int tokens, int inter) {
  using namespace llmp_b200;
  if (used < 1 || used > kMaxUsed || tokens < 1 || tokens > kMaxTokens || inter < 1) return 0;
  return ChoiceBytes() + (static_cast<size_t>(used) * tokens * 3 * inter * 2);
}

int llmp_b200_moe_layer(const llmp_b200_moe_layer_desc* desc, void* stream) {
  using namespace llmp_b200;
  if (desc == nullptr) return Reject("moe_layer: null descriptor");
  const llmp_b200_moe_layer_desc& d = *desc;
  if (const int status = CheckMatrix(d.gate_up, "moe_layer gate_up"); status != 0) return status;
  if (const int status = CheckMatrix(d.down, "moe_layer down"); status != 0) return status;
  const int hidden = d.gate_up.k, inter = d.gate_up.n / 2, experts = d.gate_up.experts;
  if (d.gate_up.glu != 1 || d.down.glu != 0) return Reject("moe_layer: gate_up a GLU slab, down a plain one");
  if (d.down.n != hidden || d.down.k != inter || d.down.experts != experts) {
    return Reject("moe_layer: down [experts][hidden][inter] to gate_up [experts][2 inter][hidden]");
  }
  if (hidden > 16384 || inter > 65536 || experts > kMaxExperts) {
    return Reject("moe_layer: hidden up to 16384, inter up to 65536, up to 512 experts");
  }
  if (d.used < 1 || d.used > kMaxUsed || d.used > experts) return Reject("moe_layer: 1 to 16 experts a token, no more than there are");
  if (d.tokens == 0) return 0;
  if (d.tokens < 0 || d.tokens > kMaxTokens) return Reject("moe_layer: 1 to 16 tokens");
  if (d.x == nullptr || d.router == nullptr || d.y == nullptr || d.ids == nullptr || d.weights == nullptr || d.scratch == nullptr) {
    return Reject("moe_layer: activations, a router, an output, ids, weights and scratch");
  }
  if (!FloatType(d.x_type) || !FloatType(d.router_type) || !FloatType(d.y_type)) {
    return Reject("moe_layer: F32, F16 or BF16 activations, router and output");
  }
  if (d.glu < LLMP_B200_GLU_SWIGLU || d.glu > LLMP_B200_GLU_GEGLU) return Reject("moe_layer: a GLU");
  if (d.score != LLMP_B200_SCORE_SOFTMAX && d.score != LLMP_B200_SCORE_SIGMOID) return Reject("moe_layer: score %d", d.score);
  const int xb = TypeBytes(d.x_type), rb = TypeBytes(d.router_type);
  if (!Aligned(d.x, xb) || !Aligned(d.router, rb) || !Aligned(d.y, TypeBytes(d.y_type)) || !Aligned(d.bias, 4) ||
      !Aligned(d.ids, 4) || !Aligned(d.weights, 4) || !Aligned(d.scratch, 256) ||
      (d.tokens > 1 && (d.x_stride < hidden || d.y_stride < hidden)) || (experts > 1 && d.router_stride < hidden)) {
    return Reject("moe_layer: aligned rows at least hidden values apart, 256-byte aligned scratch");
  }
  if (const int status = DeviceStatus(); status != 0) return status;
  LayerArgs a{};
  a.x = d.x, a.x_stride = d.x_stride;
  a.x_vec = Aligned(d.x, 16) && (d.tokens == 1 || (d.x_stride * xb) % 16 == 0);
  a.router = d.router, a.router_stride = d.router_stride, a.router_type = d.router_type;
  a.router_vec = Aligned(d.router, 16) && (experts == 1 || (d.router_stride * rb) % 16 == 0);
  a.bias = d.bias, a.score = d.score, a.renormalize = d.renormalize, a.scale = d.scale;
  a.gate_up = static_cast<const std::uint8_t*>(d.gate_up.slab);
  a.down = static_cast<const std::uint8_t*>(d.down.slab);
  a.experts = experts, a.used = d.used, a.tokens = d.tokens, a.hidden = hidden, a.inter = inter;
  a.tiles_up = Tiles(d.gate_up.n, 1), a.steps_up = Steps(hidden);
  // (Tiles of 8 and 16: 60 experts in F32, five tokens 30.4 and 30.9 us; in bf16, one token, 32 experts of 2560 values 23.5 and 22.9, 64 of 1024
  // 14.8 and 14.4: an MMA has 16 rows either way.)
  a.router_rows = d.router_type == kF32 && experts <= 8 * kCluster ? 8 : 16;
  a.tiles_down = Tiles(d.down.n, 0), a.steps_down = Steps(inter);
  a.glu = d.glu, a.limit = d.limit;
  a.y = d.y, a.y_stride = d.y_stride, a.y_type = d.y_type;
  a.ids = d.ids, a.weights = d.weights;
  a.choice = static_cast<Choice*>(d.scratch);
  a.h = reinterpret_cast<unsigned short*>(static_cast<std::uint8_t*>(d.scratch) + ChoiceBytes());
  a.x_pitch = (a.steps_up * kStep * 2) + 64;
  // A warp's run of a tile is four steps and more where hidden allows it (each round costs a warp about two steps'
  // instructions besides), but a tile has at least four warps: few tokens name few tiles.  Not by the number of tokens:
  // a token's sums stay the same whatever its company.
  int tile_warps = 4;
  while (tile_warps < kWarps && a.steps_up >= 8 * tile_warps) tile_warps *= 2;
  a.round_tiles = kWarps / tile_warps;
  a.parts = std::min(tile_warps, a.steps_up);
  a.glu_pieces = GluPieces(d.x_type, d.y_type);
  a.cap = d.tokens;
  a.group_cap = std::min(d.tokens, GroupTokens(d.x_type));
  auto bytes = [&]() {
    return FirstLayout(BlockBytes(d.gate_up.group), a.cap, a.group_cap, BfloatPieces(d.x_type), a.x_pitch, d.tokens, experts).bytes;
  };
  while (a.cap > 1 && bytes() > kFirstSmemLimit) {
    --a.cap;
    a.group_cap = std::min(a.group_cap, a.cap);
  }
  const auto s = static_cast<cudaStream_t>(stream);
  if (d.x_type == kF32) return LaunchLayer<kF32>(d.gate_up.group, d.down.group, a, s);
  if (d.x_type == kF16) return LaunchLayer<kF16>(d.gate_up.group, d.down.group, a, s);
  return LaunchLayer<kBF16>(d.gate_up.group, d.down.group, a, s);
}

}  // extern "C"
