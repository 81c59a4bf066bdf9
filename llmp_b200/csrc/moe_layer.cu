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
// The second kernel's CTA owns 16 output rows and adds a token's experts up in slot order, so a
// token's sums do not depend on the other tokens of the call.
#include <cooperative_groups.h>

#include <algorithm>

#include "w4.cuh"

namespace llmp_b200 {
namespace {

namespace cg = cooperative_groups;
using namespace w4;

constexpr int kThreads = 256, kWarps = 8;
constexpr int kCluster = 8;
constexpr int kMaxTokens = 16, kMaxUsed = 16, kMaxExperts = 512;
constexpr int kMaxPairs = kMaxTokens * kMaxUsed;
constexpr int kXBudget = 100 * 1024;  // staged activations a CTA: two CTAs an SM

// The choice as the first kernel leaves it for the second: the named experts in ascending order, expert
// i's (token, slot) pairs (t * used + j, in token order) being pairs[first[i]] .. pairs[first[i + 1] - 1].
struct Choice {
  std::int32_t named;
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
  int cap;            // tokens staged at a time
  int x_pitch;        // bytes of a staged piece of a token
};

// Pieces of a GLU value: 16-bit activations keep 16 bits of it, F32 ones all 24.
__host__ __device__ constexpr int GluPieces(int type) { return type == kF32 ? 3 : 2; }

// Unsigned order of floats: NaN below everything, the two zeros alike; 0 is no float's.
__device__ __forceinline__ std::uint32_t OrderKey(float v) {
  if (v != v) return 1u;
  const std::uint32_t b = __float_as_uint(v + 0.0f);
  return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

struct FirstShared {
  double partial[kWarps][kTileRows][kMaxTokens];  // the router's; the units' as floats, twice
  std::int32_t ids[kMaxPairs];
  float weights[kMaxPairs];
  std::uint32_t mask[kMaxExperts];  // tokens that name the expert
  std::int32_t start[kMaxExperts];
  std::int32_t group_expert[kMaxPairs], group_first[kMaxPairs], group_count[kMaxPairs];
  std::int32_t groups;
  Choice choice;
};

// kPieces of the router's elements: 16 experts' logits for the staged tokens, this warp's share of
// hidden.  Products of two bf16 pieces are exact; a 32-value block's sum is F32 and the blocks are
// added in 64 bits, because the choice compares values that may lie next to each other.
template <int kType, int kRouter, int kTiles>
__device__ __forceinline__ void RouterTile(const LayerArgs& a, const std::uint8_t* staged, int first_expert, int tokens,
                                           int warp, int lane, double (&partial)[kTileRows][kMaxTokens]) {
  constexpr int kPieces = BfloatPieces(kType), kRouterPieces = BfloatPieces(kRouter);
  const int g = lane >> 2, t = lane & 3;
  const int piece = g % Cols(kPieces);
  const int tiles = (tokens + TokensATile(kPieces) - 1) / TokensATile(kPieces);
  double total[kTiles][4];
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) total[nt][0] = total[nt][1] = total[nt][2] = total[nt][3] = 0.0;
  const int blocks = a.hidden / 32;
  const int row_a = first_expert + g, row_b = row_a + 8;
  const auto* base = static_cast<const std::uint8_t*>(a.router);
  const std::int64_t row_bytes = a.router_stride * TypeBytes(kRouter);
  for (int b = warp * blocks / kWarps; b < (warp + 1) * blocks / kWarps; ++b) {
    uint4 qa[kRouterPieces], qb[kRouterPieces];
    const int at = (32 * b) + (8 * t);
    LoadBfloat8<kRouter>(base + (row_a * row_bytes), at, row_a < a.experts ? 8 : 0, a.router_vec, qa);
    LoadBfloat8<kRouter>(base + (row_b * row_bytes), at, row_b < a.experts ? 8 : 0, a.router_vec, qb);
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      if (nt >= tiles) break;
      const int token = (nt * TokensATile(kPieces)) + (g / Cols(kPieces));
      uint4 x = make_uint4(0, 0, 0, 0);
      if (token < tokens && piece < kPieces) {
        x = *reinterpret_cast<const uint4*>(staged + (((token * kPieces) + piece) * a.x_pitch) + (at * 2));
      }
#pragma unroll
      for (int r = 0; r < kRouterPieces; ++r) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        Mma<false, true>(sum, qa[r].x, qb[r].x, qa[r].y, qb[r].y, x.x, x.y);
        Mma<false, false>(sum, qa[r].z, qb[r].z, qa[r].w, qb[r].w, x.z, x.w);
#pragma unroll
        for (int c = 0; c < 4; ++c) total[nt][c] += sum[c];
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < kTiles; ++nt) {
    double v[2][2];
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
      const int token = (nt * TokensATile(kPieces)) + TokenOf<kPieces>(t, j);
      if (token < tokens) {
        partial[g][token] = v[0][j];
        partial[g + 8][token] = v[1][j];
      }
    }
  }
}

// Tokens token_of(0 .. count - 1) of x as pieces in shared memory.
template <int kType, typename Token>
__device__ __forceinline__ void StageTokens(const LayerArgs& a, std::uint8_t* staged, int count, Token token_of) {
  constexpr int kPieces = BfloatPieces(kType);
  const int padded = a.steps_up * kStep;
  for (int i = static_cast<int>(threadIdx.x); i < count * (padded / 8); i += kThreads) {
    const int c = i / (padded / 8), at = (i % (padded / 8)) * 8;
    uint4 quads[kPieces];
    const auto* row = static_cast<const std::uint8_t*>(a.x) + (token_of(c) * a.x_stride * TypeBytes(kType));
    LoadBfloat8<kType>(row, at, a.hidden - at, a.x_vec, quads);
#pragma unroll
    for (int s = 0; s < kPieces; ++s) {
      *reinterpret_cast<uint4*>(staged + (((c * kPieces) + s) * a.x_pitch) + (at * 2)) = quads[s];
    }
  }
}

// A warp: token t's experts, best first, and their weights from its logits.
__device__ __forceinline__ void Choose(const LayerArgs& a, float* logits, int t, int lane, FirstShared& s) {
  float* row = logits + (t * a.experts);
  float top = __uint_as_float(0xff800000u);
  for (int e = lane; e < a.experts; e += 32) top = fmaxf(top, row[e]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float total = 0.0f;
  bool bad = false;
  if (a.score == LLMP_B200_SCORE_SOFTMAX) {
    for (int e = lane; e < a.experts; e += 32) {
      bad = bad || row[e] != row[e];
      total += expf(row[e] - top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (__any_sync(0xffffffffu, bad)) total = __uint_as_float(0x7fc00000u);
  }
  auto score = [&](float l) {
    return a.score == LLMP_B200_SCORE_SOFTMAX ? expf(l - top) / total : 1.0f / (1.0f + expf(-l));
  };
  // a lane's best of its experts; the one that is taken is struck out and its lane looks again
  auto key_of = [&](int e) {
    return OrderKey(a.bias == nullptr ? row[e] : score(row[e]) + a.bias[e]);
  };
  std::uint32_t taken = 0;  // bit i: expert lane + 32 i
  std::uint32_t best = 0;
  int best_at = 0;
  auto look = [&]() {
    best = 0;
    for (int e = lane, i = 0; e < a.experts; e += 32, ++i) {
      if ((taken >> i) & 1u) continue;
      const std::uint32_t k = key_of(e);
      if (k > best) best = k, best_at = e;
    }
  };
  look();
  float sum = 0.0f, mine = 0.0f;
  for (int j = 0; j < a.used; ++j) {
    const std::uint32_t most = __reduce_max_sync(0xffffffffu, best);
    const int at = static_cast<int>(__reduce_min_sync(0xffffffffu, best == most ? static_cast<unsigned>(best_at) : 0x7fffffffu));
    const float p = score(row[at]);
    sum += p;
    if (lane == j) mine = p;
    if (lane == 0) s.ids[(t * a.used) + j] = at;
    if ((at & 31) == lane) {
      taken |= 1u << (at >> 5);
      look();
    }
  }
  if (lane < a.used) {
    const float w = a.renormalize != 0 ? mine / sum : mine;
    s.weights[(t * a.used) + lane] = w * a.scale;
  }
}

template <int kType, int kGroups>
__global__ void __launch_bounds__(kThreads)
FirstKernel(const LayerArgs a) {
  constexpr int kPieces = BfloatPieces(kType);
  constexpr int kTiles = kMaxTokens / TokensATile(kPieces);
  constexpr int kBlock = BlockBytes(kStep / kGroups);
  extern __shared__ __align__(128) std::uint8_t smem[];
  __shared__ FirstShared s;
  std::uint8_t* staged = smem;
  float* logits = reinterpret_cast<float*>(smem + (static_cast<std::size_t>(a.cap) * kPieces * a.x_pitch));
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  GridLaunchDependents();
  GridDependencyWait();
  cluster.sync();  // every CTA of the cluster has begun: its shared memory may be written

  // ---- the router's product: 16 experts at a time, CTA rank r the tiles r, r + 8, ...
  const int expert_tiles = (a.experts + 15) / 16;
  for (int first = 0; first < a.tokens; first += a.cap) {
    const int count = min(a.cap, a.tokens - first);
    __syncthreads();
    StageTokens<kType>(a, staged, count, [&](int c) { return static_cast<std::int64_t>(first + c); });
    __syncthreads();
    for (int m = rank; m < expert_tiles; m += kCluster) {
      if (a.router_type == kF32) {
        RouterTile<kType, kF32, kTiles>(a, staged, m * 16, count, warp, lane, s.partial[warp]);
      } else if (a.router_type == kF16) {
        RouterTile<kType, kF16, kTiles>(a, staged, m * 16, count, warp, lane, s.partial[warp]);
      } else {
        RouterTile<kType, kBF16, kTiles>(a, staged, m * 16, count, warp, lane, s.partial[warp]);
      }
      __syncthreads();
      for (int i = tid; i < 16 * count; i += kThreads) {
        const int row = i / count, c = i % count, e = (m * 16) + row;
        if (e >= a.experts) continue;
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += s.partial[w][row][c];
        for (int r = 0; r < kCluster; ++r) {
          cluster.map_shared_rank(logits, r)[((first + c) * a.experts) + e] = static_cast<float>(sum);
        }
      }
      __syncthreads();
    }
  }
  for (int e = tid; e < a.experts; e += kThreads) s.mask[e] = 0;
  cluster.sync();  // the cluster's logits are in every CTA

  // ---- the choice, the same in every CTA
  for (int t = warp; t < a.tokens; t += kWarps) Choose(a, logits, t, lane, s);
  __syncthreads();
  const int pairs = a.tokens * a.used;
  for (int p = tid; p < pairs; p += kThreads) atomicOr(&s.mask[s.ids[p]], 1u << (p / a.used));
  __syncthreads();
  if (warp == 0) {
    int named = 0, first = 0, groups = 0;
    for (int base = 0; base < a.experts; base += 32) {
      const int e = base + lane;
      const int count = e < a.experts ? __popc(s.mask[e]) : 0;
      const int pieces = (count + a.cap - 1) / a.cap;
      int sum_named = count > 0 ? 1 : 0, sum_first = count, sum_groups = pieces;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int n0 = __shfl_up_sync(0xffffffffu, sum_named, o), n1 = __shfl_up_sync(0xffffffffu, sum_first, o),
                  n2 = __shfl_up_sync(0xffffffffu, sum_groups, o);
        if (lane >= o) sum_named += n0, sum_first += n1, sum_groups += n2;
      }
      if (count > 0) {
        const int at = named + sum_named - 1, begin = first + sum_first - count;
        s.choice.expert[at] = e;
        s.choice.first[at] = begin;
        s.start[e] = begin;
        for (int q = 0; q < pieces; ++q) {
          const int i = groups + sum_groups - pieces + q;
          s.group_expert[i] = e;
          s.group_first[i] = begin + (q * a.cap);
          s.group_count[i] = min(a.cap, count - (q * a.cap));
        }
      }
      named += __shfl_sync(0xffffffffu, sum_named, 31);
      first += __shfl_sync(0xffffffffu, sum_first, 31);
      groups += __shfl_sync(0xffffffffu, sum_groups, 31);
    }
    if (lane == 0) {
      s.choice.named = named;
      s.choice.first[named] = first;
      s.groups = groups;
    }
  }
  __syncthreads();
  for (int p = tid; p < pairs; p += kThreads) {
    const int e = s.ids[p], t = p / a.used;
    s.choice.pairs[s.start[e] + __popc(s.mask[e] & ((1u << t) - 1u))] = p;
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    for (int p = tid; p < pairs; p += kThreads) {
      a.ids[p] = s.ids[p];
      a.weights[p] = s.weights[p];
      a.choice->pairs[p] = s.choice.pairs[p];
    }
    for (int i = tid; i < s.choice.named; i += kThreads) a.choice->expert[i] = s.choice.expert[i];
    for (int i = tid; i <= s.choice.named; i += kThreads) a.choice->first[i] = s.choice.first[i];
    if (tid == 0) a.choice->named = s.choice.named;
  }

  // ---- this CTA's units: (group, tile of 8 gate and 8 up rows), the warps a share of hidden each
  const std::int64_t units = static_cast<std::int64_t>(s.groups) * a.tiles_up;
  const int u0 = static_cast<int>(units * blockIdx.x / gridDim.x), u1 = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
  const bool all_staged = a.tokens <= a.cap;
  const int piece = g % Cols(kPieces);
  const int step0 = warp * a.steps_up / kWarps, step1 = (warp + 1) * a.steps_up / kWarps;
  auto* sums = reinterpret_cast<float*>(s.partial);  // [2][kWarps][kTileRows][kMaxTokens]
  int staged_group = -1;
  for (int u = u0; u < u1; ++u) {
    const int group = u / a.tiles_up, tile = u % a.tiles_up;
    const int e = s.group_expert[group], begin = s.group_first[group], count = s.group_count[group];
    if (!all_staged && staged_group != group) {
      __syncthreads();
      StageTokens<kType>(a, staged, count, [&](int c) { return static_cast<std::int64_t>(s.choice.pairs[begin + c] / a.used); });
      __syncthreads();
      staged_group = group;
    }
    std::uint32_t column_at[kTiles];
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const int c = (nt * TokensATile(kPieces)) + (g / Cols(kPieces));
      column_at[nt] = 0xffffffffu;
      if (c < count && piece < kPieces) {
        const int row = all_staged ? s.choice.pairs[begin + c] / a.used : c;
        column_at[nt] = static_cast<std::uint32_t>((((row * kPieces) + piece) * a.x_pitch) + (t4 * 16));
      }
    }
    const int tiles = (count + TokensATile(kPieces) - 1) / TokensATile(kPieces);
    Sums total[kTiles];
    const std::uint8_t* block =
        a.gate_up + ((((static_cast<std::size_t>(e) * a.tiles_up) + tile) * a.steps_up) + step0) * kBlock;
    for (int step = step0; step < step1; ++step, block += kBlock) {
      StepWeights<kGroups> w;
      w.Load(block, lane);
      MultiplyStep<false, kGroups, kTiles>(w, tiles, total, [&](int nt, int i) {
        if (column_at[nt] == 0xffffffffu) return make_uint4(0, 0, 0, 0);
        return *reinterpret_cast<const uint4*>(staged + column_at[nt] + (step * 256) + (i * 64));
      });
    }
    float* buffer = sums + ((u & 1) * kWarps * kTileRows * kMaxTokens);
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      if (nt >= tiles) break;
      float v[2][2];
      FoldColumns<false, kPieces>(total[nt], v);
#pragma unroll
      for (int j = 0; j < (kPieces == 1 ? 2 : 1); ++j) {
        const int c = (nt * TokensATile(kPieces)) + TokenOf<kPieces>(t4, j);
        if (c < count) {
          buffer[(((warp * kTileRows) + g) * kMaxTokens) + c] = v[0][j];
          buffer[(((warp * kTileRows) + g + 8) * kMaxTokens) + c] = v[1][j];
        }
      }
    }
    __syncthreads();
    // the other buffer's readers are past the barrier before the one that its next writers pass
    for (int i = tid; i < 8 * count; i += kThreads) {
      const int row = i % 8, c = i / 8, at = (tile * 8) + row;
      if (at >= a.inter) continue;
      float gate = 0.0f, up = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        gate += buffer[(((w * kTileRows) + row) * kMaxTokens) + c];
        up += buffer[(((w * kTileRows) + row + 8) * kMaxTokens) + c];
      }
      constexpr int kGlu = GluPieces(kType);
      std::uint32_t bits[kGlu];
      Split<kGlu>(Glu(a.glu, gate * Up(false), up * Up(false), a.limit), bits);
      unsigned short* h = a.h + (static_cast<std::size_t>(s.choice.pairs[begin + c]) * kGlu * a.inter) + at;
#pragma unroll
      for (int q = 0; q < kGlu; ++q) h[static_cast<std::size_t>(q) * a.inter] = static_cast<unsigned short>(bits[q]);
    }
  }
}

// A CTA's 16 rows of the output: its warps take (expert, half of inter) items in turn, each pair's
// sums meet in shared memory and a token's slots are added in order.
constexpr int kParts = 2;

template <int kType, int kGroups>
__global__ void __launch_bounds__(kThreads)
SecondKernel(const LayerArgs a) {
  constexpr int kGlu = GluPieces(kType);
  constexpr int kTiles = kMaxTokens / TokensATile(kGlu);
  constexpr int kBlock = BlockBytes(kStep / kGroups);
  extern __shared__ __align__(128) std::uint8_t smem[];
  auto* sums = reinterpret_cast<float*>(smem);  // [pair][part][16 rows]
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  GridLaunchDependents();
  GridDependencyWait();
  const int tile = static_cast<int>(blockIdx.x);
  const int named = __ldcg(&a.choice->named);
  const int piece = g % Cols(kGlu);
  for (int item = warp; item < named * kParts; item += kWarps) {
    const int i = item / kParts, part = item % kParts;
    const int e = __ldcg(&a.choice->expert[i]), begin = __ldcg(&a.choice->first[i]);
    const int count = __ldcg(&a.choice->first[i + 1]) - begin;
    const int step0 = part * a.steps_down / kParts, step1 = (part + 1) * a.steps_down / kParts;
    const unsigned short* column[kTiles];
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      const int c = (nt * TokensATile(kGlu)) + (g / Cols(kGlu));
      column[nt] = nullptr;
      if (c < count && piece < kGlu) {
        column[nt] = a.h + (((static_cast<std::size_t>(__ldcg(&a.choice->pairs[begin + c])) * kGlu) + piece) * a.inter) + (t4 * 8);
      }
    }
    const int tiles = (count + TokensATile(kGlu) - 1) / TokensATile(kGlu);
    Sums total[kTiles];
    const std::uint8_t* block =
        a.down + ((((static_cast<std::size_t>(e) * a.tiles_down) + tile) * a.steps_down) + step0) * kBlock;
    for (int step = step0; step < step1; ++step, block += kBlock) {
      StepWeights<kGroups> w;
      w.Load(block, lane);
      MultiplyStep<false, kGroups, kTiles>(w, tiles, total, [&](int nt, int b) {
        const int at = (step * kStep) + (32 * b);  // inter is whole 32-value blocks
        if (column[nt] == nullptr || at >= a.inter) return make_uint4(0, 0, 0, 0);
        return __ldcg(reinterpret_cast<const uint4*>(column[nt] + at));
      });
    }
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      if (nt >= tiles) break;
      float v[2][2];
      FoldColumns<false, kGlu>(total[nt], v);
      const int c = (nt * TokensATile(kGlu)) + TokenOf<kGlu>(t4, 0);
      if (c < count) {
        float* out = sums + (((__ldcg(&a.choice->pairs[begin + c]) * kParts) + part) * kTileRows);
        out[g] = v[0][0];
        out[g + 8] = v[1][0];
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < a.tokens * kTileRows; i += kThreads) {
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

constexpr int kFirstSmemLimit = 160 * 1024;

template <int kType, int kGroups>
int LaunchFirst(const LayerArgs& a, cudaStream_t stream) {
  static thread_local int configured_device = -1;
  if (const cudaError_t e = Configure(FirstKernel<kType, kGroups>, configured_device, kFirstSmemLimit); e != cudaSuccess) {
    return Failed(e, "moe_layer attribute");
  }
  const int smem = (a.cap * BfloatPieces(kType) * a.x_pitch) + (a.tokens * a.experts * 4);
  if (smem > kFirstSmemLimit) return Reject("moe_layer: %d bytes of shared memory", smem);
  const std::int64_t units = static_cast<std::int64_t>(std::min(a.experts, a.tokens * a.used)) * a.tiles_up;
  const std::int64_t most = std::max<std::int64_t>(1, static_cast<std::int64_t>(SmCount()) * 2 / kCluster);
  const std::int64_t clusters = std::max<std::int64_t>(1, std::min(most, (units + kCluster - 1) / kCluster));
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

template <int kType, int kGroups>
int LaunchSecond(const LayerArgs& a, cudaStream_t stream) {
  const int smem = a.tokens * a.used * kParts * kTileRows * 4;
  const cudaError_t e = LaunchPdl(SecondKernel<kType, kGroups>, dim3(static_cast<unsigned>(a.tiles_down)), dim3(kThreads),
                                  static_cast<std::size_t>(smem), stream, a);
  return e == cudaSuccess ? 0 : Failed(e, "moe_layer down launch");
}

template <int kType>
int LaunchLayer(int group_up, int group_down, const LayerArgs& a, cudaStream_t stream) {
  int status = group_up == 128  ? LaunchFirst<kType, 1>(a, stream)
               : group_up == 64 ? LaunchFirst<kType, 2>(a, stream)
                                : LaunchFirst<kType, 4>(a, stream);
  if (status != 0) return status;
  status = group_down == 128  ? LaunchSecond<kType, 1>(a, stream)
           : group_down == 64 ? LaunchSecond<kType, 2>(a, stream)
                              : LaunchSecond<kType, 4>(a, stream);
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
  a.tiles_down = Tiles(d.down.n, 0), a.steps_down = Steps(inter);
  a.glu = d.glu, a.limit = d.limit;
  a.y = d.y, a.y_stride = d.y_stride, a.y_type = d.y_type;
  a.ids = d.ids, a.weights = d.weights;
  a.choice = static_cast<Choice*>(d.scratch);
  a.h = reinterpret_cast<unsigned short*>(static_cast<std::uint8_t*>(d.scratch) + ChoiceBytes());
  a.x_pitch = (a.steps_up * kStep * 2) + 64;
  a.cap = std::max(1, std::min(d.tokens, kXBudget / (BfloatPieces(d.x_type) * a.x_pitch)));
  const auto s = static_cast<cudaStream_t>(stream);
  if (d.x_type == kF32) return LaunchLayer<kF32>(d.gate_up.group, d.down.group, a, s);
  if (d.x_type == kF16) return LaunchLayer<kF16>(d.gate_up.group, d.down.group, a, s);
  return LaunchLayer<kBF16>(d.gate_up.group, d.down.group, a, s);
}

}  // extern "C"
