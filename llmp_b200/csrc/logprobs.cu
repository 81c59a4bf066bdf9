// Log probabilities of given tokens with their ranks, the entropy, and the top alternatives, from a
// head's logits: what a server answers with beside the tokens, and what scores a prompt.  No
// counterpart in the reference's kernels; reads what the head's product (decode_vector, vecq,
// w4_vector) leaves.
//
// x = logit / temperature, m the largest; S = sum e^(x - m), U = sum (x - m) e^(x - m), in F32:
//   log p = x - m - log S,   entropy = log S - U / S   (two terms of one sign: nothing cancels)
// Masked logits are -inf and add nothing.  Choices and ranks compare the logits themselves.
#include <cooperative_groups.h>

#include <algorithm>

#include "w4.cuh"

namespace llmp_b200 {
namespace {

namespace cg = cooperative_groups;
using w4::LoadValue;

constexpr int kFewRows = 512, kManyRows = 128;  // threads a CTA
constexpr int kMaxGiven = 16, kMaxTop = 32;
constexpr int kMaxRanks = 8;
constexpr int kCandidates = 1024;
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr float kFar = -200.0f;  // 2^-200 is zero in F32

__device__ __forceinline__ float MinusInf() { return __uint_as_float(0xff800000u); }
__device__ __forceinline__ float Nan() { return __uint_as_float(0x7fc00000u); }
// 2^x; below 2^-126 zero.  e^(d / T) is this of one product with log2 e / T instead of expf of a quotient: fewer instructions a
// logit, for errors up to half as large again (log probabilities against 64 bits, relative, root mean square: 16 x 131072
// F32 logits 7.4e-8, by expf in F32 5.5e-8; 2048 x 32003 bf16 ones 7.2e-8 and 4.9e-8).
__device__ __forceinline__ float Exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// (logit, lowest index first) as one unsigned number: NaN below -inf, the zeros alike.
using Key = unsigned long long;
__device__ __forceinline__ Key KeyOf(float v, int index) {
  std::uint32_t k = 0;
  if (v == v) {
    const std::uint32_t b = __float_as_uint(v + 0.0f);
    k = (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
  }
  return (static_cast<Key>(k) << 32) | (0xffffffffu - static_cast<std::uint32_t>(index));
}
__device__ __forceinline__ float ValueOf(Key k) {
  const std::uint32_t b = static_cast<std::uint32_t>(k >> 32);
  return b == 0 ? Nan() : __uint_as_float((b & 0x80000000u) != 0 ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int IndexOf(Key k) { return static_cast<int>(0xffffffffu - static_cast<std::uint32_t>(k)); }

// Over some logits, in units of 1 / c = T / log2 e: the largest, sum 2^d and sum d 2^d, d = (x - m) c.  m starts at the
// lowest finite number, so a masked logit is 2^-inf = 0 whatever m is; a NaN or +inf makes s a NaN.
struct Sums {
  float m, s, u;
  __device__ __forceinline__ void Rebase(float most, float c) {
    const float d = (m - most) * c, f = Exp2(d);
    u = d > kFar ? f * fmaf(d, s, u) : u * 0.0f;
    s *= f;
    m = most;
  }
  // All lanes' sums: the largest first, one change of base, then plain sums in a fixed order.
  template <int kLanes>
  __device__ __forceinline__ void JoinLanes(float c) {
    float most = m;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (m != most) Rebase(most, c);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      u += __shfl_xor_sync(0xffffffffu, u, o);
    }
  }
};

// A row as units of eight logits whose addresses are 16-byte aligned; the first and the last may begin before the
// row or end behind it: those are read one by one, with -inf outside.
template <int kType>
struct Row {
  const std::uint8_t* base;
  int vocab, skew, units;  // skew: logits that unit 0 begins before the row
  int whole0, whole1;      // the units that lie inside the row
  __device__ __forceinline__ Row(const void* logits, std::int64_t at, int vocab_) : vocab(vocab_) {
    base = static_cast<const std::uint8_t*>(logits) + (at * w4::TypeBytes(kType));
    skew = static_cast<int>((reinterpret_cast<std::uintptr_t>(base) & 15u) / w4::TypeBytes(kType));
    units = (vocab + skew + 7) / 8;
    whole0 = skew > 0 ? 1 : 0;
    whole1 = (vocab + skew) / 8;
  }
  __device__ __forceinline__ float At(int i) const { return LoadValue(base, i, kType); }
  __device__ __forceinline__ int First(int unit) const { return (unit * 8) - skew; }
  static constexpr int kQuads = kType == w4::kF32 ? 2 : 1;
  __device__ __forceinline__ void LoadWhole(int unit, uint4 (&raw)[kQuads]) const {
    const auto* p = reinterpret_cast<const uint4*>(base + (static_cast<std::int64_t>(First(unit)) * w4::TypeBytes(kType)));
#pragma unroll
    for (int i = 0; i < kQuads; ++i) raw[i] = p[i];
  }
  static __device__ __forceinline__ void Expand(const uint4 (&raw)[kQuads], float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
      const std::uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kType == w4::kF32) {
          v[(4 * i) + j] = __uint_as_float(w[j]);
        } else if constexpr (kType == w4::kBF16) {
          v[2 * j] = __uint_as_float(w[j] << 16);
          v[(2 * j) + 1] = __uint_as_float(w[j] & 0xffff0000u);
        } else {
          v[2 * j] = HalfBitsToFloat(w[j] & 0xffffu);
          v[(2 * j) + 1] = HalfBitsToFloat(w[j] >> 16);
        }
      }
    }
  }
  // The largest of a unit that is a number (16-bit ones two at a time); NaN where none is.
  static __device__ __forceinline__ float Largest(const uint4 (&raw)[kQuads]) {
    if constexpr (kType == w4::kF32) {
      float v[8];
      Expand(raw, v);
      return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
    } else if constexpr (kType == w4::kBF16) {
      const auto* p = reinterpret_cast<const __nv_bfloat162*>(&raw[0]);
      const __nv_bfloat162 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
      return fmaxf(__low2float(m), __high2float(m));
    } else {
      const auto* p = reinterpret_cast<const __half2*>(&raw[0]);
      const __half2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
      return fmaxf(__low2float(m), __high2float(m));
    }
  }
  __device__ __forceinline__ void Load(int unit, float (&v)[8]) const {
    const int first = First(unit);
    w4::Load8<kType>(base, first, first >= 0 && first + 8 <= vocab ? 8 : 0, true, v);
    if (first < 0 || first + 8 > vocab) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = first + i >= 0 && first + i < vocab ? At(first + i) : MinusInf();
    }
  }
};

struct Part {  // of a row, by one CTA
  Sums sums;
  int above[kMaxGiven];
  int candidates;
  Key top[kMaxTop];
};

// A row is divided among the CTAs of a cluster (one, where there are rows enough): one pass over the logits, kBatch
// units of a thread in flight.  The top alternatives need no sort: the `top`-th largest of the maxima of 32 groups of threads
// is a logit that at least `top` logits reach, so the few that reach it are collected by the threads whose own
// maximum does (they look at their logits again, which L2 still holds), and a candidate's place is the number of
// keys above its own.  Ranks are counted in the pass, the given logits being fetched before it.  Each CTA stores its
// sums, counts and best keys into rank 0's shared memory, which joins them in rank order after one cluster barrier.
//
// Measured: 32000 bf16 logits, twenty alternatives 7.7 us, bound by its chain of barriers; 16 x 131072 F32 13.4 us; 2048 x
// 32003 bf16 49 us (2.7 TB/s, issue slots 66 % full): some 10 instructions a logit, an exponential among them, and a
// row's joining and alternatives, about a third as much again.
template <int kType, int kGiven, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads)
LogprobsKernel(const llmp_b200_logprobs_desc a) {
  constexpr int kWarps = kThreads / 32, kGroup = kThreads / 32;  // threads whose maximum is one of 32
  constexpr int kBatch = kType == w4::kF32 ? 2 : 4;
  __shared__ Sums warp_sums[kWarps];
  __shared__ float maxima[32];
  __shared__ int warp_above[kWarps][kGiven > 0 ? kGiven : 1];
  __shared__ Key candidates[kCandidates];
  __shared__ Key best[kWarps];
  __shared__ Key merged[kMaxRanks * kMaxTop];
  __shared__ Part part, parts[kMaxRanks];
  __shared__ float given_logit[kMaxGiven];
  __shared__ int given_token[kMaxGiven];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const std::int64_t row_index = static_cast<std::int64_t>(blockIdx.x) / ranks;
  const float c = kLog2E / a.temperature;
  GridLaunchDependents();
  GridDependencyWait();
  const Row<kType> row(a.logits, row_index * a.stride, a.vocab);
  const int unit0 = static_cast<int>(static_cast<std::int64_t>(row.units) * rank / ranks);
  const int unit1 = static_cast<int>(static_cast<std::int64_t>(row.units) * (rank + 1) / ranks);
  if (ranks > 1) cluster.barrier_arrive();  // this CTA has begun: its shared memory may be written
  for (int i = 0; i < kBatch; ++i) {  // on their way while the given logits are looked up
    const int ahead = unit0 + tid + (i * kThreads);
    if (ahead < unit1 && ahead >= row.whole0) {
      asm volatile("prefetch.global.L2 [%0];" ::"l"(row.base + (static_cast<std::int64_t>(row.First(ahead)) * w4::TypeBytes(kType))));
    }
  }
  float given[kGiven > 0 ? kGiven : 1];
  int above[kGiven > 0 ? kGiven : 1];
  if constexpr (kGiven > 0) {
    if (tid < kGiven) {
      const int token = tid < a.given ? a.tokens[(row_index * a.given) + tid] : -1;
      given_token[tid] = token;
      given_logit[tid] = token >= 0 && token < a.vocab ? row.At(token) : Nan();  // nothing is above a NaN
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kGiven; ++j) above[j] = 0, given[j] = given_logit[j];
  }
  if (tid == 0) part.candidates = 0;

  Sums mine = {-3.402823466e38f, 0.0f, 0.0f};
  float most = MinusInf();  // this thread's largest, of any number
  auto take = [&](const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (the difference first: the product of a large logit with c would lose the difference's last bits)
      const float d = (v[i] - mine.m) * c, e = Exp2(d);
      mine.s += e;
      mine.u = fmaf(fmaxf(d, kFar), e, mine.u);
#pragma unroll
      for (int j = 0; j < kGiven; ++j) above[j] += v[i] > given[j] ? 1 : 0;
    }
  };
  const int first_whole = max(unit0, row.whole0), end_whole = min(unit1, row.whole1);
  int unit = first_whole + tid;
  for (; unit + ((kBatch - 1) * kThreads) < end_whole; unit += kBatch * kThreads) {
    uint4 raw[kBatch][kType == w4::kF32 ? 2 : 1];
#pragma unroll
    for (int q = 0; q < kBatch; ++q) row.LoadWhole(unit + (q * kThreads), raw[q]);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) most = fmaxf(most, Row<kType>::Largest(raw[q]));
    if (most > mine.m) mine.Rebase(most, c);
#pragma unroll
    for (int q = 0; q < kBatch; ++q) {
      float v[8];
      Row<kType>::Expand(raw[q], v);
      take(v);
    }
  }
  for (; unit < end_whole; unit += kThreads) {
    uint4 raw[kType == w4::kF32 ? 2 : 1];
    row.LoadWhole(unit, raw);
    most = fmaxf(most, Row<kType>::Largest(raw));
    if (most > mine.m) mine.Rebase(most, c);
    float v[8];
    Row<kType>::Expand(raw, v);
    take(v);
  }
  // the units that reach over an end of the row, by two threads
  const int edge = tid == 0 && unit0 < row.whole0 ? 0 : tid == 32 && unit1 > row.whole1 && row.whole1 >= row.whole0 ? row.whole1 : -1;
  if (edge >= unit0 && edge < unit1) {
    float v[8];
    row.Load(edge, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) most = fmaxf(most, v[i]);
    if (most > mine.m) mine.Rebase(most, c);
    take(v);
  }

  // ---- this CTA's sums and counts
  mine.JoinLanes<32>(c);
  if (lane == 0) warp_sums[warp] = mine;
#pragma unroll
  for (int j = 0; j < kGiven; ++j) {
    const int sum = __reduce_add_sync(0xffffffffu, above[j]);
    if (lane == 0) warp_above[warp][j] = sum;
  }
  if (a.top > 0) {
    float group = most;
#pragma unroll
    for (int o = kGroup / 2; o > 0; o >>= 1) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, o));
    if (tid % kGroup == 0) maxima[tid / kGroup] = group;
  }
  __syncthreads();
  if (warp == 0) {
    Sums sum = warp_sums[lane % kWarps];
    sum.JoinLanes<kWarps>(c);
    if (lane == 0) part.sums = sum;
    if constexpr (kGiven > 0) {
      if (lane < kGiven) {
        int count = 0;
        for (int w = 0; w < kWarps; ++w) count += warp_above[w][lane];
        part.above[lane] = count;
      }
    }
  }

  // ---- this CTA's best keys
  if (a.top > 0) {
    const int logits = min(unit1 * 8 - row.skew, a.vocab) - max(unit0 * 8 - row.skew, 0);
    const int wanted = min(a.top, max(logits, 0));
    float reach = MinusInf();  // at least `wanted` logits reach it
    {
      const float mine_max = maxima[lane];
      int larger = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float other = maxima[i];
        larger += other > mine_max || (other == mine_max && i < lane) ? 1 : 0;
      }
      const unsigned int which = __ballot_sync(0xffffffffu, larger == wanted - 1);
      if (which != 0) reach = __shfl_sync(0xffffffffu, mine_max, __ffs(which) - 1);
    }
    // collected: the logits that reach it, or all above -inf (few logits, or few that are not masked)
    auto collect = [&](int at) {
      float v[8];
      row.Load(at, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (v[i] >= reach && v[i] > MinusInf()) {
          const int place = atomicAdd(&part.candidates, 1);
          if (place < kCandidates) candidates[place] = KeyOf(v[i], row.First(at) + i);
        }
      }
    };
    const bool flagged_me = most >= reach && most > MinusInf();
    if (flagged_me && edge >= unit0 && edge < unit1) collect(edge);
    if (end_whole - first_whole <= 2 * kThreads) {  // a thread's own one or two units
      if (flagged_me) {
        for (int at = first_whole + tid; at < end_whole; at += kThreads) collect(at);
      }
    } else {  // a warp goes over the units of each of its threads whose maximum does
      for (unsigned int flagged = __ballot_sync(0xffffffffu, flagged_me); flagged != 0; flagged &= flagged - 1) {
        const int owner = (warp * 32) + __ffs(flagged) - 1;
        for (int at = first_whole + owner + (lane * kThreads); at < end_whole; at += 32 * kThreads) collect(at);
      }
    }
    __syncthreads();
    const int found = part.candidates;
    if (found <= kCandidates) {
      for (int i = tid; i < found; i += kThreads) {
        const Key key = candidates[i];
        int larger = 0;
        for (int j = 0; j < found; ++j) larger += candidates[j] > key ? 1 : 0;
        if (larger < wanted) part.top[larger] = key;
      }
      if (found < wanted && warp == 0) {  // the masked logits in order of their index, then the NaNs
        int have = found;
        const int begin = max(row.First(unit0), 0), end = min(row.First(unit1), a.vocab);
        for (int nan = 0; nan < 2; ++nan) {
          for (int first = begin; first < end && have < wanted; first += 32) {
            const int i = first + lane;
            const float x = i < end ? row.At(i) : 0.0f;
            const bool takes = i < end && (nan == 0 ? x == MinusInf() : x != x);
            const unsigned int takers = __ballot_sync(0xffffffffu, takes);
            const int place = have + __popc(takers & ((1u << lane) - 1u));
            if (takes && place < wanted) part.top[place] = KeyOf(x, i);
            have += __popc(takers);
          }
        }
      }
    } else {
      // More that reach it than there is room for (a row masked by the type's lowest value that leaves fewer logits than
      // `top`: all the masked ones do): one key at a time, each pass the largest below the one before.  20 of 131072 F32 logits,
      // three of them not masked: 97 us instead of 10.4; masked by -inf 8.1, as those are never candidates.
      Key below = ~0ull;
      for (int n = 0; n < wanted; ++n) {
        Key largest = 0;
        for (int unit = unit0 + tid; unit < unit1; unit += kThreads) {
          float v[8];
          row.Load(unit, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = row.First(unit) + i;
            const Key key = KeyOf(v[i], at);
            if (at >= 0 && at < a.vocab && key < below && key > largest) largest = key;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const Key other = __shfl_xor_sync(0xffffffffu, largest, o);
          largest = other > largest ? other : largest;
        }
        __syncthreads();
        if (lane == 0) best[warp] = largest;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) largest = best[w] > largest ? best[w] : largest;
        below = largest;
        if (tid == 0) part.top[n] = largest;
      }
    }
    __syncthreads();
    if (tid == 0) part.candidates = wanted;
  }
  __syncthreads();
  const Part* joined = &part;
  if (ranks > 1) {
    cluster.barrier_wait();
    constexpr int kWords = sizeof(Part) / 4;
    auto* to = reinterpret_cast<std::uint32_t*>(cluster.map_shared_rank(&parts[rank], 0));
    for (int i = tid; i < kWords; i += kThreads) to[i] = reinterpret_cast<const std::uint32_t*>(&part)[i];
    cluster.sync();
    joined = parts;
  }
  if (rank != 0) return;

  // ---- rank 0: the parts in rank order
  Sums sum = joined[lane % ranks].sums;  // (ranks is a power of two; every warp for itself)
  if (ranks == 2) sum.JoinLanes<2>(c);
  if (ranks == 4) sum.JoinLanes<4>(c);
  if (ranks == 8) sum.JoinLanes<8>(c);
  const bool bad = sum.s != sum.s, nothing = sum.s == 0.0f;
  const float log_s = logf(sum.s);
  auto log_p = [&](float x) {
    if (bad) return Nan();
    if (nothing || x == MinusInf()) return MinusInf();
    return ((x - sum.m) / a.temperature) - log_s;
  };
  if (tid == 0) a.entropy[row_index] = bad ? Nan() : nothing ? 0.0f : log_s - (kLn2 * (sum.u / sum.s));
  if constexpr (kGiven > 0) {
    if (tid < a.given) {
      const bool inside = given_token[tid] >= 0 && given_token[tid] < a.vocab;
      int count = 1;
      for (int r = 0; r < ranks; ++r) count += joined[r].above[tid];
      a.logprobs[(row_index * a.given) + tid] = inside ? log_p(given_logit[tid]) : Nan();
      a.ranks[(row_index * a.given) + tid] = inside ? count : 0;
    }
  }
  if (a.top > 0) {
    // keys of all parts; a place is the number of larger ones
    int total = 0;
    for (int r = 0; r < ranks; ++r) {
      const int count = joined[r].candidates;
      for (int i = tid; i < count; i += kThreads) merged[total + i] = joined[r].top[i];
      total += count;
    }
    __syncthreads();
    for (int i = tid; i < total; i += kThreads) {
      const Key key = merged[i];
      int larger = 0;
#pragma unroll 8
      for (int j = 0; j < total; ++j) larger += merged[j] > key ? 1 : 0;
      if (larger < a.top) {
        a.top_ids[(row_index * a.top) + larger] = IndexOf(key);
        a.top_logprobs[(row_index * a.top) + larger] = log_p(ValueOf(key));
      }
    }
  }
}

template <int kType, int kGiven, int kThreads>
int LaunchThreads(const llmp_b200_logprobs_desc& a, int ranks, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(a.rows * ranks));
  config.blockDim = dim3(kThreads);
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[0].val.programmaticStreamSerializationAllowed = 1;
  attribute[1].id = cudaLaunchAttributeClusterDimension;
  attribute[1].val.clusterDim.x = static_cast<unsigned>(ranks);
  attribute[1].val.clusterDim.y = attribute[1].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, LogprobsKernel<kType, kGiven, kThreads>, a);
  return e == cudaSuccess ? 0 : Failed(e, "logprobs launch");
}

template <int kType, int kGiven>
int LaunchGiven(const llmp_b200_logprobs_desc& a, cudaStream_t stream) {
  // Many rows: a small CTA each, eight an SM, so that one row's short steps between its barriers run beside another's
  // pass.  (Small CTAs and those of 512 threads, bf16: 450 rows of 32003 logits 23.2 and 21.8 us, 600 24.8 and 27.9, 1200
  // 35.7 and 47.6; of 131072 logits 580 59 and 49, 600 64 and 58, 1200 103 and 98: the rule follows the shorter rows.)
  // Few: as many CTAs a row as fill the device twice over, with 4096 logits each.  (With 2048, 4096 and 8192, bf16:
  // one row of 32000 6.6, 6.9 and 7.8 us; 32 rows 10.5, 8.7 and 9.2; 16 of 16384 7.7, 7.0 and 6.8.)
  if (a.rows >= 4 * SmCount()) return LaunchThreads<kType, kGiven, kManyRows>(a, 1, stream);
  int ranks = 1;
  while (ranks < kMaxRanks && a.rows * ranks < 2 * SmCount() && a.vocab / (2 * ranks) >= 4096) ranks *= 2;
  return LaunchThreads<kType, kGiven, kFewRows>(a, ranks, stream);
}

template <int kType>
int LaunchType(const llmp_b200_logprobs_desc& a, cudaStream_t stream) {
  if (a.given == 0) return LaunchGiven<kType, 0>(a, stream);
  if (a.given == 1) return LaunchGiven<kType, 1>(a, stream);
  if (a.given <= 4) return LaunchGiven<kType, 4>(a, stream);
  return LaunchGiven<kType, 16>(a, stream);
}

}  // namespace
}  // namespace llmp_b200

extern "C" int llmp_b200_logprobs(const llmp_b200_logprobs_desc* desc, void* stream) {
  using namespace llmp_b200;
  if (desc == nullptr) return Reject("logprobs: null descriptor");
  const llmp_b200_logprobs_desc& a = *desc;
  if (!w4::FloatType(a.type)) return Reject("logprobs: F32, F16 or BF16 logits");
  if (a.vocab < 1 || a.vocab > (1 << 24)) return Reject("logprobs: rows of 1 to 2^24 logits");
  if (a.rows < 0 || a.rows > 0x0fffffffLL) return Reject("logprobs: 0 to 2^28 - 1 rows");
  if (a.given < 0 || a.given > kMaxGiven || a.top < 0 || a.top > kMaxTop || a.top > a.vocab) {
    return Reject("logprobs: up to 16 given tokens a row and up to 32 alternatives, no more than there are logits");
  }
  if (!(a.temperature >= 1e-6f && a.temperature <= 1e6f)) return Reject("logprobs: a temperature of 1e-6 to 1e6");
  if (a.rows == 0) return 0;
  if (a.logits == nullptr || a.entropy == nullptr ||
      (a.given > 0 && (a.tokens == nullptr || a.logprobs == nullptr || a.ranks == nullptr)) ||
      (a.top > 0 && (a.top_ids == nullptr || a.top_logprobs == nullptr))) {
    return Reject("logprobs: logits and the outputs that are asked for");
  }
  if (!Aligned(a.logits, w4::TypeBytes(a.type)) || !Aligned(a.tokens, 4) || !Aligned(a.logprobs, 4) || !Aligned(a.ranks, 4) ||
      !Aligned(a.entropy, 4) || !Aligned(a.top_ids, 4) || !Aligned(a.top_logprobs, 4) || (a.rows > 1 && a.stride < 0)) {
    return Reject("logprobs: operands aligned to their elements, no negative stride");
  }
  if (const int status = DeviceStatus(); status != 0) return status;
  const auto s = static_cast<cudaStream_t>(stream);
  if (a.type == w4::kF32) return LaunchType<w4::kF32>(a, s);
  if (a.type == w4::kF16) return LaunchType<w4::kF16>(a, s);
  return LaunchType<w4::kBF16>(a, s);
}
