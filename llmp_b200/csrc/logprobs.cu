// Log probabilities of given tokens with their ranks, the entropy, and the top alternatives, from a
// head's logits: what a server answers with beside the tokens, and what scores a prompt.  No
// counterpart in the reference's kernels; reads what the head's product (decode_vector, vecq,
// w4_vector) leaves.
//
// x = logit / temperature, m the largest; S = sum e^(x - m), U = sum (x - m) e^(x - m), in F32:
//   log p = x - m - log S,   entropy = log S - U / S   (two terms of one sign: nothing cancels)
// Masked logits are -inf and add nothing.  Choices and ranks compare the logits themselves.
#include <algorithm>

#include "w4.cuh"

namespace llmp_b200 {
namespace {

using w4::LoadValue;

constexpr int kThreads = 512;
constexpr int kMaxGiven = 16, kMaxTop = 32;

// (logit, lowest index first) as one unsigned number: NaN below -inf, the zeros alike.
__device__ __forceinline__ unsigned long long Key(float v, int index) {
  std::uint32_t k = 0;
  if (v == v) {
    const std::uint32_t b = __float_as_uint(v + 0.0f);
    k = (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
  }
  return (static_cast<unsigned long long>(k) << 32) | (0xffffffffu - static_cast<std::uint32_t>(index));
}

struct Sums {
  float m, s, u;
  bool bad;  // a NaN or +inf: no distribution
};
__device__ __forceinline__ Sums Join(const Sums& a, const Sums& b, float scale) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  r.bad = a.bad || b.bad;
  const float da = a.m == r.m ? 0.0f : (a.m - r.m) * scale, db = b.m == r.m ? 0.0f : (b.m - r.m) * scale;
  const float ea = expf(da), eb = expf(db);
  r.s = (a.s * ea) + (b.s * eb);
  // (x - m') e^(x - m') = e^(m - m') ((x - m) + (m - m')) e^(x - m); a side without weight adds nothing,
  // however far below it lies (a mask of the type's lowest value)
  r.u = (a.s * ea != 0.0f ? ea * fmaf(da, a.s, a.u) : 0.0f) + (b.s * eb != 0.0f ? eb * fmaf(db, b.s, b.u) : 0.0f);
  return r;
}

__global__ void __launch_bounds__(kThreads)
LogprobsKernel(const llmp_b200_logprobs_desc a) {
  __shared__ Sums sums[kThreads / 32];
  __shared__ unsigned long long best[kThreads / 32];
  __shared__ int counts[kMaxGiven];
  GridLaunchDependents();
  GridDependencyWait();
  const std::int64_t row = blockIdx.x;
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const std::int64_t base = row * a.stride;
  const float scale = 1.0f / a.temperature;
  const float kNan = __uint_as_float(0x7fc00000u), kMinusInf = __uint_as_float(0xff800000u);
  auto logit = [&](int i) { return LoadValue(a.logits, base + i, a.type); };

  Sums mine = {kMinusInf, 0.0f, 0.0f, false};
  for (int i = tid; i < a.vocab; i += kThreads) {
    const float x = logit(i);
    if (x != x || x == -kMinusInf) mine.bad = true;
    if (!(x > kMinusInf)) continue;
    mine = Join(mine, Sums{x, 1.0f, 0.0f, false}, scale);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Sums other;
    other.m = __shfl_xor_sync(0xffffffffu, mine.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, mine.s, o);
    other.u = __shfl_xor_sync(0xffffffffu, mine.u, o);
    other.bad = __shfl_xor_sync(0xffffffffu, mine.bad ? 1 : 0, o) != 0;
    mine = Join(mine, other, scale);
  }
  if (lane == 0) sums[warp] = mine;
  if (tid < kMaxGiven) counts[tid] = 0;
  __syncthreads();
  Sums all = sums[0];
  for (int w = 1; w < kThreads / 32; ++w) all = Join(all, sums[w], scale);
  const float log_s = logf(all.s);
  auto log_p = [&](float x) {
    if (all.bad) return kNan;
    if (x == kMinusInf) return kMinusInf;
    return ((x - all.m) / a.temperature) - log_s;
  };
  if (tid == 0) a.entropy[row] = all.bad ? kNan : all.s == 0.0f ? 0.0f : log_s - (all.u / all.s);

  for (int j = 0; j < a.given; ++j) {
    const int token = a.tokens[(row * a.given) + j];
    const bool inside = token >= 0 && token < a.vocab;
    if (inside) {
      const float x = logit(token);
      int above = 0;
      for (int i = tid; i < a.vocab; i += kThreads) above += logit(i) > x ? 1 : 0;
      above = __reduce_add_sync(0xffffffffu, above);
      if (lane == 0) atomicAdd(&counts[j], above);
    }
    __syncthreads();
    if (tid == 0) {
      a.logprobs[(row * a.given) + j] = inside ? log_p(logit(token)) : kNan;
      a.ranks[(row * a.given) + j] = inside ? counts[j] + 1 : 0;
    }
  }

  unsigned long long below = ~0ull;
  for (int n = 0; n < a.top; ++n) {
    unsigned long long most = 0;
    for (int i = tid; i < a.vocab; i += kThreads) {
      const unsigned long long k = Key(logit(i), i);
      if (k < below && k > most) most = k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, most, o);
      most = other > most ? other : most;
    }
    __syncthreads();
    if (lane == 0) best[warp] = most;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) most = best[w] > most ? best[w] : most;
    below = most;
    if (tid == 0) {
      const int id = static_cast<int>(0xffffffffu - static_cast<std::uint32_t>(most));
      a.top_ids[(row * a.top) + n] = id;
      a.top_logprobs[(row * a.top) + n] = log_p(logit(id));
    }
  }
}

}  // namespace
}  // namespace llmp_b200

extern "C" int llmp_b200_logprobs(const llmp_b200_logprobs_desc* desc, void* stream) {
  using namespace llmp_b200;
  if (desc == nullptr) return Reject("logprobs: null descriptor");
  const llmp_b200_logprobs_desc& a = *desc;
  if (!w4::FloatType(a.type)) return Reject("logprobs: F32, F16 or BF16 logits");
  if (a.vocab < 1 || a.vocab > (1 << 24)) return Reject("logprobs: rows of 1 to 2^24 logits");
  if (a.rows < 0 || a.rows > 0x7fffffffLL) return Reject("logprobs: 0 to 2^31 - 1 rows");
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
  const cudaError_t e = LaunchPdl(LogprobsKernel, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0,
                                  static_cast<cudaStream_t>(stream), a);
  return e == cudaSuccess ? 0 : Failed(e, "logprobs launch");
}
