// 4-bit weights with group scales: the slab that the products read, and the product of a tile.
//
// A weight is scale * (code - zero), code and zero in 0..15, one scale and zero a group of 32, 64
// or 128 values of a row.  The slab (llmp_b200_w4_relayout, once at load time) holds, per expert,
// tiles of 16 weight rows x steps of 128 values, steps of a tile back to back, each
//
//   [2][32 lanes][16 bytes]  codes: lane (g, t) = (lane / 4, lane % 4) holds row g's and row g + 8's
//                            values 32 i + 8 t .. + 7 of the step in word i = 0..3, the even values'
//                            nibbles in the low half and the odd ones' in the high half
//   [16 rows][128 / group]   words: the scale in F32, whose last byte the 16-bit types leave free for the zero
//
// so a warp reads a step with two 16-byte copies a lane and a few of its rows' words.  Codes multiply
// as exact small integers: word & 0x000f000f, or'ed with 0x6400 (1024 in f16, whose last four mantissa
// bits then are the code), plus -(1024 + zero), whose two bytes are 0xe4 and the zero, is a pair of neighbouring
// values in one addition; & 0x00f000f0 the same way is 1024 + 16 code, a pair in one multiply-add; a shift by 8 serves the other
// two.  In bf16, 0x4300 is 128, every pair needs its shift, and the multiply-add takes 2^-11 into the pair.  They are
// the A fragment of mma.sync.m16n8k16, whose k order is free as long as B's is the same.  With a
// GLU a tile's rows 0..7 are gate rows and 8..15 the same rows of up, so a lane's sums hold both.
//
// The tokens are the MMA's 8 columns.  Sums are F32 and the scale multiplies a group's F32 sum: nothing of
// the weights is rounded.  BF16 and F16 activations multiply as they are, in their own type; a group's sum
// comes before its scale and may be 15 * 128 times an activation, hence bf16's 2^-11 (taken back in
// the result): it overflows only where the scaled product would.  F32 activations are two f16
// pieces of the value times a power of two a row, which brings the row's largest finite value to 2^14..2^15: the second
// piece 2^11 larger, the two within a unit of the value's last bit (below 2^-29 of the row's largest within 2^-51
// of that), and exact bf16 pieces (3, without a scale) where values must not lose that.
#ifndef LLMP_B200_CSRC_W4_CUH_
#define LLMP_B200_CSRC_W4_CUH_

#include <cuda_bf16.h>

#include "common.cuh"

namespace llmp_b200 {
namespace w4 {

constexpr int kStep = 128;       // values of a row in a step
constexpr int kTileRows = 16;

__host__ __device__ constexpr int BlockBytes(int group) { return 1024 + (64 * (kStep / group)); }
__host__ __device__ constexpr int Steps(int k) { return (k + kStep - 1) / kStep; }
// Tiles of a matrix of n rows (with a GLU: n / 2 gate rows, then n / 2 up rows).
__host__ __device__ constexpr int Tiles(int n, int glu) {
  return glu ? ((n / 2) + 7) / 8 : (n + 15) / 16;
}

// Element types of activations and outputs (GGML's numbers).
constexpr int kF32 = LLMP_B200_TYPE_F32, kF16 = LLMP_B200_TYPE_F16, kBF16 = LLMP_B200_TYPE_BF16;
inline bool FloatType(int t) { return t == kF32 || t == kF16 || t == kBF16; }
__host__ __device__ constexpr int TypeBytes(int t) { return t == kF32 ? 4 : 2; }
// The f16 pieces, and the bf16 pieces, that a value of the type is the sum of.
__host__ __device__ constexpr int HalfPieces(int t) { return t == kF32 ? 2 : 1; }
__host__ __device__ constexpr int BfloatPieces(int t) { return t == kF32 ? 3 : t == kF16 ? 2 : 1; }

// Columns a token takes, tokens an MMA's 8 columns hold.
__host__ __device__ constexpr int Cols(int pieces) { return pieces == 3 ? 4 : pieces; }
__host__ __device__ constexpr int TokensATile(int pieces) { return 8 / Cols(pieces); }

// ---- the vector product's shared memory (w4.cu): rings, two buffers of sums, the staged activations
// Two CTAs of eight warps an SM, or one of sixteen where the activations take the shared memory of both; rings of what fits.
__host__ __device__ constexpr int Warps(bool wide) { return wide ? 16 : 8; }
__host__ __device__ constexpr int Reducers(bool wide) { return wide ? 2 : 1; }
__host__ __device__ constexpr int Slots(bool wide) { return wide ? 3 : 5; }
__host__ __device__ constexpr int Threads(bool wide) { return (Warps(wide) + Reducers(wide)) * 32; }
// Staged activations: a column's values at a pitch of 64 more bytes than whole steps, so the two
// columns that a quarter warp reads (64 bytes each) lie in different halves of the banks.
__host__ __device__ constexpr int Pitch(int steps) { return (steps * kStep * 2) + 64; }
// Column tiles that the kernel for `rows` rows multiplies, all of them: 1, 2 or 4.
__host__ __device__ constexpr int ColumnTiles(int rows, int pieces) {
  return rows <= TokensATile(pieces) ? 1 : rows <= 2 * TokensATile(pieces) ? 2 : 4;
}
// The staged column that an MMA column reads, for the token and piece that it stands for.  Where the tiles hold more tokens
// than there are rows, a column of zeros follows the rows' for the tokens that are none.
__host__ __device__ constexpr bool ZeroColumn(int rows, int pieces) {
  return rows < ColumnTiles(rows, pieces) * TokensATile(pieces);
}
__host__ __device__ constexpr int StagedColumn(int token, int piece, int rows, int pieces) {
  return token < rows ? (token * pieces) + piece : rows * pieces;
}
__host__ __device__ constexpr int StagedAt(bool wide, int rows, int block_bytes) {
  return (Warps(wide) * Slots(wide) * block_bytes) + (2 * Warps(wide) * kTileRows * rows * 4);
}
constexpr std::int64_t SmemBytes(bool wide, int ranks, int rows, int steps, int pieces, int block_bytes) {
  const int columns = (rows * pieces) + (ZeroColumn(rows, pieces) ? 1 : 0);
  return StagedAt(wide, rows, block_bytes) + (columns * static_cast<std::int64_t>(Pitch((steps + ranks - 1) / ranks)));
}

// A product in bf16 leaves this much larger.
__host__ __device__ constexpr float Up(bool half) { return half ? 1.0f : 0x1p+11f; }

// Shape and alignment of a matrix whose slab a product reads: 0 or a refusal.
int CheckMatrix(const llmp_b200_w4_matrix& m, const char* what);

#ifdef __CUDACC__
__device__ __forceinline__ float LoadValue(const void* p, std::int64_t i, int type) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  const std::uint32_t bits = static_cast<const unsigned short*>(p)[i];
  return type == kBF16 ? __uint_as_float(bits << 16) : HalfBitsToFloat(bits);
}
__device__ __forceinline__ void StoreValue(void* p, std::int64_t i, int type, float v) {
  if (type == kF32) {
    static_cast<float*>(p)[i] = v;
  } else if (type == kBF16) {
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  } else {
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  }
}

// common.cuh's GLU with clamps that keep a NaN: fminf and fmaxf, as the reference's products have them, return the
// other operand, and a gate that is no number would come out as silu(limit).
__device__ __forceinline__ float GluOf(int glu, float gate, float up, float limit) {
  if (glu != LLMP_B200_GLU_SWIGLU_CLAMP) return Glu(glu, gate, up, limit);
  gate = gate > limit ? limit : gate;
  up = up > limit ? limit : up;
  up = up < -limit ? -limit : up;
  return Silu(gate) * up;
}

// The pieces of x, in bf16 bits: truncations, so each remainder is exact and none overflows.
template <int kPieces>
__device__ __forceinline__ void Split(float x, std::uint32_t (&bits)[kPieces]) {
  float rest = x;
#pragma unroll
  for (int s = 0; s < kPieces; ++s) {
    const std::uint32_t b = __float_as_uint(rest);
    bits[s] = b >> 16;
    rest -= __uint_as_float(b & 0xffff0000u);
  }
  if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) {  // inf - inf: the first piece says it all
    if ((__float_as_uint(x) & 0x007fffffu) != 0) bits[0] |= 0x0040u;  // a NaN stays one
#pragma unroll
    for (int s = 1; s < kPieces; ++s) bits[s] = 0;
  }
}

// Eight consecutive values (zero from `valid` on).
template <int kType>
__device__ __forceinline__ void Load8(const void* row, std::int64_t at, int valid, bool vec, float (&v)[8]) {
  if (vec && valid >= 8) {
    if constexpr (kType == kF32) {
      const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + at);
      const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(row) + at + 4);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(row) + at);
      const std::uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kType == kF16) {
          v[2 * i] = HalfBitsToFloat(w[i] & 0xffffu);
          v[(2 * i) + 1] = HalfBitsToFloat(w[i] >> 16);
        } else {
          v[2 * i] = __uint_as_float(w[i] << 16);
          v[(2 * i) + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? LoadValue(row, at + i, kType) : 0.0f;
  }
}
// ... as bf16 pieces, a 16-byte quad a piece.
template <int kPieces>
__device__ __forceinline__ void PackBfloat8(const float (&v)[8], uint4 (&quads)[kPieces]) {
  std::uint32_t packed[kPieces][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    std::uint32_t lo[kPieces], hi[kPieces];
    Split<kPieces>(v[2 * i], lo);
    Split<kPieces>(v[(2 * i) + 1], hi);
#pragma unroll
    for (int s = 0; s < kPieces; ++s) packed[s][i] = lo[s] | (hi[s] << 16);
  }
#pragma unroll
  for (int s = 0; s < kPieces; ++s) quads[s] = make_uint4(packed[s][0], packed[s][1], packed[s][2], packed[s][3]);
}
template <int kType>
__device__ __forceinline__ void LoadBfloat8(const void* row, std::int64_t at, int valid, bool vec,
                                            uint4 (&quads)[BfloatPieces(kType)]) {
  float v[8];
  Load8<kType>(row, at, valid, vec, v);
  PackBfloat8(v, quads);
}
// Eight F32 values times `scale` as two f16 pieces.
__device__ __forceinline__ void LoadHalf8(const void* row, std::int64_t at, int valid, bool vec, float scale, uint4 (&quads)[2]) {
  float v[8];
  Load8<kF32>(row, at, valid, vec, v);
  std::uint32_t packed[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[2 * i] * scale, b = v[(2 * i) + 1] * scale;
    const __half2 first = __floats2half2_rn(a, b);
    packed[0][i] = *reinterpret_cast<const std::uint32_t*>(&first);
    const float2 f = __half22float2(first);  // the remainders are exact; of an infinity there is none
    const __half2 second = __floats2half2_rn(isinf(f.x) ? 0.0f : (a - f.x) * 2048.0f, isinf(f.y) ? 0.0f : (b - f.y) * 2048.0f);
    packed[1][i] = *reinterpret_cast<const std::uint32_t*>(&second);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) quads[s] = make_uint4(packed[s][0], packed[s][1], packed[s][2], packed[s][3]);
}
// The largest finite magnitude's bits among eight F32 values, and the power of two that brings it to 2^14..2^15.
__device__ __forceinline__ std::uint32_t Magnitude8(const void* row, std::int64_t at, int valid, bool vec) {
  float v[8];
  Load8<kF32>(row, at, valid, vec, v);
  std::uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const std::uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
    if (b < 0x7f800000u) most = max(most, b);
  }
  return most;
}
__device__ __forceinline__ int ScaleExponent(std::uint32_t magnitude) {
  return min(126, 141 - static_cast<int>(magnitude >> 23));  // 14 - (exponent - 127); at least 14 - 127
}
__device__ __forceinline__ float PowerOfTwo(int e) { return __uint_as_float(static_cast<std::uint32_t>(e + 127) << 23); }

// c += A B, or c = A B (kFirst: no registers to clear); kHalf: f16 operands, else bf16.
template <bool kHalf, bool kFirst>
__device__ __forceinline__ void Mma(float (&c)[4], std::uint32_t a0, std::uint32_t a1, std::uint32_t a2,
                                    std::uint32_t a3, std::uint32_t b0, std::uint32_t b1) {
  if constexpr (kFirst && kHalf) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  } else if constexpr (kFirst) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  } else if constexpr (kHalf) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ std::uint32_t SharedAddress(const void* p) {
  return static_cast<std::uint32_t>(__cvta_generic_to_shared(p));
}
// The zero points of a row's group as the pairs take them.
template <bool kHalf>
struct Zeros {
  std::uint32_t near, far;  // f16: -(1024 + zero), -(64 + zero); bf16: -2^-11 (128 + zero), unused
  __device__ __forceinline__ explicit Zeros(std::uint32_t word) {
    near = __byte_perm(word, 0xe4e4e4e4u, 0x4040);
    if constexpr (kHalf) {
      const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&near), __floats2half2_rn(960.0f, 960.0f));
      far = *reinterpret_cast<const std::uint32_t*>(&v);
    } else {
      near -= 0x26802680u;  // 0xe400 + zero to 0xbd80 + zero
      far = 0;
    }
  }
};
// (w & mask) | bits, one instruction (two constants in an expression become two).
__device__ __forceinline__ std::uint32_t AndOr(std::uint32_t w, std::uint32_t mask, std::uint32_t bits) {
  std::uint32_t v;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(w), "r"(mask), "r"(bits));
  return v;
}
// A word's codes less the zero point: pairs[j] holds values 2 j and 2 j + 1.
template <bool kHalf>
__device__ __forceinline__ void Pairs(std::uint32_t w, const Zeros<kHalf>& z, std::uint32_t (&pairs)[4]) {
  if constexpr (kHalf) {
    const __half2 near = *reinterpret_cast<const __half2*>(&z.near), far = *reinterpret_cast<const __half2*>(&z.far);
    const __half2 sixteenth = __floats2half2_rn(0.0625f, 0.0625f);
#pragma unroll
    for (int j = 0; j < 4; j += 2, w >>= 8) {
      const std::uint32_t a = AndOr(w, 0x000f000fu, 0x64006400u), b = AndOr(w, 0x00f000f0u, 0x64006400u);
      const __half2 va = __hadd2(*reinterpret_cast<const __half2*>(&a), near);
      const __half2 vb = __hfma2(*reinterpret_cast<const __half2*>(&b), sixteenth, far);
      pairs[j] = *reinterpret_cast<const std::uint32_t*>(&va);
      pairs[j + 1] = *reinterpret_cast<const std::uint32_t*>(&vb);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const std::uint32_t a = AndOr(w >> (4 * j), 0x000f000fu, 0x43004300u);
      const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a), __float2bfloat162_rn(0x1p-11f),
                                       *reinterpret_cast<const __nv_bfloat162*>(&z.near));
      pairs[j] = *reinterpret_cast<const std::uint32_t*>(&v);
    }
  }
}
// Copies that complete behind the thread's back, counted in groups.
template <int kOffset = 0>
__device__ __forceinline__ void CopyAsync16(std::uint32_t shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%2], 16;" ::"r"(shared), "l"(global), "n"(kOffset) : "memory");
}
__device__ __forceinline__ void CopyAsyncCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void CopyAsyncWait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}

// Barriers of some of a CTA's warps: those that wait, and those that only arrive.
__device__ __forceinline__ void BarrierSync(int id, int threads) {
  asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void BarrierArrive(int id, int threads) {
  asm volatile("barrier.cta.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Eight 16-bit values as they are (zero from `valid` on) into shared memory: in the thread's open group of copies
// where they may be copied 16 bytes at a time.
__device__ __forceinline__ void Stage8(void* shared, const void* row, std::int64_t at, int valid, bool vec) {
  const auto* p = static_cast<const unsigned short*>(row) + at;
  if (vec && valid >= 8) {
    CopyAsync16(SharedAddress(shared), p);
    return;
  }
  std::uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = (2 * i) < valid ? p[2 * i] : 0u;
    if ((2 * i) + 1 < valid) w[i] |= static_cast<std::uint32_t>(p[(2 * i) + 1]) << 16;
  }
  *reinterpret_cast<uint4*>(shared) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float Scale(std::uint32_t word) { return __uint_as_float(word & 0xffffff00u); }

// A step of a tile as a lane holds it.
template <int kGroups>
struct StepWeights {
  uint4 a, b;                                // rows g and g + 8
  std::uint32_t word_a[kGroups], word_b[kGroups];
  __device__ __forceinline__ void LoadShared(const std::uint8_t* block, int lane) {
    a = *reinterpret_cast<const uint4*>(block + (lane * 16));
    b = *reinterpret_cast<const uint4*>(block + 512 + (lane * 16));
    const std::uint8_t* words = block + 1024 + ((lane >> 2) * (kGroups * 4));
    if constexpr (kGroups == 1) {
      word_a[0] = *reinterpret_cast<const std::uint32_t*>(words);
      word_b[0] = *reinterpret_cast<const std::uint32_t*>(words + 32);
    } else if constexpr (kGroups == 2) {
      const uint2 wa = *reinterpret_cast<const uint2*>(words), wb = *reinterpret_cast<const uint2*>(words + 64);
      word_a[0] = wa.x, word_a[1] = wa.y, word_b[0] = wb.x, word_b[1] = wb.y;
    } else {
      const uint4 wa = *reinterpret_cast<const uint4*>(words), wb = *reinterpret_cast<const uint4*>(words + 128);
      word_a[0] = wa.x, word_a[1] = wa.y, word_a[2] = wa.z, word_a[3] = wa.w;
      word_b[0] = wb.x, word_b[1] = wb.y, word_b[2] = wb.z, word_b[3] = wb.w;
    }
  }
};

// Two floats in a register pair: multiply-adds take both at once.
using Float2 = unsigned long long;
__device__ __forceinline__ Float2 Pack(float a, float b) {
  Float2 v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void Unpack(Float2 v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ Float2 Fma2(Float2 a, Float2 b, Float2 c) {
  Float2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
// A column tile's sums of a lane: row g's two columns, row g + 8's.
struct Sums {
  Float2 a, b;
  __device__ __forceinline__ Sums() : a(0), b(0) {}
};

// total += the step's products: column quads come from column(nt, i), the 16 bytes that hold
// values 32 i + 8 t .. + 7 of the step for column lane / 4 of column tile nt.
template <bool kHalf, int kGroups, int kTiles, typename Column>
__device__ __forceinline__ void MultiplyStep(const StepWeights<kGroups>& w, int tiles, Sums (&total)[kTiles],
                                             Column column) {
  const std::uint32_t wa[4] = {w.a.x, w.a.y, w.a.z, w.a.w}, wb[4] = {w.b.x, w.b.y, w.b.z, w.b.w};
  constexpr int kBlocks = 4 / kGroups;  // 32-value blocks a group
#pragma unroll
  for (int group = 0; group < kGroups; ++group) {
    const Zeros<kHalf> za(w.word_a[group]), zb(w.word_b[group]);
    float sum[kTiles][4];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      const int i = (group * kBlocks) + b;
      std::uint32_t pa[4], pb[4];
      Pairs<kHalf>(wa[i], za, pa);
      Pairs<kHalf>(wb[i], zb, pb);
#pragma unroll
      for (int nt = 0; nt < kTiles; ++nt) {
        if (nt == 0 || nt < tiles) {
          const uint4 x = column(nt, i);
          if (b == 0) {
            Mma<kHalf, true>(sum[nt], pa[0], pb[0], pa[1], pb[1], x.x, x.y);
          } else {
            Mma<kHalf, false>(sum[nt], pa[0], pb[0], pa[1], pb[1], x.x, x.y);
          }
          Mma<kHalf, false>(sum[nt], pa[2], pb[2], pa[3], pb[3], x.z, x.w);
        }
      }
    }
    const float sa = Scale(w.word_a[group]), sb = Scale(w.word_b[group]);
    const Float2 sa2 = Pack(sa, sa), sb2 = Pack(sb, sb);
#pragma unroll
    for (int nt = 0; nt < kTiles; ++nt) {
      if (nt == 0 || nt < tiles) {
        total[nt].a = Fma2(sa2, Pack(sum[nt][0], sum[nt][1]), total[nt].a);
        total[nt].b = Fma2(sb2, Pack(sum[nt][2], sum[nt][3]), total[nt].b);
      }
    }
  }
}

// A lane's sums of one column tile with a token's columns added up: values[r][j] is row g + 8 r,
// token TokenOf(j); with 2 or 3 pieces only j = 0 counts.  An f16 value's second piece is 2^11 larger.
template <bool kHalf, int kPieces>
__device__ __forceinline__ void FoldColumns(const Sums& sums, float (&values)[2][2]) {
  float total[4];
  Unpack(sums.a, total[0], total[1]);
  Unpack(sums.b, total[2], total[3]);
  if constexpr (kPieces == 1) {
    values[0][0] = total[0], values[0][1] = total[1], values[1][0] = total[2], values[1][1] = total[3];
  } else {
    constexpr float kSecond = kHalf ? 0x1p-11f : 1.0f;
    // (the fourth column of three pieces stands for nothing and may hold anything)
    if (kPieces == 3 && (threadIdx.x & 1) != 0) total[1] = total[3] = 0.0f;
    values[0][0] = fmaf(total[1], kSecond, total[0]);
    values[1][0] = fmaf(total[3], kSecond, total[2]);
    values[0][1] = values[1][1] = 0.0f;
    if constexpr (kPieces == 3) {  // columns 0, 1 in an even lane, 2 in the next
#pragma unroll
      for (int r = 0; r < 2; ++r) values[r][0] += __shfl_xor_sync(0xffffffffu, values[r][0], 1);
    }
  }
}
// The token (within a column tile) of values[.][j] in lane t = lane % 4; every value is valid in
// some lanes more than once with 3 pieces (t and t ^ 1 hold the same).
template <int kPieces>
__device__ __forceinline__ int TokenOf(int t, int j) {
  return kPieces == 1 ? (2 * t) + j : kPieces == 2 ? t : t >> 1;
}
#endif  // __CUDACC__

}  // namespace w4
}  // namespace llmp_b200

#endif  // LLMP_B200_CSRC_W4_CUH_
