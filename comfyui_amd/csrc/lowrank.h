// Products with a narrow side (the rank of an adapter, the experts of a router), 1 to 256 wide, on the matrix cores: operands, their
// transposes in registers, and fp32 values as pairs of bf16.
//
// v_mfma_f32_16x16x32: lane l holds row (column) l % 16 of an operand and its elements k = 8 (l / 16) .. + 7, and of the result column
// l % 16 and rows 4 (l / 16) .. + 3. Which k, row or column of the problem these stand for is free as long as both operands agree: loads are
// 16 bytes along whatever runs contiguously.
//
// fp32 values (the narrow intermediate h, gradients of logits) enter as hi + lo, bf16 each: 16 significant bits, products exact, sums fp32; what is left
// out is 2^-16 of a value. fp16 weights or rows that meet them are hi + lo in bf16 too, which is exact (11 bits in 16, and bf16
// has the range); lo times lo, 2^-16 of the product, is left out. Rows times weights of the same 16-bit type are multiplied as they are.
#pragma once
#include "common.h"
#include "numfmt.h"

namespace lowrank {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct Bf16 {
  static constexpr bool HALF = false;
  static __device__ __forceinline__ f4 mul(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float lo(uint32_t u) { return HdmoeBf16::lo(u); }
  static __device__ __forceinline__ float hi(uint32_t u) { return HdmoeBf16::hi(u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return HdmoeBf16::pack(a, b); }
};

struct F16 {
  static constexpr bool HALF = true;
  static __device__ __forceinline__ f4 mul(u4 a, u4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ float lo(uint32_t u) { return HdmoeF16::lo(u); }
  static __device__ __forceinline__ float hi(uint32_t u) { return HdmoeF16::hi(u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return HdmoeF16::pack(a, b); }
};

// Eight 16-bit values from any address; those from `have` on are 0 and not read.
__device__ __forceinline__ u4 load8(const uint16_t* p) {
  u4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
// Nobody has a part of eight where rows are multiples of eight long: the wave then passes over those loads
__device__ __forceinline__ u4 load8(const uint16_t* p, int have) {
  u4 v = {0, 0, 0, 0};
  if (have >= 8) {
    v = load8(p);
  } else if (have > 0) {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < have) v[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
  }
  return v;
}
__device__ __forceinline__ void store8(uint16_t* p, u4 v, int have) {
  if (have >= 8) {
    __builtin_memcpy(p, &v, 16);
  } else if (have > 0) {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < have) p[j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
  }
}

// v[j] value q <-> v[q] value j: eight rows of eight values become eight columns.
__device__ __forceinline__ void transpose8(u4 (&v)[8]) {
  u4 o[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int w = 0; w < 4; ++w)
      o[j][w] = __builtin_amdgcn_perm(v[2 * w + 1][j / 2], v[2 * w][j / 2], j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = o[j];
}

// v[i] of lane c <-> v[c] of lane i among four neighbouring lanes: 32 instructions. The matrix instructions want one row a lane and its neighbour's
// next to it, memory wants neighbouring lanes on neighbouring addresses: a load or store whose four neighbours take 64 bytes of one row goes through
// the address unit four times as fast as one where every lane has a row of its own (62 accesses each, counted; 16384 x 6912 in and out, rank 64: 147 us).
__device__ __forceinline__ void quad_transpose(u4 (&v)[4]) {
  const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
  for (int i = 0; i < 4; i += 2)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int a = (int)v[i][w], b = (int)v[i + 1][w];
      const int a1 = __builtin_amdgcn_mov_dpp(a, 0xb1, 0xf, 0xf, true), b1 = __builtin_amdgcn_mov_dpp(b, 0xb1, 0xf, 0xf, true);   // the lane's neighbour in its pair
      v[i][w] = (uint32_t)(odd ? b1 : a);
      v[i + 1][w] = (uint32_t)(odd ? b : a1);
    }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int a = (int)v[i][w], b = (int)v[i + 2][w];
      const int a2 = __builtin_amdgcn_mov_dpp(a, 0x4e, 0xf, 0xf, true), b2 = __builtin_amdgcn_mov_dpp(b, 0x4e, 0xf, 0xf, true);   // in the other pair
      v[i][w] = (uint32_t)(high ? b2 : a);
      v[i + 2][w] = (uint32_t)(high ? b : a2);
    }
}

// v[i] of lane l <-> v[c] of lane l - 4 c + 4 i, c = l / 4 % 4: the same among lanes four apart.
__device__ __forceinline__ void row_transpose(u4 (&v)[4]) {
  const bool odd = threadIdx.x & 4, high = threadIdx.x & 8;
#pragma unroll
  for (int i = 0; i < 4; i += 2)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int a = (int)v[i][w], b = (int)v[i + 1][w];
      const int a1 = __builtin_amdgcn_mov_dpp(a, 0x104, 0xf, 0xf, true), b1 = __builtin_amdgcn_mov_dpp(b, 0x114, 0xf, 0xf, true);   // of lane l + 4, l - 4
      v[i][w] = (uint32_t)(odd ? b1 : a);
      v[i + 1][w] = (uint32_t)(odd ? b : a1);
    }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int a = (int)v[i][w], b = (int)v[i + 2][w];
      const int a2 = __builtin_amdgcn_mov_dpp(a, 0x128, 0xf, 0xf, true), b2 = __builtin_amdgcn_mov_dpp(b, 0x128, 0xf, 0xf, true);   // l + 8 or l - 8
      v[i][w] = (uint32_t)(high ? b2 : a);
      v[i + 2][w] = (uint32_t)(high ? b : a2);
    }
}

// Operands of 16 rows and 128 k: lane l loads 16 bytes of row 4 i + l / 4 % 4, k = 8 (4 (l / 16) + l % 4), i = 0 .. 3; transposed, instruction n has
// k = 32 (l / 16) + 8 n .. + 7 of row 4 (l % 4) + l / 4 % 4 in lane l. row_of(l % 16) is that row.
constexpr int K_BLOCK = 128;
__device__ __forceinline__ int row_of(int col) { return (col & 3) * 4 + (col >> 2); }

// Two fp32 values as packed bf16 pairs, hi + lo.
__device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = HdmoeBf16::pack(a, b);
  lo = HdmoeBf16::pack(a - HdmoeBf16::lo(hi), b - HdmoeBf16::hi(hi));
}

// Eight values of type A in bf16: themselves, or hi and lo of fp16 ones.
template <class A>
__device__ __forceinline__ void to_bf16(u4 v, u4& hi, u4& lo) {
  if constexpr (A::HALF) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t h, l;
      split(A::lo(v[w]), A::hi(v[w]), h, l);
      hi[w] = h, lo[w] = l;
    }
  } else {
    hi = v;
  }
}

// c += a (qh + ql) for an operand of type A in bf16 (ah, and al where A is fp16).
template <class A>
__device__ __forceinline__ f4 mul_split(u4 ah, u4 al, u4 qh, u4 ql, f4 c) {
  c = Bf16::mul(ah, ql, c);
  if constexpr (A::HALF) c = Bf16::mul(al, qh, c);
  return Bf16::mul(ah, qh, c);
}

// Sums of `splits` parts, each group of parts in its order and the groups in theirs, rounded once; no parts: zeros. Four values a thread; GROUPS threads share
// them where there are many parts (103 parts of 10240 values 28 us with one, 4 with 16).
struct SumArgs {
  const float* part[2];
  uint16_t* out[2];
  size_t n[2];
  int splits;
  const int32_t* there;     // [splits, groups]: parts that were written, of equal shares of n; NULL: all
  int groups;
};
template <class A, int GROUPS>
static __global__ __launch_bounds__(GROUPS == 1 ? 256 : 64 * GROUPS) void sum_parts_kernel(SumArgs p) {
  constexpr int LANES = GROUPS == 1 ? 256 : 64;
  __shared__ f4 lds[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? 64 : 1];
  const size_t blocks = (p.n[0] + LANES * 4 - 1) / (LANES * 4);
  const int side = blockIdx.x >= blocks, lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const size_t n = p.n[side], i = ((size_t)blockIdx.x - (side ? blocks : 0)) * LANES * 4 + lane * 4;
  f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  const int each = (p.splits + GROUPS - 1) / GROUPS, hi = min(p.splits, (group + 1) * each);
  const float* from = p.part[side] + i;
  if (p.there != nullptr) {
    const size_t share = n / p.groups;
    const size_t end = i + 3 < n ? i + 3 : n - 1;
    const int first = i >= n ? -1 : n < ((size_t)1 << 32) ? (int)((uint32_t)i / (uint32_t)share) : (int)(i / share);
    const int one = __builtin_amdgcn_readfirstlane(first);
    const bool simple = i >= n || (first == one && end < ((size_t)one + 1) * share && i + 4 <= n);
    if (one >= 0 && __all(simple)) {          // the wave's values are of one group: its parts, four at a time
      for (int s0 = group * each; s0 < hi; s0 += 64) {
        const int s = s0 + (threadIdx.x & 63);
        uint64_t left = __ballot(s < hi && p.there[(size_t)s * p.groups + one] != 0);
        while (left != 0) {
          f4 q[4] = {};
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (left != 0) {
              if (i < n) __builtin_memcpy(&q[j], from + (size_t)(s0 + __builtin_ctzll(left)) * n, 16);
              left &= left - 1;
            }
#pragma unroll
          for (int j = 0; j < 4; ++j) v += q[j];
        }
      }
    } else if (i < n) {                       // of several: flags and values of four parts at a time, whatever the flags say
      int of[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const size_t at = i + j < n ? i + j : n - 1;
        of[j] = n < ((size_t)1 << 32) ? (int)((uint32_t)at / (uint32_t)share) : (int)(at / share);
      }
#pragma unroll 4
      for (int s = group * each; s < hi; ++s) {
        f4 q = {0.0f, 0.0f, 0.0f, 0.0f};
        if (i + 4 <= n) {
          __builtin_memcpy(&q, from + (size_t)s * n, 16);
        } else {
          for (int j = 0; j < 4; ++j)
            if (i + j < n) q[j] = from[(size_t)s * n + j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (p.there[(size_t)s * p.groups + of[j]] != 0) v[j] += q[j];
      }
    }
  } else if (i + 4 <= n) {
#pragma unroll 8
    for (int s = group * each; s < hi; ++s) {
      f4 q;
      __builtin_memcpy(&q, from + (size_t)s * n, 16);
      v += q;
    }
  } else if (i < n) {
    for (int s = group * each; s < hi; ++s)
      for (int j = 0; j < 4; ++j)
        if (i + j < n) v[j] += from[(size_t)s * n + j];
  }
  if constexpr (GROUPS > 1) {
    lds[group][lane] = v;
    __syncthreads();
    if (group != 0) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) v += lds[g][lane];
  }
  uint16_t* to = p.out[side] + i;
  const uint32_t o[2] = {A::pack(v[0], v[1]), A::pack(v[2], v[3])};
  if (i + 4 <= n) __builtin_memcpy(to, o, 8);
  else
    for (int j = 0; j < 4; ++j)
      if (i + j < n) to[j] = (uint16_t)(o[j / 2] >> (16 * (j & 1)));
}

template <class A>
static void launch_sum_parts(const SumArgs& p, hipStream_t s) {
  auto blocks = [&](size_t lanes) { return dim3((unsigned)((p.n[0] + lanes * 4 - 1) / (lanes * 4) + (p.n[1] + lanes * 4 - 1) / (lanes * 4))); };
  if (p.splits > 16) hipLaunchKernelGGL((sum_parts_kernel<A, 16>), blocks(64), dim3(1024), 0, s, p);
  else hipLaunchKernelGGL((sum_parts_kernel<A, 1>), blocks(256), dim3(256), 0, s, p);
}

}  // namespace lowrank
