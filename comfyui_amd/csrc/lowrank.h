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
__device__ __forceinline__ u4 load8(const uint16_t* p, int have) {
  if (have >= 8) return load8(p);
  u4 v = {0, 0, 0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < have) v[j / 2] |= (uint32_t)p[j] << (16 * (j & 1));
  return v;
}
__device__ __forceinline__ void store8(uint16_t* p, u4 v, int have) {
  if (have >= 8) {
    __builtin_memcpy(p, &v, 16);
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < have) p[j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
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

// Sums of `splits` parts in their order, rounded once; no parts: zeros.
struct SumArgs {
  const float* part[2];
  uint16_t* out[2];
  size_t n[2];
  int splits;
};
template <class A>
static __global__ __launch_bounds__(256) void sum_parts_kernel(SumArgs p) {
  size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const int side = i >= p.n[0];
  if (side) i -= p.n[0];
  if (i >= p.n[side]) return;
  float v = 0.0f;
  for (int s = 0; s < p.splits; ++s) v += p.part[side][s * p.n[side] + i];
  p.out[side][i] = (uint16_t)A::pack(v, 0.0f);
}

}  // namespace lowrank
