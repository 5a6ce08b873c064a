// Linears in e4m3fn with a scale for each block of 128: activations with one fp32 scale for every 128 consecutive values of a
// row, weights [N,K] with one for every 128 x 128 block (scale_weight [ceil(N/128), ceil(K/128)]):
//   y[r, n] = sum_b s[r, b] * sw[n / 128, b] * ( sum_{k in block b} q[r, k] * w[n, k] ) + bias[n]
// The inner sums run on the matrix cores, the outer one in fp32 on the vector units: a K step is one block, its MFMA starts from
// zero, and the four results a lane gets join its accumulators with one fma each (the lane's column of the MFMA result is a token
// and its rows are features of one weight block, so one product s * sw serves all of them).
//
// The cast of a row block: top = max(max|x|, 2^-96), s = top / 448, q = e4m3fn(x * (448 / top)), every operation rounded to
// fp32 once. 2^-96 keeps both quotients normal numbers. The maximum is taken on the bit patterns, where NaN orders above every
// number: a block that holds NaN becomes NaN, as does one that holds an infinity (0 * inf).
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "numfmt.h"

namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));

constexpr int BLK = 128;                     // values (and K bytes) of a scale block
constexpr int MAX_E = HDMOE_BLOCK_MAX_EXPERTS;
constexpr float TOP_FLOOR = 0x1p-96f;

// ---- cast ---------------------------------------------------------------------------------------------------------
// Sources of a cast: eight values of a lane and the largest magnitude among them as a bit pattern.
template <class Act>
struct Half {   // bf16 or fp16
  u32x4 v;
  __device__ __forceinline__ void load(const void* x, size_t i) { v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(x) + i); }
  __device__ __forceinline__ void clear() { v = u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(v[i] & 0x7fffu, (v[i] >> 16) & 0x7fffu));
    return m;
  }
  static __device__ __forceinline__ float value(uint32_t m) { return Act::lo(m); }
  __device__ __forceinline__ float get(int i) const { return i & 1 ? Act::hi(v[i >> 1]) : Act::lo(v[i >> 1]); }
};
struct Full {   // fp32
  v4f v[2];
  __device__ __forceinline__ void load(const void* x, size_t i) {
    const v4f* const p = reinterpret_cast<const v4f*>(static_cast<const float*>(x) + i);
    v[0] = p[0];
    v[1] = p[1];
  }
  __device__ __forceinline__ void clear() { v[0] = v[1] = v4f{0, 0, 0, 0}; }
  __device__ __forceinline__ uint32_t largest() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(get(i)) & 0x7fffffffu);
    return m;
  }
  static __device__ __forceinline__ float value(uint32_t m) { return __uint_as_float(m); }
  __device__ __forceinline__ float get(int i) const { return v[i >> 2][i & 3]; }
};

// Eight values of a block that 16 lanes hold -> their bytes and the block's scale.
template <class Src>
__device__ __forceinline__ void cast_unit(const Src& x, uint32_t (&o)[2], float& s) {
  uint32_t m = x.largest();
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 16));
  const float top_in = Src::value(m);
  const float top = top_in < TOP_FLOOR ? TOP_FLOOR : top_in;
  const float r = 448.0f / top;
#pragma unroll
  for (int i = 0; i < 2; ++i) o[i] = hdmoe_dev_pack4_e4m3fn(x.get(4 * i) * r, x.get(4 * i + 1) * r, x.get(4 * i + 2) * r, x.get(4 * i + 3) * r);
  s = top / 448.0f;
}

// 16 lanes hold a block of a row, 8 values each; a wave takes 4 neighbouring blocks. Bound by memory: 3.03 bytes per value of 16 bits
// (32768 x 6912: 126 us, 5.4 TB/s).
// bounds: NULL, or only the rows from bounds[0] to bounds[nbounds - 1] are cast.
template <class Src>
__global__ __launch_bounds__(256) void block_cast_kernel(const void* __restrict__ x, int rows, int K, int KB, uint8_t* __restrict__ q,
                                                         float* __restrict__ s, long long ld_s, const int32_t* __restrict__ bounds, int nbounds) {
  const long long n = (long long)rows * KB;
  const long long u = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (u >= n) return;
  const int row = (int)(u / KB), b = (int)(u - (long long)row * KB);
  if (bounds != nullptr && (row < bounds[0] || row >= bounds[nbounds - 1])) return;
  const int k = b * BLK + (threadIdx.x & 15) * 8;
  const bool in = k < K;   // K is a multiple of 16: eight values lie inside or outside together
  Src v;
  v.clear();
  if (in) v.load(x, (size_t)row * K + k);
  uint32_t o[2];
  float scale;
  cast_unit(v, o, scale);
  if (in) *reinterpret_cast<u32x2*>(q + (size_t)row * K + k) = u32x2{o[0], o[1]};
  if ((threadIdx.x & 15) == 0) s[(size_t)b * ld_s + row] = scale;
}

// ---- contraction --------------------------------------------------------------------------------------------------
struct Group {
  const uint8_t* w0;    // [N,K]; gate/up: w1
  const float* s0;
  const uint8_t* w1;    // gate/up: w3
  const float* s1;
  const uint16_t* bias; // [N] or NULL
};

// Rows and sizes that the experts' groups share, and those of the static one.
struct Operand {
  const uint8_t* a;     // e4m3fn rows of K bytes (few rows, cast inside: 16-bit rows of K values)
  const float* sa;      // scale of block b of row r at sa[b * ld_sa + r]
  const int32_t* gather;  // NULL, or sorted row r is row gather[r] >> 1 of a
  long long ld_sa;
  int a_rows;           // rows of a
  int rows;             // rows of the segments (or of the static group)
  int K, N;
  void* out;            // 16-bit [rows,N]; gate/up: e4m3fn [rows,N]
  float* h;             // gate/up of few rows: fp32 [rows,N] in front of the cast
  float* s_out;         // gate/up: scale of block b of row r at s_out[b * ld_out + r]
  long long ld_out;
};

struct BlockArgs {
  Group g[MAX_E + 1];   // the static group is g[E]
  Operand op[2];        // the experts' operand, the static group's
  const int32_t* offsets;
  int E;
  int lds_rows;         // few rows, cast inside: rows that a tile can have (the tile's height at most)
  int parts;            // tiles of 256 rows: 64-row parts that a tile can have (4 at most)
};

__device__ __forceinline__ int swz(int row) { return ((row >> 1) & 7) ^ ((row & 1) << 2); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, bytes, 0x00020000);
}
typedef __attribute__((address_space(3))) void* lds_ptr_t;

struct Tile { int g, row0, rows_here, n0; };

// The list of tiles: group by group (lane g holds group g), in a group bands of GROUP_M row tiles, in a band feature tile by feature
// tile. Blocks congruent mod 8 (one XCD) walk a contiguous eighth of it.
template <int BM, int FEAT>
struct Tiles {
  int begin, end, ntiles, last;   // per lane
  int total;
  __device__ __forceinline__ Tiles(const BlockArgs& args, int lane) {
    begin = end = 0;
    ntiles = 0;
    if (lane < args.E) {
      const int rows = args.op[0].rows;
      begin = min(max(args.offsets[lane], 0), rows);
      end = min(max(args.offsets[lane + 1], begin), rows);
      ntiles = (args.op[0].N + FEAT - 1) / FEAT;
    } else if (lane == args.E) {
      end = args.op[1].rows;
      ntiles = (args.op[1].N + FEAT - 1) / FEAT;
    }
    last = (end - begin + BM - 1) / BM * ntiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(last, d, 64);
      if (lane >= d) last += v;
    }
    total = __builtin_amdgcn_readlane(last, 63);
  }
  // tile L of [0, total)
  __device__ __forceinline__ Tile get(int L) const {
    constexpr int GROUP_M = 4;
    const int g = __ffsll((long long)__ballot(last > L)) - 1;
    const int rb = __builtin_amdgcn_readlane(begin, g), re = __builtin_amdgcn_readlane(end, g), nt = __builtin_amdgcn_readlane(ntiles, g);
    const int mt = (re - rb + BM - 1) / BM;
    L -= __builtin_amdgcn_readlane(last, g) - mt * nt;
    const int nbands = max(1, (mt + GROUP_M / 2) / GROUP_M);
    const int band = min(L / (GROUP_M * nt), nbands - 1);
    const int gm = band == nbands - 1 ? mt - band * GROUP_M : GROUP_M;
    const int within = L - band * GROUP_M * nt;
    const int n = within / gm;
    Tile t;
    t.g = g;
    t.row0 = rb + (band * GROUP_M + within - n * gm) * BM;
    t.rows_here = min(re - t.row0, BM);
    t.n0 = n * FEAT;
    return t;
  }
};

// The lane, formed anew: nothing that depends on it has to live across the K loop, which takes nearly all registers.
__device__ __forceinline__ int lane_now() {
  int v;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(v));
  return v;
}

// The tiles of block_gemm8_kernel: a group's rows are cut into as few tiles of up to `parts` parts of 64 rows as they fill. Blocks are persistent.
// Up to two rounds of them: a group's tiles are as even as parts allow, the groups with the highest ones come first, and the second round is
// dealt backwards, so that who had a high tile gets a low one, over all XCDs by fours (the row tiles of a feature tile): one XCD alone reads
// 0.6 MB/us. More rounds, or tiles of one height: full tiles, an eighth of the list to each XCD, which keeps its rows in L2.
// Four segments of 1021 rows, 2560 x 6912 x 2560: 111-113 us (full tiles by eighths 116); seven of 3001, 2048 x 8192: 72.5 (75.4; the second round to whole
// XCDs 74); 7656 x 3728 x 2752 in tiles of 3 parts 106 (of 4: 137); 16384 rows in four, 6912 x 2560, three rounds: by eighths 322, in turn 336.
template <int FEAT>
struct Deal {
  int begin, end, start, cut, wide;   // per lane: rows of group `lane`, its first tile in the list, its row tiles << 3 | the parts of the lowest, its feature tiles
  int next, then, step, stop;   // this block's next tile, if it is below `stop`, the one after it, and the way to others
  __device__ __forceinline__ Deal(const BlockArgs& args, int lane) {
    begin = end = 0;
    if (lane < args.E) {
      const int rows = args.op[0].rows;
      begin = min(max(args.offsets[lane], 0), rows);
      end = min(max(args.offsets[lane + 1], begin), rows);
    } else if (lane == args.E) {
      end = args.op[1].rows;
    }
    wide = (args.op[lane == args.E ? 1 : 0].N + FEAT - 1) / FEAT;
    const int p = (end - begin + 63) / 64, mt = (p + args.parts - 1) / args.parts, count = mt * wide;
    int total = 0;
    for (int o = 0; o <= args.E; ++o) total += __builtin_amdgcn_readlane(count, o);
    const bool even = total <= 2 * HDMOE_NUM_CU && mt > 0;
    const int low = even ? p / mt : args.parts, high = even ? (p + mt - 1) / mt : min(p, low);
    cut = mt << 3 | low;
    start = 0;
    int top = 0, least = 8;
    for (int o = 0; o <= args.E; ++o) {
      const int n = __builtin_amdgcn_readlane(count, o), h = __builtin_amdgcn_readlane(high, o);
      if (h > high || (h == high && o < lane)) start += n;
      top = max(top, h);
      if (n > 0) least = min(least, h);
    }
    const int slots = (int)(gridDim.x / HDMOE_NUM_XCD), xcd = (int)(blockIdx.x % HDMOE_NUM_XCD), slot = (int)(blockIdx.x / HDMOE_NUM_XCD);
    if (gridDim.x == HDMOE_NUM_CU && total > HDMOE_NUM_CU && total <= 2 * HDMOE_NUM_CU && top > least) {
      auto at = [&](int t) { return (t / 4 * HDMOE_NUM_XCD + xcd) * 4 + t % 4; };
      next = at(slot);
      then = at(2 * slots - 1 - slot);
      step = stop = total;   // no third one
    } else {
      const int each = (total + HDMOE_NUM_XCD - 1) / HDMOE_NUM_XCD;
      next = xcd * each + slot;
      then = next + slots;
      step = slots;
      stop = min((xcd + 1) * each, total);
    }
  }
  __device__ __forceinline__ bool more() const { return next < stop; }
  // The block's next tile
  __device__ __forceinline__ Tile take() {
    constexpr int GROUP_M = 4;
    int L = next;
    next = then;
    then += step;
    const int g = __ffsll((long long)__ballot(L >= start && L < start + (cut >> 3) * wide)) - 1;
    const int rb = __builtin_amdgcn_readlane(begin, g), re = __builtin_amdgcn_readlane(end, g), nt = __builtin_amdgcn_readlane(wide, g);
    const int mt = __builtin_amdgcn_readlane(cut, g) >> 3, low = __builtin_amdgcn_readlane(cut, g) & 7;
    const int more = max((re - rb + 63) / 64 - mt * low, 0);   // row tiles with a part more
    L -= __builtin_amdgcn_readlane(start, g);
    const int nbands = max(1, (mt + GROUP_M / 2) / GROUP_M);
    const int band = min(L / (GROUP_M * nt), nbands - 1);
    const int gm = band == nbands - 1 ? mt - band * GROUP_M : GROUP_M;
    const int within = L - band * GROUP_M * nt;
    const int n = within / gm, m = band * GROUP_M + within - n * gm;
    Tile t;
    t.g = g;
    t.row0 = rb + 64 * (m * low + min(m, more));
    t.rows_here = min(re - t.row0, 64 * (m < more ? low + 1 : low));
    t.n0 = n * FEAT;
    return t;
  }
};

// One block of 128: p = A B^T of 16 x 16. The e4m3fn instruction cuts each product at 2^-13 of the largest of its eight neighbours, which leaves a
// sum off by 6e-5 of itself. That drowns in the rounding of a 16-bit output, but not where the sum is cast again: 0.23 % of an intermediate's
// codes then are a step off (0.003 % with exact products), and the feed-forward's output by 0.0013 of itself: below bf16's rounding, six times fp16's.
// EXACT: the values as fp16, which holds them, at half the rate and behind a conversion; products and sums are fp32. Gate/up has it up to EXACT_ROWS
// rows, where a handful of codes can be much of an output (2560 x 6912, four experts: 2 rows 34.4 us, 33.7 without, gate/up and down; gate/up of
// 64 rows 45 us, 40 without, of a layer of 4 to 32 tokens with its shared expert 46 and 41.5), and on any number where the caller asks for it or the activations are
// fp16 (600 rows in eight segments, 1024 x 1024 x 1024, 30.7 and 27.1; 16384 in four, 2560 x 4096 x 2560, 1258 us, 521 on the 256-row tiles, whose loop has none).
template <bool EXACT>
__device__ __forceinline__ v4f block_product(const v8i& a, const v8i& b) {
  v4f c = {0, 0, 0, 0};
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (EXACT) {
    typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
    auto wide = [](int lo, int hi) -> half8_t {
      const half2_t x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
      const half2_t x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
      return half8_t{x0.x, x0.y, x1.x, x1.y, x2.x, x2.y, x3.x, x3.y};
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(wide(a[2 * i], a[2 * i + 1]), wide(b[2 * i], b[2 * i + 1]), c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  }
#endif
  return c;
}
__device__ __forceinline__ float silu(float g) { return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)); }

// The end of a tile, for a wave that holds acc(f, tt, i) as laid out below: bias, rounding and stores, or SiLU * mul and the cast.
struct BiasWords { u32x4 w[4]; };   // of the lane's 4 FT features
template <int FT>
__device__ __forceinline__ BiasWords load_bias(const Operand& op, const Group& grp, const Tile& t, int wf, int lane) {
  BiasWords b = {};
  const uint16_t* const p = grp.bias;
  if (p != nullptr) {
    const int f0 = t.n0 + wf * FT * 16 + (lane >> 4) * 8;
#pragma unroll
    for (int c = 0; c < FT / 2; ++c)
      if (f0 + c * 32 < op.N) b.w[c] = *reinterpret_cast<const u32x4*>(p + f0 + c * 32);   // N is a multiple of 16
#pragma unroll
    for (int c = 0; c < FT / 2; ++c) asm volatile("" : "+v"(b.w[c]));   // what waits for them does so here, not where there is no bias
  }
  return b;
}

template <class Act, bool SWIGLU, int BM, int WF, int FT, int TT, class Acc>
__device__ __forceinline__ void store_tile(const Operand& op, const BiasWords& bias, const Tile& t, uint8_t* exchange, int wf, int wt, int lane, Acc acc) {
  const int N = op.N, quad = lane >> 4;
  constexpr int OUTSIDE = (int)0x80000000u, WT = BM / (TT * 16);
  if constexpr (!SWIGLU) {
    const int f0 = t.n0 + wf * FT * 16 + quad * 8;    // eight features from f0 + 32 c on
    // rows of the tile; what lies past its rows or features gets an offset past the buffer and is not written
    const __amdgpu_buffer_rsrc_t out = make_rsrc(static_cast<uint16_t*>(op.out) + (size_t)t.row0 * N, (uint32_t)t.rows_here * (uint32_t)N * 2u);
#pragma unroll
    for (int c = 0; c < FT / 2; ++c) {
      const int f = f0 + c * 32;
      const u32x4 b = bias.w[c];
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const int r = (tt * WT + wt) * 16 + (lane & 15);
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = Act::pack(acc(2 * c + i / 2, tt, i % 2 * 2) + Act::lo(b[i]), acc(2 * c + i / 2, tt, i % 2 * 2 + 1) + Act::hi(b[i]));
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4i, v), out, r < t.rows_here && f < N ? (r * N + f) * 2 : OUTSIDE, 0, 0);
      }
    }
  } else {
    // silu(g) * u, then the cast of the 128 features: 2 FT in a lane, 8 FT in the four lanes of a token, WF waves. The exponential and
    // the reciprocal are the hardware's, 1 ulp each beside half an e4m3 step of 2^-4.
    uint32_t* const tops = reinterpret_cast<uint32_t*>(exchange);   // [WF][BM]
    float h[TT][FT * 2];
    uint32_t top[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      top[tt] = 0;
#pragma unroll
      for (int f = 0; f < FT / 2; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = silu(acc(f, tt, i)) * acc(f + FT / 2, tt, i);
          h[tt][f * 4 + i] = v;
          top[tt] = max(top[tt], __float_as_uint(v) & 0x7fffffffu);
        }
      top[tt] = max(top[tt], (uint32_t)__shfl_xor((int)top[tt], 16, 64));
      top[tt] = max(top[tt], (uint32_t)__shfl_xor((int)top[tt], 32, 64));
      if (quad == 0) tops[wf * BM + (tt * WT + wt) * 16 + lane] = top[tt];
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
    const int f0 = t.n0 + wf * FT * 8 + quad * FT * 2;
    const __amdgpu_buffer_rsrc_t out = make_rsrc(static_cast<uint8_t*>(op.out) + (size_t)t.row0 * N, (uint32_t)t.rows_here * (uint32_t)N);
    const __amdgpu_buffer_rsrc_t outs = make_rsrc(op.s_out + (size_t)(t.n0 / BLK) * op.ld_out + t.row0, (uint32_t)t.rows_here * 4u);
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const int r = (tt * WT + wt) * 16 + (lane & 15);
#pragma unroll
      for (int w = 1; w < WF; ++w) top[tt] = max(top[tt], tops[(wf + w) % WF * BM + r]);
      const float both = __uint_as_float(top[tt]);
      const float tp = both < TOP_FLOOR ? TOP_FLOOR : both;
      const float m = 448.0f / tp;
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(tp / 448.0f), outs, r < t.rows_here && wf == 0 && quad == 0 ? r * 4 : OUTSIDE, 0, 0);
      const int at = r < t.rows_here && f0 < N ? r * N + f0 : OUTSIDE;
      int v[FT / 2];
#pragma unroll
      for (int i = 0; i < FT / 2; ++i)
        v[i] = (int)hdmoe_dev_pack4_e4m3fn(h[tt][4 * i] * m, h[tt][4 * i + 1] * m, h[tt][4 * i + 2] * m, h[tt][4 * i + 3] * m);
      if constexpr (FT == 8) __builtin_amdgcn_raw_buffer_store_b128(v4i{v[0], v[1], v[2], v[3]}, out, at, 0, 0);
      else __builtin_amdgcn_raw_buffer_store_b64(u32x2{(uint32_t)v[0], (uint32_t)v[1]}, out, at, 0, 0);
    }
  }
}

// The feature (of its wave's) that row r of MFMA tile f holds: one that puts 8 consecutive features (gate/up: 2 FT) in a lane's
// accumulators and 32 (8 FT) in the four lanes of a token, so that stores are 16 bytes each and 64 of them lie next to each other. Gate/up:
// tiles below FT / 2 are w1, the others the same features of w3.
template <bool SWIGLU, int FT>
__device__ __forceinline__ int tile_feature(int f, int r) {
  return SWIGLU ? (r >> 2) * FT * 2 + f % (FT / 2) * 4 + (r & 3) : (f >> 1) * 32 + (r >> 2) * 8 + (f & 1) * 4 + (r & 3);
}

// Tiles of 128 tokens x 128 features (gate/up: 64 tokens x 128 of w1 and of w3), for launches whose 256-row tiles would leave CUs idle.
// WF x WT waves, each FT * 16 weight rows x TT * 16 tokens in MFMA tiles of 16 x 16 x 128; the results of a weight tile join the
// accumulators behind the MFMAs of the next one. STAGES K steps in LDS, STAGES - 1 of them asked for ahead: with two, two blocks share
// a CU and one fills the other's waits; with more, for launches that have at most a block for every CU, a step does not last as long as
// its loads are on their way (128 x 6912 x 2560: 32 us, 41.5 with two stages).
// Gate/up: Act says whether products are exact (HdmoeF16) or not; nothing of its type is read or written.
template <class Act, bool SWIGLU, int WF, int WT, int FT, int TT, int STAGES>
__global__ __launch_bounds__(64 * WF * WT, STAGES == 2 ? 4 : 2) void block_gemm_kernel(const BlockArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)   // (the host pass leaves out stubs of kernels whose lambdas hold arrays of dependent size)
  constexpr int NT = 64 * WF * WT;
  constexpr int BM = WT * TT * 16, BN = WF * FT * 16;
  constexpr int FEAT = SWIGLU ? BN / 2 : BN;
  static_assert(FEAT == BLK, "one block of weight scales, one of the cast output");
  constexpr int STAGE = (BM + BN) * BLK + 2048;      // and the scales of the tokens
  constexpr int ROWS_PER_LOAD = NT / 8;               // rows that one load of every wave moves
  constexpr int LA = BM / ROWS_PER_LOAD, LB = BN / ROWS_PER_LOAD;
  static_assert(LA * ROWS_PER_LOAD == BM && LB * ROWS_PER_LOAD == BN && ROWS_PER_LOAD % 16 == 0, "whole loads");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave % WF, wt = wave / WF;

  const Tiles<BM, FEAT> tiles(args, lane);
  const int per_xcd = (tiles.total + HDMOE_NUM_XCD - 1) / HDMOE_NUM_XCD;
  const int slot = blockIdx.x / HDMOE_NUM_XCD;
  const int L = (int)(blockIdx.x % HDMOE_NUM_XCD) * per_xcd + slot;
  if (slot >= per_xcd || L >= tiles.total) return;
  const Tile t = tiles.get(L);
  const Group& grp = args.g[t.g];
  const Operand& op = args.op[t.g == args.E ? 1 : 0];
  const int K = op.K, N = op.N;
  const int KB = (K + BLK - 1) / BLK;
  const int32_t* const gather = op.gather;
  const int a_rows = op.a_rows;

  // ---- global -> LDS: lane i of a load lands in 16-byte chunk i & 7 of row i >> 3 and fetches the chunk that the swizzle puts there.
  // Rows and chunks that do not exist get an offset past the buffer and read as zero.
  const int ld_row = wave * 8 + (lane >> 3);
  const int ld_chunk = (lane & 7) ^ swz(ld_row);
  constexpr int OUTSIDE = (int)0x80000000u;
  int va[LA], vb[LB];
  const __amdgpu_buffer_rsrc_t ra = gather != nullptr ? make_rsrc(op.a, (uint32_t)a_rows * (uint32_t)K)
                                                      : make_rsrc(op.a + (size_t)t.row0 * K, (uint32_t)t.rows_here * (uint32_t)K);
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = j * ROWS_PER_LOAD + ld_row;
    va[j] = OUTSIDE;
    if (r < t.rows_here) {
      const int from = gather != nullptr ? gather[t.row0 + r] >> 1 : r;   // a bad index of the permutation reads as a row of zeros
      if (gather == nullptr || (unsigned)from < (unsigned)a_rows) va[j] = from * K + ld_chunk * 16;
    }
  }
  const int feats = min(N - t.n0, FEAT);
  const __amdgpu_buffer_rsrc_t rb0 = make_rsrc(grp.w0 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K);
  const __amdgpu_buffer_rsrc_t rb1 = SWIGLU ? make_rsrc(grp.w1 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K) : rb0;
  // gate/up: whether load j of this wave fetches rows of w3 (one answer for its 8 rows)
  auto upper = [&](int j) { return SWIGLU && ((j * ROWS_PER_LOAD + wave * 8) / 16) % FT >= FT / 2; };
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int p = j * ROWS_PER_LOAD + ld_row;         // LDS row of the weight tile
    const int w = p / (FT * 16), f = w * (SWIGLU ? FT * 8 : FT * 16) + tile_feature<SWIGLU, FT>(p / 16 % FT, p & 15);
    vb[j] = f < feats ? f * K + ld_chunk * 16 : OUTSIDE;
  }
  // Scales go through LDS as well, 64 words a wave: of the tile's tokens, and (one value for all lanes) of the weight block by wave 7,
  // gate/up: of w3's by wave 6. The other waves ask for none. (Scalar loads return out of order with LDS reads, and a wait for one is a
  // wait for all.)
  const int ld_s = __builtin_amdgcn_readfirstlane((int)op.ld_sa * 4);
  const bool of_w = wave == 7 || (SWIGLU && wave == 6);
  const float* const sw = (SWIGLU && wave == 6 ? grp.s1 : grp.s0) + (size_t)(t.n0 / BLK) * KB;
  const __amdgpu_buffer_rsrc_t rs = of_w ? make_rsrc(sw, (uint32_t)KB * 4u) : make_rsrc(op.sa, (uint32_t)(KB - 1) * (uint32_t)ld_s + (uint32_t)a_rows * 4u);
  const int s_step = __builtin_amdgcn_readfirstlane(of_w ? 4 : ld_s);
  int tok = of_w ? 0 : OUTSIDE;
  {
    const int r = wave * 64 + lane;
    if (r < t.rows_here && r < BM) {
      const int from = gather != nullptr ? gather[t.row0 + r] >> 1 : t.row0 + r;
      if ((unsigned)from < (unsigned)a_rows) tok = from * 4;
    }
  }
  static_assert(BM <= 6 * 64, "waves 6 and 7 load the weights' scales");
  // The loads are written by hand so that the compiler, which takes any of them for one that a later LDS read may want, does not wait.
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)smem;
  auto to_lds = [](const __amdgpu_buffer_rsrc_t& r, uint32_t lds, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(lds), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
  };
  // load i of the step kb into `stage`
  auto load = [&](int i, int stage, int kb) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + wave * 8 * BLK);
    const int k0 = kb * BLK;
    const int mask = k0 + ld_chunk * 16 < K ? 0 : OUTSIDE;   // (none past the last step)
    if (i < LA) {
      to_lds(ra, at + i * ROWS_PER_LOAD * BLK, va[i] | mask, k0);
    } else if (i < LA + LB) {
      const int j = i - LA;
      if (upper(j)) to_lds(rb1, at + (BM + j * ROWS_PER_LOAD) * BLK, vb[j] | mask, k0);
      else to_lds(rb0, at + (BM + j * ROWS_PER_LOAD) * BLK, vb[j] | mask, k0);
    } else {
      const uint32_t ss = __builtin_amdgcn_readfirstlane(lds0 + stage * STAGE + (BM + BN) * BLK + wave * 256);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" : : "s"(ss), "v"(tok), "s"(rs), "s"(min(kb, KB - 1) * s_step) : "memory", "m0");
    }
  };
  constexpr int LOADS = LA + LB + 1;
  auto issue = [&](int stage, int kb) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) load(i, stage, kb);
  };

  const int fr = lane & 15, fs = swz(fr), c0 = lane >> 4;
  v4f acc[FT][TT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[f][tt] = v4f{0, 0, 0, 0};
  // What a wave reads of a step. The addresses are those of the step's stage and move on in place: formed anew for every read they take
  // registers that reads on their way are still to fill, and each of those is waited for.
  struct Step { v8i a[FT], b[TT]; float x[TT], s0, s1; };
  typedef const __attribute__((address_space(3))) v4i* lds_v4i;
  typedef const __attribute__((address_space(3))) float* lds_float;
  uint32_t at_a[2], at_b[2], at_x = lds0 + (BM + BN) * BLK + (wt * 16 + fr) * 4, at_s = lds0 + (BM + BN) * BLK + lane * 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = ((c0 + 4 * h) ^ fs) << 4;
    at_b[h] = lds0 + (wt * 16 + fr) * BLK + c;
    at_a[h] = lds0 + (BM + wf * FT * 16 + fr) * BLK + c;
  }
  int stage = 0;
  auto read = [&](Step& st) {
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) st.x[tt] = *(lds_float)(at_x + tt * WT * 64);
    st.s0 = *(lds_float)(at_s + 7 * 256);
    st.s1 = SWIGLU ? *(lds_float)(at_s + 6 * 256) : 0.0f;
    auto frag = [&](const uint32_t (&at)[2], int off) -> v8i {
      const v4i lo = *(lds_v4i)(at[0] + off), hi = *(lds_v4i)(at[1] + off);
      return v8i{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    };
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) st.b[tt] = frag(at_b, tt * WT * 16 * BLK);
#pragma unroll
    for (int f = 0; f < FT; ++f) st.a[f] = frag(at_a, f * 16 * BLK);
    const int on = stage + 1 == STAGES ? -(STAGES - 1) * STAGE : STAGE;
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    at_x += on;
    at_s += on;
#pragma unroll
    for (int h = 0; h < 2; ++h) { at_a[h] += on; at_b[h] += on; }
  };
  // (with one block on a CU the loads go between the MFMAs: a burst of them in front keeps the waves at the memory queue)
  auto multiply = [&](const Step& st, int next, int kb) {
    v4f p[2][TT];
    float m0[TT], m1[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) { m0[tt] = st.x[tt] * st.s0; m1[tt] = st.x[tt] * st.s1; }
    auto join = [&](int f) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][tt][i] = __builtin_fmaf(p[f & 1][tt][i], SWIGLU && f >= FT / 2 ? m1[tt] : m0[tt], acc[f][tt][i]);
    };
#pragma unroll
    for (int f = 0; f < FT; ++f) {
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) p[f & 1][tt] = block_product<SWIGLU && std::is_same_v<Act, HdmoeF16>>(st.a[f], st.b[tt]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = f * LOADS / FT; i < (f + 1) * LOADS / FT; ++i)
        if (STAGES > 2) load(i, next, kb);
      if (f > 0) join(f - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    join(FT - 1);
  };
  auto ring = [](int stage) { return stage + 1 == STAGES ? 0 : stage + 1; };

#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st) issue(st, st);
  int next = STAGES - 1;
  if constexpr (STAGES == 2) {
    for (int kb = 0; kb < KB; ++kb) {
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" : : : "memory");
      Step st;
      read(st);
      issue(next, kb + 1);
      next = ring(next);
      multiply(st, 0, KB);
    }
  } else {
    // a step's operands are read while the one before is multiplied
    Step st[2];
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((STAGES - 2) * LOADS) : "memory");
    read(st[0]);
    auto step = [&](Step& here, Step& there, int kb) {
      asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" : : "n"((STAGES - 3) * LOADS) : "memory");
      read(there);
      __builtin_amdgcn_sched_barrier(0);
      multiply(here, next, kb + STAGES - 1);
      next = ring(next);
    };
    int kb = 0;
    for (; kb + 2 <= KB; kb += 2) {
      step(st[0], st[1], kb);
      step(st[1], st[0], kb + 1);
    }
    if (kb < KB) step(st[0], st[1], kb);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");   // LDS is read and written no more
  store_tile<Act, SWIGLU, BM, WF, FT, TT>(op, SWIGLU ? BiasWords{} : load_bias<FT>(op, grp, t, wf, lane), t, smem, wf, wt, lane,
                                          [&](int f, int tt, int i) -> float { return acc[f][tt][i]; });
#endif
}

// Tiles of 256 x 256 (gate/up: 256 x 128 of w1 and of w3) with the K loop of gen_block_fp8.py, for segments that fill them; one block of 160 KiB of
// LDS per CU. The first loads of a block's next tile go out before the end of this one. Bound by MFMA issue at the clock that the power limit
// leaves: a K step is 2470 cycles of which the MFMAs take 2048, at 1.6 GHz, and a tile's start and stores 6 us (16384 x 4096 x 8192 454-480 us,
// 2.3-2.4 PFLOP/s; the 8-wave loop left to the compiler 650). Two waves a SIMD on 128 x 64 each: 4 x 8 tiles' accumulators and a step's fragments
// are all of the 256 registers.
#include "block_fp8_asm.inc"
#define HDMOE_BLOCK_ACC \
  "={v[128:143]}"(acc[0]), "={v[144:159]}"(acc[1]), "={v[160:175]}"(acc[2]), "={v[176:191]}"(acc[3]), "={v[192:207]}"(acc[4]), \
      "={v[208:223]}"(acc[5]), "={v[224:239]}"(acc[6]), "={v[240:255]}"(acc[7])
template <class Act, bool SWIGLU>
__global__ __launch_bounds__(512) void block_gemm8_kernel(const BlockArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int BM = 256, FEAT = SWIGLU ? 128 : 256, TT = 4;
  constexpr int OUTSIDE = (int)0x80000000u;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];   // tokens of two stages, weights of three, 32 KiB each

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wf = wave & 1, wt = wave >> 1;

  Deal<FEAT> tiles(args, lane);
  if (!tiles.more()) return;

  typedef int v32i __attribute__((ext_vector_type(32)));
  typedef float v16f __attribute__((ext_vector_type(16)));
  typedef float v8f __attribute__((ext_vector_type(8)));
  auto sgpr = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  auto rsrc = [&](const void* p, uint32_t bytes) -> v4i {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    return v4i{sgpr((int)(uint32_t)a), sgpr((int)((uint32_t)(a >> 32) & 0xffffu)), sgpr((int)bytes), 0x00020000};
  };
  auto buffer = [](const v4i& r) {
    return make_rsrc(reinterpret_cast<const void*>((uint64_t)(uint32_t)r.y << 32 | (uint32_t)r.x), (uint32_t)r.z);
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)smem;

  // What the loop is given for a tile, and its first two steps on their way into LDS; the registers' names are those of gen_block_fp8.py.
  struct Source { v4i ra, rb0, rb1, rs, rw0, rw1; int KB, ld_s; };
  int tail = 0;
  v4i addr, tok, va, vb;
  v4f x0, sx;
  float s0, s1 = 0.0f, sw[2] = {0.0f, 0.0f};
  auto start = [&](const Tile& t, int lane) -> Source {
    const Group& grp = args.g[t.g];
    const Operand& op = args.op[t.g == args.E ? 1 : 0];
    const int K = op.K, N = op.N;
    const int32_t* const gather = op.gather;
    const int a_rows = op.a_rows;
    const int KB = (K + BLK - 1) / BLK;
    const int feats = min(N - t.n0, FEAT);
    const int nblk = SWIGLU ? t.n0 / BLK : min(t.n0 / BLK + wf, (N - 1) / BLK);
    Source s;
    s.KB = KB;
    s.ra = gather != nullptr ? rsrc(op.a, (uint32_t)a_rows * (uint32_t)K) : rsrc(op.a + (size_t)t.row0 * K, (uint32_t)t.rows_here * (uint32_t)K);
    s.rb0 = rsrc(grp.w0 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K);
    s.rb1 = SWIGLU ? rsrc(grp.w1 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K) : s.rb0;
    s.ld_s = sgpr((int)op.ld_sa * 4);   // bytes between the scales of two blocks of a row
    s.rs = rsrc(op.sa, (uint32_t)(KB - 1) * (uint32_t)s.ld_s + (uint32_t)a_rows * 4u);
    s.rw0 = rsrc(grp.s0 + (size_t)nblk * KB, (uint32_t)KB * 4u);
    s.rw1 = SWIGLU ? rsrc(grp.s1 + (size_t)nblk * KB, (uint32_t)KB * 4u) : s.rw0;

    const int ld_row = wave * 8 + (lane >> 3);
    const int ld_chunk = (lane & 7) ^ swz(ld_row);
    tail = (KB - 1) * BLK + ld_chunk * 16 < K ? 0 : OUTSIDE;   // of the last block this lane fetches nothing
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = j * 64 + ld_row;
      va[j] = tok[j] = OUTSIDE;
      if (r < t.rows_here) {
        const int from = gather != nullptr ? gather[t.row0 + r] >> 1 : r;   // a bad index of the permutation reads as a row of zeros
        if (gather == nullptr || (unsigned)from < (unsigned)a_rows) va[j] = from * K + ld_chunk * 16;
      }
      const int f = (r >> 7) * (SWIGLU ? 64 : 128) + tile_feature<SWIGLU, 8>(r / 16 % 8, r & 15);
      vb[j] = f < feats ? f * K + ld_chunk * 16 : OUTSIDE;
      const int x = (j * 4 + wt) * 16 + (lane & 15);
      if (x < t.rows_here) {
        const int from = gather != nullptr ? gather[t.row0 + x] >> 1 : t.row0 + x;
        if ((unsigned)from < (unsigned)a_rows) tok[j] = from * 4;
      }
    }
    // the scales first: requests come back in order
    auto word = [&](const v4i& r, int off, int so) { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(buffer(r), off, so, 0)); };
    const int second = min(1, KB - 1);
    s0 = word(s.rw0, 0, 0);
    if (SWIGLU) s1 = word(s.rw1, 0, 0);
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      x0[tt] = word(s.rs, tok[tt], 0);
      sx[tt] = word(s.rs, tok[tt], second * s.ld_s);
    }
    sw[0] = word(s.rw0, 0, second * 4);
    if (SWIGLU) sw[1] = word(s.rw1, 0, second * 4);
    asm volatile("" : : : "memory");
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int mask = st >= KB ? OUTSIDE : st == KB - 1 ? tail : 0;
      uint8_t* const sa = smem + st * 32768 + wave * 1024;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer(s.ra), (lds_ptr_t)(sa + j * 8192), 16, va[j] | mask, st * BLK, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer(SWIGLU && (j & 1) ? s.rb1 : s.rb0), (lds_ptr_t)(sa + 65536 + j * 8192), 16, vb[j] | mask, st * BLK, 0, 0);
      }
    }
    const int fr = lane & 15, quad = lane >> 4, fs = swz(fr);
    if (KB <= 2) tail = OUTSIDE;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = ((quad + 4 * h) ^ fs) * 16;
      addr[h] = (int)lds0 + (wt * 16 + fr) * BLK + c;
      addr[2 + h] = (int)lds0 + 65536 + (wf * 128 + fr) * BLK + c;
    }
    return s;
  };

  Tile cur = tiles.take();
  Source src = start(cur, lane);
  const int ldsw = sgpr((int)lds0 + wave * 1024);
  // between a tile's first loads and its loop: nothing, or the stores of the tile before, which need not have arrived
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" : : : "memory");
  for (;;) {
    // the first step's factors; not before the end of the tile before, which would wait for all of the loads above
    asm volatile("" : "+v"(x0), "+v"(s0), "+v"(s1));
    v4f m0, m1 = {};
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      m0[tt] = x0[tt] * s0;
      if (SWIGLU) m1[tt] = x0[tt] * s1;
    }
    v16f acc[8];
    const int second = min(1, src.KB - 1);
    int n = sgpr(src.KB), left = sgpr(src.KB - 2), so = sgpr(BLK), ss = sgpr(second * src.ld_s), so_w = sgpr(second * 4), ws = sgpr(0);
    v32i fa, fb;
    v8f last;
    v16f p;
#define HDMOE_BLOCK_LOOP(TEXT) \
    asm volatile(TEXT : HDMOE_BLOCK_ACC, "={v[96:127]}"(fb), "={v[64:95]}"(fa), "={v[48:63]}"(p), "={v[40:47]}"(last), "+{v[32:35]}"(m0), "+{v[36:39]}"(m1), \
                        "+{v[26:29]}"(sx), "+{v30}"(sw[0]), "+{v31}"(sw[1]), "+{v8}"(tail), "+{v[10:13]}"(addr), "+{v[18:21]}"(va), "+{v[22:25]}"(vb), \
                        [n] "+s"(n), [left] "+s"(left), [so] "+s"(so), [ss] "+s"(ss), [sw] "+s"(so_w), [ws] "+s"(ws) \
                      : "{v[14:17]}"(tok), [ra] "s"(src.ra), [rb0] "s"(src.rb0), [rb1] "s"(src.rb1), [rs] "s"(src.rs), [rw0] "s"(src.rw0), [rw1] "s"(src.rw1), \
                        [ssi] "s"(src.ld_s), [ldsw] "s"(ldsw), [steps] "s"(src.KB), [nt] "s"((cur.rows_here + 63) / 64) \
                      : "memory", "m0", "scc", "s60", "s61", "s62")
    if constexpr (SWIGLU) HDMOE_BLOCK_LOOP(HDMOE_BLOCK_SWIGLU);
    else HDMOE_BLOCK_LOOP(HDMOE_BLOCK_PLAIN);

    const Tile done = cur;
    const bool more = tiles.more();
    if (more) {
      cur = tiles.take();
      src = start(cur, lane_now());
    }
    asm volatile("" : : : "memory");
    const Operand& op = args.op[done.g == args.E ? 1 : 0];
    const BiasWords bias = SWIGLU ? BiasWords{} : load_bias<8>(op, args.g[done.g], done, wf, lane_now());
    store_tile<Act, SWIGLU, BM, 2, 8, TT>(op, bias, done, smem + 131072, wf, wt, lane_now(),
                                    [&](int f, int tt, int i) -> float { return acc[f][tt * 4 + i]; });
    if (!more) return;
    // a tile ends in 16 stores (gate/up: 8); the loads in front of them have come back
    if constexpr (SWIGLU) asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" : : : "memory");
    else asm volatile("s_waitcnt vmcnt(16)\n\ts_barrier" : : : "memory");
  }
#endif
}

// ---- few rows -----------------------------------------------------------------------------------------------------
// Segments of up to a few dozen rows: the weights are read once from memory. A wave multiplies FT strips of 16 weight rows with TT * 16
// tokens; KW waves deal the K blocks of the same strips out, each through a ring of its own in LDS, so none waits for another before
// the end, where their sums meet.
// What a CU fetches in a microsecond is the bound. Lanes that hold a row each would ask for 16 bytes of a cache line 4 at a time, one line a
// cycle: 39 KB/us. Through LDS 8 neighbouring lanes ask for 128 bytes of a row: 80 KB/us (48 x 6912 x 2560
// with the cast 10.7 us, 15.7 the other way; 128 rows in four segments 25.6 and 30.0, the weights at 3.6 TB/s).
// More strips a wave read the activations less often (they come out of L2, 16 TT rows for every 16 FT of the weights), fewer make more
// blocks: a CU has only so many requests on their way, so all 256 have to take part.
//   gate/up: half of the strips are w1's, half the same features of w3; silu(g) * u leaves in fp32, and a second launch casts it. (One
//            launch needs the 128 features of a cast block in one thread block, 54 blocks an expert at 6912.)
// CAST: the activations are 16-bit rows; the block casts its own into LDS (rows of K + 16 bytes: 16 rows then hit all banks) while the
// first weights are on their way, instead of a launch of its own in front.
constexpr int STREAM_WAVES = 4, CAST_UNITS = 128;   // CAST: blocks of 128 values that a thread block can cast
// Blocks that rings are sized for on a CU: two where half of the LDS holds enough on its way, so that one starts while the other streams. What the
// blocks cast for themselves comes on top (stream_blocks).
constexpr int stream_rings(int ft, int tt, bool cast) { return cast || ft * tt <= 2 ? 2 : 1; }
// Of a wave: a K block of weights and activations with their scales, and how many of them its ring has
constexpr int stream_slot(int ft, int tt, bool swiglu, bool cast) { return 2048 * (ft + (cast ? 0 : tt)) + 256 * (1 + (swiglu ? 1 : 0) + (cast ? 0 : 1)); }
constexpr int stream_depth(int ft, int tt, bool swiglu, bool cast) {
  const int budget = stream_rings(ft, tt, cast) == 1 ? 159744 : cast ? 73728 : 81920, n = budget / (STREAM_WAVES * stream_slot(ft, tt, swiglu, cast));
  return n > 8 ? 8 : n;
}

// CAST: cast rows and scales, and in front of the 16-bit ones
__host__ __device__ constexpr int stream_cast_bytes(int rows, int KB) { return (rows * (KB * BLK + 16 + KB * 4) + 255) / 256 * 256; }
constexpr int stream_raw_bytes(int rows, int KB) { return (rows * KB + 4 * STREAM_WAVES - 1) / (4 * STREAM_WAVES) * STREAM_WAVES * 1024; }
// LDS of a block: its waves' rings, whose place their sums take at the end, and where it casts `rows` rows (at most) of KB blocks for itself, these
constexpr int stream_lds(int ft, int tt, bool swiglu, bool cast, int rows, int KB) {
  return STREAM_WAVES * stream_depth(ft, tt, swiglu, cast) * stream_slot(ft, tt, swiglu, cast) + (cast ? stream_cast_bytes(rows, KB) + stream_raw_bytes(rows, KB) : 0);
}
// Blocks that a CU holds at once. Casting, two of gate/up only for one row (2560 values: 80640 bytes; two rows 87296).
constexpr int stream_blocks(int ft, int tt, bool swiglu, bool cast, int rows, int KB) { return 163840 / stream_lds(ft, tt, swiglu, cast, rows, KB) >= 2 ? 2 : 1; }

template <class Act, bool SWIGLU, int FT, int TT, bool CAST>
__global__ __launch_bounds__(64 * STREAM_WAVES) void block_stream_kernel(const BlockArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int KW = STREAM_WAVES;
  static_assert(!SWIGLU || FT % 2 == 0, "w1 and w3 by halves");
  constexpr int BM = TT * 16;
  constexpr int STRIPS = SWIGLU ? FT / 2 : FT;   // of one matrix
  constexpr int FEAT = 16 * STRIPS;
  constexpr int XT = CAST ? 0 : TT;              // strips of activations in a slot
  constexpr int SLOT = stream_slot(FT, TT, SWIGLU, CAST), DEPTH = stream_depth(FT, TT, SWIGLU, CAST), RING = DEPTH * SLOT;
  constexpr int LOADS = 2 * (FT + XT) + 1 + (SWIGLU ? 1 : 0) + (CAST ? 0 : 1);   // of a step
  static_assert(DEPTH >= 2 && (DEPTH - 1) * LOADS < 64, "two K blocks at least, and their loads counted in 6 bits");
  constexpr int OUTSIDE = (int)0x80000000u;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int fr = lane & 15, quad = lane >> 4;
  const int kw = wave;

  const Tiles<BM, FEAT> tiles(args, lane);
  const int per_xcd = (tiles.total + HDMOE_NUM_XCD - 1) / HDMOE_NUM_XCD;
  const int slot_x = blockIdx.x / HDMOE_NUM_XCD;
  const int L = (int)(blockIdx.x % HDMOE_NUM_XCD) * per_xcd + slot_x;
  if (slot_x >= per_xcd || L >= tiles.total) return;
  const Tile t = tiles.get(L);
  const Group& grp = args.g[t.g];
  const Operand& op = args.op[t.g == args.E ? 1 : 0];
  const int K = op.K, N = op.N;
  const int KB = (K + BLK - 1) / BLK;
  const int32_t* const gather = op.gather;
  const int a_rows = op.a_rows;

  // global -> LDS: lane i of a load lands in 16-byte chunk i & 7 of row i >> 3 of a strip's half and fetches the chunk that the swizzle puts
  // there. Rows and chunks that do not exist read as zero.
  const int feats = min(N - t.n0, FEAT);
  const __amdgpu_buffer_rsrc_t rw0 = make_rsrc(grp.w0 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K);
  const __amdgpu_buffer_rsrc_t rw1 = SWIGLU ? make_rsrc(grp.w1 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K) : rw0;
  const __amdgpu_buffer_rsrc_t rs0 = make_rsrc(grp.s0 + (size_t)(t.n0 / BLK) * KB, (uint32_t)KB * 4u);
  const __amdgpu_buffer_rsrc_t rs1 = SWIGLU ? make_rsrc(grp.s1 + (size_t)(t.n0 / BLK) * KB, (uint32_t)KB * 4u) : rs0;
  const __amdgpu_buffer_rsrc_t ra = gather != nullptr ? make_rsrc(op.a, (uint32_t)a_rows * (uint32_t)K)
                                                      : make_rsrc(op.a + (size_t)t.row0 * K, (uint32_t)t.rows_here * (uint32_t)K);
  const int ld_s = __builtin_amdgcn_readfirstlane((int)op.ld_sa * 4);
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(op.sa, (uint32_t)(KB - 1) * (uint32_t)ld_s + (uint32_t)a_rows * 4u);
  int vw[2], last[2], vx[CAST ? 1 : TT][2], tok = OUTSIDE;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = j * 8 + (lane >> 3), c = (lane & 7) ^ swz(r);
    vw[j] = r * K + c * 16;
    last[j] = (KB - 1) * BLK + c * 16 < K ? 0 : OUTSIDE;
#pragma unroll
    for (int tt = 0; tt < XT; ++tt) {
      const int x = tt * 16 + r;
      vx[tt][j] = OUTSIDE;
      if (x < t.rows_here) {
        const int from = gather != nullptr ? gather[t.row0 + x] >> 1 : x;   // a bad index of the permutation reads as a row of zeros
        if (gather == nullptr || (unsigned)from < (unsigned)a_rows) vx[tt][j] = from * K + c * 16;
      }
    }
  }
  if (!CAST && lane < BM && lane < t.rows_here) {
    const int from = gather != nullptr ? gather[t.row0 + lane] >> 1 : t.row0 + lane;
    if ((unsigned)from < (unsigned)a_rows) tok = from * 4;
  }
  const uint32_t ring = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr_t)smem + wave * RING);
  // (by hand: the compiler takes any of them for one that a later LDS read may want)
  auto to_lds = [](const __amdgpu_buffer_rsrc_t& r, uint32_t lds, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" : : "s"(lds), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
  };
  auto word_to_lds = [](const __amdgpu_buffer_rsrc_t& r, uint32_t lds, int voff, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" : : "s"(lds), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
  };
  constexpr int SCALES = 2048 * (FT + XT);   // of a slot: w1's, w3's, the tokens', 64 words each
  auto issue = [&](int slot, int kb) {   // (past the last K block as well, asking for nothing: the loads on their way are counted)
    const uint32_t at = ring + slot * SLOT;
    const int kc = min(kb, KB - 1);
    int mask[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) mask[j] = kb >= KB ? OUTSIDE : kb == KB - 1 ? last[j] : 0;
#pragma unroll
    for (int f = 0; f < FT; ++f)
#pragma unroll
      for (int j = 0; j < 2; ++j) to_lds(f >= STRIPS ? rw1 : rw0, at + f * 2048 + j * 1024, (vw[j] + f % STRIPS * 16 * K) | mask[j], kc * BLK);
#pragma unroll
    for (int tt = 0; tt < XT; ++tt)
#pragma unroll
      for (int j = 0; j < 2; ++j) to_lds(ra, at + (FT + tt) * 2048 + j * 1024, vx[tt][j] | mask[j], kc * BLK);
    word_to_lds(rs0, at + SCALES, 0, kc * 4);
    if (SWIGLU) word_to_lds(rs1, at + SCALES + 256, 0, kc * 4);
    if (!CAST) word_to_lds(rs, at + SCALES + (SWIGLU ? 512 : 256), tok, kc * ld_s);
  };

  // CAST: the 16-bit rows first, 16 lanes for each block of 128; [rows][ld_x] cast rows, [KB][rows] scales. A column without a row reads the
  // last one's and is never stored.
  const int ld_x = KB * BLK + 16, R = args.lds_rows;
  uint8_t* const lx = smem + KW * RING;
  float* const ls = reinterpret_cast<float*>(lx + (size_t)R * ld_x);
  uint8_t* const raw = lx + stream_cast_bytes(R, KB);
  if constexpr (CAST) {
    const __amdgpu_buffer_rsrc_t rx = gather != nullptr ? make_rsrc(op.a, (uint32_t)a_rows * (uint32_t)K * 2u)
                                                        : make_rsrc(op.a + (size_t)t.row0 * K * 2, (uint32_t)t.rows_here * (uint32_t)K * 2u);
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_ptr_t)raw + wave * 1024);
    for (int i = 0; i * 4 * KW < R * KB; ++i) {
      const int u = i * 4 * KW + (tid >> 4), r = u / KB, k = (u - r * KB) * BLK + (tid & 15) * 8;
      int off = OUTSIDE;
      if (r < t.rows_here && k < K) {
        const int from = gather != nullptr ? gather[t.row0 + r] >> 1 : r;
        if (gather == nullptr || (unsigned)from < (unsigned)a_rows) off = (from * K + k) * 2;
      }
      to_lds(rx, at + i * KW * 1024, off, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < DEPTH; ++i) issue(i, kw + i * KW);

  if constexpr (CAST) {
    static_assert(DEPTH * LOADS < 64, "counted in 6 bits");
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(DEPTH * LOADS) : "memory");   // a thread casts what it asked for itself
    for (int i = 0; i * 4 * KW < R * KB; ++i) {
      const int u = i * 4 * KW + (tid >> 4), r = u / KB, b = u - r * KB;
      Half<Act> v;
      v.load(raw, (size_t)(i * 64 * KW + tid) * 8);
      uint32_t o[2];
      float s;
      cast_unit(v, o, s);
      if (r < R) {
        *reinterpret_cast<u32x2*>(lx + r * ld_x + b * BLK + (tid & 15) * 8) = u32x2{o[0], o[1]};
        if ((tid & 15) == 0) ls[b * R + r] = s;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
  }

  v4f acc[FT][TT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[f][tt] = v4f{0, 0, 0, 0};
  typedef const __attribute__((address_space(3))) v4i* lds_v4i;
  typedef const __attribute__((address_space(3))) float* lds_float;
  const int c0 = (quad ^ swz(fr)) * 16, c1 = ((quad + 4) ^ swz(fr)) * 16;
  auto strip = [&](uint32_t at) -> v8i {
    const v4i lo = *(lds_v4i)(at + fr * BLK + c0), hi = *(lds_v4i)(at + fr * BLK + c1);
    return v8i{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  };
  const int steps = kw < KB ? (KB - kw + KW - 1) / KW : 0;
  for (int j0 = 0; j0 < steps; j0 += DEPTH) {
#pragma unroll
    for (int i = 0; i < DEPTH; ++i) {
      if (j0 + i >= steps) break;
      const int kb = kw + (j0 + i) * KW;
      const uint32_t at = ring + i * SLOT;
      asm volatile("s_waitcnt vmcnt(%0)" : : "n"((DEPTH - 1) * LOADS) : "memory");
      v8i fa[FT], fb[TT];
      float m0[TT], m1[TT];
#pragma unroll
      for (int f = 0; f < FT; ++f) fa[f] = strip(at + f * 2048);
      const float s0 = *(lds_float)(at + SCALES + lane * 4), s1 = SWIGLU ? *(lds_float)(at + SCALES + 256 + lane * 4) : 0.0f;
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        float sx;
        if constexpr (CAST) {
          const int r = min(tt * 16 + fr, R - 1);
          const uint8_t* const row = lx + r * ld_x + kb * BLK + quad * 16;
          const v4i lo = *reinterpret_cast<const v4i*>(row), hi = *reinterpret_cast<const v4i*>(row + 64);
          fb[tt] = v8i{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          sx = ls[kb * R + r];
        } else {
          fb[tt] = strip(at + (FT + tt) * 2048);
          sx = *(lds_float)(at + SCALES + (SWIGLU ? 512 : 256) + (tt * 16 + fr) * 4);
        }
        m0[tt] = sx * s0;
        m1[tt] = SWIGLU ? sx * s1 : 0.0f;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");   // the slot is read: its next K block may come
      issue(i, kb + DEPTH * KW);
#pragma unroll
      for (int f = 0; f < FT; ++f) {
        v4f p[TT];
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) p[tt] = block_product<SWIGLU>(fa[f], fb[tt]);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[f][tt][c] = __builtin_fmaf(p[tt][c], SWIGLU && f >= STRIPS ? m1[tt] : m0[tt], acc[f][tt][c]);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");   // of the loads that asked for nothing: their zeros land in the ring too

  // the waves' sums, each in its own ring: [strip][token tile][lane] of 16 bytes
  constexpr int CELLS = FT * TT;
  static_assert(CELLS * 1024 <= RING, "a wave's sums take its ring's place");
  auto parts = [&](int w, int cell) -> v4f& { return reinterpret_cast<v4f*>(smem + w * RING)[cell * 64 + lane]; };
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) parts(kw, f * TT + tt) = acc[f][tt];
  __syncthreads();
  auto total = [&](int cell) {
    v4f y = parts(0, cell);
#pragma unroll
    for (int w = 1; w < KW; ++w) {
      const v4f v = parts(w, cell);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] += v[i];
    }
    return y;
  };
#pragma unroll
  for (int c0 = 0; c0 < STRIPS * TT; c0 += KW) {
    const int cell = c0 + wave, f = cell / TT, tt = cell - f * TT;
    if (cell >= STRIPS * TT) break;
    v4f y = total(cell);
    const int r = tt * 16 + fr, n = t.n0 + f * 16 + quad * 4;
    if constexpr (SWIGLU) {
      const v4f u = total(cell + STRIPS * TT);
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = silu(y[i]) * u[i];
    }
    if (r >= t.rows_here || n >= N) continue;
    const size_t at = (size_t)(t.row0 + r) * N + n;
    if constexpr (SWIGLU) {
      *reinterpret_cast<v4f*>(op.h + at) = y;
    } else {
      if (grp.bias != nullptr) {
        const u32x2 b = *reinterpret_cast<const u32x2*>(grp.bias + n);
        y[0] += Act::lo(b.x); y[1] += Act::hi(b.x); y[2] += Act::lo(b.y); y[3] += Act::hi(b.y);
      }
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(op.out) + at) = u32x2{Act::pack(y[0], y[1]), Act::pack(y[2], y[3])};
    }
  }
#endif
}

// ---- launch -------------------------------------------------------------------------------------------------------
// The opt-in for more than 64 KiB of LDS, once per kernel and device.
template <class Kernel>
int allow_lds(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done, const char* what) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return hdmoe_fail(HDMOE_E_LAUNCH, "%s: no HIP device", what);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return HDMOE_OK;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != hipSuccess) return hdmoe_fail(HDMOE_E_LAUNCH, "%s: %s", what, hipGetErrorString(e));
  done.fetch_or(bit, std::memory_order_relaxed);
  return HDMOE_OK;
}

// At most this many tiles, whatever the segments: every one of them can end in a tile that is not full. Rounded up to the XCDs.
long long grid_of(const BlockArgs& args, int bm, int feat) {
  long long tiles = 0;
  if (args.E > 0) {
    const long long rows = args.op[0].rows, ends = rows < args.E ? rows : args.E;   // the ends take a row each at least
    tiles += ((rows - ends) / bm + ends) * ((args.op[0].N + feat - 1) / feat);
  }
  tiles += ((long long)args.op[1].rows + bm - 1) / bm * ((args.op[1].N + feat - 1) / feat);
  return (tiles + HDMOE_NUM_XCD - 1) / HDMOE_NUM_XCD * HDMOE_NUM_XCD;
}

constexpr int low_stage(bool swiglu) { return (swiglu ? 64 + 256 : 128 + 128) * BLK + 2048; }   // LDS of a K step of block_gemm_kernel

template <class Act, bool SWIGLU, int STAGES>
int launch_gemm(const BlockArgs& args, const char* what, hipStream_t stream) {
  constexpr int BM = SWIGLU ? 64 : 128, BN = SWIGLU ? 256 : 128;
  constexpr size_t SMEM = STAGES * low_stage(SWIGLU);
  static_assert(low_stage(SWIGLU) == (BM + BN) * BLK + 2048, "a stage of the kernel's");
  const auto kernel = block_gemm_kernel<Act, SWIGLU, SWIGLU ? 4 : 2, SWIGLU ? 2 : 4, 4, 2, STAGES>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_lds(kernel, SMEM, done, what)) return rc;
  const long long grid = grid_of(args, BM, BLK);
  if (grid > 0x7fffffffll) return hdmoe_fail(HDMOE_E_SHAPE, "%s: %lld tiles", what, grid);
  kernel<<<(unsigned)grid, 512, SMEM, stream>>>(args);
  return hdmoe_check_launch(what);
}

constexpr int HIGH_LDS = 5 * 32768;   // tokens of two K steps, weights of three

template <class Act, bool SWIGLU>
int launch_gemm8(const BlockArgs& args, const char* what, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_lds(block_gemm8_kernel<Act, SWIGLU>, HIGH_LDS, done, what)) return rc;
  const long long grid = grid_of(args, 64 * args.parts, SWIGLU ? 128 : 256);
  if (grid > 0x7fffffffll) return hdmoe_fail(HDMOE_E_SHAPE, "%s: %lld tiles", what, grid);
  block_gemm8_kernel<Act, SWIGLU><<<(unsigned)(grid < HDMOE_NUM_CU ? grid : HDMOE_NUM_CU), 512, HIGH_LDS, stream>>>(args);
  return hdmoe_check_launch(what);
}

template <class Act, bool SWIGLU, int FT, int TT, bool CAST>
int launch_stream(const BlockArgs& args, const char* what, hipStream_t stream) {
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_lds(block_stream_kernel<Act, SWIGLU, FT, TT, CAST>, stream_lds(FT, TT, SWIGLU, CAST, 16, CAST_UNITS / 16), done, what)) return rc;
  const int K = args.op[0].K > args.op[1].K ? args.op[0].K : args.op[1].K;
  const size_t bytes = stream_lds(FT, TT, SWIGLU, CAST, args.lds_rows, (K + BLK - 1) / BLK);
  const long long grid = grid_of(args, TT * 16, SWIGLU ? 8 * FT : 16 * FT);
  if (grid > 0x7fffffffll) return hdmoe_fail(HDMOE_E_SHAPE, "%s: %lld tiles", what, grid);
  block_stream_kernel<Act, SWIGLU, FT, TT, CAST><<<(unsigned)grid, 64 * STREAM_WAVES, bytes, stream>>>(args);
  return hdmoe_check_launch(what);
}

int check_sizes(const char* what, const char* which, long long rows, int K, int N) {
  if (rows < 0 || K <= 0 || N <= 0 || K % 16 != 0 || N % 16 != 0)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s%s: rows=%lld K=%d N=%d (K and N must be multiples of 16)", what, which, rows, K, N);
  if ((long long)N * K > 0x7fffffffll || (long long)256 * K > 0x7fffffffll)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s%s: K=%d N=%d: a weight must be smaller than 2 GiB", what, which, K, N);
  if ((long long)256 * N * 2 > 0x7fffffffll) return hdmoe_fail(HDMOE_E_SHAPE, "%s%s: N=%d: at most 4194288", what, which, N);   // a tile's rows of the output
  return HDMOE_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int hdmoe_quant_block_fp8(int src_dtype, const void* x, int64_t rows, int K, void* out_e4m3fn, float* scale,
                                     int64_t scale_stride, hdmoe_stream_t stream) {
  const char* what = "hdmoe_quant_block_fp8";
  if (src_dtype != HDMOE_W_BF16 && src_dtype != HDMOE_W_F16)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: src_dtype=%d", what, src_dtype);
  if (rows < 0 || rows > 0x7fffffffll || K <= 0 || K % 16 != 0 || scale_stride < rows)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%lld K=%d scale_stride=%lld", what, (long long)rows, K, (long long)scale_stride);
  if (rows == 0) return HDMOE_OK;
  HDMOE_REQUIRE_PTR(x);
  HDMOE_REQUIRE_PTR(out_e4m3fn);
  HDMOE_REQUIRE_PTR(scale);
  if (!aligned16(x) || (reinterpret_cast<uintptr_t>(out_e4m3fn) & 7))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: x must start on 16 bytes, out on 8", what);
  const int KB = (K + BLK - 1) / BLK;
  const long long blocks = (rows * KB * 16 + 255) / 256;
  if (blocks > 0x7fffffffll) return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%lld K=%d", what, (long long)rows, K);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (src_dtype == HDMOE_W_BF16)
    block_cast_kernel<Half<HdmoeBf16>><<<(unsigned)blocks, 256, 0, s>>>(x, (int)rows, K, KB, static_cast<uint8_t*>(out_e4m3fn), scale, scale_stride, nullptr, 0);
  else
    block_cast_kernel<Half<HdmoeF16>><<<(unsigned)blocks, 256, 0, s>>>(x, (int)rows, K, KB, static_cast<uint8_t*>(out_e4m3fn), scale, scale_stride, nullptr, 0);
  return hdmoe_check_launch(what);
}

namespace {

// How a call runs: the few-row kernels on tiles of 16 * tt rows and ft strips (tt > 0; with the cast inside or not), block_gemm_kernel with
// `stages` K steps in LDS (stages > 0), or block_gemm8_kernel.
struct Plan { int tt, ft; bool cast_inside; int lds_rows; int stages, parts; bool exact; };

// What a launch is likely to take in microseconds, by what the kernels measured over 1 to 16384 rows of 2560 and 6912 wide Linears. Where the
// segments end is not known here; on average half a tile of each is empty.
struct Sizes { int rows, E, rows_static, K, N, K_static, N_static; };
double tiles_of(const Sizes& z, int bm, int feat) {   // in tiles of the experts' K
  double t = 0;
  if (z.rows > 0) {
    const int n = z.E < z.rows ? z.E : z.rows;
    const double m = z.E == 1 ? (double)((z.rows + bm - 1) / bm) : (double)z.rows / bm + 0.5 * n;
    t += (m > n ? m : n) * ((z.N + feat - 1) / feat);
  }
  if (z.rows_static > 0) {
    const double share = z.rows > 0 ? (double)z.K_static / z.K : 1.0;
    t += (double)((z.rows_static + bm - 1) / bm) * ((z.N_static + feat - 1) / feat) * share;
  }
  return t;
}
// Few rows. 3.5 us to a block's first operands and behind its last, 80 KB/us of weights and activations for a CU (32 x 6912 x 2560 with its cast, 1, 2 and 4 strips a
// block: 12.1, 10.6, 13.1 us); 55 KB/us where a wave multiplies 16 tiles of each K block and has only one more on its way (100 x 2560 x 6912: 13.9, 17.9 in
// two rounds of 8 tiles).
double few_us(const Sizes& z, bool swiglu, int tt, int ft, bool cast, int lds_rows) {
  const double blocks = tiles_of(z, 16 * tt, swiglu ? 8 * ft : 16 * ft);
  const int per = z.rows > 0 ? (z.rows + z.E - 1) / z.E : 0, most = per > z.rows_static ? per : z.rows_static;
  const int rows = most < 16 * tt ? most : 16 * tt, K = z.rows > 0 ? z.K : z.K_static;
  return 1.7 + ceil(blocks / (HDMOE_NUM_CU * stream_blocks(ft, tt, swiglu, cast, lds_rows, (K + BLK - 1) / BLK))) * 3.5 + ceil(blocks / HDMOE_NUM_CU) * (16.0 * ft + rows) * K / (ft * tt == 16 ? 55e3 : 80e3) + (swiglu ? 3.5 : 0.0);
}
// Low tiles. 128 x 6912 x 2560: 32.7 us with four stages (two 41.6), where a step lasts half as long as memory's answer; from a block for every CU on
// two blocks share one (1024 x 2560 x 6912: 32.6 against 25.8).
double low_us(const Sizes& z, bool swiglu, int stages) {
  const double t = tiles_of(z, swiglu ? 64 : 128, BLK), kb = ((z.rows > 0 ? z.K : z.K_static) + BLK - 1) / BLK;
  if (stages > 2) return 5.0 + ceil(t / HDMOE_NUM_CU) * (2.0 + kb * (swiglu ? 0.82 : 0.5));
  const double over = t <= HDMOE_NUM_CU ? 0.0 : t >= 2 * HDMOE_NUM_CU ? 1.0 : t / HDMOE_NUM_CU - 1.0;
  // A round that is begun lasts three quarters of a whole one at least (1407 x 2800 x 6208, 539 tiles: 59.2 us, 40.6 on 256-row tiles), but where
  // segments are so short that the weights' way from memory is what lasts
  double rounds = t / (2 * HDMOE_NUM_CU);
  if (rounds > 1.0 && (z.rows == 0 || z.rows / z.E >= 64) && rounds - floor(rounds) < 0.75 && rounds > floor(rounds)) rounds = floor(rounds) + 0.75;
  return 5.0 + (rounds > 1.0 ? 1.1 * rounds : 1.0) * kb * (0.63 + 0.45 * over);
}
// Tiles of 64 * cap x 256: a step lasts 0.49, 0.63, 0.85 or 1.07 us with 1 to 4 parts of 64 rows, and 1.5 where every CU multiplies a full one: the
// clock falls. A CU with a tile more than others has lower ones.
double high_us(const Sizes& z, bool swiglu, int cap) {
  const int feat = swiglu ? 128 : 256;
  const double t = tiles_of(z, 64 * cap, feat), parts = tiles_of(z, 64, feat), kb = ((z.rows > 0 ? z.K : z.K_static) + BLK - 1) / BLK;
  const double rounds = ceil(t / HDMOE_NUM_CU), full = t < HDMOE_NUM_CU ? t / HDMOE_NUM_CU : 1.0, mean = parts / t;
  const int segments = (z.rows > 0 ? z.E : 0) + (z.rows_static > 0 ? 1 : 0);
  const double top = segments == 1 ? ceil(mean) : 1.5 * mean < cap ? 1.5 * mean : (double)cap;
  const double low = segments == 1 || rounds < 2 ? mean : mean - (top - mean) * (rounds - t / HDMOE_NUM_CU) / (rounds - 1);
  auto tile = [&](double p) { return 5.0 + kb * (0.3 + (0.19 + 0.1 * full) * p); };
  const double one = tile(top), most = rounds * tile(low);
  return 4.0 + (one > most ? one : most);
}

// Gate/up: rows of either group up to which its products are exact in every type
constexpr int EXACT_ROWS = 64;
// fixed: the kernels whose sums go block after block of K, in fp32 on the matrix instruction's result for each (the tile kernels: low and high ones
// give a row the same bytes), and products of one kind, whatever the sizes. exact: gate/up's products are.
Plan plan_of(bool swiglu, int a_dtype, const Sizes& z, bool fixed, bool exact) {
  const bool x16 = a_dtype != HDMOE_W_E4M3FN;
  exact = swiglu && (exact || a_dtype == HDMOE_W_F16 || (!fixed && z.rows <= EXACT_ROWS && z.rows_static <= EXACT_ROWS));
  Plan best = {0, 0, false, 0, 0, 4, false};
  double us = exact ? 1e30 : high_us(z, swiglu, 4);   // (that kernel's loop has no exact products)
  Plan rows16 = best;   // of the few-row kernels on tiles of 16 rows
  double us16 = 1e30;
  auto offer = [&](double t, const Plan& p) {
    if (t < us) {
      us = t;
      best = p;
    }
  };
  for (int cap = 3; !exact && cap >= 2; --cap) offer(high_us(z, swiglu, cap), Plan{0, 0, false, 0, 0, cap, exact});
  if (swiglu) {
    offer(low_us(z, true, 3), Plan{0, 0, false, 0, 3, 0, exact});
  } else {
    offer(low_us(z, false, 4), Plan{0, 0, false, 0, 4, 0, exact});
    offer(low_us(z, false, 2), Plan{0, 0, false, 0, 2, 0, exact});
  }
  const int K = z.rows > 0 ? z.K : z.K_static;
  for (int tt = 1; !fixed && tt <= 4; tt *= 2)
    for (int ft = swiglu ? 2 : 1; ft <= 4; ft *= 2) {
      Plan p = {tt, ft, false, 0, 0, 0, swiglu};
      if (x16 && tt == 1) {
        // a block casts for itself what takes its threads 8 trips at most: a launch (4 us) less
        const int whole = z.rows > z.rows_static ? z.rows : z.rows_static;
        p.lds_rows = whole < 16 ? whole : 16;
        p.cast_inside = (long long)p.lds_rows * ((K + BLK - 1) / BLK) <= CAST_UNITS && (long long)whole * K * 2 <= 0x7fffffff;
      }
      double t = few_us(z, swiglu, tt, ft, p.cast_inside, p.lds_rows);
      if (p.cast_inside) t -= 4.0;
      offer(t, p);
      if (tt == 1 && (p.cast_inside ? p.lds_rows <= 4 : z.rows_static == 0) && t < us16) {
        us16 = t;
        rows16 = p;
      }
    }
  // Exact products take the low tiles 0.45 us more a step (600 rows in eight segments, K 1024: 27.1 -> 30.7 us), for empty rows too: segments of up to 16
  // rows go to tiles of 16 (8 to 32 rows of four experts, 2560 x 6912: 36 us, low tiles 42; 15 of eight, 1392 x 5456: 44 and 57; 143 of sixteen,
  // 2304 x 1648: 4 % less). Not beside a shared expert (8 tokens, 3584 wide: 49 us, low tiles 46), not for up to 8 steps, and where blocks cast
  // their rows over and over only up to four of them (a layer of 2 tokens: 38 us, low tiles 43; 5 rows of eight, 1600 x 5536: 10 % more).
  const int kb = (K + BLK - 1) / BLK;
  if (exact && best.stages > 0 && kb > 8 && z.rows <= 16 * z.E && us16 < us + 0.45 * kb) best = rows16;
  return best;
}

size_t cast_bytes(long long rows, int K) { return hdmoe_align_up((size_t)rows * K, 256) + hdmoe_align_up((size_t)rows * ((K + BLK - 1) / BLK) * 4, 256); }

// Working memory: the cast rows of 16-bit activations, unless the contraction casts them itself; gate/up of few rows: silu(g) * u in fp32.
size_t work_bytes(bool swiglu, bool x16, const Plan& plan, int rows, int T, int rows_static, int K, int N, int N_static) {
  size_t n = x16 && !plan.cast_inside ? cast_bytes(rows > 0 ? (T > 0 ? T : rows) : rows_static, K) : 0;
  if (swiglu && plan.tt > 0) n += hdmoe_align_up((size_t)rows * N * 4, 256) + hdmoe_align_up((size_t)rows_static * N_static * 4, 256);
  return n;
}

// Arguments of both contractions -> those of the kernels; checks everything but what only the device knows. 16-bit activations are
// cast into the workspace here unless the contraction does that itself.
int fill(const char* what, const hdmoe_block_args* p, bool swiglu, BlockArgs& args, Plan& plan, hipStream_t stream) {
  HDMOE_REQUIRE_PTR(p);
  const bool x16 = p->a_dtype == HDMOE_W_BF16 || p->a_dtype == HDMOE_W_F16;
  if ((p->out_dtype != HDMOE_W_BF16 && p->out_dtype != HDMOE_W_F16) || (!x16 && p->a_dtype != HDMOE_W_E4M3FN) ||
      (x16 && !swiglu && p->a_dtype != p->out_dtype))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: a_dtype=%d out_dtype=%d", what, p->a_dtype, p->out_dtype);
  if (p->E < 0 || p->E > MAX_E || p->rows < 0 || p->rows_static < 0 || (p->E == 0 && p->rows > 0))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: E=%d (at most %d) rows=%d rows_static=%d", what, p->E, MAX_E, p->rows, p->rows_static);
  args = BlockArgs{};
  auto weights = [&](const hdmoe_block_weights& w, Group& g) -> int {
    if (w.weight == nullptr || w.scale == nullptr || (swiglu && (w.weight3 == nullptr || w.scale3 == nullptr)))
      return hdmoe_fail(HDMOE_E_NULL, "%s: a weight or scale is NULL", what);
    if (!aligned16(w.weight) || !aligned16(w.weight3) || !aligned16(w.bias))
      return hdmoe_fail(HDMOE_E_SHAPE, "%s: weights and biases must start on 16 bytes", what);
    g.w0 = static_cast<const uint8_t*>(w.weight);
    g.s0 = w.scale;
    g.w1 = static_cast<const uint8_t*>(w.weight3);
    g.s1 = w.scale3;
    g.bias = static_cast<const uint16_t*>(w.bias);
    return HDMOE_OK;
  };
  auto operand = [&](const hdmoe_block_rows& r, int rows, int K, int N, const int32_t* perm, int T, Operand& op) -> int {
    const int a_rows = perm != nullptr ? T : rows;
    if (r.a == nullptr || (!x16 && r.scale_a == nullptr) || r.out == nullptr || (swiglu && r.scale_out == nullptr))
      return hdmoe_fail(HDMOE_E_NULL, "%s: activations, their scales or the output are NULL", what);
    if (!aligned16(r.a) || !aligned16(r.out)) return hdmoe_fail(HDMOE_E_SHAPE, "%s: activations and outputs must start on 16 bytes", what);
    if ((!x16 && r.scale_a_stride < a_rows) || (swiglu && r.scale_out_stride < rows))
      return hdmoe_fail(HDMOE_E_SHAPE, "%s: scale strides %lld, %lld for %d rows", what, (long long)r.scale_a_stride, (long long)r.scale_out_stride, a_rows);
    if ((x16 ? (long long)a_rows : r.scale_a_stride) * ((K + BLK - 1) / BLK) * 4 > 0x7fffffffll)
      return hdmoe_fail(HDMOE_E_SHAPE, "%s: %d rows of K=%d: their scales must be smaller than 2 GiB", what, a_rows, K);
    if (perm != nullptr && (long long)a_rows * K > 0x7fffffffll)
      return hdmoe_fail(HDMOE_E_SHAPE, "%s: %d rows of K=%d read through a permutation: at most 2 GiB", what, a_rows, K);
    op.a = static_cast<const uint8_t*>(r.a);
    op.sa = r.scale_a;
    op.gather = perm;
    op.ld_sa = r.scale_a_stride;
    op.a_rows = a_rows;
    op.rows = rows;
    op.K = K;
    op.N = N;
    op.out = r.out;
    op.s_out = r.scale_out;
    op.ld_out = r.scale_out_stride;
    return HDMOE_OK;
  };
  const bool routed = p->E > 0 && p->rows > 0;
  if (routed) {
    if (int rc = check_sizes(what, "", p->rows, p->K, p->N)) return rc;
    HDMOE_REQUIRE_PTR(p->offsets);
    HDMOE_REQUIRE_PTR(p->experts);
    if (p->perm != nullptr && (p->T <= 0 || (long long)p->T * HDMOE_TOPK != p->rows))
      return hdmoe_fail(HDMOE_E_SHAPE, "%s: T=%d rows=%d with perm", what, p->T, p->rows);
    args.E = p->E;
    args.offsets = p->offsets;
    for (int e = 0; e < p->E; ++e)
      if (int rc = weights(p->experts[e], args.g[e])) return rc;
    if (int rc = operand(p->routed, p->rows, p->K, p->N, p->perm, p->T, args.op[0])) return rc;
  }
  if (p->rows_static > 0) {
    if (int rc = check_sizes(what, " (static)", p->rows_static, p->K_static, p->N_static)) return rc;
    HDMOE_REQUIRE_PTR(p->shared);
    if (int rc = weights(*p->shared, args.g[args.E])) return rc;
    if (int rc = operand(p->fixed, p->rows_static, p->K_static, p->N_static, nullptr, 0, args.op[1])) return rc;
  }
  const int a_rows = routed ? args.op[0].a_rows : p->rows_static, K = routed ? p->K : p->K_static;
  if (x16 && routed && p->rows_static > 0 && (p->fixed.a != p->routed.a || p->rows_static != a_rows || p->K_static != K))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: 16-bit activations of the experts and of the static group must be the same rows", what);
  plan = plan_of(swiglu, p->a_dtype, Sizes{routed ? p->rows : 0, p->E, p->rows_static, p->K, p->N, p->K_static, p->N_static}, p->fixed_k_cut != 0, p->exact != 0);
  args.lds_rows = plan.lds_rows;
  args.parts = plan.parts;
  const size_t need = work_bytes(swiglu, x16, plan, routed ? p->rows : 0, routed && p->perm != nullptr ? p->T : 0, p->rows_static, K,
                                 routed ? p->N : 0, p->rows_static > 0 ? p->N_static : 0);
  if (need > 0 && (p->workspace == nullptr || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255)))
    return hdmoe_fail(HDMOE_E_WORKSPACE, "%s: workspace %zu bytes, need %zu (256-byte aligned)", what, p->workspace_bytes, need);
  uint8_t* ws = static_cast<uint8_t*>(p->workspace);
  if (a_rows > 0 && x16 && !plan.cast_inside) {
    float* const s = reinterpret_cast<float*>(ws + hdmoe_align_up((size_t)a_rows * K, 256));
    if (int rc = hdmoe_quant_block_fp8(p->a_dtype, routed ? p->routed.a : p->fixed.a, a_rows, K, ws, s, a_rows, stream)) return rc;
    for (Operand& op : args.op) {
      op.a = ws;
      op.sa = s;
      op.ld_sa = a_rows;
    }
    ws += cast_bytes(a_rows, K);
  }
  if (swiglu && plan.tt > 0) {
    args.op[0].h = reinterpret_cast<float*>(ws);
    if (routed) ws += hdmoe_align_up((size_t)p->rows * p->N * 4, 256);
    args.op[1].h = reinterpret_cast<float*>(ws);
  }
  return HDMOE_OK;
}

template <class Act, bool SWIGLU, int FT>
int launch_strips(const BlockArgs& args, const Plan& plan, const char* what, hipStream_t s) {
  if (plan.cast_inside) return launch_stream<Act, SWIGLU, FT, 1, true>(args, what, s);
  using Out = std::conditional_t<SWIGLU, HdmoeBf16, Act>;   // (gate/up: the type of what is cast, not looked at here)
  if (plan.tt == 1) return launch_stream<Out, SWIGLU, FT, 1, false>(args, what, s);
  return plan.tt == 2 ? launch_stream<Out, SWIGLU, FT, 2, false>(args, what, s) : launch_stream<Out, SWIGLU, FT, 4, false>(args, what, s);
}

template <class Act, bool SWIGLU>
int launch_few(const BlockArgs& args, const Plan& plan, const char* what, hipStream_t s) {
  if (plan.ft == 4) return launch_strips<Act, SWIGLU, 4>(args, plan, what, s);
  if constexpr (!SWIGLU)
    if (plan.ft == 1) return launch_strips<Act, false, 1>(args, plan, what, s);
  return launch_strips<Act, SWIGLU, 2>(args, plan, what, s);
}

// The cast behind the gate/up of few rows.
int launch_cast(const BlockArgs& args, const char* what, hipStream_t s) {
  for (int i = 0; i < 2; ++i) {
    const Operand& op = args.op[i];
    if (op.rows == 0) continue;
    const int HB = (op.N + BLK - 1) / BLK;
    const long long blocks = ((long long)op.rows * HB * 16 + 255) / 256;
    block_cast_kernel<Full><<<(unsigned)blocks, 256, 0, s>>>(op.h, op.rows, op.N, HB, static_cast<uint8_t*>(op.out), op.s_out, op.ld_out,
                                                             i == 0 ? args.offsets : nullptr, args.E + 1);
    if (int rc = hdmoe_check_launch(what)) return rc;
  }
  return HDMOE_OK;
}

}  // namespace

extern "C" size_t hdmoe_block_workspace_bytes(const hdmoe_block_args* p, int swiglu) {
  if (p == nullptr || p->rows < 0 || p->E < 0 || p->T < 0 || p->rows_static < 0) return 0;
  const bool x16 = p->a_dtype != HDMOE_W_E4M3FN, routed = p->E > 0 && p->rows > 0;
  if (!routed && p->rows_static == 0) return 0;
  const int K = routed ? p->K : p->K_static, N = routed ? p->N : 0, Ns = p->rows_static > 0 ? p->N_static : 0;
  if (K <= 0 || N < 0 || Ns < 0) return 0;
  const Plan plan = plan_of(swiglu != 0, p->a_dtype, Sizes{routed ? p->rows : 0, p->E, p->rows_static, p->K, N, p->K_static, Ns}, p->fixed_k_cut != 0, p->exact != 0);
  return work_bytes(swiglu != 0, x16, plan, routed ? p->rows : 0, routed && p->perm != nullptr ? p->T : 0, p->rows_static, K, N, Ns);
}

extern "C" int hdmoe_block_plan_get(const hdmoe_block_args* p, int swiglu, hdmoe_block_plan* out) {
  const char* what = "hdmoe_block_plan_get";
  HDMOE_REQUIRE_PTR(p);
  HDMOE_REQUIRE_PTR(out);
  const bool routed = p->E > 0 && p->rows > 0, fixed = p->rows_static > 0;
  if (p->E < 0 || p->E > MAX_E || p->rows < 0 || p->rows_static < 0 || !(routed || fixed))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: E=%d rows=%d rows_static=%d", what, p->E, p->rows, p->rows_static);
  if (routed)
    if (int rc = check_sizes(what, "", p->rows, p->K, p->N)) return rc;
  if (fixed)
    if (int rc = check_sizes(what, " (static)", p->rows_static, p->K_static, p->N_static)) return rc;
  const Sizes z = {routed ? p->rows : 0, p->E, p->rows_static, p->K, p->N, p->K_static, p->N_static};
  const Plan plan = plan_of(swiglu != 0, p->a_dtype, z, p->fixed_k_cut != 0, p->exact != 0);
  const int Kr = routed ? p->K : 0, Ks = fixed ? p->K_static : 0, K = Kr > Ks ? Kr : Ks;
  *out = hdmoe_block_plan{};
  if (plan.tt > 0) {
    out->kernel = HDMOE_BLOCK_FEW_ROWS;
    out->tile_rows = 16 * plan.tt;
    out->strips = plan.ft;
    out->cast_inside = plan.cast_inside;
    out->lds_bytes = stream_lds(plan.ft, plan.tt, swiglu != 0, plan.cast_inside, plan.lds_rows, (K + BLK - 1) / BLK);
    out->blocks_per_cu = stream_blocks(plan.ft, plan.tt, swiglu != 0, plan.cast_inside, plan.lds_rows, (K + BLK - 1) / BLK);
  } else if (plan.stages > 0) {
    out->kernel = HDMOE_BLOCK_LOW_TILES;
    out->tile_rows = swiglu ? 64 : 128;
    out->stages = plan.stages;
    out->lds_bytes = plan.stages * low_stage(swiglu != 0);
    out->blocks_per_cu = plan.stages == 2 ? 2 : 1;
  } else {
    out->kernel = HDMOE_BLOCK_HIGH_TILES;
    out->tile_rows = 64 * plan.parts;
    out->lds_bytes = HIGH_LDS;
    out->blocks_per_cu = 1;
  }
  out->exact = plan.exact;
  return HDMOE_OK;
}

extern "C" int hdmoe_block_linear(const hdmoe_block_args* p, hdmoe_stream_t stream) {
  const char* what = "hdmoe_block_linear";
  BlockArgs args;
  Plan plan;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = fill(what, p, false, args, plan, s)) return rc;
  if (args.op[0].rows + (long long)args.op[1].rows == 0) return HDMOE_OK;
  const bool bf16 = p->out_dtype == HDMOE_W_BF16;
  if (plan.tt > 0) return bf16 ? launch_few<HdmoeBf16, false>(args, plan, what, s) : launch_few<HdmoeF16, false>(args, plan, what, s);
  if (plan.stages == 2) return bf16 ? launch_gemm<HdmoeBf16, false, 2>(args, what, s) : launch_gemm<HdmoeF16, false, 2>(args, what, s);
  if (plan.stages == 4) return bf16 ? launch_gemm<HdmoeBf16, false, 4>(args, what, s) : launch_gemm<HdmoeF16, false, 4>(args, what, s);
  return bf16 ? launch_gemm8<HdmoeBf16, false>(args, what, s) : launch_gemm8<HdmoeF16, false>(args, what, s);
}

extern "C" int hdmoe_block_swiglu(const hdmoe_block_args* p, hdmoe_stream_t stream) {
  const char* what = "hdmoe_block_swiglu";
  BlockArgs args;
  Plan plan;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int rc = fill(what, p, true, args, plan, s)) return rc;
  if (args.op[0].rows + (long long)args.op[1].rows == 0) return HDMOE_OK;
  if (plan.tt > 0) {
    if (int rc = p->a_dtype == HDMOE_W_F16 ? launch_few<HdmoeF16, true>(args, plan, what, s) : launch_few<HdmoeBf16, true>(args, plan, what, s)) return rc;
    return launch_cast(args, what, s);
  }
  if (plan.stages > 0) return plan.exact ? launch_gemm<HdmoeF16, true, 3>(args, what, s) : launch_gemm<HdmoeBf16, true, 3>(args, what, s);
  return launch_gemm8<HdmoeBf16, true>(args, what, s);
}
