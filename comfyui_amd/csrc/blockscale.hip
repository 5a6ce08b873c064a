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
// 16 lanes hold a block of a row, 8 values each; a wave takes 4 neighbouring blocks. Bound by memory: 3.03 bytes per value.
template <class Act>
__global__ __launch_bounds__(256) void block_cast_kernel(const uint16_t* __restrict__ x, int rows, int K, int KB,
                                                         uint8_t* __restrict__ q, float* __restrict__ s, long long ld_s) {
  const long long n = (long long)rows * KB;
  const long long u = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
  if (u >= n) return;
  const int row = (int)(u / KB), b = (int)(u - (long long)row * KB);
  const int k = b * BLK + (threadIdx.x & 15) * 8;
  const bool in = k < K;   // K is a multiple of 16: eight values lie inside or outside together
  u32x4 v = {0, 0, 0, 0};
  if (in) v = *reinterpret_cast<const u32x4*>(x + (size_t)row * K + k);
  // the largest magnitude as an integer of 16 bits
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = v[i] & 0x7fffu, hi = (v[i] >> 16) & 0x7fffu;
    m = max(m, max(lo, hi));
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d, 16));
  const float top_in = Act::lo(m);
  const float top = top_in < TOP_FLOOR ? TOP_FLOOR : top_in;
  const float r = 448.0f / top;
  if (in) {
    u32x2 o;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      o[i] = hdmoe_dev_pack4_e4m3fn(Act::lo(v[2 * i]) * r, Act::hi(v[2 * i]) * r, Act::lo(v[2 * i + 1]) * r, Act::hi(v[2 * i + 1]) * r);
    *reinterpret_cast<u32x2*>(q + (size_t)row * K + k) = o;
  }
  if ((threadIdx.x & 15) == 0) s[(size_t)b * ld_s + row] = top / 448.0f;
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
  const uint8_t* a;     // e4m3fn rows of K bytes
  const float* sa;      // scale of block b of row r at sa[b * ld_sa + r]
  const int32_t* gather;  // NULL, or sorted row r is row gather[r] >> 1 of a
  long long ld_sa;
  int a_rows;           // rows of a
  int rows;             // rows of the segments (or of the static group)
  int K, N;
  void* out;            // 16-bit [rows,N]; gate/up: e4m3fn [rows,N]
  float* s_out;         // gate/up: scale of block b of row r at s_out[b * ld_out + r]
  long long ld_out;
};

struct BlockArgs {
  Group g[MAX_E + 1];   // the static group is g[E]
  Operand op[2];        // the experts' operand, the static group's
  const int32_t* offsets;
  int E;
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

// WF x WT waves, each FT * 16 = 128 weight rows x TT * 16 tokens in MFMA tiles of 16 x 16 x 128. Weight rows of a wave are features
// of one weight block (gate/up: 64 of w1 and the same 64 of w3). LDS row 16 ft + r of a wave's weights holds the feature that puts
// 4 FT consecutive ones (gate/up: 2 FT) in a lane's accumulators: stores of 16 bytes without a transposition.
template <class Act, bool SWIGLU, int WF, int WT, int TT>
__global__ __launch_bounds__(64 * WF * WT) void block_gemm_kernel(const BlockArgs args) {
#if defined(__HIP_DEVICE_COMPILE__)   // (the host pass leaves out stubs of kernels whose lambdas hold arrays of dependent size)
  constexpr int FT = 8;
  constexpr int NT = 64 * WF * WT;
  constexpr int BM = WT * TT * 16, BN = WF * BLK;
  constexpr int FEAT = SWIGLU ? BN / 2 : BN;
  static_assert(!SWIGLU || WF == 2, "a block of the cast output is 128 features");
  constexpr int STAGE = (BM + BN) * BLK;
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

  // ---- global -> LDS: lane i of a load lands in 16-byte chunk i & 7 of row i >> 3 and fetches the chunk that the swizzle puts there.
  // Rows and chunks that do not exist get an offset past the buffer and read as zero.
  const int ld_row = wave * 8 + (lane >> 3);
  const int ld_chunk = (lane & 7) ^ swz(ld_row);
  constexpr int OUTSIDE = (int)0x80000000u;
  int va[LA], vb[LB];
  const bool gathers = op.gather != nullptr;
  const __amdgpu_buffer_rsrc_t ra = gathers ? make_rsrc(op.a, (uint32_t)op.a_rows * (uint32_t)K)
                                            : make_rsrc(op.a + (size_t)t.row0 * K, (uint32_t)t.rows_here * (uint32_t)K);
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = j * ROWS_PER_LOAD + ld_row;
    va[j] = OUTSIDE;
    if (r < t.rows_here) {
      const int from = gathers ? op.gather[t.row0 + r] >> 1 : r;   // a bad index of the permutation reads as a row of zeros
      if (!gathers || (unsigned)from < (unsigned)op.a_rows) va[j] = from * K + ld_chunk * 16;
    }
  }
  const int feats = min(N - t.n0, FEAT);
  const __amdgpu_buffer_rsrc_t rb0 = make_rsrc(grp.w0 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K);
  const __amdgpu_buffer_rsrc_t rb1 = SWIGLU ? make_rsrc(grp.w1 + (size_t)t.n0 * K, (uint32_t)feats * (uint32_t)K) : rb0;
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int p = j * ROWS_PER_LOAD + ld_row;         // LDS row of the weight tile
    const int w = p >> 7, ft = (p >> 4) & 7, r = p & 15;
    const int f = SWIGLU ? w * 64 + (r >> 2) * 16 + (ft & 3) * 4 + (r & 3) : w * 128 + (r >> 2) * 32 + ft * 4 + (r & 3);
    vb[j] = f < feats ? f * K + ld_chunk * 16 : OUTSIDE;
  }
  auto issue = [&](int stage, int kb) {
    uint8_t* sa = smem + stage * STAGE + wave * 8 * BLK;
    uint8_t* sb = sa + BM * BLK;
    const int k0 = kb * BLK;
    const bool ok = k0 + ld_chunk * 16 < K;
#pragma unroll
    for (int j = 0; j < LA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr_t)(sa + j * ROWS_PER_LOAD * BLK), 16, ok ? va[j] : OUTSIDE, k0, 0, 0);
#pragma unroll
    for (int j = 0; j < LB; ++j) {
      // gate/up: the w3 rows are the upper 64 of every wave's 128; a load's rows lie on one side for a given wave
      const bool up = SWIGLU && (((j * ROWS_PER_LOAD + wave * 8) >> 6) & 1);
      if (up) __builtin_amdgcn_raw_ptr_buffer_load_lds(rb1, (lds_ptr_t)(sb + j * ROWS_PER_LOAD * BLK), 16, ok ? vb[j] : OUTSIDE, k0, 0, 0);
      else __builtin_amdgcn_raw_ptr_buffer_load_lds(rb0, (lds_ptr_t)(sb + j * ROWS_PER_LOAD * BLK), 16, ok ? vb[j] : OUTSIDE, k0, 0, 0);
    }
  };

  // ---- scales: of the lane's token in every token tile, of the wave's weight block
  int tok[TT];   // row of sa, -1: none
#pragma unroll
  for (int tt = 0; tt < TT; ++tt) {
    const int r = wt * TT * 16 + tt * 16 + (lane & 15);
    tok[tt] = r < t.rows_here ? (gathers ? op.gather[t.row0 + r] >> 1 : t.row0 + r) : -1;
    if (tok[tt] >= op.a_rows) tok[tt] = -1;
  }
  const int nblk = SWIGLU ? t.n0 / BLK : min(t.n0 / BLK + wf, (N - 1) / BLK);
  const float* sw0 = grp.s0 + (size_t)nblk * KB;
  const float* sw1 = SWIGLU ? grp.s1 + (size_t)nblk * KB : sw0;
  float sx[TT], s0 = 0.0f, s1 = 0.0f;
  auto load_scales = [&](int kb) {
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) sx[tt] = tok[tt] >= 0 ? op.sa[(size_t)kb * op.ld_sa + tok[tt]] : 0.0f;
    s0 = sw0[kb];
    if (SWIGLU) s1 = sw1[kb];
  };

  const int fr = lane & 15, fs = swz(fr), c0 = lane >> 4;
  v4f acc[FT][TT];
#pragma unroll
  for (int f = 0; f < FT; ++f)
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) acc[f][tt] = v4f{0, 0, 0, 0};

  auto frag = [&](const uint8_t* row) -> v8i {
    const v4i lo = *reinterpret_cast<const v4i*>(row + ((c0 ^ fs) << 4)), hi = *reinterpret_cast<const v4i*>(row + (((c0 + 4) ^ fs) << 4));
    return v8i{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  };

  issue(0, 0);
  load_scales(0);
  for (int kb = 0; kb < KB; ++kb) {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
    float m0[TT], m1[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) { m0[tt] = sx[tt] * s0; m1[tt] = SWIGLU ? sx[tt] * s1 : m0[tt]; }
    if (kb + 1 < KB) {
      issue((kb + 1) & 1, kb + 1);
      load_scales(kb + 1);
    }
    const uint8_t* sa = smem + (kb & 1) * STAGE + (wt * TT * 16 + fr) * BLK;
    const uint8_t* sb = smem + (kb & 1) * STAGE + (BM + wf * BLK + fr) * BLK;
    v8i fb[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) fb[tt] = frag(sa + tt * 16 * BLK);
#pragma unroll
    for (int f = 0; f < FT; ++f) {
      const v8i fa = frag(sb + f * 16 * BLK);
#pragma unroll
      for (int tt = 0; tt < TT; ++tt) {
        const v4f p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fa, fb[tt], v4f{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
        const float m = SWIGLU && f >= FT / 2 ? m1[tt] : m0[tt];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[f][tt][i] = __builtin_fmaf(p[i], m, acc[f][tt][i]);
      }
    }
  }

  const int quad = lane >> 4;
  if constexpr (!SWIGLU) {
    const int f0 = t.n0 + wf * BLK + quad * 32;       // the lane's 32 features
    float bias[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) bias[i] = 0.0f;
    if (grp.bias != nullptr) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (f0 + c * 8 < N) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(grp.bias + f0 + c * 8);
#pragma unroll
          for (int i = 0; i < 4; ++i) { bias[c * 8 + 2 * i] = Act::lo(v[i]); bias[c * 8 + 2 * i + 1] = Act::hi(v[i]); }
        }
    }
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const int r = wt * TT * 16 + tt * 16 + (lane & 15);
      if (r >= t.rows_here) continue;
      uint16_t* out = static_cast<uint16_t*>(op.out) + (size_t)(t.row0 + r) * N + f0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (f0 + c * 8 >= N) continue;                // N is a multiple of 16
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const v4f& q = acc[2 * c + i / 2][tt];
          v[i] = Act::pack(q[i % 2 * 2] + bias[c * 8 + 2 * i], q[i % 2 * 2 + 1] + bias[c * 8 + 2 * i + 1]);
        }
        *reinterpret_cast<u32x4*>(out + c * 8) = v;
      }
    }
  } else {
    // silu(g) * u in place of g, then the cast of the 128 features: 16 in a lane, 64 in the four lanes of a token, two waves
    __syncthreads();                                  // LDS is read no more
    uint32_t* const tops = reinterpret_cast<uint32_t*>(smem);   // [WF][BM]
    float h[TT][16];
    uint32_t top[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      top[tt] = 0;
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float g = acc[f][tt][i], u = acc[f + 4][tt][i];
          const float v = g / (1.0f + __expf(-g)) * u;
          h[tt][f * 4 + i] = v;
          top[tt] = max(top[tt], __float_as_uint(v) & 0x7fffffffu);
        }
      top[tt] = max(top[tt], (uint32_t)__shfl_xor((int)top[tt], 16, 64));
      top[tt] = max(top[tt], (uint32_t)__shfl_xor((int)top[tt], 32, 64));
      if (quad == 0) tops[wf * BM + wt * TT * 16 + tt * 16 + lane] = top[tt];
    }
    __syncthreads();
    const int f0 = t.n0 + wf * 64 + quad * 16;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt) {
      const int r = wt * TT * 16 + tt * 16 + (lane & 15);
      const float both = __uint_as_float(max(top[tt], tops[(1 - wf) * BM + r]));
      const float tp = both < TOP_FLOOR ? TOP_FLOOR : both;
      const float m = 448.0f / tp;
      if (r >= t.rows_here) continue;
      if (wf == 0 && quad == 0) op.s_out[(size_t)(t.n0 / BLK) * op.ld_out + t.row0 + r] = tp / 448.0f;
      if (f0 >= N) continue;
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = hdmoe_dev_pack4_e4m3fn(h[tt][4 * i] * m, h[tt][4 * i + 1] * m, h[tt][4 * i + 2] * m, h[tt][4 * i + 3] * m);
      *reinterpret_cast<u32x4*>(static_cast<uint8_t*>(op.out) + (size_t)(t.row0 + r) * N + f0) = v;
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

template <class Act, bool SWIGLU, int WF, int WT, int TT>
int launch_gemm(const BlockArgs& args, const char* what, hipStream_t stream) {
  constexpr int BM = WT * TT * 16, FEAT = SWIGLU ? WF * BLK / 2 : WF * BLK;
  constexpr size_t SMEM = 2 * (size_t)(BM + WF * BLK) * BLK;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_lds(block_gemm_kernel<Act, SWIGLU, WF, WT, TT>, SMEM, done, what)) return rc;
  // at most this many tiles, whatever the segments: every one of them can end in a tile that is not full
  long long tiles = 0;
  if (args.E > 0) tiles += ((long long)args.op[0].rows / BM + (args.op[0].rows < args.E ? args.op[0].rows : args.E)) * ((args.op[0].N + FEAT - 1) / FEAT);
  tiles += ((long long)args.op[1].rows + BM - 1) / BM * ((args.op[1].N + FEAT - 1) / FEAT);
  const long long grid = (tiles + HDMOE_NUM_XCD - 1) / HDMOE_NUM_XCD * HDMOE_NUM_XCD;
  if (grid > 0x7fffffffll) return hdmoe_fail(HDMOE_E_SHAPE, "%s: %lld tiles", what, tiles);
  block_gemm_kernel<Act, SWIGLU, WF, WT, TT><<<(unsigned)grid, 64 * WF * WT, SMEM, stream>>>(args);
  return hdmoe_check_launch(what);
}

int check_sizes(const char* what, const char* which, long long rows, int K, int N) {
  if (rows < 0 || K <= 0 || N <= 0 || K % 16 != 0 || N % 16 != 0)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s%s: rows=%lld K=%d N=%d (K and N must be multiples of 16)", what, which, rows, K, N);
  if ((long long)N * K > 0x7fffffffll || (long long)256 * K > 0x7fffffffll)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s%s: K=%d N=%d: a weight must be smaller than 2 GiB", what, which, K, N);
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
    block_cast_kernel<HdmoeBf16><<<(unsigned)blocks, 256, 0, s>>>(static_cast<const uint16_t*>(x), (int)rows, K, KB, static_cast<uint8_t*>(out_e4m3fn), scale, scale_stride);
  else
    block_cast_kernel<HdmoeF16><<<(unsigned)blocks, 256, 0, s>>>(static_cast<const uint16_t*>(x), (int)rows, K, KB, static_cast<uint8_t*>(out_e4m3fn), scale, scale_stride);
  return hdmoe_check_launch(what);
}

namespace {

// Arguments of both contractions -> those of the kernels; checks everything but what only the device knows.
int fill(const char* what, const hdmoe_block_args* p, bool swiglu, BlockArgs& args) {
  HDMOE_REQUIRE_PTR(p);
  if (p->out_dtype != HDMOE_W_BF16 && p->out_dtype != HDMOE_W_F16) return hdmoe_fail(HDMOE_E_SHAPE, "%s: out_dtype=%d", what, p->out_dtype);
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
    if (r.a == nullptr || r.scale_a == nullptr || r.out == nullptr || (swiglu && r.scale_out == nullptr))
      return hdmoe_fail(HDMOE_E_NULL, "%s: activations, their scales or the output are NULL", what);
    if (!aligned16(r.a) || !aligned16(r.out)) return hdmoe_fail(HDMOE_E_SHAPE, "%s: activations and outputs must start on 16 bytes", what);
    if (r.scale_a_stride < a_rows || (swiglu && r.scale_out_stride < rows))
      return hdmoe_fail(HDMOE_E_SHAPE, "%s: scale strides %lld, %lld for %d rows", what, (long long)r.scale_a_stride, (long long)r.scale_out_stride, a_rows);
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
  if (p->E > 0 && p->rows > 0) {
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
  return HDMOE_OK;
}

}  // namespace

extern "C" int hdmoe_block_linear(const hdmoe_block_args* p, hdmoe_stream_t stream) {
  BlockArgs args;
  if (int rc = fill("hdmoe_block_linear", p, false, args)) return rc;
  if (args.op[0].rows + (long long)args.op[1].rows == 0) return HDMOE_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return p->out_dtype == HDMOE_W_BF16 ? launch_gemm<HdmoeBf16, false, 2, 4, 4>(args, "hdmoe_block_linear", s)
                                      : launch_gemm<HdmoeF16, false, 2, 4, 4>(args, "hdmoe_block_linear", s);
}

extern "C" int hdmoe_block_swiglu(const hdmoe_block_args* p, hdmoe_stream_t stream) {
  BlockArgs args;
  if (int rc = fill("hdmoe_block_swiglu", p, true, args)) return rc;
  if (args.op[0].rows + (long long)args.op[1].rows == 0) return HDMOE_OK;
  return launch_gemm<HdmoeBf16, true, 2, 4, 4>(args, "hdmoe_block_swiglu", static_cast<hipStream_t>(stream));
}
