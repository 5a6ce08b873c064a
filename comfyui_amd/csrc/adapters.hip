// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out[t] = base[t] + s_a B_a (A_a x[t]),  a = index[t / rows_per] (outside 0 .. n - 1: none, out[t] = base[t])
//   h = A x, g = dy B      dx = s g A      dA_a = s sum_t g[t]^T x[t]      dB_a = s sum_t dy[t]^T h[t]
//
// Three products with a narrow side, in as many kernels: `narrow` (rows to rank), `wide` (rank to rows) and `outer` (sums over rows). Rows of
// one tile may have different adapters: a tile is gone through once for every adapter in it, and values of rows that have another one are
// never multiplied, not even by zero.
//
// Narrow values go from one kernel to the next as fp32 parts where the contraction is cut over blocks (few rows), added up by the reader; else
// scaled and split into bf16 hi and lo (lowrank.h) in the order in which the next product loads its operand: along the rank for `wide`, along the
// rows for `outer`. Both then run without LDS and barriers.
#include <type_traits>

#include "lowrank.h"

using namespace lowrank;

namespace {

constexpr int WAVES = 4;                   // of `wide_run`
constexpr int WIDE_WAVES = 2;              // of `wide`
constexpr int NARROW_WAVES = 8;
constexpr int RUN = 256;                   // tokens of a block of `wide_run` at most
constexpr int OUTER_BLOCKS = 160;          // of `outer`, about
constexpr size_t OUTER_BYTES = (size_t)1 << 30;   // of its parts at most
constexpr int STAGE = 128;                 // tokens that `outer` looks at the adapters of at a time

struct Requests {
  const int32_t* index;
  const float* scale;
  int T, rows_per, n;
  __device__ __forceinline__ int of(int t) const {
    if (t >= T) return -1;
    const int a = index[t / rows_per];
    return a >= 0 && a < n ? a : -1;
  }
};

// The adapters of up to 64 rows, one a lane (-1: none): f(adapter, lanes that have it) for each, those of turn `z` of `turns`.
template <class F>
__device__ __forceinline__ void each_adapter(int mine, int z, int turns, F f) {
  uint64_t left = __ballot(mine >= 0);
  int turn = 0;
  while (left != 0) {
    const int a = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    const uint64_t has = __ballot(mine == a);
    left &= ~has;
    if (turn == z) f(a, has);
    turn = turn + 1 == turns ? 0 : turn + 1;
  }
}

// Where narrow values end up, split: pieces of 1 KB, what the 64 lanes of an instruction load.
//   rank  [T / 16][R / 32][hi, lo][64][8]: lane 16 q + c has r = 8 q .. + 7 of token c (0 from R on)
//   rows  [T / 32][R / 16][hi, lo][64][8]: lane 16 q + c has tokens 8 q .. + 7 of r = c
// What rows without an adapter, or past T, and r past R of `rows` hold is not written and not used.
struct Planes {
  uint16_t *rank, *rows;
  int steps, tiles;     // R / 32, R / 16, filled up
};

// Eight r from r on of token t, scaled, into the planes.
__device__ __forceinline__ void put_planes(const Planes& to, int R, int t, int r, const float (&v)[8]) {
  u4 vh, vl;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h, l;
    split(v[2 * j], v[2 * j + 1], h, l);
    vh[j] = h, vl[j] = l;
  }
  if (to.rank != nullptr) {
    uint16_t* at = to.rank + (((size_t)(t >> 4) * to.steps + (r >> 5)) * 128 + ((r >> 3) & 3) * 16 + (t & 15)) * 8;
    *reinterpret_cast<u4*>(at) = vh;
    *reinterpret_cast<u4*>(at + 512) = vl;
  }
  if (to.rows != nullptr && r < R) {
    uint16_t* at = to.rows + (((size_t)(t >> 5) * to.tiles + (r >> 4)) * 128 + ((t >> 3) & 3) * 16 + (r & 15)) * 8 + (t & 7);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      at[8 * j] = (uint16_t)(vh[j / 2] >> (16 * (j & 1)));
      at[8 * j + 512] = (uint16_t)(vl[j / 2] >> (16 * (j & 1)));
    }
  }
}

struct NarrowArgs {
  Requests q;
  const uint16_t *x, *w;    // x [T, K]; w [n, R, K], or [n, K, R] (ACROSS, ACROSS32)
  float* part;              // [slices, T, R] fp32, or NULL: to the planes (one slice)
  Planes to;
  int K, R, slice, slices, turns;
};

// sum over the slice's k of x[t][k] w[a][r][k]. A tile is 16 TM tokens; the block's waves take blocks of 128 k of the slice in turn and join their sums in
// LDS. Where w runs along r, eight k of eight r a lane are transposed in registers: ACROSS has 128 r side by side in eight instructions, whatever R is;
// ACROSS32 has 32, four k blocks side by side instead, which are then dealt to instructions of 16 r each: a quarter
// of the loads and instructions (8192 x 6912 rows, rank 32: 49 -> 44 us, 36 with the rows of the next block on their way).
enum { ALONG, ACROSS, ACROSS32 };
template <class A, int MODE, int RT, int TM>
struct NarrowTile {
  static_assert(MODE == ALONG || RT == (MODE == ACROSS ? 8 : 2), "128 or 32 r");
  static_assert(RT * TM <= 16, "64 KB of LDS");
  static constexpr int EIGHTS = RT == 1 ? 4 : RT * 2;     // of r; `rank` holds 32 r at least
  typedef f4 Joined[NARROW_WAVES / 2][RT * TM][64];
  // Sums of tokens t0 .. for adapter a, r0 .. and k from lo to hi into joined[0], for every wave to read.
  static __device__ __forceinline__ void sums(const NarrowArgs& p, int a, int t0, int r0, int lo, int hi, Joined& joined) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    const int lane_row = col >> 2, lane_k = (quad * 4 + (col & 3)) * 8;      // of a load
    f4 acc[RT][TM] = {};
    const uint16_t* w = p.w + (size_t)a * p.R * p.K;
    auto load = [&](int k0, u4 (&x)[TM][4], auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      const int k = k0 + lane_k;
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint16_t* from = p.x + (size_t)min(t0 + m * 16 + i * 4 + lane_row, p.q.T - 1) * p.K + k;
          x[m][i] = WHOLE ? load8(from) : load8(from, hi - k);
        }
    };
    auto multiply = [&](int k0, u4 (&x)[TM][4], auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      const int k = k0 + lane_k;
      if constexpr (MODE == ALONG) {
        constexpr int RB = RT < 2 || TM == 4 ? 1 : 2;     // r tiles at a time: registers
#pragma unroll
        for (int rb = 0; rb < RT; rb += RB) {
          u4 wv[RB][4];
#pragma unroll
          for (int r = 0; r < RB; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint16_t* from = w + (size_t)min(r0 + (rb + r) * 16 + i * 4 + lane_row, p.R - 1) * p.K + k;
              wv[r][i] = WHOLE ? load8(from) : load8(from, hi - k);
            }
          if (rb == 0)
#pragma unroll
            for (int m = 0; m < TM; ++m) quad_transpose(x[m]);
#pragma unroll
          for (int r = 0; r < RB; ++r) quad_transpose(wv[r]);
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int r = 0; r < RB; ++r)
#pragma unroll
              for (int m = 0; m < TM; ++m) acc[rb + r][m] = A::mul(wv[r][n], x[m][n], acc[rb + r][m]);
          if (RB < RT) __builtin_amdgcn_sched_barrier(0);
        }
      } else if constexpr (MODE == ACROSS32) {
        const int r = r0 + (col & 3) * 8;
        u4 wv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {   // past the end x is 0: the last row again
          const int kk = k0 + quad * 32 + (col >> 2) * 8 + j;
          const uint16_t* from = w + (size_t)(WHOLE ? kk : min(kk, p.K - 1)) * p.R;
          wv[j] = p.R % 8 == 0 ? load8(from + min(r, p.R - 8)) : load8(from + r, p.R - r);   // r past R is not stored
        }
        transpose8(wv);
        u4 (*half)[4] = reinterpret_cast<u4 (*)[4]>(wv);      // instruction 4 h + n: block n, r = 8 (l % 4) + 4 h + l / 4 % 4
        row_transpose(half[0]);
        row_transpose(half[1]);
#pragma unroll
        for (int m = 0; m < TM; ++m) quad_transpose(x[m]);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < TM; ++m) acc[h][m] = A::mul(wv[4 * h + n], x[m][n], acc[h][m]);
      } else {
        const int r = r0 + col * 8;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          u4 wv[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {   // past the end x is 0: the last row again
            const int kk = k0 + quad * 32 + n * 8 + j;
            wv[j] = u4{0, 0, 0, 0};
            if (r < p.R) {
              const uint16_t* from = w + (size_t)(WHOLE ? kk : min(kk, p.K - 1)) * p.R + r;
              wv[j] = p.R % 8 == 0 ? load8(from) : load8(from, p.R - r);
            }
          }
          transpose8(wv);
          if (n == 0)
#pragma unroll
            for (int m = 0; m < TM; ++m) quad_transpose(x[m]);
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int m = 0; m < TM; ++m) acc[j][m] = A::mul(wv[j], x[m][n], acc[j][m]);
        }
      }
    };
    // the rows of the next block are on their way while one is multiplied
    constexpr int EACH = NARROW_WAVES * K_BLOCK;
    constexpr int AHEAD = TM < 4;
    u4 x[1 + AHEAD][TM][4];
    int k0 = lo + wave * K_BLOCK;
    if (AHEAD && k0 + K_BLOCK <= hi) load(k0, x[0], std::true_type());
    while (k0 + K_BLOCK <= hi) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (k0 + K_BLOCK <= hi) {
          if (!AHEAD) load(k0, x[0], std::true_type());
          if (AHEAD && k0 + EACH + K_BLOCK <= hi) load(k0 + EACH, x[(1 - i) * AHEAD], std::true_type());
          multiply(k0, x[i * AHEAD], std::true_type());
          k0 += EACH;
        }
    }
    if (k0 < hi) {
      load(k0, x[0], std::false_type());
      multiply(k0, x[0], std::false_type());
    }
    // the upper half of the waves into the lower one, and so on
#pragma unroll
    for (int half = NARROW_WAVES / 2; half > 0; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half)
#pragma unroll
        for (int i = 0; i < RT * TM; ++i) joined[wave - half][i][lane] = acc[i / TM][i % TM];
      __syncthreads();
      if (wave < half)
#pragma unroll
        for (int i = 0; i < RT * TM; ++i) {
          acc[i / TM][i % TM] += joined[wave][i][lane];
          if (half == 1) joined[0][i][lane] = acc[i / TM][i % TM];
        }
    }
    __syncthreads();
  }
  // Eight r of token `bit` of the tile, 0 from R on
  static __device__ __forceinline__ void eight(const Joined& joined, int R, int r0, int bit, int eight, float scale, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      // r of a result: ACROSS 8 row + tile, ACROSS32 8 (row % 4) + 4 tile + row / 4, else 16 tile + row_of(row) (which undoes itself, as for tokens)
      const int row = MODE == ACROSS ? eight : MODE == ACROSS32 ? (j & 3) * 4 + (eight & 3) : row_of((eight & 1) * 8 + j);
      const int tile_r = MODE == ACROSS ? j : MODE == ACROSS32 ? j >> 2 : min(eight >> 1, RT - 1);
      v[j] = r0 + eight * 8 + j < R ? joined[0][tile_r * TM + (bit >> 4)][(row >> 2) * 16 + row_of(bit & 15)][row & 3] * scale : 0.0f;
    }
  }
  // One block's share of the whole product: tile, slice and turn from `block`.
  static __device__ __forceinline__ void run(const NarrowArgs& p, int block, int r0, Joined& joined) {
    const int lane = threadIdx.x & 63;
    const int tiles = (p.q.T + 16 * TM - 1) / (16 * TM);
    const int tile = block % tiles, slice = (block / tiles) % p.slices, z = block / tiles / p.slices;
    const int t0 = tile * 16 * TM, lo = slice * p.slice, hi = min(p.K, lo + p.slice);
    const int mine = lane < 16 * TM ? p.q.of(t0 + lane) : -1;
    each_adapter(mine, z, p.turns, [&](int a, uint64_t has) {
      sums(p, a, t0, r0, lo, hi, joined);
      const float scale = p.part != nullptr ? 1.0f : p.q.scale[a];
      for (int u = threadIdx.x; u < 16 * TM * EIGHTS; u += NARROW_WAVES * 64) {
        const int e = u / (16 * TM), bit = u % (16 * TM), r = r0 + e * 8, t = t0 + bit;
        if (!((has >> bit) & 1)) continue;
        float v[8];
        eight(joined, p.R, r0, bit, e, scale, v);
        if (p.part == nullptr) {
          if (r < p.to.steps * 32) put_planes(p.to, p.R, t, r, v);
          continue;
        }
        float* to = p.part + ((size_t)slice * p.q.T + t) * p.R + r;
        if (r + 8 <= p.R) __builtin_memcpy(to, v, 32);
        else
          for (int j = 0; j < 8; ++j)
            if (r + j < p.R) to[j] = v[j];
      }
    });
  }
};

template <class A, int RT, int TM>
__global__ __launch_bounds__(NARROW_WAVES * 64) void narrow_kernel(NarrowArgs p) {
  typedef NarrowTile<A, ALONG, RT, TM> Tile;
  __shared__ typename Tile::Joined joined;
  Tile::run(p, blockIdx.x, blockIdx.y * 16 * RT, joined);
}

// h and g of the backward pass in one launch: the shorter one's blocks fill what the longer one's leave.
template <class A, int MODE, int RT, int RTG, int TM>
__global__ __launch_bounds__(NARROW_WAVES * 64) void narrow_pair_kernel(NarrowArgs h, NarrowArgs g, int blocks_g) {
  typedef NarrowTile<A, ALONG, RT, TM> H;
  typedef NarrowTile<A, MODE, RTG, TM> G;
  __shared__ union {
    typename H::Joined h;
    typename G::Joined g;
  } joined;
  if ((int)blockIdx.x < blocks_g) G::run(g, blockIdx.x, blockIdx.y * 16 * RTG, joined.g);
  else H::run(h, blockIdx.x - blocks_g, blockIdx.y * 16 * RT, joined.h);
}

// v += eight values of each of `slices` parts, `next` apart (`have` of them).
__device__ __forceinline__ void add_parts(const float* from, int slices, size_t next, int have, float (&v)[8]) {
  if (have >= 8) {
#pragma unroll 4
    for (int s = 0; s < slices; ++s) {
      f4 q[2];
      __builtin_memcpy(q, from + s * next, 32);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += q[j / 4][j % 4];
    }
  } else {
    for (int s = 0; s < slices; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < have) v[j] += from[s * next + j];
  }
}

// Parts to planes: sums of the slices, scaled and split. Eight r of a row a thread.
struct JoinArgs {
  Requests q;
  const float* part[2];     // h, g; NULL: planes are there
  Planes to[2];
  int slices[2], R;
};
__global__ __launch_bounds__(64) void join_kernel(JoinArgs p) {
  const int side = blockIdx.y;
  if (p.part[side] == nullptr) return;
  const int eights = p.to[side].steps * 4;
  const int64_t u = (int64_t)blockIdx.x * 64 + threadIdx.x;
  const int t = (int)(u % p.q.T), r = (int)(u / p.q.T) * 8;
  if (r >= eights * 8) return;
  const int a = p.q.of(t);
  if (a < 0) return;
  float v[8] = {};
  add_parts(p.part[side] + (size_t)t * p.R + r, p.slices[side], (size_t)p.q.T * p.R, p.R - r, v);
  const float f = p.q.scale[a];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] *= f;
  put_planes(p.to[side], p.R, t, r, v);
}

struct WideArgs {
  Requests q;
  const float* part;                  // [slices, T, R] (wide_kernel)
  const uint16_t* rank;               // Planes::rank (wide_run_kernel; wide_kernel without parts)
  const uint16_t *w, *base;           // w [n, C, R] and base [T, C], or w [n, R, C] and no base (TURNED)
  uint16_t* out;                      // [T, C]
  int C, R, slices, turns;
};

// out[t][c] = base[t][c] + s sum_r h[t][r] w[a][c][r] of 16 tokens and 128 columns, of which a lane has 32 of token l % 16 next to each other in the products. Base
// and out are loaded and stored transposed among four lanes: piece j of lane l is 16 bytes of token 4 (l / 4 % 4) + j.
template <class A, bool TURNED>
struct Wide {
  static constexpr int COLS = 128;
  const WideArgs& p;
  int c0, col, quad, c, have;
  bool whole;
  __device__ __forceinline__ Wide(const WideArgs& args, int first, int lane) : p(args), c0(first), col(lane & 15), quad(lane >> 4) {
    // The last 128 for a wave that would have fewer (10220 x 1120, rank 104, 36 -> 22.7 us): without a base a column may be written twice.
    if (TURNED && first < p.C && p.C >= COLS) c0 = min(first, p.C - COLS);
    c = c0 + quad * 32 + (col & 3) * 8;      // of a load or store
    have = p.C - c;
    whole = c0 + COLS <= p.C;
  }
  __device__ __forceinline__ int token(int j) const { return (col & 12) + j; }
  // Weights of 32 r from r0 on, in bf16. r past R meets values of 0: the row's last ones again, so that nothing but the lane's own column enters.
  __device__ __forceinline__ void weights(int a, int r0, u4 (&wh)[8], u4 (&wl)[8]) const {
    const uint16_t* w = p.w + (size_t)a * p.R * p.C;
    const int r = r0 + quad * 8;
    if constexpr (TURNED) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = c0 + col * 8;     // result row 4 quad + e of instruction j: value 8 e + j of the lane's 32
        const uint16_t* from = w + (size_t)min(r + j, p.R - 1) * p.C + at;
        wh[j] = whole ? load8(from) : load8(from, p.C - at);
      }
      transpose8(wh);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {      // value 4 j + e
        const uint16_t* from = w + (size_t)min(c0 + (col >> 2) * 32 + j * 4 + (col & 3), p.C - 1) * p.R;
        wh[j] = p.R % 8 == 0 ? load8(from + min(r, p.R - 8)) : load8(from + r, p.R - r);
      }
    }
    if constexpr (A::HALF)
#pragma unroll
      for (int j = 0; j < 8; ++j) to_bf16<A>(wh[j], wh[j], wl[j]);
  }
  // base of the tokens t + 0 .. 15 that `want` says (bits)
  __device__ __forceinline__ void base(int t, uint32_t want, u4 (&b)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (TURNED) continue;
      b[j] = u4{0, 0, 0, 0};
      if ((want >> token(j)) & 1) {
        const uint16_t* from = p.base + (size_t)(t + token(j)) * p.C + c;
        b[j] = whole ? load8(from) : load8(from, have);
      }
    }
  }
  __device__ __forceinline__ void put(int t, uint32_t want, const f4 (&acc)[8], u4 (&b)[4]) const {
    if constexpr (!TURNED) quad_transpose(b);
    u4 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int u = 8 * i + 2 * w;
        const float v0 = TURNED ? acc[u % 8][u / 8] : acc[u / 4][u % 4], v1 = TURNED ? acc[u % 8 + 1][u / 8] : acc[u / 4][u % 4 + 1];
        if constexpr (TURNED) o[i][w] = A::pack(v0, v1);
        else o[i][w] = A::pack(v0 + A::lo(b[i][w]), v1 + A::hi(b[i][w]));
      }
    quad_transpose(o);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((want >> token(j)) & 1) {
        uint16_t* to = p.out + (size_t)(t + token(j)) * p.C + c;
        if (whole) __builtin_memcpy(to, &o[j], 16);
        else store8(to, o[j], have);
      }
  }
  // rows without an adapter: the base as it is, bit for bit
  __device__ __forceinline__ void copy(int t, uint32_t want) const {
    if ((const void*)p.out == (const void*)p.base || want == 0) return;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if ((want >> token(j)) & 1) {
        const size_t at = (size_t)(t + token(j)) * p.C + c;
        u4 v = {0, 0, 0, 0};
        if constexpr (!TURNED) v = load8(p.base + at, have);
        store8(p.out + at, v, have);
      }
  }
};

// Few rows, or rows of many adapters: 16 tokens a tile, whose adapters are dealt to `turns` blocks. Their narrow values are added up from the parts and
// split in LDS, or loaded as `rank` has them (p.part NULL).
template <class A, bool TURNED>
__global__ __launch_bounds__(WIDE_WAVES * 64) void wide_kernel(WideArgs p) {
  typedef Wide<A, TURNED> W;
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];   // [2][16][stride]: hi, lo of s h
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int steps = (p.R + 31) / 32, stride = steps * 32 + 8;
  const int tiles = (p.q.T + 15) / 16, chunks = (p.C + WIDE_WAVES * W::COLS - 1) / (WIDE_WAVES * W::COLS);
  const int chunk = blockIdx.x % chunks, tile = (blockIdx.x / chunks) % tiles, z = blockIdx.x / chunks / tiles;
  const int t0 = tile * 16;
  const int mine = lane < 16 ? p.q.of(t0 + lane) : -1;
  const W w(p, (chunk * WIDE_WAVES + wave) * W::COLS, lane);
  // the first adapter's weights and base are on their way meanwhile
  int early = -1;
  u4 wh[8], wl[8], b[4];
  each_adapter(mine, z, p.turns, [&](int a, uint64_t has) {
    if (early >= 0 || w.c0 >= p.C) return;
    early = a;
    w.weights(a, 0, wh, wl);
    w.base(t0, (uint32_t)has, b);
  });
  for (int u = threadIdx.x; p.part != nullptr && u < 16 * steps * 4; u += WIDE_WAVES * 64) {   // eight values a thread
    const int row = u / (steps * 4), r = (u - row * (steps * 4)) * 8, t = t0 + row;
    const int a = p.q.of(t);
    float v[8] = {};
    if (a >= 0) {
      const float f = p.q.scale[a];
      add_parts(p.part + (size_t)t * p.R + r, p.slices, (size_t)p.q.T * p.R, p.R - r, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= f;
    }
    u4 vh, vl;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t h, l;
      split(v[2 * j], v[2 * j + 1], h, l);
      vh[j] = h, vl[j] = l;
    }
    *reinterpret_cast<u4*>(lds + (size_t)row * stride + r) = vh;
    *reinterpret_cast<u4*>(lds + (size_t)(16 + row) * stride + r) = vl;
  }
  __syncthreads();
  if (w.c0 >= p.C) return;
  if (z == 0) w.copy(t0, (uint32_t)__ballot(lane < 16 && mine < 0 && t0 + lane < p.q.T));
  each_adapter(mine, z, p.turns, [&](int a, uint64_t has) {
    if (a != early) w.base(t0, (uint32_t)has, b);
    f4 acc[8] = {};
    for (int s = 0; s < steps; ++s) {
      if (a != early || s > 0) w.weights(a, s * 32, wh, wl);
      u4 qh, ql;
      if (p.part != nullptr) {
        qh = *reinterpret_cast<const u4*>(lds + (size_t)col * stride + s * 32 + quad * 8);
        ql = *reinterpret_cast<const u4*>(lds + (size_t)(16 + col) * stride + s * 32 + quad * 8);
      } else {
        const uint16_t* from = p.rank + (((size_t)tile * steps + s) * 128 + lane) * 8;
        qh = *reinterpret_cast<const u4*>(from);
        ql = *reinterpret_cast<const u4*>(from + 512);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = mul_split<A>(wh[j], wl[j], qh, ql, acc[j]);
    }
    w.put(t0, (uint32_t)has, acc, b);
  });
}

// Very few rows: both products in one launch. Every block goes through the whole contraction for its tile and turn, whose weights come out of the
// caches, and two of its waves have 128 columns each; one launch fewer is worth 3 us.
template <class A, int RT>
__global__ __launch_bounds__(NARROW_WAVES * 64) void few_kernel(NarrowArgs np, WideArgs p) {
  typedef NarrowTile<A, ALONG, RT, 1> Tile;
  typedef Wide<A, false> W;
  __shared__ typename Tile::Joined joined;
  __shared__ __attribute__((aligned(16))) uint16_t values[2][RT < 2 ? 1 : RT / 2][64][8];     // as Planes::rank of one tile
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int tiles = (p.q.T + 15) / 16, chunks = (p.C + WIDE_WAVES * W::COLS - 1) / (WIDE_WAVES * W::COLS), steps = (p.R + 31) / 32;
  const int chunk = blockIdx.x % chunks, tile = (blockIdx.x / chunks) % tiles, z = blockIdx.x / chunks / tiles;
  const int t0 = tile * 16;
  const int mine = lane < 16 ? p.q.of(t0 + lane) : -1;
  const W w(p, (chunk * WIDE_WAVES + wave) * W::COLS, lane);
  const bool writes = wave < WIDE_WAVES && w.c0 < p.C;
  if (writes && z == 0) w.copy(t0, (uint32_t)__ballot(lane < 16 && mine < 0 && t0 + lane < p.q.T));
  each_adapter(mine, z, p.turns, [&](int a, uint64_t has) {
    u4 wh[8], wl[8], b[4];
    if (writes) {      // on their way meanwhile
      w.weights(a, 0, wh, wl);
      w.base(t0, (uint32_t)has, b);
    }
    Tile::sums(np, a, t0, 0, 0, np.K, joined);
    const float scale = p.q.scale[a];
    for (int u = threadIdx.x; u < 16 * steps * 4; u += NARROW_WAVES * 64) {
      float v[8];
      Tile::eight(joined, p.R, 0, u & 15, u >> 4, scale, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t h, l;
        split(v[2 * j], v[2 * j + 1], h, l);
        *reinterpret_cast<uint32_t*>(&values[0][u >> 6][u & 63][2 * j]) = h;
        *reinterpret_cast<uint32_t*>(&values[1][u >> 6][u & 63][2 * j]) = l;
      }
    }
    __syncthreads();
    if (!writes) return;
    f4 acc[8] = {};
    for (int s = 0; s < steps; ++s) {
      if (s > 0) w.weights(a, s * 32, wh, wl);
      const u4 qh = *reinterpret_cast<const u4*>(values[0][s][lane]), ql = *reinterpret_cast<const u4*>(values[1][s][lane]);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = mul_split<A>(wh[j], wl[j], qh, ql, acc[j]);
    }
    w.put(t0, (uint32_t)has, acc, b);
  });
}

// Many rows: a block has up to RUN tokens, 16 at a time; a wave keeps the weights of its columns in registers for as long as the adapter stays the same (R up to
// 32 STEPS; `parts` times that are gone through one after the other, for GROUPS times 16 tokens at a time). Bound by base and out: R of 64 takes 32 instructions
// (512 cycles of one of four units) for 8 KB of them. Where the whole run has one adapter, values and base of the AHEAD 16 tokens to come are on
// their way while some are multiplied; of longer ranks the next weights (16384 x 2560, rank 128, 112 -> 86 us).
template <class A, bool TURNED, int STEPS, int GROUPS>
__global__ __launch_bounds__(WAVES * 64) void wide_run_kernel(WideArgs p, int parts, int run) {
  typedef Wide<A, TURNED> W;
  constexpr int AHEAD = 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunks = (p.C + WAVES * W::COLS - 1) / (WAVES * W::COLS), steps = (p.R + 31) / 32;
  const int chunk = blockIdx.x % chunks, t0 = blockIdx.x / chunks * run;
  const W w(p, (chunk * WAVES + wave) * W::COLS, lane);
  if (w.c0 >= p.C) return;
  const int end = min(p.q.T, t0 + run);
  int of[RUN / 64];
  const int first = p.q.of(t0);
  bool same = first >= 0;
#pragma unroll
  for (int i = 0; i < RUN / 64; ++i) {
    const int t = t0 + i * 64 + lane;
    of[i] = t < end ? p.q.of(t) : -1;
    same = same && (t >= end || of[i] == first);
  }
  const int groups = (end - t0 + 15) / 16;
  auto in = [&](int g) { return end - t0 - g * 16 >= 16 ? 0xffffu : (1u << (end - t0 - g * 16)) - 1; };   // tokens of the group that there are
  struct Tokens {
    u4 q[2][STEPS], b[4];
  };
  auto values = [&](int g, int part, u4 (&q)[2][STEPS]) {
    const uint16_t* from = p.rank + ((size_t)(t0 / 16 + g) * steps * 128 + lane) * 8;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int at = min(part * STEPS + s, steps - 1);     // past the last step the weights are
      q[0][s] = *reinterpret_cast<const u4*>(from + (size_t)at * 1024);
      q[1][s] = *reinterpret_cast<const u4*>(from + (size_t)at * 1024 + 512);
      if (part * STEPS + s >= steps) q[0][s] = q[1][s] = u4{0, 0, 0, 0};
    }
  };
  u4 wh[STEPS][8], wl[STEPS][8];
  auto multiply = [&](const u4 (&q)[2][STEPS], f4 (&acc)[8]) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = mul_split<A>(wh[s][j], wl[s][j], q[0][s], q[1][s], acc[j]);
  };
  if constexpr (GROUPS > 1) {
    static_assert(STEPS == 1);
    if (__all(same)) {
      u4 nh[8], nl[8];       // weights of the next part, on their way
      w.weights(first, 0, nh, nl);
      for (int g = 0; g < groups; g += GROUPS) {
        f4 acc[GROUPS][8] = {};
        for (int part = 0; part < parts; ++part) {
          u4 q[GROUPS][2][STEPS];
#pragma unroll
          for (int i = 0; i < GROUPS; ++i) values(min(g + i, groups - 1), part, q[i]);
#pragma unroll
          for (int j = 0; j < 8; ++j) wh[0][j] = nh[j], wl[0][j] = nl[j];
          w.weights(first, (part + 1 < parts ? part + 1 : 0) * 32, nh, nl);
#pragma unroll
          for (int i = 0; i < GROUPS; ++i) multiply(q[i], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < GROUPS; ++i)
          if (g + i < groups) {
            u4 b[4];
            w.base(t0 + (g + i) * 16, in(g + i), b);
            w.put(t0 + (g + i) * 16, in(g + i), acc[i], b);
          }
      }
      return;
    }
  } else if (__all(same)) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) w.weights(first, s * 32, wh[s], wl[s]);
    Tokens k[AHEAD];
    auto load = [&](int g, Tokens& v) {
      values(g, 0, v.q);
      w.base(t0 + g * 16, in(g), v.b);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (i < groups) load(i, k[i]);
    for (int g = 0; g < groups; g += AHEAD)
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (g + i < groups) {
          f4 acc[8] = {};
          multiply(k[i].q, acc);
          w.put(t0 + (g + i) * 16, in(g + i), acc, k[i].b);
          if (g + i + AHEAD < groups) load(g + i + AHEAD, k[i]);
        }
    return;
  }
  int held = -1;
  for (int g = 0; g < groups; ++g) {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < RUN / 64; ++i)
      if (g / 4 == i) mine = of[i];
    mine = __shfl(mine, (g & 3) * 16 + (lane & 15), 64);
    w.copy(t0 + g * 16, (uint32_t)__ballot(mine < 0) & in(g));
    each_adapter(mine, 0, 1, [&](int a, uint64_t has) {
      Tokens k;
      w.base(t0 + g * 16, (uint32_t)has & 0xffff, k.b);
      f4 acc[8] = {};
      for (int part = 0; part < parts; ++part) {
        values(g, part, k.q);
        if (a != held || parts > 1) {
#pragma unroll
          for (int s = 0; s < STEPS; ++s) w.weights(a, (part * STEPS + s) * 32, wh[s], wl[s]);
          held = a;
        }
        multiply(k.q, acc);
      }
      w.put(t0 + g * 16, (uint32_t)has & 0xffff, acc, k.b);
    });
  }
}

struct OuterSide {
  const uint16_t* v;        // [T, C]
  const uint16_t* rows;     // Planes::rows
  void* out;                // fp32 parts [splits, n, R, C] (flip: [splits, n, C, R]), or the result itself
  int C, flip, blocks;      // blocks of 512 columns
};

struct OuterArgs {
  Requests q;
  OuterSide side[2];
  int32_t* there;           // [splits, n]: whether a part was written; NULL with one split
  int R, splits, per_split, tiles, turns;   // per_split: tokens, a multiple of STAGE
};

// out[a][r][c] = s sum over the rows t of adapter a of q[t][r] v[t][c], 16 RT of the r. A block has one run of rows and the adapters that it finds there, one
// after the other (or every turns-th): what rows share an adapter, and how many adapters have none, changes nothing in how the rows are dealt to blocks. A
// wave has 128 columns and one half of the rows: eight rows of eight columns a lane are loaded as they lie and transposed in registers; the halves are joined in LDS.
template <class A, int RT>
__global__ __launch_bounds__(512, 2) void outer_kernel(OuterArgs p) {
  static_assert(RT <= 2, "64 KB of LDS; four r tiles do not fit the registers beside the rows to come either");
  constexpr int WORDS = HDMOE_ADAPTER_MAX / 32;
  static_assert(WORDS == 128, "two words a lane");
  __shared__ union {
    uint32_t seen[WORDS];
    f4 joined[4][8 * RT][64];
  } lds;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const bool second = (int)blockIdx.x >= p.side[0].blocks;
  const OuterSide side = second ? p.side[1] : p.side[0];
  const int block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
  const int turn = blockIdx.y % p.turns, r0 = blockIdx.y / p.turns * 16 * RT, split = blockIdx.z;
  // The last 128 columns for a wave that would have fewer: the same loads for all (10220 rows of 1120 and 488 columns, rank 104, 70 -> 36 us). What two waves
  // have of them is the same sum twice.
  const int own = (block * 4 + (wave & 3)) * 128;
  const bool on = own < side.C;
  const int c0 = on && side.C >= 128 ? min(own, side.C - 128) : own, c = c0 + col * 8, have = side.C - c;
  const bool whole = c0 + 128 <= side.C;
  const int64_t start = (int64_t)split * p.per_split;
  const int64_t begin = start + (wave >> 2) * (p.per_split / 2);
  const int end = (int)min((int64_t)p.q.T, begin + p.per_split / 2);
  // the adapters of the run, a bit each: word l and l + 64 in lane l
  uint32_t seen_low = 0, seen_high = 0;
  const int64_t stop = min((int64_t)p.q.T, start + p.per_split);
  const int head = (int)(start / p.q.rows_per), last = start < p.q.T ? (int)((stop - 1) / p.q.rows_per) : head - 1;
  if (head == last) {       // one request
    const int a = p.q.index[head];
    if (a >= 0 && a < p.q.n) {
      if ((a >> 5) == lane) seen_low = 1u << (a & 31);
      if ((a >> 5) == lane + 64) seen_high = 1u << (a & 31);
    }
  } else {
    if (threadIdx.x < WORDS) lds.seen[threadIdx.x] = 0;
    __syncthreads();
    for (int i = head + threadIdx.x; i <= last; i += 512) {
      const int a = p.q.index[i];
      if (a >= 0 && a < p.q.n) atomicOr(&lds.seen[a >> 5], 1u << (a & 31));
    }
    __syncthreads();
    seen_low = lds.seen[lane];
    seen_high = lds.seen[lane + 64];
    __syncthreads();
  }
  if (p.there != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && wave == 0)
#pragma unroll
    for (int h = 0; h < 2; ++h)
      for (int j = 0; j < 32; ++j) {
        const int a = (lane + 64 * h) * 32 + j;
        if (a < p.q.n) p.there[(size_t)split * p.q.n + a] = ((h == 0 ? seen_low : seen_high) >> j) & 1;
      }
  // f of every adapter whose bit is `bit`, those of the block's turn
  auto each = [&](uint32_t flip, auto f) {
    int at = 0;
    for (int w = 0; w * 32 < p.q.n; ++w) {
      const int there = w < 64 ? __builtin_amdgcn_readlane(seen_low, w) : __builtin_amdgcn_readlane(seen_high, w - 64);
      uint32_t word = (uint32_t)there ^ flip;
      if (p.q.n - w * 32 < 32) word &= (1u << (p.q.n - w * 32)) - 1;
      for (; word != 0; word &= word - 1) {
        if (at == turn) f(w * 32 + __builtin_ctz(word));
        at = at + 1 == p.turns ? 0 : at + 1;
      }
    }
  };
  // values of 32 rows, r tile r
  auto value = [&](int t, int r, int lo) {
    return *reinterpret_cast<const u4*>(side.rows + (((size_t)(t >> 5) * p.tiles + min((r0 >> 4) + r, p.tiles - 1)) * 128 + 64 * lo + lane) * 8);
  };
  auto accumulate = [&](int a, f4 (&acc)[RT][8]) {
    if (on)
      for (int t0 = (int)min(begin, (int64_t)p.q.T); t0 < end; t0 += STAGE) {
        const uint64_t first = __ballot(t0 + lane < end && p.q.of(t0 + lane) == a), next = __ballot(t0 + 64 + lane < end && p.q.of(t0 + 64 + lane) == a);
        if ((first | next) == 0) continue;
        const bool all = whole && (first & next) == ~0ull;
        auto multiply = [&](u4 (&v)[8], u4 (&qh)[RT], u4 (&ql)[RT]) {
          transpose8(v);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            u4 vh, vl;
            to_bf16<A>(v[j], vh, vl);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              acc[r][j] = Bf16::mul(ql[r], vh, acc[r][j]);
              if constexpr (A::HALF) acc[r][j] = Bf16::mul(qh[r], vl, acc[r][j]);
              acc[r][j] = Bf16::mul(qh[r], vh, acc[r][j]);
            }
          }
        };
        const uint16_t* from = side.v + (size_t)(t0 + quad * 8) * side.C + c;
        if (all) {
          u4 v[2][8];
          auto load = [&](int st, u4 (&x)[8]) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = load8(from + (size_t)(st * 32 + j) * side.C);
          };
          load(0, v[0]);
#pragma unroll
          for (int st = 0; st < STAGE / 32; ++st) {
            u4 qh[RT], ql[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              qh[r] = value(t0 + st * 32, r, 0);
              ql[r] = value(t0 + st * 32, r, 1);
            }
            if (st + 1 < STAGE / 32) load(st + 1, v[(st + 1) & 1]);
            multiply(v[st & 1], qh, ql);
          }
          continue;
        }
        for (int st = 0; st < STAGE / 32; ++st) {
          const uint32_t has = (uint32_t)((st < 2 ? first : next) >> (32 * (st & 1)));
          if (has == 0) continue;
          const uint32_t eight = (has >> (quad * 8)) & 0xff;
          // rows of another adapter, or past the last one, are 0 on both sides
          u4 v[8], qh[RT], ql[RT], keep;
#pragma unroll
          for (int j = 0; j < 4; ++j) keep[j] = ((eight >> (2 * j)) & 1 ? 0xffffu : 0u) | ((eight >> (2 * j + 1)) & 1 ? 0xffff0000u : 0u);
          if (whole && has == ~0u) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = load8(from + (size_t)(st * 32 + j) * side.C);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[j] = u4{0, 0, 0, 0};
              if ((eight >> j) & 1) v[j] = load8(from + (size_t)(st * 32 + j) * side.C, have);
            }
          }
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            qh[r] = value(t0 + st * 32, r, 0) & keep;
            ql[r] = value(t0 + st * 32, r, 1) & keep;
          }
          multiply(v, qh, ql);
        }
      }
  };
  // One adapter's result, 4 r and 8 columns a lane
  auto store = [&](int a, const f4 (&acc)[RT][8]) {
    const size_t at = ((size_t)split * p.q.n + a) * p.R * side.C;
    const bool direct = p.there == nullptr;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int row = r0 + r * 16 + quad * 4;
      if (side.flip) {        // a column's four r next to each other
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= have || row >= p.R) continue;
          const size_t i = at + (size_t)(c + j) * p.R + row;
          if (direct) {
            uint16_t* to = static_cast<uint16_t*>(side.out) + i;
            const uint32_t o[2] = {A::pack(acc[r][j][0], acc[r][j][1]), A::pack(acc[r][j][2], acc[r][j][3])};
            if (row + 4 <= p.R) __builtin_memcpy(to, o, 8);
            else
              for (int e = 0; e < 4; ++e)
                if (row + e < p.R) to[e] = (uint16_t)(o[e / 2] >> (16 * (e & 1)));
          } else {
            float* to = static_cast<float*>(side.out) + i;
            if (row + 4 <= p.R) __builtin_memcpy(to, &acc[r][j], 16);
            else
              for (int e = 0; e < 4; ++e)
                if (row + e < p.R) to[e] = acc[r][j][e];
          }
        }
      } else {                // a row's eight columns
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (row + e >= p.R || have <= 0) continue;
          const size_t i = at + (size_t)(row + e) * side.C + c;
          if (direct) {
            u4 o;
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] = A::pack(acc[r][2 * k][e], acc[r][2 * k + 1][e]);
            store8(static_cast<uint16_t*>(side.out) + i, o, have);
          } else {
            float* to = static_cast<float*>(side.out) + i;
            if (have >= 8) {
              const f4 o[2] = {{acc[r][0][e], acc[r][1][e], acc[r][2][e], acc[r][3][e]}, {acc[r][4][e], acc[r][5][e], acc[r][6][e], acc[r][7][e]}};
              __builtin_memcpy(to, o, 32);
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (j < have) to[j] = acc[r][j][e];
            }
          }
        }
      }
    }
  };
  each(0, [&](int a) {
    f4 acc[RT][8] = {};
    accumulate(a, acc);
    if (wave >= 4)
#pragma unroll
      for (int j = 0; j < 8 * RT; ++j) lds.joined[wave - 4][j][lane] = acc[j / 8][j % 8];
    __syncthreads();
    if (wave < 4 && on) {
#pragma unroll
      for (int j = 0; j < 8 * RT; ++j) acc[j / 8][j % 8] += lds.joined[wave][j][lane];
      store(a, acc);
    }
    __syncthreads();
  });
  if (p.there != nullptr || wave >= 4 || !on) return;
  const f4 zero[RT][8] = {};
  each(~0u, [&](int a) { store(a, zero); });      // adapters without rows
}

// ---- sizes ---------------------------------------------------------------------------------------------------------

struct Side {                 // a narrow product
  int slices, slice;
  size_t part, rank, rows;    // bytes of its parts and planes in the workspace
};

struct Plan {
  int tm, turns, run, few, mixed, fine;   // run: many rows; few: one launch; mixed: rows of several adapters to a tile; fine: 32 r a block of `narrow`
  Side h, g;
  int steps, tiles, splits, per_split, rt, outer_turns;
  size_t da_bytes, db_bytes, there_bytes, total;
};

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

size_t bytes_of(size_t n) { return hdmoe_align_up(n, 256); }

constexpr int64_t FEW_BYTES = 64 << 20;   // that the blocks of `few` may read
constexpr int64_t LANES_MAX = (int64_t)1 << 32;
constexpr int MANY_ROWS = 512;            // from here on `wide` keeps its weights over runs of tokens

// The contraction is cut over blocks until the card has about one a CU, in slices of a block of each wave at least; `whole`: not at all. A whole one has one
// order of its additions in every kernel here (each wave's blocks of 128 k in turn, the waves' sums by halves), and so have the sums over the rank.
void cut(int tiles, int turns, int K, int rblocks, bool whole, Side& s) {
  const int most = div_up(K, NARROW_WAVES * K_BLOCK);
  int want = whole ? 1 : div_up(HDMOE_NUM_CU, (int64_t)tiles * turns * rblocks);
  if (want > most) want = most;
  if (want > 8) want = 8;
  s.slice = div_up(div_up(K, want), NARROW_WAVES * K_BLOCK) * NARROW_WAVES * K_BLOCK;
  s.slices = div_up(K, s.slice);
}

Plan plan_of(const hdmoe_adapter_args& a, bool backward) {
  Plan p = {};
  const int rows_per = a.rows / a.requests;
  p.mixed = rows_per < 16 && a.n > 1 && a.requests > 1;
  p.run = a.rows >= MANY_ROWS && !p.mixed;
  // tokens of a tile of `narrow`: 16, and more where there are tiles for every CU all the same and a tile's rows share an adapter
  p.tm = rows_per < 64 || a.rows < 32 * HDMOE_NUM_CU ? 1 : a.rows < 64 * HDMOE_NUM_CU || a.R > 64 ? 2 : 4;
  const int tile = 16 * p.tm;
  p.turns = div_up(tile, rows_per);          // adapters of a tile at most, as tiles go
  if (p.turns > a.n) p.turns = a.n;
  if (p.turns > a.requests) p.turns = a.requests;
  const int tiles = div_up(a.rows, tile);
  // Long ranks over more blocks where there are few: up to 128 r a block load their weights in turns (130 rows of 416 columns, rank 88, 12.0 -> 6.2 us, 1860 of
  // 2568, rank 80, 351 blocks, 27 -> 19; but 4000 of 2560, rank 64, 500 blocks, 11.3 -> 14.7: each reads the rows again).
  p.fine = a.R > 32 && (int64_t)tiles * p.turns * div_up(a.R, 32) <= HDMOE_NUM_CU * 3 / 2;
  const int rblocks = div_up(a.R, p.fine ? 32 : 128);
  cut(tiles, p.turns, a.K, rblocks, !backward && (p.run || a.fixed_k_cut), p.h);
  p.steps = div_up(a.R, 32), p.tiles = div_up(a.R, 16);
  const size_t part = (size_t)a.rows * a.R * sizeof(float), rank = (size_t)div_up(a.rows, 16) * p.steps * 2048;
  const size_t rows = (size_t)div_up(a.rows, STAGE) * (STAGE / 32) * p.tiles * 2048;
  if (!backward) {
    // One launch, whose blocks each read x and w for themselves, while all of them run at once and that is little for the caches: 1 row of 2560 x 6912, rank 16,
    // 9.4 -> 6.5 us, 8 rows of 8 adapters (34 MB) 10.7 -> 6.9, 64 rows of one 10.0 -> 6.6; 16 rows of 16 adapters, 432 blocks, 12.4 -> 12.3.
    const int64_t blocks = (int64_t)div_up(a.N, 128 * WIDE_WAVES) * tiles * p.turns;
    p.few = a.R <= 64 && !p.run && blocks <= HDMOE_NUM_CU && blocks * (a.R + 16) * a.K * 2 <= FEW_BYTES;
    if (p.few) return p;
    if (p.run) p.h.rank = rank;
    else p.h.part = bytes_of(part * p.h.slices);
    p.total = p.h.part + p.h.rank;
    return p;
  }
  cut(tiles, p.turns, a.N, rblocks, false, p.g);
  p.h.part = p.h.slices > 1 ? bytes_of(part * p.h.slices) : 0;
  p.g.part = p.g.slices > 1 ? bytes_of(part * p.g.slices) : 0;
  p.h.rows = p.g.rows = rows;
  p.g.rank = rank;
  p.rt = a.R <= 16 ? 1 : 2;
  // Rows are cut over blocks, 128 each at least, until there are 160 of these: parts are written and read again, and a run is whole stages of both halves (two
  // adapters of 4096 rows, 2560 and 6912 columns, rank 32: 152 blocks 33 us, 247 39, 133 46); a run's adapters over as many blocks as there
  // can be adapters in it, if there are CUs for them.
  const int64_t blocks = (int64_t)(div_up(a.K, 512) + div_up(a.N, 512)) * div_up(a.R, 16 * p.rt);
  const int cus = div_up(OUTER_BLOCKS, blocks), most = div_up(a.rows, STAGE);
  const int all = a.n < a.requests ? a.n : a.requests;      // adapters of all rows at most
  // Parts are of all adapters, those of other rows too: with many of them, fewer runs and in the end none.
  const size_t one = (size_t)a.n * a.R * ((size_t)a.K + a.N) * sizeof(float);
  int splits = cus < most ? cus : most;
  if (one * splits > OUTER_BYTES) splits = one < OUTER_BYTES ? (int)(OUTER_BYTES / one) : 1;
  for (int i = 0; i < 2; ++i) {
    const int each = div_up(a.rows, splits), unit = each > 2 * STAGE ? 2 * STAGE : STAGE;
    p.per_split = div_up(each, unit) * unit;
    p.outer_turns = div_up(p.per_split, rows_per);
    if (p.outer_turns > all) p.outer_turns = all;
    if (i == 0 && p.outer_turns > 1) splits = div_up(splits, p.outer_turns);
  }
  p.splits = div_up(a.rows, p.per_split);
  // A run that ends inside a request can hold one adapter more. Where runs are one or two stages that is as much again for their blocks, and it gets blocks of
  // its own (999 rows of 3 requests, 2048 and 8192 columns, rank 24: 17.2 -> 13.9 us; all of 324 rows of 2, 35.5 -> 30.8, of 760 rows of 5, rank 72, 50.4 -> 52.5);
  // in longer ones it is a stage of many (all of 8190 rows of 6, 77 -> 81).
  if (p.per_split <= 2 * STAGE && p.per_split % rows_per != 0 && rows_per % p.per_split != 0) {
    p.outer_turns = div_up(p.per_split - 1, rows_per) + 1;
    if (p.outer_turns > all) p.outer_turns = all;
  }
  if (p.splits > 1) {
    p.da_bytes = bytes_of((size_t)p.splits * a.n * a.R * a.K * sizeof(float));
    p.db_bytes = bytes_of((size_t)p.splits * a.n * a.R * a.N * sizeof(float));
    p.there_bytes = bytes_of((size_t)p.splits * a.n * sizeof(int32_t));
  }
  p.total = p.there_bytes + p.h.part + p.g.part + p.h.rows + p.g.rows + p.g.rank + p.da_bytes + p.db_bytes;
  return p;
}

// f(r tiles of 16, mode and r tiles of the turned product, tokens of a tile in 16) as constants; fine: 32 r a block at most; PAIR: both products run
template <bool PAIR, class F>
void narrow_shape(int R, bool fine, int tm, F f) {
  using std::integral_constant;
  auto tokens = [&](auto rt, auto mode, auto rtg) {
    constexpr int most = decltype(rt)::value > 4 || (PAIR && decltype(rtg)::value > 4) ? 2 : 4;
    if (tm == 1) f(rt, mode, rtg, integral_constant<int, 1>());
    else if (tm == 2 || most == 2) f(rt, mode, rtg, integral_constant<int, 2>());
    else f(rt, mode, rtg, integral_constant<int, most>());
  };
  const integral_constant<int, ACROSS32> narrow;
  const integral_constant<int, ACROSS> wide;
  const integral_constant<int, 2> two;
  const integral_constant<int, 8> eight;
  if (R <= 16) tokens(integral_constant<int, 1>(), narrow, two);
  else if (R <= 32 || fine) tokens(two, narrow, two);
  else if (R <= 64) tokens(integral_constant<int, 4>(), wide, eight);
  else tokens(eight, wide, eight);
}

int narrow_blocks(const NarrowArgs& p, int tm) { return div_up(p.q.T, 16 * tm) * p.slices * p.turns; }

template <class A, bool TURNED>
void launch_wide_run(const WideArgs& p, hipStream_t s) {
  auto go = [&](auto steps, auto groups) {
    constexpr int STEPS = decltype(steps)::value, GROUPS = decltype(groups)::value;
    // The shortest runs that leave no more blocks than two a CU, or three without a base (8192 x 2560, rank 32: 235 blocks 20.8 us, 430 15.1, 640 12.8, 855
    // 14.2). That is what the card holds at once of bf16 up to rank 64 with a base and up to 32 without; by their registers it holds two of the other instances
    // without a base (fp16 over 64: one), and one with a base of fp16 over 32 and of all over 64, whose blocks then come in two turns or more.
    constexpr int HELD = (TURNED ? 3 : 2) * HDMOE_NUM_CU;
    const int chunks = div_up(p.C, WAVES * Wide<A, TURNED>::COLS), most = chunks < HELD ? HELD / chunks : 1;
    int run = div_up(p.q.T, (int64_t)16 * most) * 16;
    if (run > RUN) run = RUN;
    hipLaunchKernelGGL((wide_run_kernel<A, TURNED, STEPS, GROUPS>), dim3(chunks * div_up(p.q.T, run)), dim3(WAVES * 64), 0, s, p, div_up(p.R, 32 * STEPS), run);
  };
  using std::integral_constant;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  if (p.R <= 32) go(one, one);
  else if (p.R <= 64) go(two, one);
  else go(one, integral_constant<int, A::HALF ? 3 : 4>());
}

template <class A, bool TURNED>
void launch_wide(const WideArgs& p, hipStream_t s) {
  const dim3 grid(div_up(p.C, WIDE_WAVES * Wide<A, TURNED>::COLS) * div_up(p.q.T, 16) * p.turns);
  const size_t bytes = p.part != nullptr ? (size_t)2 * 16 * ((p.R + 31) / 32 * 32 + 8) * 2 : 0;
  hipLaunchKernelGGL((wide_kernel<A, TURNED>), grid, dim3(WIDE_WAVES * 64), bytes, s, p);
}

// Sizes alone: what the workspace depends on
int check_sizes(const hdmoe_adapter_args* a, const char* what) {
  if (a == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: args is NULL", what);
  if (a->dtype != HDMOE_T_BF16 && a->dtype != HDMOE_T_F16) return hdmoe_fail(HDMOE_E_SHAPE, "%s: dtype=%d", what, a->dtype);
  if (a->rows < 0 || a->K < 1 || a->N < 1 || a->n < 1 || a->n > HDMOE_ADAPTER_MAX || a->R < 1 || a->R > HDMOE_ADAPTER_MAX_RANK ||
      a->requests < 0 || (a->rows > 0 && (a->requests == 0 || a->rows % a->requests != 0)))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%d requests=%d K=%d N=%d n=%d (1 to %d) R=%d (1 to %d)", what, a->rows, a->requests, a->K, a->N,
                      a->n, HDMOE_ADAPTER_MAX, a->R, HDMOE_ADAPTER_MAX_RANK);
  if (a->K > (1 << 24) || a->N > (1 << 24) || a->rows > (1 << 30))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%d (at most 2^30) K=%d N=%d (at most 2^24)", what, a->rows, a->K, a->N);
  if (a->rows == 0) return HDMOE_OK;
  // A launch has fewer than 2^32 threads, along each of its dimensions: both narrow products of a pair, the planes' groups, and the products back where
  // tiles have a block for each adapter that they can hold.
  const int64_t rows_per = a->rows / a->requests, tiles = div_up(a->rows, 16), most = rows_per < 16 ? 16 : 1;
  const int64_t turns = most < a->n ? most : a->n, narrow = tiles * turns * 2 * NARROW_WAVES * 64 + 16 * NARROW_WAVES * 64 * HDMOE_NUM_CU;
  const int64_t wide = tiles * turns * div_up(a->K > a->N ? a->K : a->N, 128 * WIDE_WAVES) * WIDE_WAVES * 64, join = (int64_t)a->rows * div_up(a->R, 32) * 4 + 64;
  if (narrow >= LANES_MAX || join >= LANES_MAX || ((rows_per < 16 || a->rows < MANY_ROWS) && wide >= LANES_MAX))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%d requests=%d K=%d N=%d: more threads than a launch has", what, a->rows, a->requests, a->K, a->N);
  return HDMOE_OK;
}

int check_args(const hdmoe_adapter_args* a, const char* what) {
  if (int rc = check_sizes(a, what)) return rc;
  if (a->a == nullptr || a->b == nullptr || a->scale == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: a, b or scale is NULL", what);
  if (a->rows > 0 && (a->x == nullptr || a->index == nullptr)) return hdmoe_fail(HDMOE_E_NULL, "%s: x or index is NULL", what);
  return HDMOE_OK;
}

Requests requests_of(const hdmoe_adapter_args* a) { return {a->index, a->scale, a->rows, a->rows / a->requests, a->n}; }

template <class F>
void typed(int dtype, F f) {
  if (dtype == HDMOE_T_BF16) f(Bf16());
  else f(lowrank::F16());
}

const uint16_t* bits(const void* p) { return static_cast<const uint16_t*>(p); }

}  // namespace

extern "C" size_t hdmoe_adapters_workspace_bytes(const hdmoe_adapter_args* a, int backward) {
  if (check_sizes(a, "hdmoe_adapters_workspace_bytes") != HDMOE_OK || a->rows == 0) return 0;
  return plan_of(*a, backward != 0).total;
}

static int check_workspace(const hdmoe_adapter_args* a, const Plan& plan, const char* what) {
  if (plan.total == 0) return HDMOE_OK;
  if (a->workspace == nullptr || a->workspace_bytes < plan.total || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return hdmoe_fail(HDMOE_E_WORKSPACE, "%s: workspace of %zu bytes on 16 needed, got %zu", what, plan.total, a->workspace_bytes);
  return HDMOE_OK;
}

extern "C" int hdmoe_add_adapters(const hdmoe_adapter_args* a, hdmoe_stream_t stream) {
  if (int rc = check_args(a, "hdmoe_add_adapters")) return rc;
  if (a->rows == 0) return HDMOE_OK;
  if (a->base == nullptr || a->out == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_add_adapters: base or out is NULL");
  const Plan plan = plan_of(*a, false);
  if (int rc = check_workspace(a, plan, "hdmoe_add_adapters")) return rc;
  // `out` may be `base`: a value is read once, by the wave that writes it afterwards. All else is read by several blocks.
  const size_t value = sizeof(uint16_t), rows = a->rows, out_bytes = rows * a->N * value;
  auto meets = [&](const void* p, size_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), out = reinterpret_cast<uintptr_t>(a->out);
    return at < out + out_bytes && out < at + bytes;
  };
  if (meets(a->x, rows * a->K * value) || meets(a->a, (size_t)a->n * a->R * a->K * value) || meets(a->b, (size_t)a->n * a->R * a->N * value) ||
      meets(a->scale, a->n * sizeof(float)) || meets(a->index, a->requests * sizeof(int32_t)) || (a->base != a->out && meets(a->base, out_bytes)))
    return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_add_adapters: out overlaps an input (it may be base, as a whole)");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const Requests q = requests_of(a);
  float* part = plan.run ? nullptr : static_cast<float*>(a->workspace);
  const Planes planes = {plan.run ? static_cast<uint16_t*>(a->workspace) : nullptr, nullptr, plan.steps, plan.tiles};
  const NarrowArgs np = {q, bits(a->x), bits(a->a), part, planes, a->K, a->R, plan.h.slice, plan.h.slices, plan.turns};
  const WideArgs wp = {q, part, planes.rank, bits(a->b), bits(a->base), static_cast<uint16_t*>(a->out), a->N, a->R, plan.h.slices, plan.turns};
  typed(a->dtype, [&](auto t) {
    typedef decltype(t) A;
    if (plan.few) {
      const dim3 grid(div_up(a->N, WIDE_WAVES * Wide<A, false>::COLS) * div_up(a->rows, 16) * plan.turns);
      if (a->R <= 16) hipLaunchKernelGGL((few_kernel<A, 1>), grid, dim3(NARROW_WAVES * 64), 0, s, np, wp);
      else if (a->R <= 32) hipLaunchKernelGGL((few_kernel<A, 2>), grid, dim3(NARROW_WAVES * 64), 0, s, np, wp);
      else hipLaunchKernelGGL((few_kernel<A, 4>), grid, dim3(NARROW_WAVES * 64), 0, s, np, wp);
      return;
    }
    narrow_shape<false>(a->R, plan.fine, plan.tm, [&](auto rt, auto, auto, auto tm) {
      constexpr int RT = decltype(rt)::value, TM = decltype(tm)::value;
      hipLaunchKernelGGL((narrow_kernel<A, RT, TM>), dim3(narrow_blocks(np, TM), div_up(a->R, 16 * RT)), dim3(NARROW_WAVES * 64), 0, s, np);
    });
    if (plan.run) launch_wide_run<A, false>(wp, s);
    else launch_wide<A, false>(wp, s);
  });
  return hdmoe_check_launch("hdmoe_add_adapters");
}

extern "C" int hdmoe_add_adapters_backward(const hdmoe_adapter_args* a, hdmoe_stream_t stream) {
  if (int rc = check_args(a, "hdmoe_add_adapters_backward")) return rc;
  if (a->da == nullptr || a->db == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_add_adapters_backward: da or db is NULL");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  SumArgs sp = {};
  sp.out[0] = static_cast<uint16_t*>(a->da), sp.out[1] = static_cast<uint16_t*>(a->db);
  sp.n[0] = (size_t)a->n * a->R * a->K, sp.n[1] = (size_t)a->n * a->R * a->N;
  if (sp.n[0] + sp.n[1] >= (size_t)1 << 33) return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_add_adapters_backward: n=%d R=%d K=%d N=%d", a->n, a->R, a->K, a->N);
  if (a->rows == 0) {   // gradients of zero
    typed(a->dtype, [&](auto t) { launch_sum_parts<decltype(t)>(sp, s); });
    return hdmoe_check_launch("hdmoe_add_adapters_backward");
  }
  if (a->dy == nullptr || a->dx == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_add_adapters_backward: dy or dx is NULL");
  const Plan plan = plan_of(*a, true);
  if (int rc = check_workspace(a, plan, "hdmoe_add_adapters_backward")) return rc;
  char* ws = static_cast<char*>(a->workspace);
  auto take = [&](size_t n) {
    void* at = n > 0 ? ws : nullptr;
    ws += n;
    return at;
  };
  const Requests q = requests_of(a);
  JoinArgs jp = {};
  jp.q = q, jp.R = a->R, jp.slices[0] = plan.h.slices, jp.slices[1] = plan.g.slices;
  float* h = static_cast<float*>(take(plan.h.part));
  float* g = static_cast<float*>(take(plan.g.part));
  jp.part[0] = h, jp.part[1] = g;
  jp.to[0] = {nullptr, static_cast<uint16_t*>(take(plan.h.rows)), plan.steps, plan.tiles};
  uint16_t* grows = static_cast<uint16_t*>(take(plan.g.rows));
  jp.to[1] = {static_cast<uint16_t*>(take(plan.g.rank)), grows, plan.steps, plan.tiles};
  const NarrowArgs hp = {q, bits(a->x), bits(a->a), h, jp.to[0], a->K, a->R, plan.h.slice, plan.h.slices, plan.turns};
  const NarrowArgs gp = {q, bits(a->dy), bits(a->b), g, jp.to[1], a->N, a->R, plan.g.slice, plan.g.slices, plan.turns};
  const WideArgs wp = {q, nullptr, jp.to[1].rank, bits(a->a), nullptr, static_cast<uint16_t*>(a->dx), a->K, a->R, 1, plan.turns};
  OuterArgs op = {};
  op.q = q, op.R = a->R, op.splits = plan.splits, op.per_split = plan.per_split, op.tiles = plan.tiles, op.turns = plan.outer_turns;
  op.there = static_cast<int32_t*>(take(plan.there_bytes));
  float* da = static_cast<float*>(take(plan.da_bytes));
  float* db = static_cast<float*>(take(plan.db_bytes));
  op.side[0] = {bits(a->x), jp.to[1].rows, plan.splits == 1 ? a->da : da, a->K, 0, div_up(a->K, 512)};
  op.side[1] = {bits(a->dy), jp.to[0].rows, plan.splits == 1 ? a->db : db, a->N, 1, div_up(a->N, 512)};
  sp.part[0] = da, sp.part[1] = db, sp.splits = plan.splits;
  sp.there = op.there, sp.groups = a->n;
  const dim3 grid(op.side[0].blocks + op.side[1].blocks, plan.outer_turns * div_up(a->R, 16 * plan.rt), plan.splits);
  typed(a->dtype, [&](auto t) {
    typedef decltype(t) A;
    narrow_shape<true>(a->R, plan.fine, plan.tm, [&](auto rt, auto mode, auto rtg, auto tm) {
      constexpr int RT = decltype(rt)::value, MODE = decltype(mode)::value, RTG = decltype(rtg)::value, TM = decltype(tm)::value;
      const int nh = narrow_blocks(hp, TM), ng = narrow_blocks(gp, TM);
      hipLaunchKernelGGL((narrow_pair_kernel<A, MODE, RT, RTG, TM>), dim3(nh + ng, div_up(a->R, MODE == ACROSS32 ? 32 : 128)), dim3(NARROW_WAVES * 64), 0, s, hp, gp, ng);
    });
    if (h != nullptr || g != nullptr)
      hipLaunchKernelGGL(join_kernel, dim3(div_up((int64_t)a->rows * plan.steps * 4, 64), 2), dim3(64), 0, s, jp);
    if (plan.mixed) launch_wide<A, true>(wp, s);
    else launch_wide_run<A, true>(wp, s);
    if (plan.rt == 1) hipLaunchKernelGGL((outer_kernel<A, 1>), grid, dim3(512), 0, s, op);
    else hipLaunchKernelGGL((outer_kernel<A, 2>), grid, dim3(512), 0, s, op);
    if (plan.splits > 1) launch_sum_parts<A>(sp, s);
  });
  return hdmoe_check_launch("hdmoe_add_adapters_backward");
}
