// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out[t] = base[t] + s_a B_a (A_a x[t]),  a = index[t / rows_per] (outside 0 .. n - 1: none, out[t] = base[t])
//   h = A x, g = dy B      dx = s g A      dA_a = s sum_t g[t]^T x[t]      dB_a = s sum_t dy[t]^T h[t]
//
// Three products with a narrow side, in as many kernels: `narrow` (rows to rank), `wide` (rank to rows) and `outer` (sums over rows). The
// narrow results stay fp32 (lowrank.h says how they are multiplied). Rows of one tile may have different adapters: a tile is gone
// through once for every adapter in it, and values of rows that have another one are never multiplied, not even by zero.
#include <type_traits>

#include "lowrank.h"

using namespace lowrank;

namespace {

constexpr int WAVES = 4;
constexpr int K_STEP = 64;                 // along the contraction, of a wave: 128 bytes of each row
constexpr int STAGE = 128;                 // tokens whose narrow values `outer` holds in LDS

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

// First of the eight r that lane `col` of a transposed operand holds: where they would pass R, the last eight once more (the same values
// then come out in two places). Below 8: 0.
__device__ __forceinline__ int across_r(int r0, int col, int R) { return max(0, min(r0 + col * 8, R - 8)); }

struct NarrowArgs {
  Requests q;
  const uint16_t *x, *w;    // x [T, K]; w [n, R, K], or [n, K, R] (ACROSS)
  float* part;              // [slices, T, R]
  int K, R, slice, slices, turns;
};

// part[slice][t][r] = sum over the slice's k of x[t][k] w[a][r][k]. A tile is 16 TM tokens; the block's waves take steps of the slice in
// turn and join their sums in LDS. ACROSS: w runs along r: eight k of eight r at a time, transposed in registers, 128 r of them (those past R are
// not loaded) whatever R is.
template <class A, bool ACROSS, int RT, int TM>
__global__ __launch_bounds__(WAVES * 64) void narrow_kernel(NarrowArgs p) {
  static_assert(!ACROSS || RT == 8, "128 r");
  __shared__ f4 joined[2][RT * TM][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int tiles = (p.q.T + 16 * TM - 1) / (16 * TM);
  const int tile = blockIdx.x % tiles, slice = (blockIdx.x / tiles) % p.slices, z = blockIdx.x / tiles / p.slices;
  const int t0 = tile * 16 * TM, r0 = blockIdx.y * 16 * RT;
  const int lo = slice * p.slice, hi = min(p.K, lo + p.slice);
  const uint16_t* rows[TM];
#pragma unroll
  for (int m = 0; m < TM; ++m) rows[m] = p.x + (size_t)min(t0 + m * 16 + col, p.q.T - 1) * p.K;
  const int mine = lane < 16 * TM ? p.q.of(t0 + lane) : -1;
  each_adapter(mine, z, p.turns, [&](int a, uint64_t has) {
    f4 acc[RT][TM] = {};
    const uint16_t* w = p.w + (size_t)a * p.R * p.K;
    auto step = [&](int k0, auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
      // a lane's 16 values of a row: two instructions' worth
      const int k = k0 + quad * 16, have = WHOLE ? 16 : hi - k;
      u4 xv[TM][2];
#pragma unroll
      for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) xv[m][i] = WHOLE ? load8(rows[m] + k + 8 * i) : load8(rows[m] + k + 8 * i, have - 8 * i);
      if constexpr (!ACROSS) {
        u4 wv[RT][2];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint16_t* wr = w + (size_t)min(r0 + r * 16 + col, p.R - 1) * p.K + k;
#pragma unroll
          for (int i = 0; i < 2; ++i) wv[r][i] = WHOLE ? load8(wr + 8 * i) : load8(wr + 8 * i, have - 8 * i);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int m = 0; m < TM; ++m) acc[r][m] = A::mul(wv[r][i], xv[m][i], acc[r][m]);
      } else {
        const int r = across_r(r0, col, p.R);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          u4 wv[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {   // past the end x is 0: the last row again
            const uint16_t* from = w + (size_t)(WHOLE ? k + 8 * i + j : min(k + 8 * i + j, p.K - 1)) * p.R + r;
            wv[j] = p.R >= 8 ? load8(from) : load8(from, p.R);
          }
          transpose8(wv);
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int m = 0; m < TM; ++m) acc[j][m] = A::mul(wv[j], xv[m][i], acc[j][m]);
        }
      }
    };
    int k0 = lo + wave * K_STEP;
    for (; k0 + K_STEP <= hi; k0 += WAVES * K_STEP) step(k0, std::true_type());
    if (k0 < hi) step(k0, std::false_type());
    // waves 2 and 3 into 0 and 1, 1 into 0
#pragma unroll
    for (int half = 2; half > 0; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half)
#pragma unroll
        for (int i = 0; i < RT * TM; ++i) joined[wave - half][i][lane] = acc[i / TM][i % TM];
      __syncthreads();
      if (wave < half)
#pragma unroll
        for (int i = 0; i < RT * TM; ++i) acc[i / TM][i % TM] += joined[wave][i][lane];
    }
    if (wave != 0) return;
#pragma unroll
    for (int m = 0; m < TM; ++m) {
      if (!((has >> (m * 16 + col)) & 1)) continue;
      float* to = p.part + ((size_t)slice * p.q.T + t0 + m * 16 + col) * p.R;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = ACROSS ? across_r(r0, quad * 4 + e, p.R) + i : r0 + i * 16 + quad * 4 + e;
          if (r < p.R) to[r] = acc[i][m][e];
        }
    }
  });
}

struct WideArgs {
  Requests q;
  const float* part;                  // [slices, T, R]
  const uint16_t *w, *base;           // w [n, C, R], or [n, R, C] (ACROSS); base [T, C] or NULL
  uint16_t* out;                      // [T, C]
  int C, R, slices, turns;
};

// out[t][c] = base[t][c] + s sum_r h[t][r] w[a][c][r]. A tile is 16 TM tokens; a wave has 64 columns (ACROSS: 128), which a lane holds 16 (32) next to each
// other of, so that it loads and stores whole 16-byte pieces and a token's 128 bytes are one wave's.
// Bound by base and out: R of 64 takes 16 matrix instructions (256 cycles of one of four units) for 4 KB of them.
template <class A, bool ACROSS, int TM>
__global__ __launch_bounds__(WAVES * 64) void wide_kernel(WideArgs p) {
  constexpr int NT = ACROSS ? 8 : 4;           // instructions side by side
  extern __shared__ __attribute__((aligned(16))) uint16_t lds[];   // [2][16 TM][stride]: hi, lo of s h
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int steps = (p.R + 31) / 32, stride = steps * 32 + 8;
  const int tiles = (p.q.T + 16 * TM - 1) / (16 * TM), chunks = (p.C + WAVES * NT * 16 - 1) / (WAVES * NT * 16);
  const int chunk = blockIdx.x % chunks, tile = (blockIdx.x / chunks) % tiles, z = blockIdx.x / chunks / tiles;
  const int t0 = tile * 16 * TM, c0 = (chunk * WAVES + wave) * NT * 16;
  const int mine = lane < 16 * TM ? p.q.of(t0 + lane) : -1;
  // the narrow values of the tile, eight a thread at a time
  for (int u = threadIdx.x; u < 16 * TM * steps * 4; u += WAVES * 64) {
    const int row = u / (steps * 4), r = (u - row * (steps * 4)) * 8, t = t0 + row;
    const int a = p.q.of(t);
    float v[8] = {};
    if (a >= 0) {
      for (int s = 0; s < p.slices; ++s) {
        const float* from = p.part + ((size_t)s * p.q.T + t) * p.R + r;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (r + j < p.R) v[j] += from[j];
      }
      const float f = p.q.scale[a];
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
    *reinterpret_cast<u4*>(lds + (size_t)(16 * TM + row) * stride + r) = vl;
  }
  __syncthreads();
  if (c0 >= p.C) return;
  // the lane's columns: 4 NT next to each other
  const int c = c0 + quad * 4 * NT, have = p.C - c;
  const bool whole = c0 + 16 * NT <= p.C;
  auto put = [&](int m, f4 (&acc)[NT], u4 (&b)[NT / 2]) {
    uint16_t* to = p.out + (size_t)(t0 + m * 16 + col) * p.C + c;
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) {
      u4 o;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // ACROSS: instruction j, element e are column 8 e + j, else 4 j + e
        const int u = 8 * i + 2 * w;
        const float v0 = ACROSS ? acc[u % 8][u / 8] : acc[u / 4][u % 4], v1 = ACROSS ? acc[u % 8 + 1][u / 8] : acc[u / 4][u % 4 + 1];
        o[w] = p.base != nullptr ? A::pack(v0 + A::lo(b[i][w]), v1 + A::hi(b[i][w])) : A::pack(v0, v1);
      }
      store8(to + 8 * i, o, have - 8 * i);
    }
  };
  auto bases = [&](int m, u4 (&b)[NT / 2], bool want) {
    const uint16_t* from = p.base + (size_t)(t0 + m * 16 + col) * p.C + c;
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) b[i] = want && p.base != nullptr ? load8(from + 8 * i, have - 8 * i) : u4{0, 0, 0, 0};
  };
  if (z == 0) {   // rows without an adapter
    const uint64_t none = __ballot(lane < 16 * TM && t0 + lane < p.q.T && mine < 0);
    if (none != 0 && (const void*)p.out != (const void*)p.base)
#pragma unroll
      for (int m = 0; m < TM; ++m)
        if ((none >> (m * 16 + col)) & 1) {
          f4 zero[NT] = {};
          u4 b[NT / 2];
          const uint16_t* from = p.base + (size_t)(t0 + m * 16 + col) * p.C + c;
          if (p.base == nullptr) {
            put(m, zero, b);
          } else {   // as it is, bit for bit
#pragma unroll
            for (int i = 0; i < NT / 2; ++i)
              store8(p.out + (size_t)(t0 + m * 16 + col) * p.C + c + 8 * i, load8(from + 8 * i, have - 8 * i), have - 8 * i);
          }
        }
  }
  each_adapter(mine, z, p.turns, [&](int a, uint64_t has) {
    u4 b[TM][NT / 2];
#pragma unroll
    for (int m = 0; m < TM; ++m) bases(m, b[m], (has >> (m * 16 + col)) & 1);
    f4 acc[TM][NT] = {};
    const uint16_t* w = p.w + (size_t)a * p.R * p.C;
    for (int s = 0; s < steps; ++s) {
      const int r = s * 32 + quad * 8;
      u4 wh[NT], wl[NT];
      // r past R meets h of 0: the row's last values again, so that nothing but the lane's own column enters
      if constexpr (ACROSS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint16_t* from = w + (size_t)min(r + j, p.R - 1) * p.C + c0 + col * 8;
          wh[j] = whole ? load8(from) : load8(from, p.C - c0 - col * 8);
        }
        transpose8(wh);
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const uint16_t* from = w + (size_t)min(c0 + (col >> 2) * 16 + j * 4 + (col & 3), p.C - 1) * p.R;
          wh[j] = p.R % 8 == 0 ? load8(from + min(r, p.R - 8)) : load8(from + r, p.R - r);
        }
      }
      if constexpr (A::HALF)
#pragma unroll
        for (int j = 0; j < NT; ++j) to_bf16<A>(wh[j], wh[j], wl[j]);
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        const u4 qh = *reinterpret_cast<const u4*>(lds + (size_t)(m * 16 + col) * stride + r);
        const u4 ql = *reinterpret_cast<const u4*>(lds + (size_t)((TM + m) * 16 + col) * stride + r);
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[m][j] = mul_split<A>(wh[j], wl[j], qh, ql, acc[m][j]);
      }
    }
#pragma unroll
    for (int m = 0; m < TM; ++m)
      if ((has >> (m * 16 + col)) & 1) put(m, acc[m], b[m]);
  });
}

struct OuterSide {
  const uint16_t* v;        // [T, C]
  const float* part;        // [slices, T, R]
  void* out;                // fp32 parts [splits, n, R, C] (flip: [splits, n, C, R]), or the result itself
  int C, slices, flip, blocks;   // blocks of 512 columns
};

struct OuterArgs {
  Requests q;
  OuterSide side[2];
  int R, splits, per_split, direct;   // per_split: tokens, a multiple of STAGE
};

// out[a][r][c] = s sum over the rows t of adapter a of q[t][r] v[t][c], 16 RT of the r. A wave has 128 columns; eight rows of eight columns
// a lane are loaded as they lie and transposed in registers.
template <class A, int RT>
__global__ __launch_bounds__(WAVES * 64, 2) void outer_kernel(OuterArgs p) {
  __shared__ uint16_t lds[2][16 * RT][STAGE + 8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const bool second = (int)blockIdx.x >= p.side[0].blocks;
  const OuterSide side = second ? p.side[1] : p.side[0];
  const int block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
  const int a = blockIdx.y % p.q.n, r0 = blockIdx.y / p.q.n * 16 * RT, split = blockIdx.z;
  const int c0 = (block * WAVES + wave) * 128, c = c0 + col * 8, have = side.C - c;
  const float f = p.q.scale[a];
  const bool whole = c0 + 128 <= side.C;
  f4 acc[RT][8] = {};
  const int end = (int)min((int64_t)p.q.T, (int64_t)(split + 1) * p.per_split);
  for (int t0 = split * p.per_split; t0 < end; t0 += STAGE) {
    const uint64_t first = __ballot(t0 + lane < end && p.q.of(t0 + lane) == a), next = __ballot(t0 + 64 + lane < end && p.q.of(t0 + 64 + lane) == a);
    if ((first | next) == 0) continue;
    __syncthreads();
    for (int u = threadIdx.x; u < STAGE * 4 * RT; u += WAVES * 64) {   // two rows of one r .. + 3 a thread, transposed
      const int row = u % (STAGE / 2) * 2, r = u / (STAGE / 2) * 2;
      float v[2][2] = {};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!(((row + i < 64 ? first : next) >> ((row + i) & 63)) & 1)) continue;
        for (int s = 0; s < side.slices; ++s) {
          const float* from = side.part + ((size_t)s * p.q.T + t0 + row + i) * p.R + r0 + r;
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (r0 + r + j < p.R) v[i][j] += from[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t h, l;
        lowrank::split(v[0][j] * f, v[1][j] * f, h, l);
        *reinterpret_cast<uint32_t*>(&lds[0][r + j][row]) = h;
        *reinterpret_cast<uint32_t*>(&lds[1][r + j][row]) = l;
      }
    }
    __syncthreads();
    if (c0 >= side.C) continue;
#pragma unroll 2
    for (int st = 0; st < STAGE / 32; ++st) {
      const uint32_t has = (uint32_t)((st < 2 ? first : next) >> (32 * (st & 1)));
      if (has == 0) continue;
      const uint32_t eight = (has >> (quad * 8)) & 0xff;
      u4 v[8];
      const uint16_t* from = side.v + (size_t)(t0 + st * 32 + quad * 8) * side.C + c;
      if (has == 0xffffffffu && whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = load8(from + (size_t)j * side.C);
      } else {   // rows of another adapter are 0, not multiplied by it
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v[j] = u4{0, 0, 0, 0};
          if ((eight >> j) & 1) v[j] = load8(from + (size_t)j * side.C, have);
        }
      }
      transpose8(v);
      u4 qh[RT], ql[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        qh[r] = *reinterpret_cast<const u4*>(&lds[0][r * 16 + col][st * 32 + quad * 8]);
        ql[r] = *reinterpret_cast<const u4*>(&lds[1][r * 16 + col][st * 32 + quad * 8]);
      }
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
    }
  }
  if (c0 >= side.C) return;
  const size_t at = ((size_t)split * p.q.n + a) * p.R * side.C;
  auto put = [&](size_t i, float v) {
    if (p.direct) static_cast<uint16_t*>(side.out)[at + i] = (uint16_t)A::pack(v, 0.0f);
    else static_cast<float*>(side.out)[at + i] = v;
  };
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int row = r0 + r * 16 + quad * 4 + e;
      if (row >= p.R) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < have) put(side.flip ? (size_t)(c + j) * p.R + row : (size_t)row * side.C + c + j, acc[r][j][e]);
    }
}

// ---- sizes ---------------------------------------------------------------------------------------------------------

struct Plan {
  int tm_narrow, slices_x, slice_x, slices_y, slice_y, turns, tm_wide, turns_wide, splits, per_split, rt;
  size_t h_bytes, g_bytes, da_bytes, db_bytes;
};

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Tokens a tile: 16 where rows of a tile have different adapters or where there are few; the contraction is cut until the card has about two
// blocks a CU, in slices of at least one step of each wave.
void narrow_plan(int tiles, int turns, int K, int rblocks, int& slices, int& slice) {
  const int most = div_up(K, WAVES * K_STEP);
  int want = div_up(2 * HDMOE_NUM_CU, (int64_t)tiles * turns * rblocks);
  if (want > most) want = most;
  if (want > 16) want = 16;
  slice = div_up(most, want) * WAVES * K_STEP;
  slices = div_up(K, slice);
}

Plan plan_of(const hdmoe_adapter_args& a, bool backward) {
  Plan p = {};
  const int rows_per = a.rows / a.requests;
  const bool mixed = rows_per < 64;
  p.tm_narrow = mixed || a.rows <= 512 ? 1 : a.R > 64 ? 2 : 4;
  const int tile = 16 * p.tm_narrow;
  const int distinct = rows_per >= tile ? 1 : div_up(tile, rows_per);
  p.turns = distinct < a.n ? distinct : a.n;
  if (p.turns > tile) p.turns = tile;
  const int tiles = div_up(a.rows, tile), rblocks = a.R > 128 ? 2 : 1;
  narrow_plan(tiles, p.turns, a.K, rblocks, p.slices_x, p.slice_x);
  narrow_plan(tiles, p.turns, a.N, rblocks, p.slices_y, p.slice_y);
  p.tm_wide = mixed || a.rows <= 256 ? 1 : a.R > 128 ? 2 : 4;
  p.turns_wide = p.tm_wide == 1 ? p.turns : 1;
  p.h_bytes = hdmoe_align_up((size_t)p.slices_x * a.rows * a.R * sizeof(float), 256);
  if (!backward) return p;
  p.g_bytes = hdmoe_align_up((size_t)p.slices_y * a.rows * a.R * sizeof(float), 256);
  p.rt = a.R <= 16 ? 1 : a.R <= 32 ? 2 : 4;
  const int blocks = (div_up(a.K, WAVES * 128) + div_up(a.N, WAVES * 128)) * a.n * div_up(a.R, 16 * p.rt);
  int splits = div_up(2 * HDMOE_NUM_CU, blocks);
  const int most = div_up(a.rows, 2 * STAGE);
  if (splits > most) splits = most;
  if (splits > 64) splits = 64;
  p.per_split = div_up(div_up(a.rows, splits), STAGE) * STAGE;
  p.splits = div_up(a.rows, p.per_split);
  if (p.splits > 1) {
    p.da_bytes = hdmoe_align_up((size_t)p.splits * a.n * a.R * a.K * sizeof(float), 256);
    p.db_bytes = hdmoe_align_up((size_t)p.splits * a.n * a.R * a.N * sizeof(float), 256);
  }
  return p;
}

template <class A, bool ACROSS>
void launch_narrow(const NarrowArgs& p, int tm, hipStream_t s) {
  auto go = [&](auto rt, auto m) {
    constexpr int RT = decltype(rt)::value, TM = decltype(m)::value;
    const dim3 grid(div_up(p.q.T, 16 * TM) * p.slices * p.turns, div_up(p.R, 16 * RT));
    hipLaunchKernelGGL((narrow_kernel<A, ACROSS, RT, TM>), grid, dim3(WAVES * 64), 0, s, p);
  };
  using std::integral_constant;
  auto rt = [&](auto r) {
    if (tm == 1) go(r, integral_constant<int, 1>());
    else if constexpr (decltype(r)::value == 8) go(r, integral_constant<int, 2>());
    else go(r, integral_constant<int, 4>());
  };
  if constexpr (ACROSS) {
    rt(integral_constant<int, 8>());
  } else {
    if (p.R <= 16) rt(integral_constant<int, 1>());
    else if (p.R <= 32) rt(integral_constant<int, 2>());
    else if (p.R <= 64) rt(integral_constant<int, 4>());
    else rt(integral_constant<int, 8>());
  }
}

template <class A, bool ACROSS>
void launch_wide(const WideArgs& p, int tm, hipStream_t s) {
  auto go = [&](auto m) {
    constexpr int TM = decltype(m)::value;
    const int chunks = div_up(p.C, WAVES * (ACROSS ? 128 : 64)), tiles = div_up(p.q.T, 16 * TM);
    const size_t bytes = (size_t)2 * 16 * TM * ((p.R + 31) / 32 * 32 + 8) * 2;
    hipLaunchKernelGGL((wide_kernel<A, ACROSS, TM>), dim3((unsigned)(chunks * tiles * p.turns)), dim3(WAVES * 64), bytes, s, p);
  };
  using std::integral_constant;
  if (tm == 1) go(integral_constant<int, 1>());
  else if constexpr (ACROSS) go(integral_constant<int, 2>());   // 128 columns: half the rows in as many registers
  else if (tm == 2) go(integral_constant<int, 2>());
  else go(integral_constant<int, 4>());
}

int check_args(const hdmoe_adapter_args* a, const char* what, bool backward) {
  if (a == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: args is NULL", what);
  if (a->dtype != HDMOE_T_BF16 && a->dtype != HDMOE_T_F16) return hdmoe_fail(HDMOE_E_SHAPE, "%s: dtype=%d", what, a->dtype);
  if (a->rows < 0 || a->K < 1 || a->N < 1 || a->n < 1 || a->n > HDMOE_ADAPTER_MAX || a->R < 1 || a->R > HDMOE_ADAPTER_MAX_RANK ||
      a->requests < 0 || (a->rows > 0 && (a->requests == 0 || a->rows % a->requests != 0)))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%d requests=%d K=%d N=%d n=%d (1 to %d) R=%d (1 to %d)", what, a->rows, a->requests, a->K, a->N,
                      a->n, HDMOE_ADAPTER_MAX, a->R, HDMOE_ADAPTER_MAX_RANK);
  const int64_t blocks = (int64_t)div_up(a->rows, 16) * 16 * (div_up(a->N, 64) + div_up(a->K, 64));
  if (blocks >= (int64_t)1 << 31) return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%d K=%d N=%d: too many tiles", what, a->rows, a->K, a->N);
  if (a->K > (1 << 24) || a->N > (1 << 24) || a->rows > (1 << 30))
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: rows=%d (at most 2^30) K=%d N=%d (at most 2^24)", what, a->rows, a->K, a->N);
  if (a->a == nullptr || a->b == nullptr || a->scale == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: a, b or scale is NULL", what);
  if (a->rows == 0) return HDMOE_OK;
  if (a->x == nullptr || a->index == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: x or index is NULL", what);
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
  if (check_args(a, "hdmoe_adapters_workspace_bytes", backward != 0) != HDMOE_OK || a->rows == 0) return 0;
  const Plan p = plan_of(*a, backward != 0);
  return p.h_bytes + p.g_bytes + p.da_bytes + p.db_bytes;
}

extern "C" int hdmoe_add_adapters(const hdmoe_adapter_args* a, hdmoe_stream_t stream) {
  if (int rc = check_args(a, "hdmoe_add_adapters", false)) return rc;
  if (a->rows == 0) return HDMOE_OK;
  if (a->base == nullptr || a->out == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_add_adapters: base or out is NULL");
  const Plan plan = plan_of(*a, false);
  if (a->workspace == nullptr || a->workspace_bytes < plan.h_bytes || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return hdmoe_fail(HDMOE_E_WORKSPACE, "hdmoe_add_adapters: workspace of %zu bytes on 16 needed, got %zu", plan.h_bytes, a->workspace_bytes);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  float* h = static_cast<float*>(a->workspace);
  const NarrowArgs np = {requests_of(a), bits(a->x), bits(a->a), h, a->K, a->R, plan.slice_x, plan.slices_x, plan.turns};
  const WideArgs wp = {requests_of(a), h, bits(a->b), bits(a->base), static_cast<uint16_t*>(a->out), a->N, a->R, plan.slices_x, plan.turns_wide};
  typed(a->dtype, [&](auto t) {
    typedef decltype(t) A;
    launch_narrow<A, false>(np, plan.tm_narrow, s);
    launch_wide<A, false>(wp, plan.tm_wide, s);
  });
  return hdmoe_check_launch("hdmoe_add_adapters");
}

extern "C" int hdmoe_add_adapters_backward(const hdmoe_adapter_args* a, hdmoe_stream_t stream) {
  if (int rc = check_args(a, "hdmoe_add_adapters_backward", true)) return rc;
  if (a->da == nullptr || a->db == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_add_adapters_backward: da or db is NULL");
  const hipStream_t s = static_cast<hipStream_t>(stream);
  SumArgs sp = {};
  sp.out[0] = static_cast<uint16_t*>(a->da), sp.out[1] = static_cast<uint16_t*>(a->db);
  sp.n[0] = (size_t)a->n * a->R * a->K, sp.n[1] = (size_t)a->n * a->R * a->N;
  if ((sp.n[0] + sp.n[1]) / 256 >= (1u << 31)) return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_add_adapters_backward: n=%d R=%d K=%d N=%d", a->n, a->R, a->K, a->N);
  auto sum = [&] {
    typed(a->dtype, [&](auto t) {
      hipLaunchKernelGGL(sum_parts_kernel<decltype(t)>, dim3((unsigned)((sp.n[0] + sp.n[1] + 255) / 256)), dim3(256), 0, s, sp);
    });
  };
  if (a->rows == 0) {   // gradients of zero
    sum();
    return hdmoe_check_launch("hdmoe_add_adapters_backward");
  }
  if (a->dy == nullptr || a->dx == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_add_adapters_backward: dy or dx is NULL");
  const Plan plan = plan_of(*a, true);
  const size_t need = plan.h_bytes + plan.g_bytes + plan.da_bytes + plan.db_bytes;
  if (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
    return hdmoe_fail(HDMOE_E_WORKSPACE, "hdmoe_add_adapters_backward: workspace of %zu bytes on 16 needed, got %zu", need, a->workspace_bytes);
  char* ws = static_cast<char*>(a->workspace);
  float *h = reinterpret_cast<float*>(ws), *g = reinterpret_cast<float*>(ws + plan.h_bytes);
  float *da = reinterpret_cast<float*>(ws + plan.h_bytes + plan.g_bytes), *db = reinterpret_cast<float*>(ws + plan.h_bytes + plan.g_bytes + plan.da_bytes);
  const Requests q = requests_of(a);
  const NarrowArgs hp = {q, bits(a->x), bits(a->a), h, a->K, a->R, plan.slice_x, plan.slices_x, plan.turns};
  const NarrowArgs gp = {q, bits(a->dy), bits(a->b), g, a->N, a->R, plan.slice_y, plan.slices_y, plan.turns};
  const WideArgs wp = {q, g, bits(a->a), nullptr, static_cast<uint16_t*>(a->dx), a->K, a->R, plan.slices_y, plan.turns_wide};
  OuterArgs op = {};
  op.q = q, op.R = a->R, op.splits = plan.splits, op.per_split = plan.per_split, op.direct = plan.splits == 1;
  op.side[0] = {bits(a->x), g, op.direct ? a->da : da, a->K, plan.slices_y, 0, div_up(a->K, WAVES * 128)};
  op.side[1] = {bits(a->dy), h, op.direct ? a->db : db, a->N, plan.slices_x, 1, div_up(a->N, WAVES * 128)};
  sp.part[0] = da, sp.part[1] = db, sp.splits = plan.splits;
  const dim3 grid(op.side[0].blocks + op.side[1].blocks, a->n * div_up(a->R, 16 * plan.rt), plan.splits);
  typed(a->dtype, [&](auto t) {
    typedef decltype(t) A;
    launch_narrow<A, false>(hp, plan.tm_narrow, s);
    launch_narrow<A, true>(gp, plan.tm_narrow, s);
    launch_wide<A, true>(wp, plan.tm_wide, s);
    if (plan.rt == 1) hipLaunchKernelGGL((outer_kernel<A, 1>), grid, dim3(WAVES * 64), 0, s, op);
    else if (plan.rt == 2) hipLaunchKernelGGL((outer_kernel<A, 2>), grid, dim3(WAVES * 64), 0, s, op);
    else hipLaunchKernelGGL((outer_kernel<A, 4>), grid, dim3(WAVES * 64), 0, s, op);
  });
  if (plan.splits > 1) sum();
  return hdmoe_check_launch("hdmoe_add_adapters_backward");
}
