// The router's balance loss, its per-expert counts, and the gradients of the loss and of the chosen scores.
//
//   p[t] = softmax(W x[t])           c[s][e] = choices of expert e among the n_s tokens of sequence s that the mask leaves
//   loss = alpha / held sum_s sum_e (E c[s][e] / (k n_s)) (1 / n_s) sum_t p[t][e]        held: sequences with tokens
//   dp[t][e] = dloss alpha E c[s][e] / (held k n_s^2) + sum of dweight[t][j] over the j with idx[t][j] = e
//   dz = p (dp - sum_e p dp)         dx = dz W        dW = sum_t dz[t]^T x[t]
//
// Bound by x: forward reads it once, backward reads it and writes dx in one kernel. The logits are fp32 (the rounding of gate_top2's to the activations'
// type counts as none in the gradient). Tokens that the mask takes out are neither counted nor multiplied, whatever they hold.
#include <type_traits>

#include "lowrank.h"

using namespace lowrank;

namespace {

constexpr int WAVES = 4;         // of the backward kernel
constexpr int SCORE_WAVES = 8;
constexpr int STAGE = 64;       // tokens whose dz a block of the backward kernel holds
constexpr int LANES_E = 16;     // experts, filled up

struct TileSums {               // of one tile of tokens
  float p[LANES_E];
  int32_t c[LANES_E];
  int32_t n, pad[3];
};

struct BalanceArgs {
  const uint16_t *x, *w;
  const int32_t* idx;
  const uint8_t* mask;
  float* scores;
  TileSums* tiles;
  int T, length, D, E, k, tiles_per_seq;
};

// Scores of 16 TM tokens of one sequence and their sums. The block's waves take steps along D in turn; subtile m of the sums is wave m's.
template <class A, int TM>
__global__ __launch_bounds__(SCORE_WAVES * 64) void gate_balance_kernel(BalanceArgs p) {
  __shared__ f4 joined[SCORE_WAVES][TM][64];
  __shared__ TileSums part[TM];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int seq = blockIdx.x / p.tiles_per_seq, l0 = (blockIdx.x - seq * p.tiles_per_seq) * 16 * TM;
  const int t0 = seq * p.length + l0;
  f4 acc[TM] = {};
  const int lane_row = col >> 2, lane_k = (quad * 4 + (col & 3)) * 8;      // of a load
  auto step = [&](int k0, auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
    const int k = k0 + lane_k;
    const bool on = WHOLE || k < p.D;             // D is a multiple of 8
    u4 wv[4], xv[TM][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wv[i] = u4{0, 0, 0, 0};
      if (on) wv[i] = load8(p.w + (size_t)min(i * 4 + lane_row, p.E - 1) * p.D + k);
#pragma unroll
      for (int m = 0; m < TM; ++m) {
        xv[m][i] = u4{0, 0, 0, 0};
        if (on) xv[m][i] = load8(p.x + (size_t)(seq * p.length + min(l0 + m * 16 + i * 4 + lane_row, p.length - 1)) * p.D + k);
      }
    }
    quad_transpose(wv);
#pragma unroll
    for (int m = 0; m < TM; ++m) quad_transpose(xv[m]);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int m = 0; m < TM; ++m) acc[m] = A::mul(wv[n], xv[m][n], acc[m]);
  };
  int k0 = wave * K_BLOCK;
  for (; k0 + K_BLOCK <= p.D; k0 += SCORE_WAVES * K_BLOCK) step(k0, std::true_type());
  if (k0 < p.D) step(k0, std::false_type());
#pragma unroll
  for (int m = 0; m < TM; ++m) joined[wave][m][lane] = acc[m];
  __syncthreads();
  if (wave < TM) {
    f4 z = {};
#pragma unroll
    for (int w = 0; w < SCORE_WAVES; ++w) z += joined[w][wave][lane];
    // token row_of(col), experts row_of(4 quad + i) = 4 i + quad: a token has its 16 logits in four lanes, 16 apart
    const int t = t0 + wave * 16 + row_of(col);
    const bool in = l0 + wave * 16 + row_of(col) < p.length;
    float top = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i * 4 + quad < p.E) top = fmaxf(top, z[i]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    float sum = 0.0f, s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = i * 4 + quad < p.E ? expf(z[i] - top) : 0.0f;
      sum += s[i];
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    const bool counts = in && (p.mask == nullptr || p.mask[t] != 0);
    int32_t c[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] /= sum;
      const int e = i * 4 + quad;
      if (in && e < p.E) p.scores[(size_t)t * p.E + e] = s[i];
      if (!counts) s[i] = 0.0f;
    }
    if (counts)
      for (int j = 0; j < p.k; ++j) {
        const int e = p.idx[(size_t)t * p.k + j];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += e == i * 4 + quad;
      }
    int n = counts;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      n += __shfl_xor(n, off, 64);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] += __shfl_xor(s[i], off, 64);
        c[i] += __shfl_xor(c[i], off, 64);
      }
    }
    if (col == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave].p[i * 4 + quad] = s[i], part[wave].c[i * 4 + quad] = c[i];
      if (quad == 0) part[wave].n = n;
    }
  }
  __syncthreads();
  if (threadIdx.x < LANES_E) {
    TileSums* to = p.tiles + blockIdx.x;
    float s = 0.0f;
    int32_t c = 0, n = 0;
#pragma unroll
    for (int m = 0; m < TM; ++m) s += part[m].p[threadIdx.x], c += part[m].c[threadIdx.x], n += part[m].n;
    to->p[threadIdx.x] = s;
    to->c[threadIdx.x] = c;
    if (threadIdx.x == 0) to->n = n;
  }
}

// The loss and the counts from the tiles' sums: 64 groups of 16 lanes, as many of them a sequence as there are sequences few, four in a wave.
__global__ __launch_bounds__(1024) void balance_finish_kernel(const TileSums* tiles, int seqs, int tiles_per_seq, int E, int k, float alpha,
                                                              float* loss, int32_t* counts) {
  __shared__ float sp[16][LANES_E], total[64];
  __shared__ int32_t sc[16][LANES_E], sn[16], held[64];
  const int e = threadIdx.x & 15, group = threadIdx.x >> 4, wave = threadIdx.x >> 6;
  int share = 64;   // groups of a sequence
  while (share > 1 && share * seqs > 64) share >>= 1;
  const int member = group & (share - 1), teams = 64 / share;
  float mine = 0.0f;
  int32_t mine_held = 0;
  for (int s0 = 0; s0 < seqs; s0 += teams) {
    const int s = s0 + group / share;
    float p = 0.0f;
    int32_t c = 0, n = 0;
    if (s < seqs) {
      const TileSums* from = tiles + (size_t)s * tiles_per_seq;
#pragma unroll 8
      for (int i = member; i < tiles_per_seq; i += share) p += from[i].p[e], c += from[i].c[e], n += from[i].n;
    }
    for (int off = 16; off < 64 && off < 16 * share; off <<= 1) {   // within the wave
      p += __shfl_xor(p, off, 64);
      c += __shfl_xor(c, off, 64);
      n += __shfl_xor(n, off, 64);
    }
    if (share > 4) {                                                // over the waves
      __syncthreads();
      if ((group & 3) == 0) {
        sp[wave][e] = p;
        sc[wave][e] = c;
        if (e == 0) sn[wave] = n;
      }
      __syncthreads();
      if (member == 0)
#pragma unroll 4
        for (int i = 1; i < share / 4; ++i) p += sp[wave + i][e], c += sc[wave + i][e], n += sn[wave + i];
    }
    if (member == 0 && s < seqs) {
      if (e < E) counts[(size_t)s * E + e] = c;
      if (n > 0) {
        const float f = 1.0f / (float)n;
        float v = e < E ? ((float)c * (f * ((float)E / (float)k))) * (p * f) : 0.0f;
#pragma unroll
        for (int off = 1; off < 16; off <<= 1) v += __shfl_xor(v, off, 16);
        mine += v;
        ++mine_held;
      }
    }
  }
  if (e == 0) total[group] = mine, held[group] = mine_held;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  float v = total[threadIdx.x];
  int32_t h = held[threadIdx.x];
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off, 64), h += __shfl_xor(h, off, 64);
  if (threadIdx.x == 0) *loss = h > 0 ? alpha * (v / (float)h) : 0.0f;
}

// Tokens that the mask leaves of each sequence.
__global__ __launch_bounds__(256) void mask_counts_kernel(const uint8_t* mask, int length, int32_t* n) {
  __shared__ int32_t part[4];
  const uint8_t* m = mask + (size_t)blockIdx.x * length;
  int c = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < length; i += 256) c += m[i] != 0;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) c += __shfl_xor(c, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = c;
  __syncthreads();
  if (threadIdx.x == 0) n[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

struct BalanceGrad {
  const uint16_t *x, *w;
  const int32_t *idx, *counts;
  const uint8_t* mask;
  const float *scores, *dloss;
  const uint16_t* dweight;        // NULL: none
  const int32_t* n;               // tokens of each sequence; NULL: length
  uint16_t* dx;
  void* dw;                       // fp32 parts [splits, E, D], or the gradient itself
  int T, length, seqs, D, E, k, per_split, direct;
  float alpha;
};

// dx and dW. A wave has 128 columns: W's of them stay in registers, transposed; x goes through registers once, eight rows of eight columns a lane,
// transposed for the sum over tokens. dz of 64 tokens lies in LDS twice, along the experts (with its hi and lo in one instruction's 32) and
// along the tokens. Bound by x and dx.
template <class A>
__global__ __launch_bounds__(WAVES * 64, 2) void gate_balance_backward_kernel(BalanceGrad p) {
  __shared__ __attribute__((aligned(16))) uint16_t along_e[STAGE][32 + 8];            // hi 0-7, lo 0-7, hi 8-15, lo 8-15
  __shared__ __attribute__((aligned(16))) uint16_t along_t[2][LANES_E][STAGE + 8];    // hi, lo
  __shared__ int live[2];                                                             // bits of 32 tokens each
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
  const int c0 = (blockIdx.x * WAVES + wave) * 128, c = c0 + col * 8;
  const bool mine = c < p.D;                       // D is a multiple of 8
  u4 wh[8], wl[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = (quad >> 1) * 8 + j;
    wh[j] = mine && e < p.E ? load8(p.w + (size_t)e * p.D + c) : u4{0, 0, 0, 0};
  }
  transpose8(wh);
  if constexpr (A::HALF)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      to_bf16<A>(wh[j], wh[j], wl[j]);
      if (quad & 1) wl[j] = u4{0, 0, 0, 0};        // these lanes hold lo of dz
    }
  float held = 0.0f;                               // sequences with tokens
  if (p.n == nullptr) held = (float)p.seqs;
  else {
    for (int s = lane; s < p.seqs; s += 64) held += p.n[s] > 0 ? 1.0f : 0.0f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) held += __shfl_xor(held, off, 64);
  }
  const float factor = held > 0.0f ? *p.dloss * p.alpha / held * ((float)p.E / (float)p.k) : 0.0f;
  f4 acc[8] = {};
  const int begin = blockIdx.y * p.per_split, end = min(p.T, begin + p.per_split);
  for (int t0 = begin; t0 < end; t0 += STAGE) {
    {   // dz of a token by four threads, four experts each
      const int row = threadIdx.x >> 2, e0 = (threadIdx.x & 3) * 4, t = t0 + row;
      const bool on = t < end && (p.mask == nullptr || p.mask[t] != 0);
      float s[4] = {}, dp[4] = {}, dot = 0.0f;
      if (on) {
        const int seq = t / p.length;
        const float n = p.n == nullptr ? (float)p.length : (float)p.n[seq];
        const float f = factor / (n * n);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e0 + i < p.E) {
            s[i] = p.scores[(size_t)t * p.E + e0 + i];
            dp[i] = f * (float)p.counts[(size_t)seq * p.E + e0 + i];
          }
        if (p.dweight != nullptr)
          for (int j = 0; j < p.k; ++j) {
            const int e = p.idx[(size_t)t * p.k + j] - e0;
            const float d = A::lo(p.dweight[(size_t)t * p.k + j]);
#pragma unroll
            for (int i = 0; i < 4; ++i) dp[i] += e == i ? d : 0.0f;
          }
      }
      // Less the first expert's dp: a softmax's gradient does not change by what all dp of a token have in common, and the sum of s is a rounding away from
      // 1. Where all dp are the same, as with every expert chosen by every token, the gradient is 0.
      const float common = __shfl(dp[0], lane & ~3, 64);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dp[i] -= common;
        dot = __builtin_fmaf(s[i], dp[i], dot);
      }
      dot += __shfl_xor(dot, 1, 64);
      dot += __shfl_xor(dot, 2, 64);
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) split(s[2 * i] * (dp[2 * i] - dot), s[2 * i + 1] * (dp[2 * i + 1] - dot), hi[i], lo[i]);
      const uint64_t bits = __ballot(on && (threadIdx.x & 3) == 0);   // every fourth lane: 16 tokens of the wave
      __syncthreads();                                                // the stage before has been read
      if (threadIdx.x < 2) live[threadIdx.x] = 0;
      const int at = (e0 >> 3) * 16 + (e0 & 7);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<uint32_t*>(&along_e[row][at + 2 * i]) = hi[i];
        *reinterpret_cast<uint32_t*>(&along_e[row][at + 8 + 2 * i]) = lo[i];
        along_t[0][e0 + 2 * i][row] = (uint16_t)hi[i], along_t[0][e0 + 2 * i + 1][row] = (uint16_t)(hi[i] >> 16);
        along_t[1][e0 + 2 * i][row] = (uint16_t)lo[i], along_t[1][e0 + 2 * i + 1][row] = (uint16_t)(lo[i] >> 16);
      }
      __syncthreads();
      if (lane == 0) {
        uint32_t m = 0;
        for (int i = 0; i < 16; ++i) m |= (uint32_t)((bits >> (4 * i)) & 1) << i;
        atomicOr(&live[wave >> 1], (int)(m << (16 * (wave & 1))));
      }
      __syncthreads();
    }
    if (c0 >= p.D) continue;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const uint32_t has = (uint32_t)live[st];
      if (t0 + st * 32 >= end) break;
      u4 v[8];
      const uint16_t* from = p.x + (size_t)(t0 + st * 32 + quad * 8) * p.D + c;
      if (has == 0xffffffffu && c0 + 128 <= p.D) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = load8(from + (size_t)j * p.D);
      } else {   // masked tokens are 0
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = mine && ((has >> (quad * 8 + j)) & 1) ? load8(from + (size_t)j * p.D) : u4{0, 0, 0, 0};
      }
      // dx of 16 tokens at a time
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const u4 q = *reinterpret_cast<const u4*>(&along_e[st * 32 + m * 16 + col][quad * 8]);
        f4 y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
          if constexpr (A::HALF) y[j] = Bf16::mul(wl[j], q, y[j]);
          y[j] = Bf16::mul(wh[j], q, y[j]);
        }
        u4 o[4];      // 32 columns of a token next to each other
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int w = 0; w < 4; ++w) o[e][w] = A::pack(y[2 * w][e], y[2 * w + 1][e]);
        quad_transpose(o);
        const int d = c0 + quad * 32 + (col & 3) * 8;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + st * 32 + m * 16 + (col & 12) + e;
          if (t < end && d < p.D) __builtin_memcpy(p.dx + (size_t)t * p.D + d, &o[e], 16);
        }
      }
      // dW
      transpose8(v);
      const u4 qh = *reinterpret_cast<const u4*>(&along_t[0][col][st * 32 + quad * 8]), ql = *reinterpret_cast<const u4*>(&along_t[1][col][st * 32 + quad * 8]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u4 vh, vl;
        to_bf16<A>(v[j], vh, vl);
        acc[j] = Bf16::mul(ql, vh, acc[j]);
        if constexpr (A::HALF) acc[j] = Bf16::mul(qh, vl, acc[j]);
        acc[j] = Bf16::mul(qh, vh, acc[j]);
      }
    }
  }
  if (!mine) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = quad * 4 + i;
    if (e >= p.E) continue;
    if (p.direct) {
      u4 o;
#pragma unroll
      for (int w = 0; w < 4; ++w) o[w] = A::pack(acc[2 * w][i], acc[2 * w + 1][i]);
      __builtin_memcpy(static_cast<uint16_t*>(p.dw) + (size_t)e * p.D + c, &o, 16);
    } else {
      float* to = static_cast<float*>(p.dw) + ((size_t)blockIdx.y * p.E + e) * p.D + c;
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = acc[j][i];
    }
  }
}

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// 16 tokens a tile while that makes at most two blocks a CU, else 64: a quarter of the reads of W
int balance_tile(int length, int seqs) { return (int64_t)div_up(length, 16) * seqs <= 2 * HDMOE_NUM_CU ? 16 : 64; }

// tokens of a block of the backward kernel
int balance_split(int T, int D) {
  const int strips = div_up(D, WAVES * 128);
  int splits = div_up(2 * HDMOE_NUM_CU, strips);
  const int each = div_up(div_up(T, splits), STAGE) * STAGE;
  return each;
}

// Sizes alone: what the workspace depends on, beside whether there is a mask
int check_sizes(const hdmoe_balance_args* a, const char* what) {
  if (a == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: args is NULL", what);
  if (a->dtype != HDMOE_T_BF16 && a->dtype != HDMOE_T_F16) return hdmoe_fail(HDMOE_E_SHAPE, "%s: dtype=%d", what, a->dtype);
  if (a->T < 0 || a->T > (1 << 30) || a->D < 8 || a->D % 8 != 0 || a->D > (1 << 24) || a->E < 1 || a->E > HDMOE_MAX_EXPERTS || a->k < 1 || a->k > HDMOE_MAX_EXPERTS ||
      a->sequences < 1 || a->T % a->sequences != 0)
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: T=%d sequences=%d D=%d (a multiple of 8) E=%d k=%d (1 to %d)", what, a->T, a->sequences, a->D, a->E, a->k,
                      HDMOE_MAX_EXPERTS);
  const int length = a->T / a->sequences;
  if ((int64_t)a->sequences * (div_up(length, balance_tile(length, a->sequences)) + 1) * SCORE_WAVES * 64 >= (int64_t)1 << 32)      // threads of a launch
    return hdmoe_fail(HDMOE_E_SHAPE, "%s: T=%d sequences=%d: too many", what, a->T, a->sequences);
  return HDMOE_OK;
}

int check_balance(const hdmoe_balance_args* a, const char* what) {
  if (int rc = check_sizes(a, what)) return rc;
  if (a->gate_w == nullptr || a->counts == nullptr) return hdmoe_fail(HDMOE_E_NULL, "%s: gate_w or counts is NULL", what);
  if (a->T > 0 && (a->x == nullptr || a->topk_idx == nullptr || a->scores == nullptr))
    return hdmoe_fail(HDMOE_E_NULL, "%s: x, topk_idx or scores is NULL", what);
  return HDMOE_OK;
}

size_t balance_bytes(const hdmoe_balance_args* a, bool backward) {
  if (!backward) {
    const int length = a->T / a->sequences;
    return a->T == 0 ? 0 : (size_t)a->sequences * div_up(length, balance_tile(length, a->sequences)) * sizeof(TileSums);
  }
  const int each = a->T > 0 ? balance_split(a->T, a->D) : 1, splits = div_up(a->T, each);
  return hdmoe_align_up(a->mask != nullptr ? (size_t)a->sequences * sizeof(int32_t) : 0, 256) + (splits > 1 ? (size_t)splits * a->E * a->D * sizeof(float) : 0);
}

template <class F>
void typed(int dtype, F f) {
  if (dtype == HDMOE_T_BF16) f(Bf16());
  else f(lowrank::F16());
}

}  // namespace

extern "C" size_t hdmoe_gate_balance_workspace_bytes(const hdmoe_balance_args* a, int backward) {
  return check_sizes(a, "hdmoe_gate_balance_workspace_bytes") == HDMOE_OK ? balance_bytes(a, backward != 0) : 0;
}

static int check_workspace(const hdmoe_balance_args* a, bool backward, const char* what) {
  const size_t need = balance_bytes(a, backward);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0))
    return hdmoe_fail(HDMOE_E_WORKSPACE, "%s: workspace of %zu bytes on 16 needed, got %zu", what, need, a->workspace_bytes);
  return HDMOE_OK;
}

extern "C" int hdmoe_gate_balance(const hdmoe_balance_args* a, hdmoe_stream_t stream) {
  if (int rc = check_balance(a, "hdmoe_gate_balance")) return rc;
  if (a->loss == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_gate_balance: loss is NULL");
  if (int rc = check_workspace(a, false, "hdmoe_gate_balance")) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  BalanceArgs p = {};
  p.x = static_cast<const uint16_t*>(a->x), p.w = static_cast<const uint16_t*>(a->gate_w), p.idx = a->topk_idx, p.mask = a->mask;
  p.scores = static_cast<float*>(a->scores), p.tiles = static_cast<TileSums*>(a->workspace);
  p.T = a->T, p.length = a->T / a->sequences, p.D = a->D, p.E = a->E, p.k = a->k;
  if (a->T > 0) {
    const int tile = balance_tile(p.length, a->sequences);
    p.tiles_per_seq = div_up(p.length, tile);
    typed(a->dtype, [&](auto t) {
      typedef decltype(t) A;
      const dim3 grid((unsigned)(p.tiles_per_seq * a->sequences));
      if (tile == 16) hipLaunchKernelGGL((gate_balance_kernel<A, 1>), grid, dim3(SCORE_WAVES * 64), 0, s, p);
      else hipLaunchKernelGGL((gate_balance_kernel<A, 4>), grid, dim3(SCORE_WAVES * 64), 0, s, p);
    });
  }
  hipLaunchKernelGGL(balance_finish_kernel, dim3(1), dim3(1024), 0, s, p.tiles, a->sequences, p.tiles_per_seq, a->E, a->k, a->alpha, a->loss, a->counts);
  return hdmoe_check_launch("hdmoe_gate_balance");
}

extern "C" int hdmoe_gate_balance_backward(const hdmoe_balance_args* a, hdmoe_stream_t stream) {
  if (int rc = check_balance(a, "hdmoe_gate_balance_backward")) return rc;
  if (a->dloss == nullptr || a->dgate_w == nullptr || (a->T > 0 && a->dx == nullptr))
    return hdmoe_fail(HDMOE_E_NULL, "hdmoe_gate_balance_backward: dloss, dgate_w or dx is NULL");
  if (int rc = check_workspace(a, true, "hdmoe_gate_balance_backward")) return rc;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int each = a->T > 0 ? balance_split(a->T, a->D) : 1, splits = div_up(a->T, each);
  char* ws = static_cast<char*>(a->workspace);
  int32_t* n = a->mask != nullptr ? reinterpret_cast<int32_t*>(ws) : nullptr;
  float* parts = reinterpret_cast<float*>(ws + hdmoe_align_up(n != nullptr ? (size_t)a->sequences * sizeof(int32_t) : 0, 256));
  SumArgs sp = {};
  sp.part[0] = parts, sp.out[0] = static_cast<uint16_t*>(a->dgate_w), sp.n[0] = (size_t)a->E * a->D, sp.splits = splits;
  BalanceGrad p = {};
  p.x = static_cast<const uint16_t*>(a->x), p.w = static_cast<const uint16_t*>(a->gate_w), p.idx = a->topk_idx, p.counts = a->counts;
  p.mask = a->mask, p.scores = static_cast<const float*>(a->scores), p.dloss = a->dloss, p.dweight = static_cast<const uint16_t*>(a->dweight);
  p.n = n, p.dx = static_cast<uint16_t*>(a->dx), p.direct = splits == 1, p.dw = p.direct ? a->dgate_w : parts;
  p.T = a->T, p.length = a->T / a->sequences, p.seqs = a->sequences, p.D = a->D, p.E = a->E, p.k = a->k, p.per_split = each, p.alpha = a->alpha;
  typed(a->dtype, [&](auto t) {
    typedef decltype(t) A;
    if (a->T > 0) {
      if (n != nullptr) hipLaunchKernelGGL(mask_counts_kernel, dim3(a->sequences), dim3(256), 0, s, a->mask, p.length, n);
      hipLaunchKernelGGL(gate_balance_backward_kernel<A>, dim3(div_up(a->D, WAVES * 128), splits), dim3(WAVES * 64), 0, s, p);
    }
    if (splits != 1) launch_sum_parts<A>(sp, s);
  });
  return hdmoe_check_launch("hdmoe_gate_balance_backward");
}
