// Layer norm over the last axis, and its gradients (an affine norm, or one that is modulated by a scale and a shift of each sequence).
//
//   n = (x - mean) r,  r = 1 / sqrt(mean((x - mean)^2) + eps)      y = n w + b
//   g = dy w           dx = r (g - mean(g) - n mean(g n))          dw = sum_rows dy n,  db = sum_rows dy
//
// A row stays in the registers of one wave, or of four or eight of a block where it is long or rows are few, so it is read once, its
// variance is that of the differences from its mean (nothing cancels), and the backward pass takes mean and r from x again instead of
// reading what a forward pass would have stored. All sums are fp32; every output is rounded once.
//
// A sum of D values times 1 / D is a few roundings off the mean, of the values' size: for equal values that alone would be their variance, and r up to
// 1 / sqrt(eps) times it (1000 values of 29952, eps 1e-5: y of 0.5 instead of 0). The sum of the differences f = x - mean goes beside that of their squares and
// says what the mean lacks: c = sum f / D, mean + c, var = sum f^2 / D - c^2, sum g (f - c) = sum g f - c sum g. Equal values then have differences of 0.
//
// The sums over rows of dw and db: a wave keeps them for its columns over all rows that it takes, the waves of a block add theirs up in
// LDS, and a second kernel adds the blocks' up, each in one fixed order (no atomics). Modulated: a block's rows are of one sequence.
#include <type_traits>

#include "common.h"
#include "numfmt.h"

namespace {

constexpr int V = 8;                 // values a lane takes at a time
constexpr int NORM_BLOCKS = 512;     // partial sums at most: two blocks a CU
constexpr int FEW_ROWS = HDMOE_NUM_CU * 8;

struct NormBf16 {
  typedef uint16_t type;
  static __device__ __forceinline__ float one(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t put(float f) { return (uint16_t)hdmoe_dev_pack_bf16(f, 0.0f); }
};
struct NormF16 {
  typedef uint16_t type;
  static __device__ __forceinline__ float one(uint16_t v) { return HdmoeF16::lo(v); }
  static __device__ __forceinline__ uint16_t put(float f) { return (uint16_t)HdmoeF16::pack(f, 0.0f); }
};
struct NormF32 {
  typedef float type;
  static __device__ __forceinline__ float one(float v) { return v; }
  static __device__ __forceinline__ float put(float f) { return f; }
};

// V values as they lie in memory. Rows start anywhere (an odd D, a view): global loads of 16 bytes take any address.
template <class A>
struct Raw {
  typename A::type v[V];
  __device__ __forceinline__ void load(const typename A::type* p, int have) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = typename A::type(0);
    if (have >= V) {
      __builtin_memcpy(v, p, sizeof(v));
    } else if (have > 0) {     // in no lane where D is a multiple of V
#pragma unroll
      for (int j = 0; j < V - 1; ++j)
        if (j < have) v[j] = p[j];
    }
  }
  __device__ __forceinline__ float at(int j) const { return A::one(v[j]); }
};

template <class A>
__device__ __forceinline__ void store(typename A::type* p, const float (&f)[V], int have) {
  typename A::type o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = A::put(f[j]);
  if (have >= V) {
    __builtin_memcpy(p, o, sizeof(o));
  } else if (have > 0) {
#pragma unroll
    for (int j = 0; j < V - 1; ++j)
      if (j < have) p[j] = o[j];
  }
}

// Sums of N values over the wave, every lane ending with the totals.
template <int N>
__device__ __forceinline__ void wave_sums(float (&v)[N]) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, 64);
}

// The same over the W waves of a block that share a row. `turn` alternates between calls: a wave may be in the next one while another
// still reads this one's.
template <int W, int M, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*lds)[W][M], int& turn) {
  static_assert(N <= M);
  wave_sums(v);
  if constexpr (W > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) lds[turn][wave][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[i] += lds[turn][w][i];
    }
    turn ^= 1;
  }
}

// r from v = sum f^2 / D and c. Past the largest number v says so and c^2 nothing.
__device__ __forceinline__ float inverse_deviation(float v, float c, float eps) {
  if (v < __builtin_inff()) v = fmaxf(__builtin_fmaf(-c, c, v), 0.0f);
  return 1.0f / __builtin_sqrtf(v + eps);
}

struct Gain {
  const void* w;      // NULL: 1
  const void* b;      // NULL: 0
  int f32;            // w and b are fp32, else of the rows' type
};

// Gains of the lane's V columns (16-byte loads where the columns are all there), 0 beyond the row.
template <class A>
__device__ __forceinline__ void gains(float (&f)[V], const void* w, int f32, size_t base, int have) {
  if (f32) {
    Raw<NormF32> r;
    r.load(static_cast<const float*>(w) + base, have);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = r.at(j);
  } else {
    Raw<A> r;
    r.load(static_cast<const typename A::type*>(w) + base, have);
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = r.at(j);
  }
}

// W waves a row (1: every wave of the block takes rows of its own), C chunks of W * 64 * V values of it.
// FULL: D is all of them.
constexpr int threads(int W) { return W > 4 ? W * 64 : 256; }

template <class A, int W, int C, bool FULL>
__global__ __launch_bounds__(threads(W)) void layer_norm_kernel(const typename A::type* __restrict__ x, Gain gain, int64_t rows, int D, float eps,
                                                         typename A::type* __restrict__ out) {
  __shared__ float lds[2][W][2];
  int turn = 0;
  constexpr int TEAMS = W > 4 ? 1 : 4 / W;
  const int lane = threadIdx.x & (W * 64 - 1);
  const float inv = 1.0f / (float)D;
  int have[C];
#pragma unroll
  for (int c = 0; c < C; ++c) have[c] = FULL ? V : min(V, max(0, D - (c * W * 64 + lane) * V));
  for (int64_t t = (int64_t)blockIdx.x * TEAMS + threadIdx.x / (W * 64); t < rows; t += (int64_t)gridDim.x * TEAMS) {
    const size_t at = (size_t)t * D + (size_t)lane * V;
    Raw<A> raw[C];
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c].load(x + at + c * W * 64 * V, have[c]);
    float f[C][V], s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) f[c][j] = raw[c].at(j), s[0] += f[c][j];
    row_sums<W>(s, lds, turn);
    const float mean = s[0] * inv;
    float q[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[c][j] = FULL || j < have[c] ? f[c][j] - mean : 0.0f;
        q[0] = __builtin_fmaf(f[c][j], f[c][j], q[0]);
        q[1] += f[c][j];
      }
    row_sums<W>(q, lds, turn);
    const float lacks = q[1] / (float)D, r = inverse_deviation(q[0] * inv, lacks, eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * W * 64 + lane) * V;
      float y[V], w[V], b[V];
      if (gain.w != nullptr) gains<A>(w, gain.w, gain.f32, col, have[c]);
      if (gain.b != nullptr) gains<A>(b, gain.b, gain.f32, col, have[c]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y[j] = (f[c][j] - lacks) * r;
        if (gain.w != nullptr) y[j] *= w[j];
        if (gain.b != nullptr) y[j] += b[j];
      }
      store<A>(out + at + c * W * 64 * V, y, have[c]);
    }
  }
}

struct NormGrad {
  const void *dy, *x, *w;
  void *dx, *dw, *db;
  float* part;            // [groups * blocks][2][D] sums of the blocks; NULL: a block's sums are the result
  int64_t per_group;      // rows that share a row of w
  int blocks;             // blocks of a group
  int D, w_f32, g_f32;    // w and dw, db are fp32, else of the rows' type
  float plus, eps;
};

template <class A>
__device__ __forceinline__ void put_grad(void* p, int f32, size_t i, float v) {
  if (f32) static_cast<float*>(p)[i] = v;
  else static_cast<typename A::type*>(p)[i] = A::put(v);
}

// Two waves of one of a CU's four units whatever registers five chunks would like: without that, 30000 x 2200 in fp16 took 270 us, with it 180.
template <class A, int W, int C, bool FULL>
__global__ __launch_bounds__(threads(W), 2) void layer_norm_backward_kernel(NormGrad p) {
  constexpr int TEAMS = W > 4 ? 1 : 4 / W;
  constexpr int WIDTH = W * 64 * V * C;
  __shared__ float lds[2][W][3];
  __shared__ __attribute__((aligned(16))) float joined[TEAMS][TEAMS > 1 ? WIDTH : 1];
  int turn = 0;
  const int lane = threadIdx.x & (W * 64 - 1), team = threadIdx.x / (W * 64), D = p.D;
  const float inv = 1.0f / (float)D;
  const typename A::type *x = static_cast<const typename A::type*>(p.x), *dy = static_cast<const typename A::type*>(p.dy);
  typename A::type* dx = static_cast<typename A::type*>(p.dx);
  const int64_t group = blockIdx.x / p.blocks;
  const int block = blockIdx.x % p.blocks;
  const bool sums = p.dw != nullptr || p.db != nullptr;
  int have[C];
#pragma unroll
  for (int c = 0; c < C; ++c) have[c] = FULL ? V : min(V, max(0, D - (c * W * 64 + lane) * V));
  float aw[C][V] = {}, ab[C][V] = {};
  for (int64_t t = (int64_t)block * TEAMS + team; t < p.per_group; t += (int64_t)p.blocks * TEAMS) {
    const size_t at = (size_t)(group * p.per_group + t) * D + (size_t)lane * V;
    Raw<A> rx[C], ry[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      rx[c].load(x + at + c * W * 64 * V, have[c]);
      ry[c].load(dy + at + c * W * 64 * V, have[c]);
    }
    float f[C][V], g[C][V], s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float w[V];
      if (p.w != nullptr) gains<A>(w, p.w, p.w_f32, (size_t)group * D + (c * W * 64 + lane) * V, have[c]);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[c][j] = rx[c].at(j);
        g[c][j] = p.w != nullptr ? ry[c].at(j) * (p.plus + w[j]) : ry[c].at(j);
        s[0] += f[c][j];
        s[1] += g[c][j];
      }
    }
    row_sums<W>(s, lds, turn);
    const float mean = s[0] * inv, mg = s[1] * inv;
    float q[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        f[c][j] = FULL || j < have[c] ? f[c][j] - mean : 0.0f;
        q[0] = __builtin_fmaf(f[c][j], f[c][j], q[0]);
        q[1] = __builtin_fmaf(f[c][j], g[c][j], q[1]);
        q[2] += f[c][j];
      }
    row_sums<W>(q, lds, turn);
    const float lacks = q[2] / (float)D, r = inverse_deviation(q[0] * inv, lacks, p.eps);
    const float mgn = __builtin_fmaf(-lacks, s[1], q[1]) * r * inv;   // mean(g n)
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float n = (f[c][j] - lacks) * r, d = ry[c].at(j);
        o[j] = r * (g[c][j] - mg - n * mgn);
        aw[c][j] = __builtin_fmaf(d, n, aw[c][j]);
        ab[c][j] += d;
      }
      store<A>(dx + at + c * W * 64 * V, o, have[c]);
    }
  }
  if (!sums) return;
  // the teams' sums, dw and then db: each thread adds up columns of its own
  auto put = [&](int which, int col, float v) {
    if (p.part != nullptr) {
      p.part[((size_t)blockIdx.x * 2 + which) * D + col] = v;
    } else {
      void* to = which == 0 ? p.dw : p.db;
      if (to != nullptr) put_grad<A>(to, p.g_f32, (size_t)group * D + col, v);
    }
  };
  if constexpr (TEAMS > 1) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 1) __syncthreads();
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) joined[team][(c * V + j) * 64 + lane] = which == 0 ? aw[c][j] : ab[c][j];   // next to the neighbours'
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WIDTH / 256; ++i) {
        // column 8 l + j of chunk c lies at (8 c + j) 64 + l
        const int col = i * 256 + threadIdx.x, at = ((col >> 9) * V + (col & 7)) * 64 + ((col >> 3) & 63);
        float v = joined[0][at];
#pragma unroll
        for (int w = 1; w < TEAMS; ++w) v += joined[w][at];
        if (col < D) put(which, col, v);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = (c * W * 64 + lane) * V;
      if (p.part != nullptr) {
        float* q = p.part + (size_t)blockIdx.x * 2 * D + col;
        store<NormF32>(q, aw[c], have[c]);
        store<NormF32>(q + D, ab[c], have[c]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (j < have[c]) put(0, col + j, aw[c][j]), put(1, col + j, ab[c][j]);
      }
    }
  }
}

// Sums of the blocks' parts: 64 columns of one group a block, its 16 waves each a run of parts, joined in their order.
template <class A>
__global__ __launch_bounds__(1024) void norm_sums_kernel(NormGrad p) {
  __shared__ float lds[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t group = blockIdx.y;
  const int col = blockIdx.x * 64 + lane;      // of [2][D]
  float s = 0.0f;
  if (col < 2 * p.D) {
    const int each = (p.blocks + 15) / 16;
    const int lo = wave * each, hi = min(p.blocks, lo + each);
    const float* q = p.part + (size_t)group * p.blocks * 2 * p.D + col;
#pragma unroll 8
    for (int b = lo; b < hi; ++b) s += q[(size_t)b * 2 * p.D];
  }
  lds[wave][lane] = s;
  __syncthreads();
  if (wave != 0 || col >= 2 * p.D) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += lds[w][lane];
  void* to = col < p.D ? p.dw : p.db;
  if (to != nullptr) put_grad<A>(to, p.g_f32, (size_t)group * p.D + (col < p.D ? col : col - p.D), s);
}

// One block a group where a second launch (2 us) costs more than the rows that its waves then take one after the other: four a wave, where a row has the
// whole block of 5120 values in all (4 x 1000 8.5 us in one block, 9.5 in four; 2 x 2560 8.1, 9.1; 4 x 2560 12.6, 9.2; 4 x 8000 21.8, 10.2).
int norm_blocks(int64_t per_group, int64_t groups, int D) {
  const int teams = D <= 512 || (per_group * groups >= FEW_ROWS && D <= 2560) ? 4 : 1;
  int64_t most = NORM_BLOCKS / (groups > 0 ? groups : 1);
  if (most < 1) most = 1;
  const int64_t each = D > 8192 ? 2 : teams, fill = (per_group + each - 1) / each;     // 300 rows of 16384: one a block 29 us, two 21
  if (per_group <= 4 * teams && (teams > 1 || per_group * D <= 5120)) return 1;
  return (int)(fill < most ? fill : most);
}

template <class A, int W, int C>
void launch_norm(bool full, int grid, hipStream_t s, const void* x, const Gain& gain, int64_t rows, int D, float eps, void* out) {
  const typename A::type* xp = static_cast<const typename A::type*>(x);
  typename A::type* op = static_cast<typename A::type*>(out);
  if (full) hipLaunchKernelGGL((layer_norm_kernel<A, W, C, true>), dim3(grid), dim3(threads(W)), 0, s, xp, gain, rows, D, eps, op);
  else hipLaunchKernelGGL((layer_norm_kernel<A, W, C, false>), dim3(grid), dim3(threads(W)), 0, s, xp, gain, rows, D, eps, op);
}

template <class A, int W, int C>
void launch_grad(bool full, int grid, hipStream_t s, const NormGrad& p) {
  if (full) hipLaunchKernelGGL((layer_norm_backward_kernel<A, W, C, true>), dim3(grid), dim3(threads(W)), 0, s, p);
  else hipLaunchKernelGGL((layer_norm_backward_kernel<A, W, C, false>), dim3(grid), dim3(threads(W)), 0, s, p);
}

// f(W, C) with the shape that a row of D values is held in: one wave where there are rows for eight waves of every CU, four where there are fewer (forward
// of 1021 x 1153 5.5 -> 4.5 us, gradients of 77 x 2560 10.3 -> 9.2) or where the row would take more than five chunks of a wave (12 x 2817 15 -> 9).
template <class F>
void norm_shape(int D, int64_t rows, F f) {
  using std::integral_constant;
  const integral_constant<int, 1> one;
  const integral_constant<int, 2> two;
  const integral_constant<int, 3> three;
  const integral_constant<int, 4> four;
  if (D <= 512) f(one, one);
  else if (rows >= FEW_ROWS && D <= 2560) {
    if (D <= 1024) f(one, two);
    else if (D <= 1536) f(one, three);
    else if (D <= 2048) f(one, four);
    else f(one, integral_constant<int, 5>());
  } else if (D <= 2048) f(four, one);
  else if (D <= 4096) f(four, two);
  else if (D <= 6144) f(four, three);
  else if (D <= 8192) f(four, four);
  else f(integral_constant<int, 8>(), four);
}

bool norm_dtype(int dtype) { return dtype == HDMOE_T_BF16 || dtype == HDMOE_T_F16 || dtype == HDMOE_T_F32; }

template <class F>
void norm_type(int dtype, F f) {
  if (dtype == HDMOE_T_BF16) f(NormBf16());
  else if (dtype == HDMOE_T_F16) f(NormF16());
  else f(NormF32());
}

}  // namespace

extern "C" int hdmoe_layer_norm(int dtype, const void* x, int64_t rows, int D, int gain_dtype, const void* weight, const void* bias,
                                float eps, void* out, hdmoe_stream_t stream) {
  if (!norm_dtype(dtype) || ((weight != nullptr || bias != nullptr) && gain_dtype != dtype && gain_dtype != HDMOE_T_F32))
    return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_layer_norm: dtype=%d gain_dtype=%d (the gains are of the rows' type or fp32)", dtype, gain_dtype);
  if (rows < 0 || D < 1 || D > HDMOE_NORM_MAX_D || !(eps >= 0.0f))
    return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_layer_norm: rows=%lld D=%d (1 to %d) eps=%g", (long long)rows, D, HDMOE_NORM_MAX_D, (double)eps);
  if (rows == 0) return HDMOE_OK;
  HDMOE_REQUIRE_PTR(x);
  HDMOE_REQUIRE_PTR(out);
  const Gain gain = {weight, bias, gain_dtype == HDMOE_T_F32};
  const hipStream_t s = static_cast<hipStream_t>(stream);
  norm_shape(D, rows, [&](auto w, auto c) {
    constexpr int W = decltype(w)::value, C = decltype(c)::value;
    constexpr int TEAMS = W > 4 ? 1 : 4 / W;
    int64_t grid = (rows + TEAMS - 1) / TEAMS;
    if (grid > HDMOE_NUM_CU * 8) grid = HDMOE_NUM_CU * 8;
    norm_type(dtype, [&](auto a) { launch_norm<decltype(a), W, C>(D == W * 64 * V * C, (int)grid, s, x, gain, rows, D, eps, out); });
  });
  return hdmoe_check_launch("hdmoe_layer_norm");
}

extern "C" size_t hdmoe_layer_norm_backward_workspace_bytes(int64_t rows, int D, int64_t rows_per_group) {
  if (rows <= 0 || D < 1 || D > HDMOE_NORM_MAX_D || rows_per_group <= 0 || rows % rows_per_group != 0) return 0;
  const int64_t groups = rows / rows_per_group;
  const int blocks = norm_blocks(rows_per_group, groups, D);
  return blocks > 1 ? (size_t)groups * blocks * 2 * D * sizeof(float) : 0;
}

extern "C" int hdmoe_layer_norm_backward(const hdmoe_norm_grad_args* a, hdmoe_stream_t stream) {
  if (a == nullptr) return hdmoe_fail(HDMOE_E_NULL, "hdmoe_layer_norm_backward: args is NULL");
  const bool sums = a->dweight != nullptr || a->dbias != nullptr;
  if (!norm_dtype(a->dtype) || ((a->weight != nullptr || sums) && a->gain_dtype != a->dtype && a->gain_dtype != HDMOE_T_F32))
    return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_layer_norm_backward: dtype=%d gain_dtype=%d (the gains are of the rows' type or fp32)", a->dtype,
                      a->gain_dtype);
  if (a->rows < 0 || a->D < 1 || a->D > HDMOE_NORM_MAX_D || !(a->eps >= 0.0f) || a->rows_per_group < 0 ||
      (a->rows > 0 && (a->rows_per_group == 0 || a->rows % a->rows_per_group != 0)))
    return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_layer_norm_backward: rows=%lld rows_per_group=%lld D=%d (1 to %d) eps=%g", (long long)a->rows,
                      (long long)a->rows_per_group, a->D, HDMOE_NORM_MAX_D, (double)a->eps);
  const int64_t groups = a->rows > 0 ? a->rows / a->rows_per_group : (a->rows_per_group == 0 ? 1 : 0);
  if (groups >= (int64_t)1 << 23)     // of 512 threads at least: a launch has fewer than 2^32
    return hdmoe_fail(HDMOE_E_SHAPE, "hdmoe_layer_norm_backward: %lld groups", (long long)groups);
  NormGrad p = {};
  p.dy = a->dy, p.x = a->x, p.w = a->weight, p.dx = a->dx, p.dw = a->dweight, p.db = a->dbias;
  p.per_group = a->rows_per_group, p.D = a->D, p.w_f32 = p.g_f32 = a->gain_dtype == HDMOE_T_F32;
  p.plus = a->one_plus ? 1.0f : 0.0f, p.eps = a->eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->rows == 0) {   // nothing to add up: gradients of zero
    if (!sums || groups == 0) return HDMOE_OK;
    p.blocks = 0;
    norm_type(a->dtype, [&](auto t) {
      hipLaunchKernelGGL(norm_sums_kernel<decltype(t)>, dim3((2 * a->D + 63) / 64, 1), dim3(1024), 0, s, p);
    });
    return hdmoe_check_launch("hdmoe_layer_norm_backward");
  }
  if (a->dy == nullptr || a->x == nullptr || a->dx == nullptr)
    return hdmoe_fail(HDMOE_E_NULL, "hdmoe_layer_norm_backward: dy, x or dx is NULL");
  p.blocks = norm_blocks(a->rows_per_group, groups, a->D);
  if (p.blocks > 1 && sums) {
    const size_t need = hdmoe_layer_norm_backward_workspace_bytes(a->rows, a->D, a->rows_per_group);
    if (a->workspace == nullptr || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16 != 0)
      return hdmoe_fail(HDMOE_E_WORKSPACE, "hdmoe_layer_norm_backward: workspace of %zu bytes on 16 needed, got %zu", need, a->workspace_bytes);
    p.part = static_cast<float*>(a->workspace);
  }
  norm_shape(a->D, a->rows, [&](auto w, auto c) {
    constexpr int W = decltype(w)::value, C = decltype(c)::value;
    norm_type(a->dtype, [&](auto t) { launch_grad<decltype(t), W, C>(a->D == W * 64 * V * C, (int)(groups * p.blocks), s, p); });
  });
  if (p.part != nullptr)
    norm_type(a->dtype, [&](auto t) {
      hipLaunchKernelGGL(norm_sums_kernel<decltype(t)>, dim3((2 * a->D + 63) / 64, (unsigned)groups), dim3(1024), 0, s, p);
    });
  return hdmoe_check_launch("hdmoe_layer_norm_backward");
}
