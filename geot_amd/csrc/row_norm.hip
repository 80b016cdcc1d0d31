// row_norm.hip -- layer normalisation of rows: geot_layer_norm and its backward pass.
//
//   mu = mean x, v = mean (x - mu)^2, s = 1 / sqrt(v + eps), h = (x - mu) s, y = h w + b
//   dx = s (g - mean g - h mean(g h)) with g = dy w;   dw = sum over rows of dy h;   db = sum over rows of dy
//
// Bound by memory: a row is read once and stays in the registers of its team of L lanes (EPL elements a lane), which holds the weight's
// and the bias's columns too and walks over rows.  The mean is taken in two steps - m = mean x in float32, then c = mean (x - m) - and
// used as m + c: the variance is mean (x - m)^2 - c^2 with c at the size of m's rounding, so rows far from zero (mean 1e4, spread 1) keep
// their digits.  The backward pass adds dw and db up in registers over its rows, joins its teams in LDS, writes one partial row a
// workgroup and a second kernel adds those in a fixed order: no atomics, the same bits every run.
//
// Measured (2.4 M rows of 128, bf16): forward 277 us (1.25 GB, 4.5 TB/s), backward 412 us (1.88 GB, 4.6 TB/s) + 11 us for the join; rows of
// 4096 float32, forward: 116 us for 16384 (4.6 TB/s).  A plain copy reaches 4.9 TB/s on the same card.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "geot_hip.h"
#include "internal.h"

namespace {

using bf16 = __bf16;
using f16 = _Float16;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), may_alias));
template <int SIZE> struct Packed;
template <> struct Packed<2> {
  typedef u32x4 x16 __attribute__((aligned(2), may_alias));
};
template <> struct Packed<4> {
  typedef u32x4 x16 __attribute__((aligned(4), may_alias));
};
template <typename T> using Packed16 = typename Packed<sizeof(T)>::x16;
constexpr int kThreads = 256;

// V consecutive elements at p, `left` of which exist (the rest read as 0), as floats
template <typename T> __device__ inline void load_vec(const T *p, int64_t left, float *out) {
  constexpr int V = 16 / sizeof(T);
  alignas(16) T tmp[V];
  if (left >= V) {
    *reinterpret_cast<u32x4 *>(tmp) = *reinterpret_cast<const Packed16<T> *>(p);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) tmp[e] = e < left ? p[e] : (T)0.0f;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) out[e] = (float)tmp[e];
}
template <typename T> __device__ inline void store_vec(T *p, int64_t left, const float *in) {
  constexpr int V = 16 / sizeof(T);
  alignas(16) T tmp[V];
#pragma unroll
  for (int e = 0; e < V; ++e) tmp[e] = (T)in[e];
  if (left >= V) {
    *reinterpret_cast<Packed16<T> *>(p) = *reinterpret_cast<const u32x4 *>(tmp);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < left) p[e] = tmp[e];
  }
}

// Sums of two values over a team of L lanes; every lane gets them.  L = 256: over the workgroup (all threads call; `lds` holds two
// alternating sets of 2 x 4 floats, so one barrier a sum is enough).
template <int L> struct Team {
  float *lds;
  int turn = 0;
  __device__ void sum(float &a, float &b) {
#pragma unroll
    for (int m = 1; m < (L < 64 ? L : 64); m *= 2) {
      a += __shfl_xor(a, m);
      b += __shfl_xor(b, m);
    }
    if constexpr (L > 64) {
      float *set = lds + turn * 8;
      turn ^= 1;
      if (threadIdx.x % 64 == 0) {
        set[threadIdx.x / 64] = a;
        set[4 + threadIdx.x / 64] = b;
      }
      __syncthreads();
      a = (set[0] + set[1]) + (set[2] + set[3]);
      b = (set[4] + set[5]) + (set[6] + set[7]);
    }
  }
};

// lane's columns: element v * V + e of its EPL sits in column (v * L + lane) * V + e
template <typename T, typename P, int L, int EPL> struct Row {
  static constexpr int V = 16 / sizeof(T), NV = EPL / V;
  static __device__ int64_t column(int v, int lane) { return (int64_t)(v * L + lane) * V; }
  static __device__ void load(const T *row, int64_t d, int lane, float (&x)[EPL]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) load_vec<T>(row + column(v, lane), d - column(v, lane), x + v * V);
  }
  static __device__ void store(T *row, int64_t d, int lane, const float (&y)[EPL]) {
#pragma unroll
    for (int v = 0; v < NV; ++v) store_vec<T>(row + column(v, lane), d - column(v, lane), y + v * V);
  }
  static __device__ void params(const P *p, int64_t d, int lane, float none, float (&w)[EPL]) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int64_t c = column(v, lane) + e;
        w[v * V + e] = p && c < d ? (float)p[c] : none;
      }
  }
};

// s / d as ONE rounded number: left to the compiler, x - s * inv becomes a fused multiply-add of the unrounded product, and the mean that
// the statistics keep is another one (seen: 3.5e-4 off at a mean of 1e4)
__device__ inline float rounded_product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

struct NormArgs {
  const void *x, *weight, *bias, *dy;
  void *y, *dx;      // forward / backward result (dx null where it is not asked for)
  float *stats;      // [3, rows]
  float *part;       // backward: [blocks, 2, feat], null where no parameter gradient is asked for
  int64_t ldx, rows, feat;
  float eps;
};

template <typename T, typename P, int L, int EPL> __global__ __launch_bounds__(kThreads) void norm_kernel(const NormArgs g) {
  using R = Row<T, P, L, EPL>;
  __shared__ float lds[16];
  constexpr int TEAMS = kThreads / L;
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const int64_t d = g.feat;
  float w[EPL], b[EPL];
  R::params(static_cast<const P *>(g.weight), d, lane, 1.0f, w);
  R::params(static_cast<const P *>(g.bias), d, lane, 0.0f, b);
  Team<L> all{lds};
  const float inv = 1.0f / (float)d;
  for (int64_t row = (int64_t)blockIdx.x * TEAMS + team; row < g.rows; row += (int64_t)gridDim.x * TEAMS) {
    float x[EPL];
    R::load(static_cast<const T *>(g.x) + row * g.ldx, d, lane, x);
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) s += x[e];
    all.sum(s, q);
    const float m = rounded_product(s, inv);
    s = q = 0.0f;
#pragma unroll
    for (int v = 0; v < R::NV; ++v)
#pragma unroll
      for (int e = 0; e < R::V; ++e) {
        const float t = R::column(v, lane) + e < d ? x[v * R::V + e] - m : 0.0f;
        x[v * R::V + e] = t;
        s += t;
        q = fmaf(t, t, q);
      }
    all.sum(s, q);
    const float c = rounded_product(s, inv);
    float var = fmaf(-c, c, q * inv);
    var = var > 0.0f || var != var ? var : 0.0f; // (a NaN stays one)
    const float r = 1.0f / sqrtf(var + g.eps);
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = fmaf((x[e] - c) * r, w[e], b[e]);
    R::store(static_cast<T *>(g.y) + row * d, d, lane, x);
    if (g.stats && lane == 0) {
      g.stats[row] = m;
      g.stats[g.rows + row] = c;
      g.stats[2 * g.rows + row] = r;
    }
  }
}

template <typename T, typename P, int L, int EPL> __global__ __launch_bounds__(kThreads) void norm_backward_kernel(const NormArgs g) {
  using R = Row<T, P, L, EPL>;
  constexpr int TEAMS = kThreads / L, WAVES = L < 256 ? 4 : 1; // waves that hold the same columns
  __shared__ float lds[L < 256 ? 4 * (L > 64 ? 64 : L) * EPL : 16];
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const int64_t d = g.feat;
  float w[EPL], dw[EPL], db[EPL];
  R::params(static_cast<const P *>(g.weight), d, lane, 1.0f, w);
#pragma unroll
  for (int e = 0; e < EPL; ++e) dw[e] = db[e] = 0.0f;
  Team<L> all{lds};
  const float inv = 1.0f / (float)d;
  for (int64_t row = (int64_t)blockIdx.x * TEAMS + team; row < g.rows; row += (int64_t)gridDim.x * TEAMS) {
    float x[EPL], dy[EPL];
    R::load(static_cast<const T *>(g.x) + row * g.ldx, d, lane, x);
    R::load(static_cast<const T *>(g.dy) + row * d, d, lane, dy);
    const float m = g.stats[row], c = g.stats[g.rows + row], r = g.stats[2 * g.rows + row];
    float s = 0.0f, q = 0.0f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) { // (columns behind the row's end have dy = 0: their h does not count)
      const float h = ((x[e] - m) - c) * r, t = dy[e] * w[e];
      x[e] = h;
      s += t;
      q = fmaf(t, h, q);
      dw[e] = fmaf(dy[e], h, dw[e]);
      db[e] += dy[e];
      dy[e] = t;
    }
    if (!g.dx) continue; // (the parameters' gradients alone)
    all.sum(s, q);
    s *= inv;
    q *= inv;
#pragma unroll
    for (int e = 0; e < EPL; ++e) dy[e] = r * ((dy[e] - s) - x[e] * q);
    R::store(static_cast<T *>(g.dx) + row * d, d, lane, dy);
  }
  if (!g.part) return;
  float *out = g.part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float v[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
      v[e] = which ? db[e] : dw[e];
#pragma unroll
      for (int k = L; k < 64; k *= 2) v[e] += __shfl_xor(v[e], k);
    }
    if constexpr (WAVES == 1) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const int64_t col = R::column(e / R::V, lane) + e % R::V;
        if (col < d) out[which * d + col] = v[e];
      }
    } else {
      __syncthreads();
      const int wave = threadIdx.x / 64;
      if (threadIdx.x % 64 < L)
#pragma unroll
        for (int e = 0; e < EPL; ++e) lds[wave * (L * EPL) + R::column(e / R::V, lane) + e % R::V] = v[e];
      __syncthreads();
      for (int col = threadIdx.x; col < d; col += kThreads)
        out[which * d + col] = (lds[col] + lds[L * EPL + col]) + (lds[2 * L * EPL + col] + lds[3 * L * EPL + col]);
    }
  }
}

// Rows wider than a workgroup's registers (feat > 8192): the row is read again for every step (it stays in the L2).
template <typename T> __device__ inline void wide_moments(const T *row, int64_t d, Team<256> &all, float inv, float &m, float &c, float &r, float eps) {
  float s = 0.0f, q = 0.0f;
  for (int64_t i = threadIdx.x; i < d; i += kThreads) s += (float)row[i];
  all.sum(s, q);
  m = rounded_product(s, inv);
  s = q = 0.0f;
  for (int64_t i = threadIdx.x; i < d; i += kThreads) {
    const float t = (float)row[i] - m;
    s += t;
    q = fmaf(t, t, q);
  }
  all.sum(s, q);
  c = rounded_product(s, inv);
  float var = fmaf(-c, c, q * inv);
  var = var > 0.0f || var != var ? var : 0.0f;
  r = 1.0f / sqrtf(var + eps);
}
template <typename T, typename P> __global__ __launch_bounds__(kThreads) void norm_wide_kernel(const NormArgs g) {
  __shared__ float lds[16];
  Team<256> all{lds};
  const int64_t d = g.feat;
  const P *w = static_cast<const P *>(g.weight), *b = static_cast<const P *>(g.bias);
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(g.x) + row * g.ldx;
    T *y = static_cast<T *>(g.y) + row * d;
    float m, c, r;
    wide_moments(x, d, all, 1.0f / (float)d, m, c, r, g.eps);
    for (int64_t i = threadIdx.x; i < d; i += kThreads)
      y[i] = (T)fmaf((((float)x[i] - m) - c) * r, w ? (float)w[i] : 1.0f, b ? (float)b[i] : 0.0f);
    if (g.stats && threadIdx.x == 0) {
      g.stats[row] = m;
      g.stats[g.rows + row] = c;
      g.stats[2 * g.rows + row] = r;
    }
  }
}
template <typename T, typename P> __global__ __launch_bounds__(kThreads) void norm_wide_backward_kernel(const NormArgs g) {
  __shared__ float lds[16];
  Team<256> all{lds};
  const int64_t d = g.feat;
  const P *w = static_cast<const P *>(g.weight);
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(g.x) + row * g.ldx, *dy = static_cast<const T *>(g.dy) + row * d;
    T *dx = static_cast<T *>(g.dx) + row * d;
    const float m = g.stats[row], c = g.stats[g.rows + row], r = g.stats[2 * g.rows + row];
    float s = 0.0f, q = 0.0f;
    for (int64_t i = threadIdx.x; i < d; i += kThreads) {
      const float t = (float)dy[i] * (w ? (float)w[i] : 1.0f);
      s += t;
      q = fmaf(t, (((float)x[i] - m) - c) * r, q);
    }
    all.sum(s, q);
    s /= (float)d;
    q /= (float)d;
    for (int64_t i = threadIdx.x; i < d; i += kThreads) {
      const float t = (float)dy[i] * (w ? (float)w[i] : 1.0f);
      dx[i] = (T)(r * ((t - s) - (((float)x[i] - m) - c) * r * q));
    }
  }
}
// ... and their parameter gradients: a workgroup takes 256 columns of every gridDim.y-th row
template <typename T> __global__ __launch_bounds__(kThreads) void norm_wide_params_kernel(const NormArgs g) {
  const int64_t col = (int64_t)blockIdx.x * kThreads + threadIdx.x, d = g.feat;
  if (col >= d) return;
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < g.rows; row += gridDim.y) {
    const float dy = (float)static_cast<const T *>(g.dy)[row * d + col];
    dw = fmaf(dy, (((float)static_cast<const T *>(g.x)[row * g.ldx + col] - g.stats[row]) - g.stats[g.rows + row]) * g.stats[2 * g.rows + row], dw);
    db += dy;
  }
  g.part[(int64_t)blockIdx.y * 2 * d + col] = dw;
  g.part[(int64_t)blockIdx.y * 2 * d + d + col] = db;
}

// part [blocks, 2, feat] -> dweight, dbias: 16 threads a column, each every 16th block, then the 16 by halves
template <typename P> __global__ __launch_bounds__(kThreads) void norm_join_kernel(const float *part, int64_t blocks, int64_t d, P *dw, P *db) {
  __shared__ float fold[kThreads];
  const int lane = threadIdx.x % 16, way = threadIdx.x / 16;
  const int64_t i = (int64_t)blockIdx.x * 16 + lane;
  float s = 0.0f;
  if (i < 2 * d)
#pragma unroll 8
    for (int64_t b = way; b < blocks; b += 16) s += part[b * 2 * d + i];
  fold[threadIdx.x] = s;
  __syncthreads();
#pragma unroll
  for (int h = 128; h >= 16; h /= 2) {
    if ((int)threadIdx.x < h) fold[threadIdx.x] += fold[threadIdx.x + h];
    __syncthreads();
  }
  if (way == 0 && i < 2 * d) (i < d ? dw[i] : db[i - d]) = (P)fold[lane];
}

// ---- launches -----------------------------------------------------------------------------------------------------------------------
constexpr int64_t kWide = 8192; // the widest row the register kernels hold
int launched(const char *name) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return geot_internal_fail(GEOT_ELAUNCH, hipGetErrorString(e));
  if (name) geot_internal_note_kernel(name);
  return GEOT_OK;
}
// lanes of a team: the fewest that hold the row at 8 elements a lane, up to a wave; then 16 and 32 elements, then the workgroup
int64_t team_lanes(int64_t feat) { return feat <= 64 ? 8 : feat <= 128 ? 16 : feat <= 256 ? 32 : feat <= 2048 ? 64 : 256; }
int64_t backward_blocks(int64_t rows, int64_t feat) {
  if (feat > kWide) return rows < 64 ? (rows > 0 ? rows : 1) : 64; // (norm_wide_params_kernel's gridDim.y)
  const int64_t teams = kThreads / team_lanes(feat), need = (rows + teams - 1) / teams;
  const int64_t most = 2048;
  return need < 1 ? 1 : (need < most ? need : most);
}

template <typename T, typename P, int L, int EPL> void run_forward(const NormArgs &g, hipStream_t st) {
  const int64_t need = (g.rows + kThreads / L - 1) / (kThreads / L);
  hipLaunchKernelGGL((norm_kernel<T, P, L, EPL>), dim3((unsigned)(need < 8192 ? need : 8192)), dim3(kThreads), 0, st, g);
}
template <typename T, typename P, int L, int EPL> void run_backward(const NormArgs &g, hipStream_t st) {
  hipLaunchKernelGGL((norm_backward_kernel<T, P, L, EPL>), dim3((unsigned)backward_blocks(g.rows, g.feat)), dim3(kThreads), 0, st, g);
}
#define NORM_SHAPES(run)                                                                                                  \
  if (d <= 64) run<T, P, 8, 8>(g, st);                                                                                    \
  else if (d <= 128) run<T, P, 16, 8>(g, st);                                                                             \
  else if (d <= 256) run<T, P, 32, 8>(g, st);                                                                             \
  else if (d <= 512) run<T, P, 64, 8>(g, st);                                                                             \
  else if (d <= 1024) run<T, P, 64, 16>(g, st);                                                                           \
  else if (d <= 2048) run<T, P, 64, 32>(g, st);                                                                           \
  else if (d <= 4096) run<T, P, 256, 16>(g, st);                                                                          \
  else run<T, P, 256, 32>(g, st)

template <typename T, typename P> int forward(const NormArgs &g, hipStream_t st) {
  const int64_t d = g.feat;
  if (d > kWide) {
    hipLaunchKernelGGL((norm_wide_kernel<T, P>), dim3((unsigned)(g.rows < 4096 ? g.rows : 4096)), dim3(kThreads), 0, st, g);
    return launched("norm_wide_kernel");
  }
  NORM_SHAPES(run_forward);
  return launched("norm_kernel");
}
template <typename T, typename P> int backward(NormArgs &g, void *dweight, void *dbias, hipStream_t st) {
  const int64_t d = g.feat, blocks = backward_blocks(g.rows, d);
  if ((g.rows > 0 && g.dx) || g.part) {
    if (d > kWide) {
      if (g.rows > 0 && g.dx) hipLaunchKernelGGL((norm_wide_backward_kernel<T, P>), dim3((unsigned)(g.rows < 4096 ? g.rows : 4096)), dim3(kThreads), 0, st, g);
      if (g.part) hipLaunchKernelGGL((norm_wide_params_kernel<T>), dim3((unsigned)((d + kThreads - 1) / kThreads), (unsigned)blocks), dim3(kThreads), 0, st, g);
    } else {
      NORM_SHAPES(run_backward);
    }
    if (const int rc = launched("norm_backward_kernel")) return rc;
  }
  if (g.part) {
    hipLaunchKernelGGL((norm_join_kernel<P>), dim3((unsigned)((2 * d + 15) / 16)), dim3(kThreads), 0, st, g.part, blocks, d, static_cast<P *>(dweight),
                       static_cast<P *>(dbias));
    return launched(nullptr);
  }
  return GEOT_OK;
}

template <typename F> int by_type(int dtype, int param, F f) {
  if (dtype == GEOT_F32 && param == GEOT_F32) return f((float *)nullptr, (float *)nullptr);
  if (dtype == GEOT_F16 && param == GEOT_F16) return f((f16 *)nullptr, (f16 *)nullptr);
  if (dtype == GEOT_F16 && param == GEOT_F32) return f((f16 *)nullptr, (float *)nullptr);
  if (dtype == GEOT_BF16 && param == GEOT_BF16) return f((bf16 *)nullptr, (bf16 *)nullptr);
  if (dtype == GEOT_BF16 && param == GEOT_F32) return f((bf16 *)nullptr, (float *)nullptr);
  return geot_internal_fail(GEOT_EUNSUPPORTED, "layer_norm takes float32, float16 and bfloat16 rows, with parameters of that type or float32");
}
bool bad(int64_t rows, int64_t feat, int64_t ldx) {
  constexpr int64_t lim = (int64_t)1 << 34, area = (int64_t)1 << 44; // (more elements than any memory)
  return rows < 0 || feat < 0 || ldx < 0 || feat > lim || rows > area || (feat > 0 && rows > area / feat);
}

} // namespace

extern "C" {

int geot_layer_norm(const void *x, int64_t ldx, const void *weight, const void *bias, void *y, float *stats, int64_t rows, int64_t feat, float eps, int dtype,
                    int param_dtype, void *stream) {
  if (bad(rows, feat, ldx)) return geot_internal_fail(GEOT_EINVAL, "geot_layer_norm: bad size");
  if (rows == 0 || feat == 0) return GEOT_OK;
  if (!x || !y) return geot_internal_fail(GEOT_EINVAL, "geot_layer_norm: null pointer");
  NormArgs g{};
  g.x = x; g.ldx = ldx; g.weight = weight; g.bias = bias; g.y = y; g.stats = stats; g.rows = rows; g.feat = feat; g.eps = eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_type(dtype, param_dtype, [&](auto *t, auto *p) {
    return forward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(p)>>(g, st);
  });
}

size_t geot_layer_norm_backward_workspace_bytes(int64_t rows, int64_t feat) {
  if (bad(rows, feat, 0)) return 0;
  return (size_t)backward_blocks(rows, feat) * 2 * (size_t)feat * sizeof(float);
}

int geot_layer_norm_backward(const void *x, int64_t ldx, const void *weight, const float *stats, const void *dy, void *dx, void *dweight, void *dbias,
                             int64_t rows, int64_t feat, int dtype, int param_dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (bad(rows, feat, ldx) || (dweight == nullptr) != (dbias == nullptr)) return geot_internal_fail(GEOT_EINVAL, "geot_layer_norm_backward: bad argument");
  if (feat == 0) return GEOT_OK;
  if (rows > 0 && (!x || !stats || !dy)) return geot_internal_fail(GEOT_EINVAL, "geot_layer_norm_backward: null pointer");
  NormArgs g{};
  g.x = x; g.ldx = ldx; g.weight = weight; g.dy = dy; g.dx = dx; g.stats = const_cast<float *>(stats); g.rows = rows; g.feat = feat;
  if (dweight) {
    if (!workspace || workspace_bytes < geot_layer_norm_backward_workspace_bytes(rows, feat) || ((uintptr_t)workspace & 3))
      return geot_internal_fail(GEOT_EWORKSPACE, "geot_layer_norm_backward: workspace too small or misaligned");
    g.part = static_cast<float *>(workspace);
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  return by_type(dtype, param_dtype, [&](auto *t, auto *p) {
    return backward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(p)>>(g, dweight, dbias, st);
  });
}

} // extern "C"
