// dense_mm.hip -- the matrix products of a layer's node and edge rows: geot_linear, geot_segment_matmul and their gradients.
//
// One tile kernel per shape of product, on the matrix cores:
//   mm_rows_kernel     y[i, :] = act(a[i, :] . B(group of i) + bias) + residual      rows grouped by a pointer array (or one group)
//   mm_weight_kernel   dW(group) = p_rows^T q_rows, the sum running over the group's rows, split into chunks of rows
//   mm_join_kernel     adds the chunks' partial products (32 bits, in chunk order: the same bits every run)
//
// Arithmetic.  16-bit operands go to v_mfma_f32_32x32x16 as they are, sums in float32.  float32 operands are split exactly into three
// bfloat16 parts, x = x1 + x2 + x3 (8 significant bits each, round to nearest), and a product takes the six partial products whose
// weight is above 2^-24 of it: x1y1, x1y2, x2y1, x2y2, x1y3, x3y1.  What is left out (x2y3, x3y2, x3y3) is at most 2^-23 of |xy| and
// 2^-26 of it on average - below the float32 rounding of the sum itself - while the bfloat16 cores run 16 times faster than the
// float32 ones (dense peaks 2.5 PFLOP/s against 0.157): six products there cost less than half of one here.  A split of an infinity
// (inf - inf) or of a value that rounds up to one is not a number: any non-finite sum is computed again in plain
// float32 (sums_again), so infinities and NaN come out as in an ordinary float32 product.  The matrix cores read a bfloat16 below 2^-133
// as 0, so a factor below 2^-110 keeps an absolute 2^-133 instead of its last bits (float32 itself ends at 2^-149).
//
// Layout in LDS.  A tile holds chunks of 8 reduction values (16 bytes) - the operand of one MFMA lane - as
// [part][chunk][row ^ ((row >> 3) & 7)], each chunk column padded: fragment reads are contiguous, and the writes of both staging forms
// hit 8 different 16-byte banks.  An operand whose reduction index is contiguous in memory is staged chunk by chunk; one whose OUTPUT
// index is contiguous is staged in blocks of 8 reduction values by VR columns that a thread transposes in its registers, so one compute
// loop serves x W^T, dz W, and x^T dz.
//
// Tiles and what they measured.  128 rows x 128 columns (64 where there are no more, or operands are split), four waves, one LDS buffer and
// three workgroups a CU: two buffers and two workgroups were 5 to 10 % slower (64 experts f16 training 846 and 783 us).  256 x 256, eight
// waves, two buffers where the reduction is long (>= 512) and there are tiles enough: 8192 x 4096 x 4096 f16 372 -> 306 us at that step, 602
// features -> 256 157 us against 172 in tiles of 128; but not for groups below 2048 rows (experts of 512 rows: 300 us against 249 - half a
// tile is empty).  Few tiles: mm_few_rows_kernel, or shares of the reduction (rows_share).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "geot_hip.h"
#include "internal.h"

namespace {

using bf16 = __bf16;
using f16 = _Float16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8), may_alias));
typedef f16 f16x8 __attribute__((ext_vector_type(8), may_alias));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2), may_alias));

constexpr int kThreads = 256; // of the kernels beside the tile kernels

// loads and stores of 16 / 8 bytes at the element's own alignment (rows of any width, views of any offset)
template <int SIZE> struct Packed;
template <> struct Packed<2> {
  typedef u32x4 x16 __attribute__((aligned(2), may_alias));
  typedef u32x2 x8 __attribute__((aligned(2), may_alias));
};
template <> struct Packed<4> {
  typedef u32x4 x16 __attribute__((aligned(4), may_alias));
  typedef u32x2 x8 __attribute__((aligned(4), may_alias));
};
template <typename T> using Packed16 = typename Packed<sizeof(T)>::x16;
template <typename T> using Packed8 = typename Packed<sizeof(T)>::x8;

template <typename T> struct Elem;
template <> struct Elem<bf16> {
  static constexpr int PARTS = 1, BK = 64;
  typedef bf16x8 Frag;
  static __device__ f32x16 mfma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<f16> {
  static constexpr int PARTS = 1, BK = 64;
  typedef f16x8 Frag;
  static __device__ f32x16 mfma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<float> {
  static constexpr int PARTS = 3, BK = 32;
  typedef bf16x8 Frag;
  static __device__ f32x16 mfma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

template <typename T> __device__ inline float as_float(T v) { return (float)v; }

__device__ inline int swizzled(int row) { return row ^ ((row >> 3) & 7); }

// ---- a tile of R rows (output index) by BK reduction values -------------------------------------------------------------------
template <typename T, int R> struct Tile {
  using E = Elem<T>;
  static constexpr int CK = E::BK / 8;        // chunks along the reduction
  static constexpr int PAD = 8 / CK;          // chunk columns 16 * PAD bytes apart in their banks
  static constexpr int COL = R + PAD;         // 16-byte slots of a chunk column
  static constexpr int BYTES = E::PARTS * CK * COL * 16;
  static __device__ int slot(int part, int chunk, int row) { return (part * CK + chunk) * COL + swizzled(row); }
};

// three bfloat16 parts of 8 floats
__device__ inline void split8(const float (&v)[8], bf16x8 (&p)[3]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bf16 a = (bf16)v[j];
    const float r = v[j] - (float)a;
    const bf16 b = (bf16)r;
    p[0][j] = a;
    p[1][j] = b;
    p[2][j] = (bf16)(r - (float)b);
  }
}

// Staging, reduction index contiguous: element (row, k) at base[row * ld + k].
template <typename T, int R, int NT> struct StageK {
  using E = Elem<T>;
  using L = Tile<T, R>;
  static constexpr int N = (R * L::CK + NT - 1) / NT;
  static constexpr bool WHOLE = (R * L::CK) % NT == 0;
  static constexpr int W = 8 * sizeof(T) / 16; // 16-byte pieces of a chunk
  u32x4 reg[N][W];
  const T *base;
  int64_t ld;
  int rows;     // rows that exist (>= 1); the others read the last one and are not stored
  int64_t k_end;

  __device__ void open(const T *b, int64_t ld_, int64_t first, int64_t rows_left, int64_t k_begin, int64_t k_end_) {
    ld = ld_;
    rows = (int)(rows_left < R ? rows_left : R);
    base = b + first * ld_ + k_begin;
    k_end = k_end_ - k_begin;
  }
  __device__ bool fast() const { return true; }
  // a whole step (k0 + BK <= k_end)
  __device__ void load_fast(int64_t k0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * NT, row = idx / L::CK;
      const T *p = base + (row < rows ? row : rows - 1) * ld + k0 + idx % L::CK * 8;
#pragma unroll
      for (int w = 0; w < W; ++w) reg[i][w] = reinterpret_cast<const Packed16<T> *>(p)[w];
    }
  }
  __device__ void load_any(int64_t k0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * NT, row = idx / L::CK;
      const int64_t k = k0 + idx % L::CK * 8;
      const T *p = base + (row < rows ? row : rows - 1) * ld + k;
      if (k + 8 <= k_end) {
#pragma unroll
        for (int w = 0; w < W; ++w) reg[i][w] = reinterpret_cast<const Packed16<T> *>(p)[w];
      } else {
        alignas(16) T tmp[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) tmp[j] = k + j < k_end ? p[j] : (T)0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) reg[i][w] = reinterpret_cast<const u32x4 *>(tmp)[w];
      }
    }
  }
  __device__ void store(char *lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * NT;
      if (!WHOLE && idx >= R * L::CK) continue;
      const int chunk = idx % L::CK, row = idx / L::CK;
      if constexpr (E::PARTS == 1) {
        reinterpret_cast<u32x4 *>(lds)[L::slot(0, chunk, row)] = reg[i][0];
      } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(reg[i][j / 4][j % 4]);
        bf16x8 p[3];
        split8(v, p);
#pragma unroll
        for (int s = 0; s < 3; ++s) reinterpret_cast<bf16x8 *>(lds)[L::slot(s, chunk, row)] = p[s];
      }
    }
  }
};

// Staging, output index contiguous: element (row, k) at base[k * ld + row], transposed in registers.  SUM: also adds up what it stages, per row.
template <typename T, int R, int NT, bool SUM, int LOAD = 8> struct StageR {
  using E = Elem<T>;
  using L = Tile<T, R>;
  static constexpr int VR = LOAD / sizeof(T), PW = LOAD / 4; // rows of a thread's block: LOAD bytes
  using Piece = typename std::conditional<PW == 4, Packed16<T>, Packed8<T>>::type;
  using Words = typename std::conditional<PW == 4, u32x4, u32x2>::type;
  static constexpr int BLOCKS = (R / VR) * L::CK;
  static constexpr int N = (BLOCKS + NT - 1) / NT;
  static constexpr bool WHOLE = BLOCKS % NT == 0;
  Words reg[N][8] = {};
  float sum[SUM ? N : 1][VR];
  const T *base;
  int64_t ld, k_end;
  int rows;
  bool add = false; // (SUM: this workgroup is the one that adds them up)

  __device__ void open(const T *b, int64_t ld_, int64_t first, int64_t rows_left, int64_t k_begin, int64_t k_end_) {
    ld = ld_;
    rows = (int)(rows_left < R ? rows_left : R);
    base = b + k_begin * ld_ + first;
    k_end = k_end_ - k_begin;
    if constexpr (SUM) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < VR; ++j) sum[i][j] = 0.0f;
    }
  }
  // columns behind the last one are never stored: a block that lies behind reads the last whole one instead, which needs the width
  // (of an edge tile) to be whole blocks
  __device__ bool fast() const { return rows == R || (rows % VR == 0 && rows > 0); }
  __device__ void load_fast(int64_t k0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * NT, row = (idx % (R / VR)) * VR, chunk = idx / (R / VR);
      if (!WHOLE && idx >= BLOCKS) continue; // (whole waves)
      const T *p = base + (k0 + chunk * 8) * ld + (row + VR <= rows ? row : rows - VR);
#pragma unroll
      for (int j = 0; j < 8; ++j) reg[i][j] = *reinterpret_cast<const Piece *>(p + j * ld);
    }
  }
  __device__ void load_any(int64_t k0, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * NT, row = (idx % (R / VR)) * VR, chunk = idx / (R / VR);
      if (!WHOLE && idx >= BLOCKS) continue;
      const T *p = base + (k0 + chunk * 8) * ld + row;
      const bool wide = row + VR <= rows;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t k = k0 + chunk * 8 + j;
        Words v = {};
        if (k < k_end && wide) {
          v = *reinterpret_cast<const Piece *>(p + j * ld);
        } else if (k < k_end && row < rows) {
          alignas(16) T tmp[VR];
#pragma unroll
          for (int r = 0; r < VR; ++r) tmp[r] = row + r < rows ? p[j * ld + r] : (T)0.0f;
          v = *reinterpret_cast<const Words *>(tmp);
        }
        reg[i][j] = v;
      }
    }
  }
  __device__ float value(int i, int j, int r) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(reg[i][j][r]);
    } else {
      const uint32_t half = (r & 1) ? reg[i][j][r / 2] >> 16 : reg[i][j][r / 2] & 0xffffu;
      return (float)__builtin_bit_cast(T, (uint16_t)half);
    }
  }
  __device__ void store(char *lds, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int idx = tid + i * NT;
      const int row = (idx % (R / VR)) * VR, chunk = idx / (R / VR);
      if (WHOLE || idx < BLOCKS) {
#pragma unroll
        for (int r = 0; r < VR; ++r) {
          if constexpr (E::PARTS == 1) {
            u32x4 out; // two of 8 reduction values a word: the halves of two neighbouring loads
#pragma unroll
            for (int j = 0; j < 4; ++j)
              out[j] = __builtin_amdgcn_perm(reg[i][2 * j + 1][r / 2], reg[i][2 * j][r / 2], (r & 1) ? 0x07060302u : 0x05040100u);
            reinterpret_cast<u32x4 *>(lds)[L::slot(0, chunk, row + r)] = out;
          } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = value(i, j, r);
            bf16x8 p[3];
            split8(v, p);
#pragma unroll
            for (int s = 0; s < 3; ++s) reinterpret_cast<bf16x8 *>(lds)[L::slot(s, chunk, row + r)] = p[s];
          }
        }
      }
      if constexpr (SUM) {
        if (add) {
#pragma unroll
          for (int r = 0; r < VR; ++r)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[i][r] += value(i, j, r);
        }
      }
    }
  }
};

// Both operands of that form, in tiles of R rows: one half of the threads stages A, the other B, each with 16-byte loads (64 experts,
// 1024 -> 2048 f16, the weight's gradient: 360 us with every thread loading 8 bytes of both).
template <typename T, int R, int NT, bool SUM> struct StagePair {
  StageR<T, R, NT / 2, SUM, 16> st;
  bool both;
  __device__ bool fast() const { return both; }
  __device__ void load_fast(int64_t k0, int tid) { st.load_fast(k0, tid % (NT / 2)); }
  __device__ void load_any(int64_t k0, int tid) { st.load_any(k0, tid % (NT / 2)); }
  __device__ void store(char *lds, int tid) { st.store(lds + tid / (NT / 2) * Tile<T, R>::BYTES, tid % (NT / 2)); }
};
struct StageNone {
  __device__ bool fast() const { return true; }
  __device__ void load_fast(int64_t, int) {}
  __device__ void load_any(int64_t, int) {}
  __device__ void store(char *, int) {}
};

__device__ inline bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
template <typename P> __device__ inline P *pointer_of_lane(P *p, int lane) {
  const uint64_t v = reinterpret_cast<uint64_t>(p);
  return reinterpret_cast<P *>(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}
// A lane's sum that came out non-finite again, in plain float32: the way of an infinity, a NaN or an overflow through a product of split
// operands.  a[i * stride_a] times b[i * stride_b], i < k; every active lane of the wave takes part, `bad` or not.  A lane walks its first 64
// terms alone, which ends most NaN; longer reductions go to the whole wave one after the other, every lane taking each n-th term (one
// infinity in a column of x makes every output's sum over that column's rows non-finite, and a chunk of rows can be all of them: 4096 x 4096
// weights, 30,000 rows, their gradient 27 ms with one, 7.7 without; lane by lane alone 93).  Fixed order: the same bits every run.
// A function of its own: inlined, its registers spilled others around the tile kernels' loops (typed nodes f32, x W 81 -> 88 us; 85 so).
__device__ __attribute__((noinline)) float sum_again(float v, bool bad, const float *a, int64_t stride_a, const float *b, int64_t stride_b, int64_t k) {
  constexpr int64_t kAlone = 64;
  constexpr int U = 8; // terms of a lane in flight
  bool left = false;
  if (bad) {
    const int64_t alone = k < kAlone ? k : kAlone;
    v = 0.0f;
    for (int64_t i = 0; i < alone && v == v; ++i) v = fmaf(a[i * stride_a], b[i * stride_b], v);
    left = k > kAlone && v == v;
  }
  const int lane = threadIdx.x % 64;
  const uint64_t on = __ballot(true);
  const int64_t helpers = __popcll(on), rank = __popcll(on & (((uint64_t)1 << lane) - 1));
  for (uint64_t todo = __ballot(left); todo; todo &= todo - 1) {
    const int src = __builtin_ctzll(todo);
    const float *pa = pointer_of_lane(a, src), *pb = pointer_of_lane(b, src);
    float s = 0.0f;
    for (int64_t i = rank; i < k; i += U * helpers) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = i + u * helpers;
        if (j < k) s = fmaf(pa[j * stride_a], pb[j * stride_b], s);
      }
      if (__ballot(s != s)) break;
    }
    float total = 0.0f;
    for (uint64_t h = on; h; h &= h - 1) total += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s), __builtin_ctzll(h)));
    v = lane == src ? total : v;
  }
  return v;
}
// ... of V elements a lane, b's `next` apart
template <int V>
__device__ inline void sums_again(float (&v)[V], int cols, const float *a, int64_t stride_a, const float *b, int64_t stride_b, int64_t next, int64_t k) {
  bool any = false;
#pragma unroll
  for (int c = 0; c < V; ++c) any |= c < cols && !finite(v[c]);
  if (__ballot(any) == 0) return;
#pragma unroll 1
  for (int c = 0; c < V; ++c) {
    float one = v[0];
#pragma unroll
    for (int e = 1; e < V; ++e) one = c == e ? v[e] : one;
    one = sum_again(one, c < cols && !finite(one), a, stride_a, b + c * next, stride_b, k);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = c == e ? one : v[e];
  }
}

// ---- the products of one staged pair of tiles -----------------------------------------------------------------------------------
// WM x WN waves over a BM x BN tile
template <typename T, int BM, int BN, int WM, int WN> struct Accum {
  using E = Elem<T>;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32; // 32 x 32 fragments of a wave
  f32x16 acc[FM][FN];

  __device__ void clear() {
    zero(acc);
  }
  // into: acc, or for split operands a sum of their own (add) - the six partial products of 16 reduction values, smallest first, so that
  // the long sum rounds once for a whole step (added to it one by one, K = 4048 came out 1.0e-6 off where a float32 product is 0.6e-6)
  __device__ static void products(f32x16 (&into)[FM][FN], const typename E::Frag (&a)[E::PARTS][FM], const typename E::Frag (&b)[E::PARTS][FN]) {
    constexpr int NP = E::PARTS == 1 ? 1 : 6;
    constexpr int PA[6] = {E::PARTS == 1 ? 0 : 2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) into[i][j] = E::mfma(a[PA[p]][i], b[PB[p]][j], into[i][j]);
  }
  static __device__ void zero(f32x16 (&t)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) t[i][j][e] = 0.0f;
  }
  __device__ void add(const f32x16 (&t)[FM][FN]) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] += t[i][j][e];
  }
  __device__ void step(const char *la, const char *lb, int wm, int wn, int lane) {
    if constexpr (E::PARTS == 1) {
      staged(acc, la, lb, wm, wn, lane);
    } else {
      f32x16 t[FM][FN];
      zero(t);
      staged(t, la, lb, wm, wn, lane);
      add(t);
    }
  }
  static __device__ void staged(f32x16 (&into)[FM][FN], const char *la, const char *lb, int wm, int wn, int lane) {
    using F = typename E::Frag;
    using LA = Tile<T, BM>;
    using LB = Tile<T, BN>;
#pragma unroll
    for (int s = 0; s < E::BK / 16; ++s) {
      const int chunk = 2 * s + lane / 32;
      F a[E::PARTS][FM], b[E::PARTS][FN];
#pragma unroll
      for (int p = 0; p < E::PARTS; ++p) {
#pragma unroll
        for (int i = 0; i < FM; ++i) a[p][i] = reinterpret_cast<const F *>(la)[LA::slot(p, chunk, wm * (BM / WM) + i * 32 + lane % 32)];
#pragma unroll
        for (int j = 0; j < FN; ++j) b[p][j] = reinterpret_cast<const F *>(lb)[LB::slot(p, chunk, wn * (BN / WN) + j * 32 + lane % 32)];
      }
      products(into, a, b);
    }
  }
  // element e of a fragment: row 8 * (e / 4) + 4 * (lane / 32) + e % 4, column lane % 32
  static __device__ int row_of(int e, int lane) { return 8 * (e / 4) + 4 * (lane / 32) + e % 4; }
  // row block i of every wave -> lds[32 * WM][BN + 4] floats (rows wm * 32 + ..); row lr of it is row tile_row(lr, i) of the tile
  __device__ void put(float *lds, int i, int wm, int wn, int lane) const {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) lds[(wm * 32 + row_of(e, lane)) * (BN + 4) + wn * (BN / WN) + j * 32 + lane % 32] = acc[i][j][e];
  }
  static __device__ int tile_row(int lr, int i) { return (lr / 32) * (BM / WM) + i * 32 + lr % 32; }
  // Non-finite sums among those that this wave has put there, computed again (sum_again).  Element (row, col) of the tile: a + row * row_a,
  // b + col * col_b, for rows < `rows`, columns < `cols`.
  __device__ void again(float *lds, int i, int wm, int wn, int lane, const float *a, int64_t row_a, int64_t stride_a, const float *b, int64_t col_b, int64_t stride_b,
                        int rows, int cols, int64_t k) const {
    float any = 0.0f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) any = fmaf(acc[i][j][e], 0.0f, any);
    if (__ballot(any != 0.0f) == 0) return; // (0, or NaN)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // (the wave's own lanes wrote what is read here)
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int at = lane; at < 32 * (BN / WN); at += 64) {
      const int lr = wm * 32 + at / (BN / WN), col = wn * (BN / WN) + at % (BN / WN), row = tile_row(lr, i);
      float &v = lds[lr * (BN + 4) + col];
      const bool bad = row < rows && col < cols && !finite(v);
      if (__ballot(bad) == 0) continue;
      v = sum_again(v, bad, a + row * row_a, stride_a, b + col * col_b, stride_b, k);
    }
  }
};

// max(z, 0) as a half sum: +inf and NaN stay, -inf becomes NaN (as -inf * 0 does)
__device__ inline float positive_part(float z) { return fmaf(0.5f, fabsf(z), 0.5f * z); }

// The normal distribution's tail, Phi(-a) = exp(-a^2 / 2) R(a) for a >= 0: R is smooth (Mills' ratio times the density's constant) and
// is taken as a polynomial in t = 1 / (1 + 0.26 a), fitted by least squares reweighted to equal ripple on [0, 14.2] (3e-8; 4e-7 with its
// float32 rounding).  The same exponential serves the density in the slope.  erfcf + expf instead bound the kernels by their vector
// instructions: a gelu layer of 2.4 M x 128 -> 256 bf16 took 1527 us forward and 1064 us for its dz, 640 and 760 us of memory time.
struct Normal {
  float tail, bell; // Phi(-|z|), exp(-z^2 / 2)
};
__device__ inline Normal normal_of(float z) {
  // (exp(-200) is 0 in float32, nothing changes behind 20 but inf - inf below; a NaN goes on in the caller's z)
  const float a = fminf(fabsf(z), 20.0f);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.26f, a, 1.0f));
  constexpr float half_log2e = 0.72134752044448170f;
  const float sq = a * a, arg = sq * half_log2e;
  float bell = __builtin_amdgcn_exp2f(-arg);
  // what the two products above rounded away (up to 24 x 2^-24 in the argument)
  const float rest = fmaf(sq, half_log2e, -arg) + fmaf(a, a, -sq) * half_log2e;
  bell = fmaf(bell * rest, -0.69314718055994531f, bell);
  float r = 0.030395518988370895f;
  r = fmaf(r, t, -0.15229645371437073f);
  r = fmaf(r, t, 0.25038889050483704f);
  r = fmaf(r, t, -0.14968349039554596f);
  r = fmaf(r, t, 0.160069078207016f);
  r = fmaf(r, t, 0.051404859870672226f);
  r = fmaf(r, t, 0.10293274372816086f);
  r = fmaf(r, t, 0.10303061455488205f);
  r = fmaf(r, t, 0.10375823080539703f);
  return {r * t * bell, bell};
}
// 16-bit results: fewer instructions (the exact form's 25 an element were 610 us of vector time in the layer above).  log2 Phi(-a) is close
// to a parabola: a polynomial in the exponent, of degree 7 for float16 (2^-17 of the value up to a = 5.8; behind that it rounds to 0) and 9
// for bfloat16, whose range holds Phi down to 2^-126 (2^-15 up to a = 10, 2^-13.8 up to 12.9, 0 behind).  Degree 7 for both was 27 %
// off at -12.
template <typename T> __device__ inline float gelu16(float z) {
  const float a = fminf(fabsf(z), 16.0f);
  float p;
  if constexpr (std::is_same<T, f16>::value) {
    p = 1.7826165503720404e-06f;
    p = fmaf(p, a, -6.053628749214113e-05f);
    p = fmaf(p, a, 0.0009219465428031981f);
    p = fmaf(p, a, -0.008472956717014313f);
    p = fmaf(p, a, 0.053884927183389664f);
    p = fmaf(p, a, 0.4585457146167755f);
    p = fmaf(p, a, 1.1512134075164795f);
  } else {
    p = 1.8970891524361377e-09f;
    p = fmaf(p, a, -1.3898932138545206e-07f);
    p = fmaf(p, a, 4.4754006012226455e-06f);
    p = fmaf(p, a, -8.38298219605349e-05f);
    p = fmaf(p, a, 0.0010227881139144301f);
    p = fmaf(p, a, -0.008678584359586239f);
    p = fmaf(p, a, 0.05400051549077034f);
    p = fmaf(p, a, 0.45869940519332886f);
    p = fmaf(p, a, 1.1510733366012573f);
  }
  p = fmaf(p, a, 1.0f);
  return fmaf(-a, __builtin_amdgcn_exp2f(-p), positive_part(z)); // max(z, 0) - a Phi(-a)
}
// gelu'(-a) = exp(-a^2 / 2) (R(a) - a / sqrt(2 pi)), gelu'(z) + gelu'(-z) = 1, R as in normal_of, of degree 5 in t = 1 / (1 + 0.35 a): 2^-16
// of the slope up to a = 13.3, and below 2^-18 absolute around its zero at -0.75.  (A polynomial of degree 7 in a for the whole bracket held
// 2^-15 absolute only: 0.7 % off at -4, 120 times the slope at -14.)
__device__ inline float gelu_slope16(float z) {
  const float a = fminf(fabsf(z), 16.0f);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, a, 1.0f));
  float q = -0.09688097983598709f;
  q = fmaf(q, t, 0.2732522487640381f);
  q = fmaf(q, t, 0.02117534540593624f);
  q = fmaf(q, t, 0.1652262806892395f);
  q = fmaf(q, t, 0.13722974061965942f);
  q = fmaf(-0.39894228040143268f, a, q * t);
  q *= __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  return z < 0.0f ? q : 1.0f - q;
}
template <bool EXACT> __device__ inline float logistic(float z) {
  constexpr float log2e = 1.44269504088896341f;
  const float arg = z * log2e;
  float e = __builtin_amdgcn_exp2f(-arg);
  if constexpr (EXACT) {
    const float rest = fmaf(z, log2e, -arg);
    if (fabsf(z) < 80.0f) e = fmaf(e * rest, -0.69314718055994531f, e);
  }
  return __builtin_amdgcn_rcpf(1.0f + e);
}
// ACT is a compile-time choice inside the loops over elements.  T: float operands take the exact forms.
// At the infinities: values as the formula gives them (z Phi(z), z / (1 + exp(-z)): +inf, and NaN at -inf), slopes as their limits (1 and 0) -
// a z saved in float16 is infinite from 65520 on, where the value that was passed on can be an ordinary 0.
template <typename T, int ACT> __device__ inline float activate(float z) {
  if constexpr (ACT == GEOT_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  else if constexpr (ACT == GEOT_ACT_GELU && sizeof(T) == 2) return gelu16<T>(z);
  else if constexpr (ACT == GEOT_ACT_GELU) { // z Phi(z) = max(z, 0) - |z| Phi(-|z|); behind 20 the tail is 0, and no infinity may meet it
    return fmaf(-fminf(fabsf(z), 20.0f), normal_of(z).tail, positive_part(z));
  }
  else if constexpr (ACT == GEOT_ACT_SILU) return z * logistic<sizeof(T) == 4>(z);
  else return z;
}
template <typename T, int ACT> __device__ inline float activation_slope(float z) {
  if constexpr (ACT == GEOT_ACT_GELU && sizeof(T) == 2) return gelu_slope16(z);
  else if constexpr (ACT == GEOT_ACT_GELU) {
    const Normal n = normal_of(z);
    const float c = fminf(fmaxf(z, -20.0f), 20.0f), s = fmaf(c * 0.39894228040143268f, n.bell, z < 0.0f ? n.tail : 1.0f - n.tail);
    return z != z ? z : s;
  } else if constexpr (ACT == GEOT_ACT_SILU) {
    const float s = logistic<sizeof(T) == 4>(z), c = fminf(fmaxf(z, -128.0f), 128.0f); // (s is 0 or 1 behind; a NaN stays in s)
    return s * fmaf(c, 1.0f - s, 1.0f);
  } else return 1.0f;
}
// dy act'(z).  relu's is a choice, not a product: where it is off, an infinite or NaN dy (a masked place) does not come through.
template <typename T, int ACT> __device__ inline float activation_gradient(float dy, float z) {
  if constexpr (ACT == GEOT_ACT_RELU) return z > 0.0f ? dy : (z != z ? z : 0.0f);
  else return dy * activation_slope<T, ACT>(z);
}
template <int V> using Const = std::integral_constant<int, V>;
template <bool ANY = true, typename F> __device__ __host__ inline void by_activation(int act, F f) {
  if constexpr (!ANY) return f(Const<GEOT_ACT_NONE>());
  switch (act) {
  case GEOT_ACT_RELU: f(Const<GEOT_ACT_RELU>()); break;
  case GEOT_ACT_GELU: f(Const<GEOT_ACT_GELU>()); break;
  case GEOT_ACT_SILU: f(Const<GEOT_ACT_SILU>()); break;
  default: f(Const<GEOT_ACT_NONE>());
  }
}

// ---- groups of rows --------------------------------------------------------------------------------------------------------------
// Rows are cut at the boundaries q_0 = 0, q_1 = ptr[0], ..., q_{G+1} = ptr[G], q_{G+2} = rows (each clamped into [0, rows]): G groups,
// and the rows in front of and behind them, whose results are zero.  Piece j starts at slot floor(q_j / unit) + j of the launch (unit a power of two): that
// leaves it at least ceil(len / unit) slots and makes the slot of a workgroup a search in ptr - no scan, no table, no second
// launch; at most G + 2 slots stay empty.  Without a pointer array there is one group, all rows.
struct Groups {
  const int64_t *ptr;
  int64_t groups, rows;
  __device__ int64_t bound(int64_t j) const { // q_j
    if (j <= 0) return 0;
    if (j >= groups + 2) return rows;
    const int64_t q = ptr[j - 1];
    return q < 0 ? 0 : (q > rows ? rows : q);
  }
};
struct Piece {
  int64_t group;      // 0 .. G-1; -1: rows outside every group
  int64_t begin, end; // the piece's rows
  int64_t index;      // which unit of the piece this slot is (may lie behind its end)
  int64_t start;      // the piece's first slot
};
// one value of the wave in scalar registers (the compiler cannot see that what depends on it is uniform)
__device__ inline int64_t uniform(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
// The last piece whose first slot is <= slot, found 64 candidates a step (one a lane): a binary search's chain of dependent loads was
// several microseconds of every workgroup.  Every lane of the wave takes part.
__device__ inline Piece piece_of(const Groups &g, int unit_log2, int64_t slot) {
  if (!g.ptr) return {0, 0, g.rows, slot, 0};
  const int lane = threadIdx.x % 64;
  int64_t lo = 0, len = g.groups + 2;
  while (len > 1) {
    const int64_t step = (len + 63) >> 6, at = lane * step;
    const bool ok = at < len && (g.bound(lo + at) >> unit_log2) + lo + at <= slot;
    int count = __popcll(__ballot(ok));
    count = count > 0 ? count : 1;
    lo = uniform(lo + (count - 1) * step);
    len = uniform(len - (count - 1) * step);
    len = len < step ? len : step;
  }
  const int64_t q0 = uniform(g.bound(lo)), q1 = uniform(g.bound(lo + 1)), start = (q0 >> unit_log2) + lo;
  if (slot < start) return {-1, 0, 0, 0, 0}; // (only where ptr does not ascend: no rows)
  return {lo >= 1 && lo <= g.groups ? lo - 1 : -1, q0, q1, slot - start, start};
}
int64_t slots_of(int64_t rows, int64_t groups, bool with_ptr, int64_t unit) {
  if (!with_ptr) return (rows + unit - 1) / unit;
  return rows / unit + groups + 2;
}

// Workgroups go to the 8 XCDs round robin; tiles that share an operand should share an L2: XCD x takes the x-th eighth of the tiles.
// (32 bits from here to the tile: a launch has fewer than 2^24 workgroups, and a 64-bit division is some 140 instructions.)
__device__ inline uint32_t xcd_contiguous(uint32_t block, uint32_t blocks) {
  const uint32_t x = block % 8, q = blocks / 8, r = blocks % 8;
  return x * q + (x < r ? x : r) + block / 8;
}

// The reduction: the next step's operands are on their way from memory while this one's are multiplied.  NBUF 2: a barrier a step.
// Whole steps run in a loop of their own: with both forms of a load behind one branch the compiler waits for the first operand's loads
// before it issues the second's (64 experts' weight gradient: 480 us, see the kernel).
template <typename T, int BM, int BN, int WM, int WN, int NBUF, typename SA, typename SB>
__device__ inline void staged_products(SA &sa, SB &sb, Accum<T, BM, BN, WM, WN> &acc, char *lds, int64_t k_len, int tid, int wm, int wn, int lane) {
  constexpr int A_BYTES = Tile<T, BM>::BYTES, STAGE = A_BYTES + Tile<T, BN>::BYTES, BK = Elem<T>::BK;
  if (k_len <= 0) return;
  const int tb = (tid + 32 * WM * WN) % (64 * WM * WN); // (where a tile is fewer blocks than threads, the other half of them stages B)
  const int64_t k_fast = sa.fast() && sb.fast() ? k_len : 0; // steps that end at or in front of it take load_fast
  if (BK <= k_fast) {
    sa.load_fast(0, tid);
    sb.load_fast(0, tb);
  } else {
    sa.load_any(0, tid);
    sb.load_any(0, tb);
  }
  int64_t k0 = 0;
  if constexpr (NBUF == 2) {
    sa.store(lds, tid);
    sb.store(lds + A_BYTES, tb);
    if (2 * BK <= k_fast) {
      sa.load_fast(BK, tid);
      sb.load_fast(BK, tb);
    } else if (BK < k_len) {
      sa.load_any(BK, tid);
      sb.load_any(BK, tb);
    }
    __syncthreads();
    char *now = lds, *next = lds + STAGE;
    auto turn = [&] {
      __syncthreads();
      char *t = now;
      now = next;
      next = t;
    };
    for (; k0 + 3 * BK <= k_fast; k0 += BK) {
      acc.step(now, now + A_BYTES, wm, wn, lane);
      sa.store(next, tid);
      sb.store(next + A_BYTES, tb);
      sa.load_fast(k0 + 2 * BK, tid);
      sb.load_fast(k0 + 2 * BK, tb);
      turn();
    }
    for (; k0 < k_len; k0 += BK) {
      acc.step(now, now + A_BYTES, wm, wn, lane);
      if (k0 + BK < k_len) {
        sa.store(next, tid);
        sb.store(next + A_BYTES, tb);
        if (k0 + 2 * BK < k_len) {
          sa.load_any(k0 + 2 * BK, tid);
          sb.load_any(k0 + 2 * BK, tb);
        }
      }
      turn();
    }
  } else {
    for (; k0 + 2 * BK <= k_fast; k0 += BK) {
      sa.store(lds, tid);
      sb.store(lds + A_BYTES, tb);
      sa.load_fast(k0 + BK, tid);
      sb.load_fast(k0 + BK, tb);
      __syncthreads();
      acc.step(lds, lds + A_BYTES, wm, wn, lane);
      __syncthreads();
    }
    for (; k0 < k_len; k0 += BK) {
      sa.store(lds, tid);
      sb.store(lds + A_BYTES, tb);
      if (k0 + BK < k_len) {
        sa.load_any(k0 + BK, tid);
        sb.load_any(k0 + BK, tb);
      }
      __syncthreads();
      acc.step(lds, lds + A_BYTES, wm, wn, lane);
      __syncthreads();
    }
  }
}

struct RowsArgs {
  const void *a, *b, *bias, *residual;
  void *z, *y;
  int64_t lda, ldb, ldr, ldy, b_group, bias_group; // strides in elements
  Groups groups;
  int64_t n, k;
  uint32_t slots, tiles_n, band; // band: row tiles of a group of tiles (tile_of)
  int act;
  float *part;     // partial sums of gridDim.y shares of the reduction, k_share values each: [shares][rows][n]
  int64_t k_share;
};

// V consecutive columns of a row, `cols` of which exist
template <typename T, int V> __device__ inline u32x4 load_cols(const T *p, int cols) {
  if (cols == V) return *reinterpret_cast<const Packed16<T> *>(p);
  alignas(16) T tmp[V];
#pragma unroll
  for (int c = 0; c < V; ++c) tmp[c] = c < cols ? p[c] : (T)0.0f;
  return *reinterpret_cast<const u32x4 *>(tmp);
}
template <typename T, int V> __device__ inline void store_cols(T *p, int cols, const float (&v)[V]) {
  alignas(16) T tmp[V];
#pragma unroll
  for (int c = 0; c < V; ++c) tmp[c] = (T)v[c];
  if (cols == V) *reinterpret_cast<Packed16<T> *>(p) = *reinterpret_cast<const u32x4 *>(tmp);
  else
#pragma unroll
    for (int c = 0; c < V; ++c)
      if (c < cols) p[c] = tmp[c];
}
// What becomes of a row's sums.  DZ false: y = act(z) + residual, z stored if asked for; `ext` is the residual's row.  DZ true:
// dz = dy act'(z), added up per column; `ext` is dy's.
template <typename T, int V, int ACT, bool DZ>
__device__ inline void finish_row(const RowsArgs &g, int64_t row, int64_t col, int cols, float (&v)[V], const float (&bias)[V], bool has_ext, u32x4 ext, float (&sum)[V]) {
  alignas(16) T tmp[V];
  *reinterpret_cast<u32x4 *>(tmp) = ext;
#pragma unroll
  for (int c = 0; c < V; ++c) v[c] += bias[c];
  if constexpr (DZ) {
#pragma unroll
    for (int c = 0; c < V; ++c) {
      v[c] = activation_gradient<T, ACT>(as_float(tmp[c]), v[c]);
      sum[c] += v[c];
    }
  } else {
    if (g.z) store_cols<T, V>(static_cast<T *>(g.z) + row * g.n + col, cols, v);
#pragma unroll
    for (int c = 0; c < V; ++c) v[c] = activate<T, ACT>(v[c]);
    if (has_ext) {
#pragma unroll
      for (int c = 0; c < V; ++c) v[c] += as_float(tmp[c]);
    }
  }
  store_cols<T, V>(static_cast<T *>(g.y) + row * g.ldy + col, cols, v);
}

// A finished tile: 32 * WM rows at a time through LDS, so that every access to memory is whole rows, V consecutive columns a thread.  What
// is read beside the sums (the residual, dy) is on its way before the barriers.  g.a and B: the operands of sums_again.
template <typename T, int BM, int BN, int WM, int WN, int ACT, bool DZ, bool BR>
__device__ inline void tile_epilogue(const RowsArgs &g, const Accum<T, BM, BN, WM, WN> &acc, float *out, const T *ext, int64_t ld_ext, const T *B, int64_t r0, int64_t rows,
                                     int64_t nc, int cols, int64_t k_len, const float (&bias)[16 / sizeof(T)], float (&sum)[16 / sizeof(T)], int tid, int wm, int wn, int lane) {
  constexpr int NT = 64 * WM * WN, V = 16 / sizeof(T), TPR = BN / V, RPP = NT / TPR, PASSES = 32 * WM / RPP;
  const int col = (tid % TPR) * V;
#pragma unroll
  for (int i = 0; i < acc.FM; ++i) {
    u32x4 pre[PASSES];
    if (ext && cols > 0) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int64_t tr = acc.tile_row(tid / TPR + p * RPP, i), row = r0 + (tr < rows ? tr : rows - 1);
        pre[p] = load_cols<T, V>(ext + row * ld_ext + nc, cols);
      }
    }
    if (i) __syncthreads();
    acc.put(out, i, wm, wn, lane);
    if constexpr (Elem<T>::PARTS == 3) {
      const int64_t n0 = nc - col;
      acc.again(out, i, wm, wn, lane, static_cast<const float *>(g.a) + r0 * g.lda, g.lda, 1, reinterpret_cast<const float *>(B) + (BR ? n0 : n0 * g.ldb), BR ? 1 : g.ldb,
                BR ? g.ldb : 1, (int)rows, (int)(g.n - n0 < BN ? g.n - n0 : BN), k_len);
    }
    __syncthreads();
    if (cols > 0) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int lr = tid / TPR + p * RPP;
        const int64_t tr = acc.tile_row(lr, i), row = r0 + tr;
        if (tr >= rows) continue;
        float v[V];
#pragma unroll
        for (int c = 0; c < V; c += 4) {
          const f32x4 q = *reinterpret_cast<const f32x4 *>(out + lr * (BN + 4) + col + c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[c + e] = q[e];
        }
        finish_row<T, V, ACT, DZ>(g, row, nc, cols, v, bias, ext != nullptr, pre[p], sum);
      }
    }
  }
}

// A workgroup's tile: groups of 8 row tiles, inside a group the column tiles one after the other with the 8 row tiles fastest - what runs
// at one time on an XCD shares both operands (8 + 8 panels for 64 tiles instead of 2 + 32 in plain order at 32 column tiles).
// Groups of rows (ptr) keep the plain order: row tiles side by side rarely share a matrix (64 groups of 512 rows, 1024 -> 2048 f16: 280 us
// in plain order, 342 in bands of 8; without groups, 8192 x 4096 x 4096: 372 and 306).
__device__ inline void tile_of(uint32_t id, uint32_t slots, uint32_t tiles_n, uint32_t band, uint32_t &slot, uint32_t &tile) {
  const uint32_t per = band * tiles_n, group = id / per, in = id % per, first = group * band;
  const uint32_t height = slots - first < band ? slots - first : band;
  slot = first + in % height;
  tile = in / height;
}

// y rows.  BR: B's output index is contiguous (element (n, k) at b[k * ldb + n]), otherwise its reduction index (b[n * ldb + k]).
// SPLIT: a workgroup takes its share of the reduction and leaves float32 sums to mm_rows_join_kernel.
template <typename T, int BM, int BN, int WM, int WN, bool BR, int NBUF, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, NBUF == 1 ? 3 : 2) void mm_rows_kernel(const RowsArgs g) {
  using E = Elem<T>;
  using LA = Tile<T, BM>;
  using LB = Tile<T, BN>;
  constexpr int NT = 64 * WM * WN, STAGE = LA::BYTES + LB::BYTES, EPI = 32 * WM * (BN + 4) * 4;
  __shared__ __attribute__((aligned(16))) char lds[NBUF * STAGE > EPI ? NBUF * STAGE : EPI];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, wm = wave / WN, wn = wave % WN;
  uint32_t slot, tile;
  tile_of(xcd_contiguous(blockIdx.x, gridDim.x), g.slots, g.tiles_n, g.band, slot, tile);
  const int64_t n0 = (int64_t)tile * BN;
  const Piece piece = piece_of(g.groups, __builtin_ctz(BM), slot);
  const int64_t r0 = piece.begin + piece.index * BM;
  if (r0 >= piece.end) return;
  const int64_t rows = piece.end - r0 < BM ? piece.end - r0 : BM;
  const bool real = piece.group >= 0;
  if (SPLIT && !real) return; // (the join writes its zeros)
  const int64_t k_begin = SPLIT ? blockIdx.y * g.k_share : 0;
  const int64_t k_end = SPLIT && k_begin + g.k_share < g.k ? k_begin + g.k_share : g.k, k_len = real ? k_end - k_begin : 0;
  const T *A = static_cast<const T *>(g.a);
  const T *B = static_cast<const T *>(g.b) + (real ? piece.group * g.b_group : 0);

  Accum<T, BM, BN, WM, WN> acc;
  acc.clear();
  StageK<T, BM, NT> sa;
  typename std::conditional<BR, StageR<T, BN, NT, false>, StageK<T, BN, NT>>::type sb;
  sa.open(A, g.lda, r0, rows, k_begin, k_begin + k_len);
  sb.open(B, g.ldb, n0, g.n - n0, k_begin, k_begin + k_len);
  staged_products<T, BM, BN, WM, WN, NBUF>(sa, sb, acc, lds, k_len, tid, wm, wn, lane);

  constexpr int V = 16 / sizeof(T), TPR = BN / V;
  const int64_t nc = n0 + (tid % TPR) * V;
  const int cols = nc + V <= g.n ? V : (nc < g.n ? (int)(g.n - nc) : 0);
  if constexpr (SPLIT) {
    float *out = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int i = 0; i < acc.FM; ++i) {
      if (i) __syncthreads();
      acc.put(out, i, wm, wn, lane);
      __syncthreads();
      for (int lr = tid / TPR; lr < 32 * WM; lr += NT / TPR) {
        const int64_t tr = acc.tile_row(lr, i);
        if (tr >= rows || cols == 0) continue;
        float *to = g.part + ((int64_t)blockIdx.y * g.groups.rows + r0 + tr) * g.n + nc;
        const float *from = out + lr * (BN + 4) + (tid % TPR) * V;
#pragma unroll
        for (int c = 0; c < V; c += 4) {
          if (c + 4 <= cols) *reinterpret_cast<Packed16<float> *>(to + c) = *reinterpret_cast<const u32x4 *>(from + c);
          else
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (c + e < cols) to[c + e] = from[c + e];
        }
      }
    }
    return;
  }
  float bias[V], none[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    bias[v] = g.bias && real && v < cols ? as_float(static_cast<const T *>(g.bias)[piece.group * g.bias_group + nc + v]) : 0.0f;
  by_activation<!BR>(g.act, [&](auto act) { // (products with B laid out that way come without an activation)
    tile_epilogue<T, BM, BN, WM, WN, decltype(act)::value, false, BR>(g, acc, reinterpret_cast<float *>(lds), static_cast<const T *>(g.residual), g.ldr, B, r0, rows, nc, cols,
                                                                     k_len, bias, none, tid, wm, wn, lane);
  });
}

// The shares of the reduction, added in their order, and what becomes of a row's sums.  A workgroup takes a quarter of a tile's rows.
template <typename T, int BN, bool BR> __global__ __launch_bounds__(kThreads) void mm_rows_join_kernel(const RowsArgs g, uint32_t shares) {
  constexpr int V = 16 / sizeof(T), TPR = BN / V, RPP = kThreads / TPR;
  const uint32_t slot = blockIdx.x / g.tiles_n, tile = blockIdx.x % g.tiles_n;
  const Piece piece = piece_of(g.groups, 7, slot);
  const int64_t r0 = piece.begin + piece.index * 128;
  if (r0 >= piece.end) return;
  const int64_t end = piece.end - r0 < 128 ? piece.end : r0 + 128;
  const bool real = piece.group >= 0;
  const int64_t nc = (int64_t)tile * BN + (threadIdx.x % TPR) * V;
  const int cols = nc + V <= g.n ? V : (nc < g.n ? (int)(g.n - nc) : 0);
  if (cols == 0) return;
  float bias[V], none[V];
#pragma unroll
  for (int v = 0; v < V; ++v)
    bias[v] = g.bias && real && v < cols ? as_float(static_cast<const T *>(g.bias)[piece.group * g.bias_group + nc + v]) : 0.0f;
  for (int64_t row = r0 + threadIdx.x / TPR + (int64_t)blockIdx.y * RPP; row < end; row += (int64_t)gridDim.y * RPP) {
    float v[V];
#pragma unroll
    for (int c = 0; c < V; ++c) v[c] = 0.0f;
    if (real) {
#pragma unroll 4
      for (uint32_t s = 0; s < shares; ++s) {
        const float *p = g.part + ((int64_t)s * g.groups.rows + row) * g.n + nc;
#pragma unroll
        for (int c = 0; c < V; c += 4) {
          const u32x4 q = load_cols<float, 4>(p + c, cols - c < 4 ? (cols > c ? cols - c : 0) : 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[c + e] += __uint_as_float(q[e]);
        }
      }
      if constexpr (Elem<T>::PARTS == 3) {
        const float *B = static_cast<const float *>(g.b) + piece.group * g.b_group;
        sums_again<V>(v, cols, static_cast<const float *>(g.a) + row * g.lda, 1, B + (BR ? nc : nc * g.ldb), BR ? g.ldb : 1, BR ? 1 : g.ldb, g.k);
      }
    }
    u32x4 ext = {0, 0, 0, 0};
    if (g.residual) ext = load_cols<T, V>(static_cast<const T *>(g.residual) + row * g.ldr + nc, cols);
    by_activation<!BR>(g.act, [&](auto act) { finish_row<T, V, decltype(act)::value, false>(g, row, nc, cols, v, bias, g.residual != nullptr, ext, none); });
  }
}

// dz = dy act'(z) with z = x W^T + b computed again instead of read: narrow layers are bound by memory, and z costs a write in the forward
// pass and a read here where x, which the weight's gradient reads anyway, is all this needs (2.4 M x 128 -> 256 bf16: 3.8 GB and 850 us
// for dz from a saved z, 3.1 GB so, and the forward pass writes 1.3 GB less).  z is not rounded on its way; dz is, to the
// operands' type, like the dz of act_backward_kernel: dx and dW take it as a matrix operand, and in float32 its write and two reads would
// move 3.8 GB more of that layer's 6.9 and double both products.  What it costs: dx and dW 2.4e-3 off in 2-norm where one rounding is 1.7e-3
// (bfloat16).  Column sums of dz - the bias's
// gradient - are taken before its rounding, one row of partial sums a row tile.  (One workgroup over several row tiles spilled 70 registers: 2057 us.)
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN, 3) void mm_preactivation_kernel(const RowsArgs g, const T *dy, float *part) {
  constexpr int NT = 64 * WM * WN, STAGE = Tile<T, BM>::BYTES + Tile<T, BN>::BYTES, EPI = 32 * WM * (BN + 4) * 4;
  __shared__ __attribute__((aligned(16))) char lds[STAGE > EPI ? STAGE : EPI];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, wm = wave / WN, wn = wave % WN;
  uint32_t slot, tile;
  tile_of(xcd_contiguous(blockIdx.x, gridDim.x), g.slots, g.tiles_n, g.band, slot, tile);
  const int64_t n0 = (int64_t)tile * BN, r0 = (int64_t)slot * BM, rows = g.groups.rows - r0 < BM ? g.groups.rows - r0 : BM;
  Accum<T, BM, BN, WM, WN> acc;
  acc.clear();
  {
    StageK<T, BM, NT> sa;
    StageK<T, BN, NT> sb;
    sa.open(static_cast<const T *>(g.a), g.lda, r0, rows, 0, g.k);
    sb.open(static_cast<const T *>(g.b), g.ldb, n0, g.n - n0, 0, g.k);
    staged_products<T, BM, BN, WM, WN, 1>(sa, sb, acc, lds, g.k, tid, wm, wn, lane);
  }
  constexpr int V = 16 / sizeof(T), TPR = BN / V, RPP = NT / TPR;
  const int col = (tid % TPR) * V;
  const int64_t nc = n0 + col;
  const int cols = nc + V <= g.n ? V : (nc < g.n ? (int)(g.n - nc) : 0);
  float bias[V], sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    bias[v] = g.bias && v < cols ? as_float(static_cast<const T *>(g.bias)[nc + v]) : 0.0f;
    sum[v] = 0.0f;
  }
  float *out = reinterpret_cast<float *>(lds);
  by_activation(g.act, [&](auto act) {
    tile_epilogue<T, BM, BN, WM, WN, decltype(act)::value, true, false>(g, acc, out, dy, g.n, static_cast<const T *>(g.b), r0, rows, nc, cols, g.k, bias, sum, tid, wm, wn,
                                                                       lane);
  });
  if (!part) return;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) out[(tid / TPR) * BN + col + v] = sum[v];
  __syncthreads();
  for (int c = tid; c < BN && n0 + c < g.n; c += NT) {
    float s = 0.0f;
    for (int r = 0; r < RPP; ++r) s += out[r * BN + c];
    part[(int64_t)slot * g.n + n0 + c] = s;
  }
}

// Few rows (or few columns): too few tiles to fill the chip, and the time of a call is that of reading one operand - for a single row of
// a 4096 x 4096 product, 32 tiles walking 64 steps each took 56 us where the weight is read in 7.  Here a workgroup takes 32 FM rows by 32
// columns, its eight waves take every eighth step of the reduction each, straight from memory into the operand registers of the matrix
// instructions (lane = row, 8 consecutive values), U steps in flight, and the eight partial tiles are added through LDS.
template <typename T, int FM> __global__ __launch_bounds__(512, 2) void mm_few_rows_kernel(const RowsArgs g) {
  using E = Elem<T>;
  using F = typename E::Frag;
  constexpr int W = 8, U = 4 / FM < 1 ? 1 : 4 / FM, P16 = 8 * sizeof(T) / 16;
  __shared__ __attribute__((aligned(16))) float part[W][32 * FM][36];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const int64_t r0 = (int64_t)(blockIdx.x / g.tiles_n) * 32 * FM, n0 = (int64_t)(blockIdx.x % g.tiles_n) * 32;
  const T *rows[FM + 1]; // of A, then of B: rows that do not exist read the last one
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int64_t r = r0 + i * 32 + lane % 32;
    rows[i] = static_cast<const T *>(g.a) + (r < g.groups.rows ? r : g.groups.rows - 1) * g.lda;
  }
  const int64_t n = n0 + lane % 32;
  rows[FM] = static_cast<const T *>(g.b) + (n < g.n ? n : g.n - 1) * g.ldb;

  Accum<T, 32 * FM, 32, 1, 1> acc;
  acc.clear();
  for (int64_t k0 = wave * 16 * U; k0 < g.k; k0 += W * 16 * U) {
    u32x4 reg[U][FM + 1][P16];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k = k0 + u * 16 + (lane / 32) * 8;
#pragma unroll
      for (int i = 0; i <= FM; ++i) {
        if (k + 8 <= g.k) {
#pragma unroll
          for (int w = 0; w < P16; ++w) reg[u][i][w] = reinterpret_cast<const Packed16<T> *>(rows[i] + k)[w];
        } else {
          alignas(16) T tmp[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) tmp[j] = k + j < g.k ? rows[i][k + j] : (T)0.0f;
#pragma unroll
          for (int w = 0; w < P16; ++w) reg[u][i][w] = reinterpret_cast<const u32x4 *>(tmp)[w];
        }
      }
    }
    f32x16 t[FM][1];
    if constexpr (E::PARTS == 3) acc.zero(t);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      F a[E::PARTS][FM], b[E::PARTS][1];
#pragma unroll
      for (int i = 0; i <= FM; ++i) {
        if constexpr (E::PARTS == 1) {
          const F f = *reinterpret_cast<const F *>(&reg[u][i][0]);
          if (i < FM) a[0][i < FM ? i : 0] = f;
          else b[0][0] = f;
        } else {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(reg[u][i][j / 4][j % 4]);
          bf16x8 p[3];
          split8(v, p);
#pragma unroll
          for (int s = 0; s < 3; ++s) (i < FM ? a[s][i < FM ? i : 0] : b[s][0]) = p[s];
        }
      }
      if constexpr (E::PARTS == 1) acc.products(acc.acc, a, b);
      else acc.products(t, a, b);
    }
    if constexpr (E::PARTS == 3) acc.add(t);
  }
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) part[wave][i * 32 + acc.row_of(e, lane)][lane % 32] = acc.acc[i][0][e];
  __syncthreads();
  constexpr int V = 16 / sizeof(T), TPR = 32 / V;
  const int col = (tid % TPR) * V;
  const int64_t nc = n0 + col;
  const int cols = nc + V <= g.n ? V : (nc < g.n ? (int)(g.n - nc) : 0);
  if (cols == 0) return;
  float bias[V], none[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = g.bias && v < cols ? as_float(static_cast<const T *>(g.bias)[nc + v]) : 0.0f;
  for (int lr = tid / TPR; lr < 32 * FM && r0 + lr < g.groups.rows; lr += 512 / TPR) {
    float v[V];
#pragma unroll
    for (int c = 0; c < V; ++c) v[c] = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int c = 0; c < V; c += 4) {
        const f32x4 q = *reinterpret_cast<const f32x4 *>(&part[w][lr][col + c]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[c + e] += q[e];
      }
    if constexpr (E::PARTS == 3)
      sums_again<V>(v, cols, static_cast<const float *>(g.a) + (r0 + lr) * g.lda, 1, static_cast<const float *>(g.b) + nc * g.ldb, 1, g.ldb, g.k);
    u32x4 ext = {0, 0, 0, 0};
    if (g.residual) ext = load_cols<T, V>(static_cast<const T *>(g.residual) + (r0 + lr) * g.ldr + nc, cols);
    by_activation(g.act, [&](auto act) { finish_row<T, V, decltype(act)::value, false>(g, r0 + lr, nc, cols, v, bias, g.residual != nullptr, ext, none); });
  }
}

// ---- gradient of the weight ---------------------------------------------------------------------------------------------------------
struct WeightArgs {
  const void *p, *q;   // [rows, np], [rows, nq]: out(i, j) = sum over rows of p[r, i] q[r, j]
  void *out, *colsum;  // [G, np, nq] in T; column sums of p (sum_p) or q [G, np or nq], may be null
  float *part;         // partial products of the chunks of groups that have several: [part_of ..][np * nq + (colsum ? ns : 0)]
  int64_t ldp, ldq, np, nq, ns;
  Groups groups;
  int64_t unit;        // rows of a chunk; with groups 1 << unit_log2
  int unit_log2;
  uint32_t tiles_p, tiles_q;
  int sum_p, compact;
  // Where chunk `index` of a group goes that starts at row q0 and has several; `slot`: the chunk's slot of the launch.  compact: a number that
  // does not grow with the groups.  floor(q0 / unit) + index ascends over all such chunks, and two of them share a value at most where one
  // group's last chunk meets the next one's first: first chunks take the odd numbers, the others the even ones, all below 2 ceil(rows / unit).
  __device__ int64_t part_of(int64_t q0, int64_t index, int64_t slot) const { return compact ? 2 * ((q0 >> unit_log2) + index) + (index == 0) : slot; }
};

template <bool PAIR, int WHICH, typename A, typename B> __device__ inline auto &pick(A &a, B &b) {
  if constexpr (PAIR) return a.st;
  else if constexpr (WHICH == 1) return a;
  else return b;
}
// SUMS: column sums of nothing (0), p (1) or q (2) beside the product
template <typename T, int BM, int BN, int WM, int WN, int SUMS>
__global__ __launch_bounds__(64 * WM * WN, BM == 64 && BN == 64 ? 4 : 3) void mm_weight_kernel(const WeightArgs g) {
  using E = Elem<T>;
  using LA = Tile<T, BM>;
  using LB = Tile<T, BN>;
  constexpr int NT = 64 * WM * WN, STAGE = LA::BYTES + LB::BYTES, EPI = 32 * WM * (BN + 4) * 4;
  __shared__ __attribute__((aligned(16))) char lds[STAGE > EPI ? STAGE : EPI];
  const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, wm = wave / WN, wn = wave % WN;
  const uint32_t tile = xcd_contiguous(blockIdx.x, gridDim.x), tiles = g.tiles_p * g.tiles_q, t = tile % tiles;
  const int64_t slot = tile / tiles, i0 = (int64_t)(t / g.tiles_q) * BM, j0 = (int64_t)(t % g.tiles_q) * BN;
  const Piece piece = piece_of(g.groups, g.unit_log2, slot);
  if (piece.group < 0) return;
  const int64_t len = piece.end - piece.begin, r0 = piece.begin + piece.index * g.unit;
  if (len > 0 ? r0 >= piece.end : piece.index > 0) return;   // (a group without rows still writes its zeros, once)
  const int64_t r1 = len <= 0 ? r0 : (r0 + g.unit < piece.end ? r0 + g.unit : piece.end);
  const bool whole = len <= g.unit;                          // this chunk is all of its group
  const T *P = static_cast<const T *>(g.p), *Q = static_cast<const T *>(g.q);
  const bool sums = SUMS == 1 ? j0 == 0 : SUMS == 2 && i0 == 0;

  Accum<T, BM, BN, WM, WN> acc;
  acc.clear();
  constexpr bool PAIR = E::PARTS == 1 && BM == 128 && BN == 128;
  typename std::conditional<PAIR, StagePair<T, BM, NT, SUMS != 0>, StageR<T, BM, NT, SUMS == 1>>::type sa;
  typename std::conditional<PAIR, StageNone, StageR<T, BN, NT, SUMS == 2>>::type sb;
  const int half = __builtin_amdgcn_readfirstlane(tid / (NT / 2));
  if constexpr (PAIR) {
    sa.st.open(half ? Q : P, half ? g.ldq : g.ldp, half ? j0 : i0, half ? g.nq - j0 : g.np - i0, r0, r1);
    sa.st.add = sums && half == SUMS - 1;
    constexpr int VR = 16 / sizeof(T);
    sa.both = (i0 + BM <= g.np || (g.np > i0 && (g.np - i0) % VR == 0)) && (j0 + BN <= g.nq || (g.nq > j0 && (g.nq - j0) % VR == 0));
  } else {
    sa.open(P, g.ldp, i0, g.np - i0, r0, r1);
    sb.open(Q, g.ldq, j0, g.nq - j0, r0, r1);
    sa.add = sb.add = sums;
  }
  const int64_t k_len = r1 - r0;
  staged_products<T, BM, BN, WM, WN, 1>(sa, sb, acc, lds, k_len, tid, wm, wn, lane);

  const int64_t per_slot = g.np * g.nq + (g.colsum ? g.ns : 0), number = g.part_of(piece.begin, piece.index, slot);
  float *out = reinterpret_cast<float *>(lds);
  const int col = (tid % (BN / 4)) * 4;
#pragma unroll
  for (int i = 0; i < acc.FM; ++i) {
    if (i) __syncthreads();
    acc.put(out, i, wm, wn, lane);
    if constexpr (E::PARTS == 3)
      acc.again(out, i, wm, wn, lane, reinterpret_cast<const float *>(P) + r0 * g.ldp + i0, 1, g.ldp, reinterpret_cast<const float *>(Q) + r0 * g.ldq + j0, 1, g.ldq,
                (int)(g.np - i0 < BM ? g.np - i0 : BM), (int)(g.nq - j0 < BN ? g.nq - j0 : BN), k_len);
    __syncthreads();
    for (int lr = tid / (BN / 4); lr < 32 * WM; lr += NT / (BN / 4)) {
      const int64_t row = i0 + acc.tile_row(lr, i);
      if (row >= g.np) continue;
      const f32x4 q = *reinterpret_cast<const f32x4 *>(out + lr * (BN + 4) + col);
      const int64_t cc = j0 + col;
      if (cc >= g.nq) continue;
      const int cols = g.nq - cc < 4 ? (int)(g.nq - cc) : 4;
      alignas(16) float v[4] = {q[0], q[1], q[2], q[3]};
      if (whole) {
        T *o = static_cast<T *>(g.out) + (piece.group * g.np + row) * g.nq + cc;
        alignas(16) T tmp[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmp[c] = (T)v[c];
        if (cols == 4) {
          if constexpr (sizeof(T) == 4) *reinterpret_cast<Packed16<T> *>(o) = *reinterpret_cast<const u32x4 *>(tmp);
          else *reinterpret_cast<Packed8<T> *>(o) = *reinterpret_cast<const u32x2 *>(tmp);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < cols) o[c] = tmp[c];
        }
      } else {
        float *o = g.part + number * per_slot + row * g.nq + cc;
        if (cols == 4) {
          *reinterpret_cast<Packed16<float> *>(o) = *reinterpret_cast<const u32x4 *>(v);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c < cols) o[c] = v[c];
        }
      }
    }
  }

  if constexpr (SUMS == 0) return;
  if (sums) { // (uniform over the workgroup) column sums: CK threads hold each column's share
    __syncthreads();
    // (as staged_products and StagePair number the threads of each operand)
    const int part_id = PAIR ? tid % (NT / 2) : SUMS == 1 ? tid : (tid + NT / 2) % NT;
    const bool mine = !PAIR || half == SUMS - 1;
    constexpr int R = SUMS == 1 ? BM : BN;
    const int64_t first = SUMS == 1 ? i0 : j0, n = SUMS == 1 ? g.np : g.nq;
    auto &st = pick<PAIR, SUMS>(sa, sb);
    using S = typename std::remove_reference<decltype(st)>::type;
#pragma unroll
    for (int i = 0; i < S::N; ++i) {
      const int idx = part_id + i * NT;
      if (mine && idx < S::BLOCKS) {
        const int row = (idx % (R / S::VR)) * S::VR, chunk = idx / (R / S::VR);
#pragma unroll
        for (int r = 0; r < S::VR; ++r) out[chunk * R + row + r] = st.sum[i][r];
      }
    }
    __syncthreads();
    for (int c = tid; c < R && first + c < n; c += NT) {
      float s = 0.0f;
      for (int k = 0; k < E::BK / 8; ++k) s += out[k * R + c];
      if (whole) static_cast<T *>(g.colsum)[piece.group * g.ns + first + c] = (T)s;
      else g.part[number * per_slot + g.np * g.nq + first + c] = s;
    }
  }
}

// The chunks of a group, added in their order by 16 threads an element (each every 16th chunk, then the 16 by halves).
// WAYS 1: at most 16 chunks, one thread an element (300 rows, 4096 -> 256: 15 of the 16 threads had nothing to add).
template <typename T, int WAYS> __global__ __launch_bounds__(kThreads) void mm_join_kernel(const WeightArgs g) {
  __shared__ float part[kThreads];
  const int64_t group = blockIdx.y;
  Piece piece;
  if (!g.groups.ptr) piece = {0, 0, g.groups.rows, 0, 0};
  else {
    const int64_t q0 = g.groups.bound(group + 1), q1 = g.groups.bound(group + 2);
    piece = {group, q0, q1, 0, (q0 >> g.unit_log2) + group + 1};
  }
  const int64_t len = piece.end - piece.begin;
  if (len <= g.unit) return;
  const int64_t chunks = (len + g.unit - 1) / g.unit;
  const int64_t size = g.np * g.nq, per_slot = size + (g.colsum ? g.ns : 0);
  const float *first = g.part + g.part_of(piece.begin, 0, piece.start) * per_slot; // (chunks behind the first: evenly spaced)
  const float *rest = g.part + (g.compact ? 2 * (piece.begin >> g.unit_log2) : piece.start) * per_slot;
  const int64_t step = (g.compact ? 2 : 1) * per_slot;
  constexpr int LANES = kThreads / WAYS;
  const int lane = threadIdx.x % LANES, way = threadIdx.x / LANES;
  for (int64_t base = (int64_t)blockIdx.x * LANES; base < per_slot; base += (int64_t)gridDim.x * LANES) {
    const int64_t i = base + lane;
    float s = 0.0f;
    if (i < per_slot) {
      if (way == 0) s = first[i];
#pragma unroll 4
      for (int64_t c = way == 0 ? WAYS : way; c < chunks; c += WAYS) s += rest[c * step + i];
    }
    if constexpr (WAYS > 1) {
      part[threadIdx.x] = s;
      __syncthreads();
#pragma unroll
      for (int h = kThreads / 2; h >= LANES; h /= 2) {
        if ((int)threadIdx.x < h) part[threadIdx.x] += part[threadIdx.x + h];
        __syncthreads();
      }
      s = part[lane];
      __syncthreads();
    }
    if (way == 0 && i < per_slot) {
      if (i < size) static_cast<T *>(g.out)[group * size + i] = (T)s;
      else static_cast<T *>(g.colsum)[group * g.ns + i - size] = (T)s;
    }
  }
}

// ---- the activation's gradient from a saved z: dz = dy * act'(z), and the column sums of dz before its rounding ------------------------
// A workgroup takes tx vectors of columns (blockDim = tx x 256 / tx) and every gridDim.y-th set of rows.
template <typename T, int ACT>
__global__ __launch_bounds__(kThreads) void act_backward_kernel(const T *dy, const T *z, T *dz, float *part, int64_t rows, int64_t n) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float fold[kThreads][V + 1];
  const int64_t col = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * V;
  const int cols = col + V <= n ? V : (col < n ? (int)(n - col) : 0);
  float sum[V];
#pragma unroll
  for (int v = 0; v < V; ++v) sum[v] = 0.0f;
  if (cols > 0) {
#pragma unroll 2
    for (int64_t row = (int64_t)blockIdx.y * blockDim.y + threadIdx.y; row < rows; row += (int64_t)gridDim.y * blockDim.y) {
      const int64_t at = row * n + col;
      alignas(16) T a[V], b[V];
      if (cols == V) {
        *reinterpret_cast<u32x4 *>(a) = *reinterpret_cast<const Packed16<T> *>(dy + at);
        *reinterpret_cast<u32x4 *>(b) = *reinterpret_cast<const Packed16<T> *>(z + at);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          a[v] = v < cols ? dy[at + v] : (T)0.0f;
          b[v] = v < cols ? z[at + v] : (T)0.0f;
        }
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float d = activation_gradient<T, ACT>(as_float(a[v]), as_float(b[v]));
        sum[v] += d;
        a[v] = (T)d;
      }
      if (cols == V) *reinterpret_cast<Packed16<T> *>(dz + at) = *reinterpret_cast<const u32x4 *>(a);
      else
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (v < cols) dz[at + v] = a[v];
    }
  }
  if (!part) return;
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
#pragma unroll
  for (int v = 0; v < V; ++v) fold[tid][v] = sum[v];
  __syncthreads();
  if (threadIdx.y != 0) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float s = 0.0f;
    for (unsigned y = 0; y < blockDim.y; ++y) s += fold[y * blockDim.x + threadIdx.x][v];
    if (v < cols) part[(int64_t)blockIdx.y * n + col + v] = s;
  }
}

// part [rows, n] -> out[n] (or, of gridDim.y > 1, a row of it per block row): 16 threads a column, each every 16th row of the block
// row's share, then the 16 by halves
template <typename T> __global__ __launch_bounds__(kThreads) void column_join_kernel(const float *part, int64_t rows, int64_t n, T *out) {
  __shared__ float fold[kThreads];
  const int lane = threadIdx.x % 16, way = threadIdx.x / 16;
  const int64_t i = (int64_t)blockIdx.x * 16 + lane, share = (rows + gridDim.y - 1) / gridDim.y, first = blockIdx.y * share;
  const int64_t last = first + share < rows ? first + share : rows;
  float s = 0.0f;
  if (i < n)
#pragma unroll 8
    for (int64_t r = first + way; r < last; r += 16) s += part[r * n + i];
  fold[threadIdx.x] = s;
  __syncthreads();
#pragma unroll
  for (int h = 128; h >= 16; h /= 2) {
    if ((int)threadIdx.x < h) fold[threadIdx.x] += fold[threadIdx.x + h];
    __syncthreads();
  }
  if (way == 0 && i < n) out[blockIdx.y * n + i] = (T)fold[lane];
}

// ---- launches -----------------------------------------------------------------------------------------------------------------------
int launched(const char *name) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return geot_internal_fail(GEOT_ELAUNCH, hipGetErrorString(e));
  if (name) geot_internal_note_kernel(name);
  return GEOT_OK;
}

constexpr int64_t kMaxBlocks = (((int64_t)1 << 32) - 1) / 512; // (a launch holds fewer than 2^32 threads)

// Reduction values of a workgroup: all of them (k) where the tiles fill the chip, or the reduction is short; else a share such that about
// two workgroups a CU run, at least four steps each.  (17 rows x 4048 -> 144 f32 in 2 groups: 5 tiles of 127 steps were 192 us.)
int64_t rows_share(int64_t rows, int64_t groups, bool with_ptr, int64_t n, int64_t k, bool f32) {
  const int64_t bn = f32 || n <= 64 ? 64 : 128, bk = f32 ? 32 : 64;
  const int64_t tiles = ((rows + 127) / 128 + (with_ptr ? (groups < rows ? groups : rows) : 0)) * ((n + bn - 1) / bn);
  if (tiles <= 0 || tiles >= 256 || k < 8 * bk) return k;
  // (workgroups that find no rows - up to one a group - count against what a launch can hold)
  const int64_t blocks = slots_of(rows, groups, with_ptr, 128) * ((n + bn - 1) / bn), room = 2 * kMaxBlocks / blocks;
  int64_t shares = (512 + tiles - 1) / tiles;
  const int64_t most = k / (4 * bk);
  shares = shares < most ? shares : most;
  if (room < 4) return k; // (mm_rows_join_kernel's four a tile)
  shares = shares < room ? shares : room;
  return ((k + shares - 1) / shares + bk - 1) / bk * bk;
}
size_t rows_workspace(int64_t rows, int64_t groups, bool with_ptr, int64_t n, int64_t k, int dtype) {
  const int64_t share = rows_share(rows, groups, with_ptr, n, k, dtype == GEOT_F32);
  return share < k ? (size_t)((k + share - 1) / share) * (size_t)rows * (size_t)n * sizeof(float) : 0;
}
template <typename T, int BM, int BN, int WM, int WN, bool BR, int NBUF> int launched_rows(bool split) {
  char name[96];
  snprintf(name, sizeof name, "mm_rows_kernel<%s, %d, %d, %d, %d, %s, %d, %s>", std::is_same<T, float>::value ? "float" : std::is_same<T, f16>::value ? "_Float16" : "__bf16",
           BM, BN, WM, WN, BR ? "true" : "false", NBUF, split ? "true" : "false");
  return launched(name);
}
template <typename T, int BM, int BN, int WM, int WN, bool BR, int NBUF> int run_rows(RowsArgs &g, hipStream_t st) {
  const int64_t tiles_n = (g.n + BN - 1) / BN, slots = slots_of(g.groups.rows, g.groups.groups, g.groups.ptr != nullptr, BM);
  if (tiles_n > kMaxBlocks / 8 || slots > kMaxBlocks / tiles_n) return geot_internal_fail(GEOT_EINVAL, "more tiles than one launch can hold");
  g.tiles_n = (uint32_t)tiles_n;
  g.slots = (uint32_t)slots;
  g.band = g.groups.ptr ? 1 : 8;
  const unsigned blocks = g.slots * g.tiles_n;
  if constexpr (BM == 128) {
    const int64_t share = rows_share(g.groups.rows, g.groups.groups, g.groups.ptr != nullptr, g.n, g.k, Elem<T>::PARTS == 3);
    if (g.part && share < g.k) {
      const unsigned shares = (unsigned)((g.k + share - 1) / share);
      g.k_share = share;
      hipLaunchKernelGGL((mm_rows_kernel<T, BM, BN, WM, WN, BR, NBUF, true>), dim3(blocks, shares), dim3(64 * WM * WN), 0, st, g);
      if (const int rc = launched_rows<T, BM, BN, WM, WN, BR, NBUF>(true)) return rc;
      hipLaunchKernelGGL((mm_rows_join_kernel<T, BN, BR>), dim3(blocks, 4), dim3(kThreads), 0, st, g, shares);
      return launched(nullptr);
    }
  }
  hipLaunchKernelGGL((mm_rows_kernel<T, BM, BN, WM, WN, BR, NBUF, false>), dim3(blocks), dim3(64 * WM * WN), 0, st, g);
  return launched_rows<T, BM, BN, WM, WN, BR, NBUF>(false);
}
template <typename T, int FM> int run_few(RowsArgs &g, hipStream_t st) {
  g.tiles_n = (uint32_t)((g.n + 31) / 32);
  const int64_t tiles_m = (g.groups.rows + 32 * FM - 1) / (32 * FM);
  hipLaunchKernelGGL((mm_few_rows_kernel<T, FM>), dim3((unsigned)(tiles_m * g.tiles_n)), dim3(512), 0, st, g);
  return launched("mm_few_rows_kernel");
}
// Few tiles and a reduction that eight waves of a workgroup walk in a few steps; a longer one of more than 32 rows is split over
// workgroups instead (bf16: 100 x 1000 -> 1000 takes 7.8 us so and 15.8 split, as its dx is; 300 x 4096 -> 256 23.6 and 18.7).
bool takes_few_rows(int64_t rows, bool with_ptr, int64_t n, int64_t k) {
  return !with_ptr && ((rows + 127) / 128) * ((n + 127) / 128) < 128 && k >= 128 && (rows <= 32 || k <= 2048);
}
template <typename T, bool BR> int rows_typed(RowsArgs &g, hipStream_t st) {
  const int64_t tiles = ((g.groups.rows + 127) / 128) * ((g.n + 127) / 128);
  if constexpr (!BR) { // (segment_matmul's gradient comes here too, with groups)
    if (takes_few_rows(g.groups.rows, g.groups.ptr != nullptr, g.n, g.k)) return g.groups.rows <= 32 ? run_few<T, 1>(g, st) : run_few<T, 2>(g, st);
  }
  // (split operands: two column fragments a wave and their six parts do not fit the registers of three workgroups a CU)
  if (Elem<T>::PARTS == 3 || g.n <= 64) return run_rows<T, 128, 64, 2, 2, BR, 1>(g, st);
  if constexpr (Elem<T>::PARTS == 1) {
    const int64_t per_group = g.groups.ptr ? g.groups.rows / (g.groups.groups > 0 ? g.groups.groups : 1) : g.groups.rows;
    if (g.n > 128 && g.k >= 512 && tiles >= 1024 && per_group >= 2048) return run_rows<T, 256, 256, 2, 4, BR, 2>(g, st);
    return run_rows<T, 128, 128, 2, 2, BR, 1>(g, st);
  }
}
int rows_product(RowsArgs &g, bool br, int dtype, hipStream_t st, void *workspace, size_t workspace_bytes) {
  if (g.groups.rows == 0 || g.n == 0) return GEOT_OK;
  const bool few = !br && takes_few_rows(g.groups.rows, g.groups.ptr != nullptr, g.n, g.k);
  const size_t need = few ? 0 : rows_workspace(g.groups.rows, g.groups.groups, g.groups.ptr != nullptr, g.n, g.k, dtype);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) return geot_internal_fail(GEOT_EWORKSPACE, "rows product: workspace too small or misaligned");
  g.part = need ? static_cast<float *>(workspace) : nullptr;
  switch (dtype) {
  case GEOT_F32: return br ? rows_typed<float, true>(g, st) : rows_typed<float, false>(g, st);
  case GEOT_F16: return br ? rows_typed<f16, true>(g, st) : rows_typed<f16, false>(g, st);
  case GEOT_BF16: return br ? rows_typed<bf16, true>(g, st) : rows_typed<bf16, false>(g, st);
  }
  return geot_internal_fail(GEOT_EUNSUPPORTED, "matrix products take float32, float16 and bfloat16");
}

// Column sums of dz: a row of partial sums per row tile (dz from x) or per block row of the grid (dz from z), joined in two steps where
// there are many.
constexpr int64_t kColumnParts = 1024, kColumnJoin = 64;
int64_t column_parts(int64_t rows) { // of either form
  const int64_t tiles = (rows + 127) / 128;
  return (tiles > kColumnParts ? tiles : kColumnParts) + kColumnJoin;
}
template <typename T, int BN> int run_preactivation(RowsArgs &g, const void *dy, float *part, hipStream_t st, int64_t &parts) {
  const int64_t tiles_n = (g.n + BN - 1) / BN;
  parts = (g.groups.rows + 127) / 128;
  if (tiles_n > kMaxBlocks / 8 || parts > kMaxBlocks / tiles_n) return geot_internal_fail(GEOT_EINVAL, "more tiles than one launch can hold");
  g.tiles_n = (uint32_t)tiles_n;
  g.slots = (uint32_t)parts;
  g.band = 8;
  hipLaunchKernelGGL((mm_preactivation_kernel<T, 128, BN, 2, 2>), dim3((unsigned)(parts * tiles_n)), dim3(256), 0, st, g, static_cast<const T *>(dy), part);
  return launched("mm_preactivation_kernel");
}
template <typename T> int preactivation_typed(RowsArgs &g, const void *dy, const void *z, float *part, void *dbias, hipStream_t st) {
  int64_t parts = 0;
  if (!z) {
    int rc;
    if constexpr (Elem<T>::PARTS == 3) rc = run_preactivation<T, 64>(g, dy, part, st, parts);
    else rc = g.n <= 64 ? run_preactivation<T, 64>(g, dy, part, st, parts) : run_preactivation<T, 128>(g, dy, part, st, parts);
    if (rc) return rc;
  } else {
    const int64_t vectors = (g.n * (int64_t)sizeof(T) + 15) / 16;
    unsigned tx = 1;
    while (tx < 256 && tx < vectors) tx *= 2;
    const unsigned ty = 256 / tx;
    const int64_t gx = (vectors + tx - 1) / tx, need = (g.groups.rows + ty - 1) / ty;
    if (gx > kMaxBlocks) return geot_internal_fail(GEOT_EINVAL, "more tiles than one launch can hold");
    parts = part ? kColumnParts : 8192;
    parts = need < parts ? need : parts;
    by_activation(g.act, [&](auto act) {
      hipLaunchKernelGGL((act_backward_kernel<T, decltype(act)::value>), dim3((unsigned)gx, (unsigned)parts), dim3(tx, ty), 0, st, static_cast<const T *>(dy),
                         static_cast<const T *>(z), static_cast<T *>(g.y), part, g.groups.rows, g.n);
    });
    if (const int rc = launched("act_backward_kernel")) return rc;
  }
  if (!part) return GEOT_OK;
  const unsigned wide = (unsigned)((g.n + 15) / 16);
  if (parts > 8 * kColumnJoin) {
    float *joined = part + parts * g.n;
    hipLaunchKernelGGL((column_join_kernel<float>), dim3(wide, (unsigned)kColumnJoin), dim3(kThreads), 0, st, part, parts, g.n, joined);
    if (const int rc = launched(nullptr)) return rc;
    part = joined;
    parts = kColumnJoin;
  }
  hipLaunchKernelGGL((column_join_kernel<T>), dim3(wide), dim3(kThreads), 0, st, part, parts, g.n, static_cast<T *>(dbias));
  return launched(nullptr);
}

// Chunks of rows: one full round of workgroups (3 a CU, 4 of the 64 x 64 tiles), and no chunk below 256 rows.  Groups of rows take chunks
// of a power of two (piece_of).
struct WeightPlan {
  int64_t tiles_p, tiles_q, unit, slots;
  int64_t parts; // partial products that need room (part_of)
  int unit_log2;
  bool compact;
};
WeightPlan weight_plan(int64_t rows, int64_t groups, bool with_ptr, int64_t np, int64_t nq, int dtype) {
  WeightPlan w;
  const int64_t bm = np <= 64 ? 64 : 128, bn = nq <= 64 || dtype == GEOT_F32 ? 64 : 128;
  w.tiles_p = np > 0 ? (np + bm - 1) / bm : 1; // (a side of width 0 still has its column sums)
  w.tiles_q = nq > 0 ? (nq + bn - 1) / bn : 1;
  const int64_t tiles = w.tiles_p * w.tiles_q;
  const int64_t round = np <= 64 && nq <= 64 ? 1024 : 768, want = round / tiles > 1 ? round / tiles : 1;
  w.unit_log2 = 8;
  if (with_ptr) {
    while (((int64_t)2 << w.unit_log2) * want <= rows) ++w.unit_log2; // the power of two at or below rows / want
    w.unit = (int64_t)1 << w.unit_log2;
  } else {
    w.unit = ((rows + want - 1) / want + 63) / 64 * 64;
    w.unit = w.unit < 256 ? 256 : w.unit;
  }
  w.slots = slots_of(rows, groups, with_ptr, w.unit);
  if (w.slots < 1) w.slots = 1;
  // (64 experts of 1024 x 2048, 32768 rows: 16 numbers of 8.4 MB where the launch has 74 slots)
  const int64_t compact = 2 * ((rows + w.unit - 1) / w.unit);
  w.compact = with_ptr && compact < w.slots;
  w.parts = rows > w.unit ? (w.compact ? compact : w.slots) : 0;
  return w;
}
template <typename T, int BM, int BN, int WM, int WN> int run_weight(WeightArgs &g, int64_t slots, hipStream_t st) {
  const int64_t tiles = (int64_t)g.tiles_p * g.tiles_q;
  const dim3 grid((unsigned)(slots * tiles)), block(64 * WM * WN);
  if (!g.colsum) hipLaunchKernelGGL((mm_weight_kernel<T, BM, BN, WM, WN, 0>), grid, block, 0, st, g);
  else if (g.sum_p) hipLaunchKernelGGL((mm_weight_kernel<T, BM, BN, WM, WN, 1>), grid, block, 0, st, g);
  else hipLaunchKernelGGL((mm_weight_kernel<T, BM, BN, WM, WN, 2>), grid, block, 0, st, g);
  if (const int rc = launched("mm_weight_kernel")) return rc;
  if (g.groups.rows > g.unit) { // some group may have several chunks
    const bool few = g.groups.rows <= 16 * g.unit;
    const int64_t lanes = few ? kThreads : 16, per = (g.np * g.nq + (g.colsum ? g.ns : 0) + lanes - 1) / lanes;
    // (which groups have several chunks only the device knows: few workgroups a group when there are many - 2048 each cost 50 us at 64
    // groups of one chunk)
    int64_t wide = 8192 / g.groups.groups;
    wide = wide < 32 ? 32 : wide > 2048 ? 2048 : wide;
    const dim3 join((unsigned)(per < wide ? per : wide), (unsigned)g.groups.groups);
    if (few) hipLaunchKernelGGL((mm_join_kernel<T, 1>), join, dim3(kThreads), 0, st, g);
    else hipLaunchKernelGGL((mm_join_kernel<T, 16>), join, dim3(kThreads), 0, st, g);
    return launched(nullptr);
  }
  return GEOT_OK;
}
template <typename T> int weight_typed(WeightArgs &g, int64_t slots, hipStream_t st) {
  if constexpr (Elem<T>::PARTS == 1) {
    if (g.nq > 64) return g.np <= 64 ? run_weight<T, 64, 128, 2, 2>(g, slots, st) : run_weight<T, 128, 128, 2, 2>(g, slots, st);
  }
  return g.np <= 64 ? run_weight<T, 64, 64, 2, 2>(g, slots, st) : run_weight<T, 128, 64, 2, 2>(g, slots, st);
}
int weight_product(WeightArgs &g, int dtype, void *workspace, size_t workspace_bytes, hipStream_t st) {
  if (g.groups.groups == 0 || (g.np * g.nq == 0 && !(g.colsum && g.ns > 0))) return GEOT_OK;
  const WeightPlan w = weight_plan(g.groups.rows, g.groups.groups, g.groups.ptr != nullptr, g.np, g.nq, dtype);
  if (w.tiles_p * w.tiles_q > kMaxBlocks / w.slots) return geot_internal_fail(GEOT_EINVAL, "more tiles than one launch can hold");
  g.unit = w.unit;
  g.unit_log2 = w.unit_log2;
  g.tiles_p = (uint32_t)w.tiles_p;
  g.tiles_q = (uint32_t)w.tiles_q;
  g.part = static_cast<float *>(workspace);
  g.compact = w.compact;
  if (w.parts > 0) {
    const size_t need = (size_t)w.parts * (size_t)(g.np * g.nq + (g.colsum ? g.ns : 0)) * sizeof(float);
    if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) return geot_internal_fail(GEOT_EWORKSPACE, "weight gradient: workspace too small or misaligned");
  }
  switch (dtype) {
  case GEOT_F32: return weight_typed<float>(g, w.slots, st);
  case GEOT_F16: return weight_typed<f16>(g, w.slots, st);
  case GEOT_BF16: return weight_typed<bf16>(g, w.slots, st);
  }
  return geot_internal_fail(GEOT_EUNSUPPORTED, "matrix products take float32, float16 and bfloat16");
}

// Sizes no operand can have: negative, or matrices of more elements than any memory (the plans' products stay inside 64 bits then)
bool bad_size(int64_t a, int64_t b, int64_t c) {
  constexpr int64_t lim = (int64_t)1 << 40, area = (int64_t)1 << 44;
  const auto large = [&](int64_t m, int64_t n) { return m > 0 && n > area / m; };
  return a < 0 || b < 0 || c < 0 || a > lim || b > lim || c > lim || large(a, b) || large(a, c) || large(b, c);
}

} // namespace

extern "C" {

size_t geot_linear_workspace_bytes(int64_t rows, int64_t in, int64_t out, int dtype) {
  return bad_size(rows, in, out) || takes_few_rows(rows, false, out, in) ? 0 : rows_workspace(rows, 1, false, out, in, dtype);
}

int geot_linear(const void *x, int64_t ldx, const void *weight, const void *bias, const void *residual, int64_t ld_residual, void *z, void *y,
                int64_t rows, int64_t in, int64_t out, int activation, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_size(rows, in, out) || ldx < 0 || ld_residual < 0) return geot_internal_fail(GEOT_EINVAL, "geot_linear: negative or impossible size");
  if (activation < GEOT_ACT_NONE || activation > GEOT_ACT_SILU) return geot_internal_fail(GEOT_EINVAL, "geot_linear: unknown activation");
  if (rows > 0 && out > 0 && (!y || (in > 0 && (!x || !weight)))) return geot_internal_fail(GEOT_EINVAL, "geot_linear: null pointer");
  RowsArgs g{};
  g.a = x; g.lda = ldx; g.b = weight; g.ldb = in; g.bias = bias; g.residual = residual; g.ldr = ld_residual; g.z = z; g.y = y; g.ldy = out;
  g.groups = {nullptr, 1, rows}; g.n = out; g.k = in; g.act = activation;
  return rows_product(g, false, dtype, static_cast<hipStream_t>(stream), workspace, workspace_bytes);
}

size_t geot_linear_grad_input_workspace_bytes(int64_t rows, int64_t in, int64_t out, int dtype) {
  return bad_size(rows, in, out) ? 0 : rows_workspace(rows, 1, false, in, out, dtype);
}

int geot_linear_grad_input(const void *dz, const void *weight, void *dx, int64_t rows, int64_t in, int64_t out, int dtype, void *workspace, size_t workspace_bytes,
                           void *stream) {
  if (bad_size(rows, in, out)) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_input: negative or impossible size");
  if (rows > 0 && in > 0 && (!dx || (out > 0 && (!dz || !weight)))) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_input: null pointer");
  RowsArgs g{};
  g.a = dz; g.lda = out; g.b = weight; g.ldb = in; g.y = dx; g.ldy = in;
  g.groups = {nullptr, 1, rows}; g.n = in; g.k = out; g.act = GEOT_ACT_NONE;
  return rows_product(g, true, dtype, static_cast<hipStream_t>(stream), workspace, workspace_bytes);
}

size_t geot_linear_grad_weight_workspace_bytes(int64_t rows, int64_t in, int64_t out, int dtype) {
  if (bad_size(rows, in, out)) return 0;
  const WeightPlan w = weight_plan(rows, 1, false, out, in, dtype);
  return (size_t)w.parts * (size_t)(in * out + out) * sizeof(float);
}

int geot_linear_grad_weight(const void *dz, const void *x, int64_t ldx, void *dweight, void *dbias, int64_t rows, int64_t in, int64_t out, int dtype,
                            void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_size(rows, in, out) || ldx < 0) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_weight: negative or impossible size");
  if (in > 0 && out > 0 && (!dweight || (rows > 0 && (!dz || !x)))) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_weight: null pointer");
  WeightArgs g{};
  g.p = dz; g.ldp = out; g.np = out; g.q = x; g.ldq = ldx; g.nq = in; g.out = dweight; g.colsum = dbias; g.ns = out; g.sum_p = 1;
  g.groups = {nullptr, 1, rows};
  return weight_product(g, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

int geot_linear_keeps_preactivation(int64_t in, int activation, int residual, int dtype) {
  if (activation == GEOT_ACT_NONE || (activation == GEOT_ACT_RELU && !residual)) return 0;
  return in > (dtype == GEOT_F32 ? 128 : 256);
}

size_t geot_linear_grad_preactivation_workspace_bytes(int64_t rows, int64_t out) {
  return bad_size(rows, out, 0) ? 0 : (size_t)column_parts(rows) * (size_t)out * sizeof(float);
}

int geot_linear_grad_preactivation(const void *dy, const void *z, const void *x, int64_t ldx, const void *weight, const void *bias, void *dz, void *dbias,
                                   int64_t rows, int64_t in, int64_t out, int activation, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_size(rows, in, out) || ldx < 0) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_preactivation: negative or impossible size");
  if (activation < GEOT_ACT_NONE || activation > GEOT_ACT_SILU) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_preactivation: unknown activation");
  if (rows == 0 || out == 0) return GEOT_OK;
  if (!dy || !dz || (!z && in > 0 && (!x || !weight))) return geot_internal_fail(GEOT_EINVAL, "geot_linear_grad_preactivation: null pointer");
  if (dbias && (!workspace || workspace_bytes < geot_linear_grad_preactivation_workspace_bytes(rows, out) || ((uintptr_t)workspace & 15)))
    return geot_internal_fail(GEOT_EWORKSPACE, "geot_linear_grad_preactivation: workspace too small or misaligned");
  RowsArgs g{};
  g.a = x; g.lda = ldx; g.b = weight; g.ldb = in; g.bias = bias; g.y = dz; g.ldy = out;
  g.groups = {nullptr, 1, rows}; g.n = out; g.k = in; g.act = activation;
  float *part = dbias ? static_cast<float *>(workspace) : nullptr;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
  case GEOT_F32: return preactivation_typed<float>(g, dy, z, part, dbias, st);
  case GEOT_F16: return preactivation_typed<f16>(g, dy, z, part, dbias, st);
  case GEOT_BF16: return preactivation_typed<bf16>(g, dy, z, part, dbias, st);
  }
  return geot_internal_fail(GEOT_EUNSUPPORTED, "matrix products take float32, float16 and bfloat16");
}

size_t geot_segment_matmul_workspace_bytes(int64_t rows, int64_t groups, int64_t in, int64_t out, int dtype) {
  return bad_size(rows, in, out) || groups < 0 || groups > 65535 ? 0 : rows_workspace(rows, groups, true, out, in, dtype);
}

int geot_segment_matmul(const void *x, int64_t ldx, const int64_t *ptr, const void *weight, const void *bias, void *y, int64_t rows, int64_t groups,
                        int64_t in, int64_t out, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_size(rows, in, out) || groups < 0 || groups > 65535 || ldx < 0) return geot_internal_fail(GEOT_EINVAL, "geot_segment_matmul: negative or impossible size, or more than 65535 groups");
  if (rows > 0 && out > 0 && (!y || !ptr || (in > 0 && groups > 0 && (!x || !weight)))) return geot_internal_fail(GEOT_EINVAL, "geot_segment_matmul: null pointer");
  RowsArgs g{};
  g.a = x; g.lda = ldx; g.b = weight; g.ldb = out; g.b_group = in * out; g.bias = bias; g.bias_group = out; g.y = y; g.ldy = out;
  g.groups = {ptr, groups, rows}; g.n = out; g.k = in; g.act = GEOT_ACT_NONE;
  return rows_product(g, true, dtype, static_cast<hipStream_t>(stream), workspace, workspace_bytes);
}

size_t geot_segment_matmul_grad_input_workspace_bytes(int64_t rows, int64_t groups, int64_t in, int64_t out, int dtype) {
  return bad_size(rows, in, out) || groups < 0 || groups > 65535 ? 0 : rows_workspace(rows, groups, true, in, out, dtype);
}

int geot_segment_matmul_grad_input(const void *dy, const int64_t *ptr, const void *weight, void *dx, int64_t rows, int64_t groups, int64_t in, int64_t out,
                                   int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_size(rows, in, out) || groups < 0 || groups > 65535) return geot_internal_fail(GEOT_EINVAL, "geot_segment_matmul_grad_input: negative or impossible size, or more than 65535 groups");
  if (rows > 0 && in > 0 && (!dx || !ptr || (out > 0 && groups > 0 && (!dy || !weight)))) return geot_internal_fail(GEOT_EINVAL, "geot_segment_matmul_grad_input: null pointer");
  RowsArgs g{};
  g.a = dy; g.lda = out; g.b = weight; g.ldb = out; g.b_group = in * out; g.y = dx; g.ldy = in;
  g.groups = {ptr, groups, rows}; g.n = in; g.k = out; g.act = GEOT_ACT_NONE;
  return rows_product(g, false, dtype, static_cast<hipStream_t>(stream), workspace, workspace_bytes);
}

size_t geot_segment_matmul_grad_weight_workspace_bytes(int64_t rows, int64_t groups, int64_t in, int64_t out, int dtype) {
  if (bad_size(rows, in, out) || groups < 0 || groups > 65535) return 0;
  const WeightPlan w = weight_plan(rows, groups, true, in, out, dtype);
  return (size_t)w.parts * (size_t)(in * out + out) * sizeof(float);
}

int geot_segment_matmul_grad_weight(const void *x, int64_t ldx, const int64_t *ptr, const void *dy, void *dweight, void *dbias, int64_t rows, int64_t groups,
                                    int64_t in, int64_t out, int dtype, void *workspace, size_t workspace_bytes, void *stream) {
  if (bad_size(rows, in, out) || groups < 0 || groups > 65535 || ldx < 0) return geot_internal_fail(GEOT_EINVAL, "geot_segment_matmul_grad_weight: negative or impossible size, or more than 65535 groups");
  if (groups > 0 && in > 0 && out > 0 && (!ptr || !dweight || (rows > 0 && (!x || !dy)))) return geot_internal_fail(GEOT_EINVAL, "geot_segment_matmul_grad_weight: null pointer");
  WeightArgs g{};
  g.p = x; g.ldp = ldx; g.np = in; g.q = dy; g.ldq = out; g.nq = out; g.out = dweight; g.colsum = dbias; g.ns = out; g.sum_p = 0;
  g.groups = {ptr, groups, rows};
  return weight_product(g, dtype, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

} // extern "C"
