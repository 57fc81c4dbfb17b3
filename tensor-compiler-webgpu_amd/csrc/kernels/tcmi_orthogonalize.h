// Newton-Schulz steps on a matrix x (M rows, N columns): X = x / (|x| + eps), |x| the
// Frobenius norm, then `steps` times
//   A = X·Xᵀ,   B = b·A + c·A·A,   X <- a·X + B·X
// from the side of the fewer rows; for a tall x (M > N) from the columns' side, A = Xᵀ·X and X <- a·X + X·B.
//
// The products are of pairs of halves (tcmi_gemm_f16x2.h), and so is what stays between the
// kernels: X, A and B are held as pairs (22 bits or more, against 24 of a float), each
// times the power of two that brings its largest possible value (from the largest singular
// value the polynomial reaches, known from its coefficients) below half's. A pair's rounding
// is as large as what the product that reads it leaves out. x keeps its layout:
// a tall X is read transposed by its products, never written so.
//
// A and B are symmetric: only tiles on and above the diagonal are computed, and written twice.
// The norm is summed in float64: no float's square overflows or vanishes.
//
// Bound: the matrix cores, s²·l + s³ + 2·s²·l flops a step (s, l: the smaller and larger of M, N).

#pragma once

#include "tcmi_gemm_f16x2.h"

namespace tcmi {

// S: the sizes of one launch as constants of its text: M, N; MP, NP padded to whole tiles of T·32 (SP: the
// smaller's); TALL; BLOCKS of the norm; SX, SA, SB exponents of the scales; VEC: N a multiple of 4; a(), b(), c(), eps().
// WS: byte offsets in one matrix's workspace, PER bytes.
template <class S>
struct Orth {
  const float* x;
  float* out;
  char* ws;
  __device__ __forceinline__ Orth(const float* x_, float* out_, float* ws_, uint32_t z)
      : x(x_ + (size_t)z * S::M * S::N), out(out_ + (size_t)z * S::M * S::N), ws(reinterpret_cast<char*>(ws_) + (size_t)z * S::PER) {}
  __device__ __forceinline__ Pairs xs(int which) const { return {ws + (which ? S::X1 : S::X0), (size_t)S::MP * S::NP * 2, S::NP * 2}; }
  __device__ __forceinline__ Pairs as() const { return {ws + S::A, (size_t)S::SP * S::SP * 2, S::SP * 2}; }
  __device__ __forceinline__ Pairs bs() const { return {ws + S::B, (size_t)S::SP * S::SP * 2, S::SP * 2}; }
};

__device__ __forceinline__ void put_pair4(const Pairs& p, size_t row, uint32_t col, const h4& hi, const h4& lo) {
  char* at = const_cast<char*>(p.hi) + row * p.ld + 2u * col;
  *reinterpret_cast<h4*>(at) = hi;
  *reinterpret_cast<h4*>(at + p.plane) = lo;
}
__device__ __forceinline__ f4 get_pair4(const Pairs& p, size_t row, uint32_t col) {
  const char* at = p.hi + row * p.ld + 2u * col;
  return join_pair(*reinterpret_cast<const h4*>(at), *reinterpret_cast<const h4*>(at + p.plane));
}

__device__ __forceinline__ double block_sum(double v, double* scratch) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = v;
  __syncthreads();
  return scratch[0] + scratch[1] + scratch[2] + scratch[3];
}

// Partial sums of squares.
template <class S>
__device__ __forceinline__ void orth_norm(const Orth<S>& o, double* scratch, uint32_t block) {
  constexpr size_t n = (size_t)S::M * S::N, step = (size_t)S::BLOCKS * 256;
  double sum = 0.0;
  for (size_t i = (size_t)block * 256 + threadIdx.x; i < n / 4; i += step) {
    const float* p = o.x + 4 * i;
    f4 v;
    if constexpr (n % 4 == 0) v = *reinterpret_cast<const f4*>(p);
    else v = f4{p[0], p[1], p[2], p[3]};
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += static_cast<double>(v[e]) * v[e];
  }
  if (block == 0 && threadIdx.x < n % 4) {
    const double v = o.x[n / 4 * 4 + threadIdx.x];
    sum += v * v;
  }
  sum = block_sum(sum, scratch);
  if (threadIdx.x == 0) reinterpret_cast<double*>(o.ws + S::NORM)[block] = sum;
}

// X = x / (|x| + eps) as pairs, padded with zeros; or (LAST: no steps) as the result.
template <class S, bool LAST>
__device__ __forceinline__ void orth_split(const Orth<S>& o, double* scratch, uint32_t block) {
  double sum = 0.0;
  for (uint32_t i = threadIdx.x; i < S::BLOCKS; i += 256) sum += reinterpret_cast<const double*>(o.ws + S::NORM)[i];
  const double by = 1.0 / (__builtin_sqrt(block_sum(sum, scratch)) + S::eps());
  constexpr uint32_t PER = 4;
  const Pairs p = o.xs(0);
  for (uint32_t u = 0; u < PER; ++u) {
    const size_t i = ((size_t)block * PER + u) * 256 + threadIdx.x;
    const size_t row = i / (S::NP / 4);
    const uint32_t col = i % (S::NP / 4) * 4;
    if (row >= S::MP) return;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    const float* q = o.x + row * S::N + col;
    if (row < S::M) {
      if (S::VEC) {
        if (col < S::N) v = *reinterpret_cast<const f4*>(q);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < S::N) v[e] = q[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = static_cast<float>(v[e] * by);
    if constexpr (LAST) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (row < S::M && col + e < S::N) o.out[row * S::N + col + e] = v[e];
    } else {
      if (row >= S::M || col >= S::N) v = f4{0.f, 0.f, 0.f, 0.f};      // 0 / (0 + 0) is not padding
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = col + e < S::N ? v[e] * static_cast<float>(1u << S::SX) : 0.f;
      h4 hi, lo;
      split_pair(v, hi, lo);
      put_pair4(p, row, col, hi, lo);
    }
  }
}

// The tile on or above the diagonal that is workgroup `id`'s (of n·(n + 1) / 2, each XCD a run of them): column by column.
__device__ __forceinline__ TileAt upper_tile(uint32_t id, uint32_t n) {
  const uint32_t all = n * (n + 1) / 2, per = all / 8u, left = all % 8u, x = id % 8u;
  const uint32_t t = x * per + min(x, left) + id / 8u;
  uint32_t col = static_cast<uint32_t>((__builtin_sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
  while (col * (col + 1) / 2 > t) --col;
  while ((col + 1) * (col + 2) / 2 <= t) ++col;
  return {t - col * (col + 1) / 2, col};
}

// f(row, col, v) of each four columns of a tile that a lane holds.
template <int T, class F>
__device__ __forceinline__ void each_four(const TileAt& tile, f4 (&acc)[T][T], F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t row0 = tile.row * 32 * T + wave / 2 * 16 * T + (lane & 15), col0 = tile.col * 32 * T + wave % 2 * 16 * T + 4 * (lane >> 4);
#pragma unroll
  for (int i = 0; i < T; ++i)
#pragma unroll
    for (int j = 0; j < T; ++j) f(row0 + i * 16, col0 + j * 16, acc[i][j]);
}

// v at (row, col ... col + 3) of a symmetric matrix, and mirrored.
__device__ __forceinline__ void put_symmetric(const Pairs& p, const TileAt& tile, uint32_t row, uint32_t col, const f4& v) {
  h4 hi, lo;
  split_pair(v, hi, lo);
  put_pair4(p, row, col, hi, lo);
  if (tile.row == tile.col) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    char* at = const_cast<char*>(p.hi) + (size_t)(col + e) * p.ld + 2u * row;
    *reinterpret_cast<_Float16*>(at) = hi[e];
    *reinterpret_cast<_Float16*>(at + p.plane) = lo[e];
  }
}

constexpr float two_to(int e) { return e < 0 ? 1.f / static_cast<float>(1ull << -e) : static_cast<float>(1ull << e); }

// A = X·Xᵀ (TALL: Xᵀ·X).
template <class S, int T, int FROM>
__device__ __forceinline__ void orth_gram(const Orth<S>& o, char* lds, uint32_t block) {
  const TileAt tile = upper_tile(block, S::SP / (32 * T));
  f4 acc[T][T];
  gemm_f16x2_sum<2, 2, T, T, !S::TALL, !S::TALL>(o.xs(FROM), o.xs(FROM), tile.row * 32 * T, tile.col * 32 * T, 0, ((S::TALL ? S::M : S::N) + 31) / 32, lds, acc);
  const Pairs p = o.as();
  each_four<T>(tile, acc, [&](uint32_t row, uint32_t col, const f4& v) { put_symmetric(p, tile, row, col, v * two_to(S::SA - 2 * S::SX)); });
}

// B = b·A + c·A·A.
template <class S, int T>
__device__ __forceinline__ void orth_poly(const Orth<S>& o, char* lds, uint32_t block) {
  const TileAt tile = upper_tile(block, S::SP / (32 * T));
  f4 acc[T][T];
  const Pairs a = o.as(), p = o.bs();
  gemm_f16x2_sum<2, 2, T, T, true, true>(a, a, tile.row * 32 * T, tile.col * 32 * T, 0, ((S::TALL ? S::N : S::M) + 31) / 32, lds, acc);
  each_four<T>(tile, acc, [&](uint32_t row, uint32_t col, const f4& v) {
    put_symmetric(p, tile, row, col, get_pair4(a, row, col) * (S::b() * two_to(S::SB - S::SA)) + v * (S::c() * two_to(S::SB - 2 * S::SA)));
  });
}

// X <- a·X + B·X (TALL: X·B), into the other X, or as the result.
template <class S, int T, int FROM, bool LAST>
__device__ __forceinline__ void orth_apply(const Orth<S>& o, char* lds, uint32_t block) {
  const TileAt tile = tile_at(block, S::MP / (32 * T), S::NP / (32 * T));
  f4 acc[T][T];
  const Pairs x = o.xs(FROM), to = o.xs(1 - FROM);
  if constexpr (S::TALL) gemm_f16x2_sum<2, 2, T, T, true, true>(x, o.bs(), tile.row * 32 * T, tile.col * 32 * T, 0, (S::N + 31) / 32, lds, acc);
  else gemm_f16x2_sum<2, 2, T, T, true, false>(o.bs(), x, tile.row * 32 * T, tile.col * 32 * T, 0, (S::M + 31) / 32, lds, acc);
  each_four<T>(tile, acc, [&](uint32_t row, uint32_t col, const f4& v) {
    const f4 y = get_pair4(x, row, col) * (S::a() * (LAST ? two_to(-S::SX) : 1.f)) + v * (LAST ? two_to(-S::SB - S::SX) : two_to(-S::SB));
    if constexpr (LAST) {
      if (row >= S::M) return;
      float* q = o.out + (size_t)row * S::N + col;
      if (S::VEC) {
        if (col < S::N) *reinterpret_cast<f4*>(q) = y;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < S::N) q[e] = y[e];
      }
    } else {
      h4 hi, lo;
      split_pair(y, hi, lo);
      put_pair4(to, row, col, hi, lo);
    }
  });
}

}  // namespace tcmi
