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
// A and B are symmetric: only tiles on and above the diagonal are computed, and written twice; all of them (HALF false) where
// that takes no longer, for few tiles, and spares the scattered mirrored writes. K is split over workgroups where tiles are few, or few are left
// over, and `join` adds the parts.
// The norm is summed in float64: no float's square overflows or vanishes.
//
// Bound: the matrix cores, s²·l + s³ + 2·s²·l flops a step (s, l: the smaller and larger of M, N). Two of 4096 x 4096, us: norm 41,
// split 45 (6.0 TB/s), and a step A 363 - 377 (380 TFLOP/s of the tiles computed), its join 16, B 370 - 387
// and 16, X 690 - 718 (390 TFLOP/s).

#pragma once

#include "tcmi_gemm_f16x2.h"

namespace tcmi {

// S: the sizes of one launch as constants of its text: M, N; KIND of tiles for A and B, AKIND for X; HALF; MP, NP padded to
// whole tiles (SP: the smaller's); GSPLIT, GCHUNKS, GEACH and BSPLIT, BCHUNKS, BEACH: A's and B's split tiles; TALL; BLOCKS of
// the norm; SX, SA, SB exponents of the scales; VEC: N a multiple of 4; a(), b(), c(), eps().
// WS: byte offsets in one matrix's workspace, PER bytes.
template <class S>
struct Orth {
  static_assert(S::SX >= 0 && S::SX <= 15 && S::SA >= 0 && S::SA <= 15 && S::SB >= -60 && S::SB <= 60, "two_to's exponents");
  const float* x;
  float* out;
  char* ws;
  __device__ __forceinline__ Orth(const float* x_, float* out_, float* ws_, uint32_t z)
      : x(x_ + (size_t)z * S::M * S::N), out(out_ + (size_t)z * S::M * S::N), ws(reinterpret_cast<char*>(ws_) + (size_t)z * S::PER) {}
  __device__ __forceinline__ Pairs xs(int which) const { return {ws + (which ? S::X1 : S::X0), S::NP * 4}; }
  __device__ __forceinline__ Pairs as() const { return {ws + S::A, S::SP * 4}; }
  __device__ __forceinline__ Pairs bs() const { return {ws + S::B, S::SP * 4}; }
};

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
      put_pairs(p, row, col, v);
    }
  }
}

// The tile on or above the diagonal that is workgroup `id`'s (of n·(n + 1) / 2): square after square of 8 x 8 tiles, column by
// column of them.
__device__ __forceinline__ TileAt upper_tile(uint32_t id, uint32_t n) {
  constexpr uint32_t SIDE = 8;
  uint32_t t = xcd_run(id, n * (n + 1) / 2);
  for (uint32_t col = 0;; col += SIDE) {
    const uint32_t wide = min(SIDE, n - col);
    const uint32_t above = col * wide, all = above + wide * (wide + 1) / 2;
    if (t >= all) {
      t -= all;
      continue;
    }
    if (t < above) return {t / (SIDE * wide) * SIDE + t % SIDE, col + t % (SIDE * wide) / SIDE};
    t -= above;
    uint32_t c = 0;
    while (t > c) t -= ++c;
    return {col + t, col + c};
  }
}

// v at (row, col ... col + 3) of a symmetric matrix, and mirrored.
template <bool HALF>
__device__ __forceinline__ void put_symmetric(const Pairs& p, const TileAt& tile, uint32_t row, uint32_t col, const f4& v) {
  h4 hi, lo;
  split_pair(v, hi, lo);
  char* at = pair_at(p, row, col);
  *reinterpret_cast<h4*>(at) = hi;
  *reinterpret_cast<h4*>(at + 64) = lo;
  if (!HALF || tile.row == tile.col) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    at = pair_at(p, col + e, row);
    *reinterpret_cast<_Float16*>(at) = hi[e];
    *reinterpret_cast<_Float16*>(at + 64) = lo[e];
  }
}

// 2^e of a normal float, -126 ... 127 (coefficients b and c near 0 take the scales' exponents past 64).
constexpr float two_to(int e) { return __builtin_bit_cast(float, static_cast<uint32_t>(e + 127) << 23); }

// One of the two symmetric products: POLY B = b·A + c·A·A, else A = X·Xᵀ (TALL: Xᵀ·X) of X number FROM.
template <class S, bool POLY, int FROM>
struct Symmetric {
  using P = Tile<S::KIND>;
  static constexpr bool KC = POLY || !S::TALL;
  static constexpr uint32_t SLICES = ((POLY == S::TALL ? S::N : S::M) + 31) / 32;
  static constexpr uint32_t LINES = S::SP / P::ROWS, TILES = S::HALF ? LINES * (LINES + 1) / 2 : LINES * LINES;
  // The last SPLIT tiles are summed in CHUNKS chunks of EACH slices.
  static constexpr uint32_t SPLIT = POLY ? S::BSPLIT : S::GSPLIT, CHUNKS = POLY ? S::BCHUNKS : S::GCHUNKS, EACH = POLY ? S::BEACH : S::GEACH;

  static __device__ __forceinline__ TileAt tile(uint32_t id) { return S::HALF ? upper_tile(id, LINES) : tile_at<P::GROUP>(id, LINES, LINES); }
  // A chunk's sums of fragment (i, 0) of this lane.
  static __device__ __forceinline__ f4* part(const Orth<S>& o, uint32_t split, uint32_t chunk, int i) {
    return reinterpret_cast<f4*>(o.ws + S::PART) + ((size_t)(chunk * SPLIT + split) * (P::TI * P::TJ) + i * P::TJ) * P::THREADS + threadIdx.x;
  }
  static __device__ __forceinline__ void put(const Orth<S>& o, const TileAt& at, uint32_t row, uint32_t col, const f4& v) {
    if constexpr (POLY) {
      put_symmetric<S::HALF>(o.bs(), at, row, col, get_pairs(o.as(), row, col) * (S::b() * two_to(S::SB - S::SA)) + v * (S::c() * two_to(S::SB - 2 * S::SA)));
    } else {
      put_symmetric<S::HALF>(o.as(), at, row, col, v * two_to(S::SA - 2 * S::SX));
    }
  }
};

template <class S, bool POLY, int FROM>
__device__ __forceinline__ void orth_symmetric(const Orth<S>& o, char* lds, uint32_t block) {
  using Y = Symmetric<S, POLY, FROM>;
  using P = typename Y::P;
  uint32_t id = block, k = 0, slices = Y::SLICES, chunk = 0;
  const bool split = Y::SPLIT > 0 && block >= Y::TILES - Y::SPLIT;
  if (split) {
    constexpr uint32_t each = Y::SPLIT > 0 ? Y::SPLIT : 1u;
    chunk = (block - (Y::TILES - Y::SPLIT)) / each;
    id = block - chunk * each;
    k = chunk * Y::EACH;
    slices = min(Y::EACH, Y::SLICES - k);
  }
  const TileAt at = Y::tile(id);
  typename P::Sums acc;
  const Pairs x = POLY ? o.as() : o.xs(FROM);
  P::template sum<Y::KC, Y::KC>(x, x, at, 32 * k, slices, lds, acc);
  if (split) {
#pragma unroll
    for (int i = 0; i < P::TI; ++i)
#pragma unroll
      for (int j = 0; j < P::TJ; ++j) Y::part(o, id - (Y::TILES - Y::SPLIT), chunk, i)[j * P::THREADS] = acc[i][j];
    return;
  }
  P::each(at, acc, [&](uint32_t row, uint32_t col, const f4& v) { Y::put(o, at, row, col, v); });
}

// The sums of the split tiles, chunk after chunk: 16 rows of each wavefront a workgroup.
template <class S, bool POLY>
__device__ __forceinline__ void orth_join(const Orth<S>& o, uint32_t block) {
  using Y = Symmetric<S, POLY, 0>;
  using P = typename Y::P;
  const uint32_t split = block / P::TI;
  const int i = block % P::TI;
  const TileAt at = Y::tile(Y::TILES - Y::SPLIT + split);
  f4 v[P::TJ];
#pragma unroll
  for (int j = 0; j < P::TJ; ++j) v[j] = Y::part(o, split, 0, i)[j * P::THREADS];
#pragma unroll 2
  for (uint32_t c = 1; c < Y::CHUNKS; ++c) {
#pragma unroll
    for (int j = 0; j < P::TJ; ++j) v[j] += Y::part(o, split, c, i)[j * P::THREADS];
  }
#pragma unroll
  for (int j = 0; j < P::TJ; ++j) Y::put(o, at, P::row(at) + 16 * i, P::col(at) + 16 * j, v[j]);
}

// X <- a·X + B·X (TALL: X·B), into the other X, or as the result.
template <class S, int FROM, bool LAST>
__device__ __forceinline__ void orth_apply(const Orth<S>& o, char* lds, uint32_t block) {
  using P = Tile<S::AKIND>;
  const TileAt tile = tile_at<P::GROUP>(block, S::MP / P::ROWS, S::NP / P::COLS);
  typename P::Sums acc;
  const Pairs x = o.xs(FROM), to = o.xs(1 - FROM);
  if constexpr (S::TALL) P::template sum<true, true>(x, o.bs(), tile, 0, (S::N + 31) / 32, lds, acc);
  else P::template sum<true, false>(o.bs(), x, tile, 0, (S::M + 31) / 32, lds, acc);
  P::each(tile, acc, [&](uint32_t row, uint32_t col, const f4& v) {
    const f4 y = get_pairs(x, row, col) * (S::a() * (LAST ? two_to(-S::SX) : 1.f)) + v * (LAST ? two_to(-S::SB - S::SX) : two_to(-S::SB));
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
      put_pairs(to, row, col, y);
    }
  });
}

}  // namespace tcmi
