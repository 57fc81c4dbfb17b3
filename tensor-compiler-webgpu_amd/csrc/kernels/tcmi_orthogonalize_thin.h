// Newton-Schulz steps (tcmi_orthogonalize.h: the formulas) on a matrix x with a side of at most 64: every step multiplies X by
// a polynomial of A = X·Xᵀ, so all of them together are Q·x (tall: x·Q) with Q made of small matrices only,
//   P = a + b·A + c·A²,   Q <- P·Q,   A <- P·A·P,
// all of them polynomials of the first A, symmetric, and interchangeable.
//
//   gram    x·xᵀ (tall: xᵀ·x), the long side over workgroups and their wavefronts
//   sum     those parts in order, where there are more than a few
//   iterate the norm (the root of A's trace) and the steps, a workgroup a matrix
//   apply   Q·x
//
// All of it is in float64 (16 x 16 x 4 matrix instructions): A holds the squares of the singular values, of which a float would lose the
// smaller half, and the steps enlarge those by a^steps. One rounding to float32 is left, of the result.
// Of the symmetric products the tiles on and above the diagonal are computed, and both halves written.
//
// Bound: launches, and `iterate`, a workgroup's chain of products and barriers: of sides up to 64 40 us for 5 steps (gram 6.0, sum
// 3.6, apply 4.8 of 64 x 4096), up to 32 11.5 (3.5, 2.8, 4.1 of 32 x 2416), up to 16 8.2. Steps on X itself by products of pairs take
// three launches a step that each read the long side.

#pragma once

#include "tcmi_orthogonalize.h"
#include "tcmi_loss_narrow.h"

namespace tcmi {

typedef double d2 __attribute__((ext_vector_type(2)));
typedef double d4 __attribute__((ext_vector_type(4)));

// S, beside M, N, TALL, VEC: T (1, 2, 4) tiles of 16 in the short side; KC of the long side a chunk, CHUNKS, SUMMED (by `sum`);
// STEPS; a(), b(), c(), eps() in float64. WS: PART, SUM, Q.
template <class S>
struct Thin {
  const float* x;
  float* out;
  char* ws;
  static constexpr uint32_t SP = 16 * S::T, PAIRS = S::T * (S::T + 1) / 2, LD = SP + 2;
  __device__ __forceinline__ Thin(const float* x_, float* out_, float* ws_, uint32_t z)
      : x(x_ + (size_t)z * S::M * S::N), out(out_ + (size_t)z * S::M * S::N), ws(reinterpret_cast<char*>(ws_) + (size_t)z * S::PER) {}
  __device__ __forceinline__ double* at(size_t off) const { return reinterpret_cast<double*>(ws + off); }
  // The row of A that line m of tile j is: a tall x is loaded by T neighbouring columns.
  static __device__ __forceinline__ uint32_t line(uint32_t j, uint32_t m) { return S::TALL ? S::T * m + j : 16 * j + m; }
  // The tile (i, j), i <= j, of pair p.
  static __device__ __forceinline__ void pair(uint32_t p, uint32_t& i, uint32_t& j) {
    j = p >= 6 ? 3u : p >= 3 ? 2u : p >= 1 ? 1u : 0u;
    i = p - j * (j + 1) / 2;
  }
};

template <class S>
__device__ __forceinline__ void thin_gram(const Thin<S>& o, double* lds, uint32_t chunk) {
  using H = Thin<S>;
  constexpr int T = S::T;
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t k0 = chunk * S::KC + wave * (S::KC / 4);
  d4 acc[H::PAIRS];
#pragma unroll
  for (int p = 0; p < H::PAIRS; ++p) acc[p] = d4{0., 0., 0., 0.};
  // 16 of the long side at a time: v[j][i] of line t of tile j, at k + 4q + i (tall: at k + 4i + q).
  auto load = [&](uint32_t k, f4 (&v)[T]) __attribute__((always_inline)) {
    if constexpr (S::TALL) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t r = k + 4 * i + q;
        const float* p = o.x + (size_t)min(r, S::M - 1) * S::N;
        if constexpr (T == 4) {
          const f4 y = raw_four<S::VEC>(p, 4 * t, S::N);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j][i] = y[j];
        } else if constexpr (T == 2) {
          const f2 y = raw_two(p, 2 * t, S::N);
          v[0][i] = y[0];
          v[1][i] = y[1];
        } else {
          v[0][i] = p[min(t, S::N - 1)];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < T; ++j) v[j] = raw_four<S::VEC>(o.x + (size_t)min(16 * j + t, S::M - 1) * S::N, k + 4 * q, S::N);
    }
  };
  auto place = [&](uint32_t k, f4 (&v)[T]) __attribute__((always_inline)) {
    if constexpr (S::TALL) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = k + 4 * i + q < S::M;
        if constexpr (T == 4) {
          const f4 y = placed<S::VEC>(f4{v[0][i], v[1][i], v[2][i], v[3][i]}, 4 * t, S::N);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j][i] = in ? y[j] : 0.f;
        } else if constexpr (T == 2) {
          const f2 y = placed_two(f2{v[0][i], v[1][i]}, 2 * t, S::N);
          v[0][i] = in ? y[0] : 0.f;
          v[1][i] = in ? y[1] : 0.f;
        } else {
          v[0][i] = in && t < S::N ? v[0][i] : 0.f;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < T; ++j) {
        v[j] = placed<S::VEC>(v[j], k + 4 * q, S::N);
        if (16 * j + t >= S::M) v[j] = f4{0.f, 0.f, 0.f, 0.f};
      }
    }
  };
  f4 v[T];
  load(k0, v);
  for (uint32_t k = k0; k < k0 + S::KC / 4; k += 16) {
    f4 next[T];
    load(k + 16, next);
    __builtin_amdgcn_sched_barrier(0);
    place(k, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      double d[T];
#pragma unroll
      for (int j = 0; j < T; ++j) d[j] = v[j][i];
#pragma unroll
      for (int j2 = 0; j2 < T; ++j2)
#pragma unroll
        for (int j1 = 0; j1 <= j2; ++j1) {
          d4& c = acc[j2 * (j2 + 1) / 2 + j1];
          c = __builtin_amdgcn_mfma_f64_16x16x4f64(d[j1], d[j2], c, 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < T; ++j) v[j] = next[j];
  }
#pragma unroll
  for (int p = 0; p < H::PAIRS; ++p) *reinterpret_cast<d4*>(lds + ((wave * H::PAIRS + p) * 64 + lane) * 4) = acc[p];
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < H::PAIRS * 256; i += 256) {
    double sum = lds[i];
#pragma unroll
    for (uint32_t w = 1; w < 4; ++w) sum += lds[w * H::PAIRS * 256 + i];
    o.at(S::PART)[(size_t)chunk * H::PAIRS * 256 + i] = sum;
  }
}

// 32 sums a workgroup: every eighth chunk a thread, then those eight.
template <class S>
__device__ __forceinline__ void thin_sum(const Thin<S>& o, double* scratch, uint32_t block) {
  const uint32_t i = block * 32 + threadIdx.x % 32, p = threadIdx.x / 32;
  double sum = 0.0;
#pragma unroll 4
  for (uint32_t c = p; c < S::CHUNKS; c += 8) sum += o.at(S::PART)[(size_t)c * Thin<S>::PAIRS * 256 + i];
  scratch[threadIdx.x] = sum;
  __syncthreads();
  if (p == 0) {
    for (uint32_t k = 1; k < 8; ++k) sum += scratch[32 * k + threadIdx.x];
    o.at(S::SUM)[i] = sum;
  }
}

// Tile (i, j) of X·Y for symmetric X and Y of SP rows in LDS: rows 16i + q + 4r, column 16j + t.
template <class H>
__device__ __forceinline__ d4 thin_product(const double* X, const double* Y, uint32_t i, uint32_t j) {
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4;
  const double* x = X + (16 * i + t) * H::LD + 2 * q;
  const double* y = Y + (16 * j + t) * H::LD + 2 * q;
  d4 acc = {0., 0., 0., 0.};
#pragma unroll
  for (uint32_t k = 0; k < H::SP; k += 8) {
    const d2 a = *reinterpret_cast<const d2*>(x + k), b = *reinterpret_cast<const d2*>(y + k);
    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[0], b[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[1], b[1], acc, 0, 0, 0);
  }
  return acc;
}

// v at (row, col) and (col, row); of a diagonal tile by the lane above the diagonal alone: the other's may differ in its last bits.
template <class H>
__device__ __forceinline__ void thin_put(double* X, bool diagonal, uint32_t row, uint32_t col, double v) {
  if (diagonal && row > col) return;
  X[row * H::LD + col] = v;
  X[col * H::LD + row] = v;
}

// lds: A, P, P·A and Q, of SP rows of LD each.
template <class S>
__device__ __forceinline__ void thin_iterate(const Thin<S>& o, double* lds) {
  using H = Thin<S>;
  constexpr uint32_t WAVES = 8, THREADS = 64 * WAVES, SIZE = H::SP * H::LD, OWN = (H::PAIRS + WAVES - 1) / WAVES;
  double *const A = lds, *const P = lds + SIZE, *const PA = P + SIZE, *const Q = PA + SIZE;
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (uint32_t i = threadIdx.x; i < H::PAIRS * 256; i += THREADS) {
    double sum;
    if constexpr (S::SUMMED) {
      sum = o.at(S::SUM)[i];
    } else {
      sum = 0.0;
      for (uint32_t c = 0; c < S::CHUNKS; ++c) sum += o.at(S::PART)[(size_t)c * H::PAIRS * 256 + i];
    }
    uint32_t ti, tj;
    H::pair(i / 256, ti, tj);
    const uint32_t l = i % 256 / 4, row = H::line(ti, l / 16 + 4 * (i % 4)), col = H::line(tj, l % 16);
    thin_put<H>(A, ti == tj, row, col, sum);
  }
  __syncthreads();
  double trace = lane < H::SP ? A[lane * H::LD + lane] : 0.0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) trace += __shfl_xor(trace, off, 64);
  const double by = 1.0 / (__builtin_sqrt(trace) + S::eps()), by2 = by * by;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < H::SP * H::SP; i += THREADS) {
    const uint32_t row = i / H::SP, col = i % H::SP;
    A[row * H::LD + col] *= by2;
    Q[row * H::LD + col] = row == col ? by : 0.0;
  }
  __syncthreads();
  for (uint32_t step = 0; step < S::STEPS; ++step) {
    for (uint32_t p = wave; p < H::PAIRS; p += WAVES) {
      uint32_t i, j;
      H::pair(p, i, j);
      const d4 v = thin_product<H>(A, A, i, j);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t row = 16 * i + q + 4 * r, col = 16 * j + t;
        const double y = S::c() * v[r] + S::b() * A[row * H::LD + col] + (row == col ? S::a() : 0.0);
        thin_put<H>(P, i == j, row, col, y);
      }
    }
    __syncthreads();
    // Q's tiles are kept until every wavefront has read the old ones.
    d4 next[OWN];
#pragma unroll
    for (uint32_t u = 0; u < OWN; ++u) {
      const uint32_t p = wave + u * WAVES;
      if (p < H::PAIRS) {
        uint32_t i, j;
        H::pair(p, i, j);
        next[u] = thin_product<H>(P, Q, i, j);
      }
    }
    if (step + 1 < S::STEPS) {
      for (uint32_t p = (wave + H::PAIRS) % WAVES; p < H::PAIRS; p += WAVES) {
        uint32_t i, j;
        H::pair(p, i, j);
        const d4 v = thin_product<H>(P, A, i, j);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t row = 16 * i + q + 4 * r, col = 16 * j + t;
          thin_put<H>(PA, i == j, row, col, v[r]);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t u = 0; u < OWN; ++u) {
      const uint32_t p = wave + u * WAVES;
      if (p < H::PAIRS) {
        uint32_t i, j;
        H::pair(p, i, j);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t row = 16 * i + q + 4 * r, col = 16 * j + t;
          thin_put<H>(Q, i == j, row, col, next[u][r]);
        }
      }
    }
    if (step + 1 < S::STEPS) {
      for (uint32_t p = wave; p < H::PAIRS; p += WAVES) {
        uint32_t i, j;
        H::pair(p, i, j);
        const d4 v = thin_product<H>(P, PA, i, j);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t row = 16 * i + q + 4 * r, col = 16 * j + t;
          thin_put<H>(A, i == j, row, col, v[r]);
        }
      }
    }
    __syncthreads();
  }
  for (uint32_t i = threadIdx.x; i < H::SP * H::SP; i += THREADS) o.at(S::Q)[i] = Q[i / H::SP * H::LD + i % H::SP];
}

// Wide: a wavefront 16 rows by 64 columns of Q·x; tall: 16 rows of x·Q. Four a workgroup.
template <class S>
__device__ __forceinline__ void thin_apply(const Thin<S>& o, uint32_t block) {
  using H = Thin<S>;
  constexpr int T = S::T;
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, task = block * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const double* Q = o.at(S::Q);
  if constexpr (S::TALL) {
    // k = 16u + 4q + i; line m of Q's tile j is its row 16j + 4·(m % 4) + m / 4, so that a lane's four results are neighbours.
    const uint32_t row = task * 16 + t;
    if (task * 16 >= S::M) return;
    const float* x = o.x + (size_t)min(row, S::M - 1) * S::N;
    f4 v[T];
#pragma unroll
    for (int u = 0; u < T; ++u) v[u] = four_of<S::VEC>(x, 16 * u + 4 * q, S::N);
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const double* p = Q + (16 * j + 4 * (t & 3) + (t >> 2)) * H::SP + 4 * q;
      d4 acc = {0., 0., 0., 0.};
#pragma unroll
      for (int u = 0; u < T; ++u) {
        const d2 a = *reinterpret_cast<const d2*>(p + 16 * u), b = *reinterpret_cast<const d2*>(p + 16 * u + 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(i < 2 ? a[i] : b[i - 2], static_cast<double>(v[u][i]), acc, 0, 0, 0);
      }
      if (row < S::M) {
        put_four_of<S::VEC>(o.out + (size_t)row * S::N, 16 * j + 4 * q, S::N,
                            f4{static_cast<float>(acc[0]), static_cast<float>(acc[1]), static_cast<float>(acc[2]), static_cast<float>(acc[3])});
      }
    }
  } else {
    const uint32_t j = task % T, col = task / T * 64;
    if (col >= S::N) return;
    f4 v[4 * T];
    double a[4 * T];
#pragma unroll
    for (int u = 0; u < 4 * T; ++u) v[u] = raw_four<S::VEC>(o.x + (size_t)min(4 * u + q, S::M - 1) * S::N, col + 4 * t, S::N);
#pragma unroll
    for (int u = 0; u < 4 * T; ++u) a[u] = Q[(16 * j + t) * H::SP + 4 * u + q];
    d4 acc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = d4{0., 0., 0., 0.};
#pragma unroll
    for (int u = 0; u < 4 * T; ++u) {
      f4 y = placed<S::VEC>(v[u], col + 4 * t, S::N);
      if (4 * u + q >= S::M) y = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_amdgcn_mfma_f64_16x16x4f64(a[u], static_cast<double>(y[e]), acc[e], 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint32_t row = 16 * j + q + 4 * r;
      if (row < S::M) {
        put_four_of<S::VEC>(o.out + (size_t)row * S::N, col + 4 * t, S::N,
                            f4{static_cast<float>(acc[0][r]), static_cast<float>(acc[1][r]), static_cast<float>(acc[2][r]), static_cast<float>(acc[3][r])});
      }
    }
  }
}

}  // namespace tcmi
