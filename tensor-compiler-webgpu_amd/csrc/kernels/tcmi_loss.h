// Softmax cross entropy of h·W + bias against class indices, and its gradients, without
// keeping the logits: the rows are taken a piece at a time, the logits of one piece in the
// workspace.
//
// With z = h·W + bias [N, V], M the row's maximum and s = sum of exp(z - M),
//   loss = M - z[target] + log s,   G = w·(exp(z - M) / s - onehot(target)),
//   dh = G·Wᵀ,   dW = hᵀ·G,   dbias = column sums of G
// (w: the loss's cotangent). A row whose target is no whole number in 0..V-1 is left out: loss 0, G 0,
// its h counted as 0. With gradients that is three products: the logits are formed once, where
// a pass over them that keeps only s would form them again for G.
//
// All products are of pairs of halves (tcmi_gemm_f16x2.h). h, W and G are split once each, W
// and h times a power of two from their largest finite magnitude, G times one from the largest
// |w|; every operand is read from the one layout it is written in.
//
//   maxima   partial maxima of |h|, |W| and |w|
//   split    h's and W's planes, padded with zeros to tiles of 128 (k to 32)
//   logits   z tile by tile; each wavefront's 64 columns of a row leave (maximum, sum of
//            exponentials), and z itself where G will be formed
//   join     a row's pairs joined in order; the losses; (M, 1/s) a row
//   spread   G's planes, and the column sums of a few rows each
//   dh, dW   products, their K split over workgroups where tiles are few; dW is added
//            up over the pieces
// The piece that a kernel works on is counted in the workspace (two slots, so that no kernel
// reads the one it writes), which keeps one kernel text and one argument block for all pieces.
//
// Bound: the matrix cores (6·N·d·V flops with gradients, 2·N·d·V without).

#pragma once

#include "tcmi_gemm_f16x2.h"

namespace tcmi {

// e^x with the product's rounding made up for: 2^t·(1 + ln 2·(x·log2 e - t)), t = x·log2 e rounded.
// Two roundings and the exponential unit's 1 ulp, at any x (op_exp loses |x|·2^-24).
__device__ __forceinline__ float exp_full(float x) {
  const float t = x * 1.4426950408889634f;
  const float e = __builtin_amdgcn_exp2f(t);
  const float low = fmaf(x, 1.9259629911266175e-8f, fmaf(x, 1.4426950408889634f, -t));
  const float r = fmaf(e * low, 0.69314718055994531f, e);
  return __builtin_isfinite(t) ? r : e;   // exp(-inf) = 0, exp(inf) = inf; NaN stays
}

// The counters at the workspace's start.
struct LossState {
  uint32_t piece, current;         // the next piece; the one being worked on
  int h, w, g;                     // exponents of the operands' scales
};

// S: the sizes of one launch as constants of its text: N, D, V; NP rows a piece, PIECES of them; DP, VP: d and V padded to
// 128; BIAS; BLOCKS partial maxima a tensor; RB rows a workgroup of `spread`; VECD, VECV: d, V multiples of 4.
// WS: byte offsets in the workspace.
template <class S>
struct Loss {
  const float *h, *W, *t, *bias, *w;
  char* ws;
  __device__ __forceinline__ LossState* state() const { return reinterpret_cast<LossState*>(ws); }
  __device__ __forceinline__ float* at(size_t off) const { return reinterpret_cast<float*>(ws + off); }
  __device__ __forceinline__ Pairs h_planes() const { return {ws + S::HP, (size_t)S::NP * S::PIECES * S::DP * 2, S::DP * 2}; }
  __device__ __forceinline__ Pairs w_planes() const { return {ws + S::WP, (size_t)S::DP * S::VP * 2, S::VP * 2}; }
  __device__ __forceinline__ Pairs g_planes() const { return {ws + S::GP, (size_t)S::NP * S::VP * 2, S::VP * 2}; }
  // Whether row r counts, and its target.
  static __device__ __forceinline__ bool is_class(float c) { return c >= 0.f && c < static_cast<float>(S::V) && c == __builtin_floorf(c); }
  __device__ __forceinline__ bool kept(uint32_t r) const { return r < S::N && is_class(t[r]); }
};

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < TCMI_INF ? a : 0.f;      // NaN too
}
// The exponent s of the scale 2^s that brings values up to `top` below 2^15.
__device__ __forceinline__ int scale_of(float top) {
  const int e = top > 0.f ? __builtin_amdgcn_frexp_expf(top) : 15;
  return 15 - e < 126 ? 15 - e : 126;
}

template <class S, bool GRAD>
__device__ __forceinline__ void loss_maxima(const Loss<S>& L, float* scratch, uint32_t block) {
  float top = 0.f;
  if (block < S::BLOCKS) {
    for (uint32_t r = block * 4 + threadIdx.x / 64; r < S::N; r += S::BLOCKS * 4) {
      if (!L.kept(r)) continue;
      const float* x = L.h + (size_t)r * S::D;
      if constexpr (S::VECD) {
        for (uint32_t c = threadIdx.x % 64 * 4; c < S::D; c += 256) {
          const f4 v = *reinterpret_cast<const f4*>(x + c);
          top = fmaxf(fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3]))), top);
        }
      } else {
        for (uint32_t c = threadIdx.x % 64; c < S::D; c += 64) top = fmaxf(top, finite_abs(x[c]));
      }
    }
  } else if (block < 2 * S::BLOCKS) {
    constexpr size_t n = (size_t)S::D * S::V, n4 = n / 4;
    const size_t i0 = (size_t)(block - S::BLOCKS) * 256 + threadIdx.x;
    constexpr size_t step = (size_t)S::BLOCKS * 256;
    for (size_t i = i0; i < n4; i += step) {
      const f4 v = reinterpret_cast<const f4*>(L.W)[i];
      top = fmaxf(fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3]))), top);
    }
    if (i0 < n % 4) top = fmaxf(top, finite_abs(L.W[4 * n4 + i0]));
  } else if constexpr (GRAD) {
    for (uint32_t r = threadIdx.x; r < S::N; r += 256)
      if (L.kept(r)) top = fmaxf(top, finite_abs(L.w[r]));
  }
  top = block_reduce<true, 256>(top, scratch);
  if (threadIdx.x == 0) L.at(S::MAXIMA)[block] = top;
}

// Four floats of row `r` of a [rows, cols] matrix from column c on, those outside it 0.
template <bool VEC>
__device__ __forceinline__ f4 four(const float* x, size_t r, uint32_t rows, uint32_t c, uint32_t cols) {
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (r >= rows) return v;
  const float* p = x + r * cols;
  if (VEC) {
    if (c < cols) v = *reinterpret_cast<const f4*>(p + c);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < cols) v[e] = p[c + e];
  }
  return v;
}
__device__ __forceinline__ void put_pairs(const Pairs& p, size_t row, uint32_t col, const f4& v) {
  h4 hi, lo;
  split_pair(v, hi, lo);
  char* at = const_cast<char*>(p.hi) + row * p.ld + 2u * col;
  *reinterpret_cast<h4*>(at) = hi;
  *reinterpret_cast<h4*>(at + p.plane) = lo;
}

constexpr uint32_t SPLIT_PER = 16;      // groups of four that a thread of `split` takes

template <class S, bool GRAD>
__device__ __forceinline__ void loss_split(const Loss<S>& L, float* scratch, uint32_t block) {
  constexpr size_t HG = (size_t)S::NP * S::PIECES * S::DP / 4, WG = (size_t)S::DP * S::VP / 4;
  constexpr uint32_t HB = (HG + 256 * SPLIT_PER - 1) / (256 * SPLIT_PER);
  const bool of_w = block >= HB;
  float top = 0.f;
  for (uint32_t i = threadIdx.x; i < S::BLOCKS; i += 256) top = fmaxf(top, L.at(S::MAXIMA)[(of_w ? S::BLOCKS : 0u) + i]);
  const int s = scale_of(block_reduce<true, 256>(top, scratch));
  if (threadIdx.x == 0) {
    LossState* st = L.state();
    if (block == 0) {
      st->piece = 0u;
      st->h = s;
      if constexpr (GRAD) st->g = scale_of(L.at(S::MAXIMA)[2 * S::BLOCKS]);
    }
    if (block == HB) st->w = s;
  }
  const Pairs p = of_w ? L.w_planes() : L.h_planes();
  for (uint32_t u = 0; u < SPLIT_PER; ++u) {
    const size_t i = ((size_t)(of_w ? block - HB : block) * SPLIT_PER + u) * 256 + threadIdx.x;
    f4 v;
    size_t row;
    uint32_t col;
    if (of_w) {
      if (i >= WG) return;
      row = i / (S::VP / 4);
      col = i % (S::VP / 4) * 4;
      v = four<S::VECV>(L.W, row, S::D, col, S::V);
    } else {
      if (i >= HG) return;
      row = i / (S::DP / 4);
      col = i % (S::DP / 4) * 4;
      v = f4{0.f, 0.f, 0.f, 0.f};
      if (L.kept(row)) v = four<S::VECD>(L.h, row, S::N, col, S::D);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], s);
    put_pairs(p, row, col, v);
  }
}

// One tile of the piece's logits.
template <class S, bool KEEP>
__device__ __forceinline__ void loss_logits(const Loss<S>& L, char* lds, uint32_t block) {
  LossState* st = L.state();
  const uint32_t piece = st->piece;
  if (block == 0 && threadIdx.x == 0) st->current = piece;
  const TileAt tile = tile_at(block, S::NP / 128, S::VP / 128);
  Pairs a = L.h_planes();
  a.hi += (size_t)piece * S::NP * a.ld;
  f4 acc[4][4];
  gemm_f16x2_sum<2, 2, 4, 4, true, false>(a, L.w_planes(), tile.row * 128, tile.col * 128, 0, (S::D + 31) / 32, lds, acc);
  const int back = -(st->h + st->w);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t16 = lane & 15, q = lane >> 4;
  const uint32_t col0 = tile.col * 128 + wave % 2 * 64 + 4 * q, row0 = tile.row * 128 + wave / 2 * 64 + t16;
  f4 b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = S::BIAS ? four<S::VECV>(L.bias, 0, 1, col0 + j * 16, S::V) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = row0 + i * 16, r = piece * S::NP + row;
    const float target = r < S::N ? L.t[r] : -1.f;
    float m = -TCMI_INF;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t col = col0 + j * 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z = ldexpf(acc[i][j][e], back) + b[j][e];
        acc[i][j][e] = z;
        if (col + e < S::V) {
          m = red_max(m, z);
          if (static_cast<float>(col + e) == target) L.at(S::PICKED)[row] = z;
        }
      }
      if constexpr (KEEP) *reinterpret_cast<f4*>(L.at(S::Z) + (size_t)row * S::VP + col) = acc[i][j];
    }
    m = quad16_reduce<true>(m);
    const float shift = m == -TCMI_INF ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (col0 + j * 16 + e < S::V) s += exp_full(acc[i][j][e] - shift);
    s = quad16_reduce<false>(s);
    if (q == 0) reinterpret_cast<float2*>(L.at(S::STATS))[(size_t)(tile.col * 2 + wave % 2) * S::NP + row] = make_float2(m, s);
  }
}

// The statistics of 16 rows, 16 threads a row.
template <class S, bool LOSS, bool LAST>
__device__ __forceinline__ void loss_join(const Loss<S>& L, float* out, float2* scratch, uint32_t block) {
  LossState* st = L.state();
  const uint32_t piece = st->current;
  constexpr uint32_t PARTS = S::VP / 64;
  const uint32_t row = block * 16 + threadIdx.x % 16, k0 = threadIdx.x / 16;
  const float2* stats = reinterpret_cast<const float2*>(L.at(S::STATS)) + row;
  float m = -TCMI_INF, s = 0.f;
  auto add = [&](const float2 x) {
    const float top = red_max(m, x.x), shift = top == -TCMI_INF ? 0.f : top;
    s = s * exp_full(m - shift) + x.y * exp_full(x.x - shift);
    m = top;
  };
  for (uint32_t k = k0; k < PARTS; k += 16) add(stats[(size_t)k * S::NP]);
  scratch[threadIdx.x] = make_float2(m, s);
  __syncthreads();
  if (k0 == 0) {
    for (uint32_t k = 1; k < 16; ++k) add(scratch[k * 16 + threadIdx.x]);
    reinterpret_cast<float2*>(L.at(S::ROWS))[row] = make_float2(m, 1.f / s);
    const uint32_t r = piece * S::NP + row;
    if constexpr (LOSS) {
      if (r < S::N) out[r] = L.kept(r) ? (m - L.at(S::PICKED)[row]) + op_log(s) : 0.f;
    }
  }
  if constexpr (LAST) {
    if (block == 0 && threadIdx.x == 0) st->piece = piece + 1;
  }
}

// RB rows of 1024 columns of G.
template <class S, bool PLANES, bool SUMS>
__device__ __forceinline__ void loss_spread(const Loss<S>& L, f4* rows, uint32_t bx, uint32_t by) {
  const LossState* st = L.state();
  const uint32_t piece = st->current;
  const int sg = st->g;
  const uint32_t row0 = by * S::RB;
  if (threadIdx.x < S::RB) {
    const uint32_t row = row0 + threadIdx.x, r = piece * S::NP + row;
    f4 c = {0.f, 0.f, 0.f, -1.f};       // M, w/s and w in G's scale, the target (-1: the row is left out)
    if (L.kept(r)) {
      const float2 x = reinterpret_cast<const float2*>(L.at(S::ROWS))[row];
      const float w = ldexpf(L.w[r], sg);
      c = f4{x.x, w * x.y, w, L.t[r]};
    }
    rows[threadIdx.x] = c;
  }
  __syncthreads();
  const uint32_t col = bx * 1024 + threadIdx.x * 4;
  if (col >= S::VP) return;
  const Pairs p = L.g_planes();
  f4 sum = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t k = 0; k < S::RB; ++k) {
    const f4 c = rows[k];
    f4 g = {0.f, 0.f, 0.f, 0.f};
    if (c[3] >= 0.f) {
      const f4 z = *reinterpret_cast<const f4*>(L.at(S::Z) + (size_t)(row0 + k) * S::VP + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (col + e < S::V) g[e] = exp_full(z[e] - c[0]) * c[1] - (static_cast<float>(col + e) == c[3] ? c[2] : 0.f);
      }
    }
    if constexpr (SUMS) sum += g;
    if constexpr (PLANES) put_pairs(p, row0 + k, col, g);
  }
  if constexpr (SUMS) *reinterpret_cast<f4*>(L.at(S::SUMS) + (size_t)by * S::VP + col) = sum;
}

// C rows x cols = the product's, scaled back by 2^back, added to what is there (ADD); chunk `z` of K to its own
// partial [DPAD, cpad] where K is split.
template <bool VEC>
__device__ __forceinline__ void put_four(float* out, size_t row, uint32_t rows, uint32_t col, uint32_t cols, f4 v, bool add) {
  if (row >= rows) return;
  float* p = out + row * cols + col;
  if (VEC) {
    if (col < cols) {
      if (add) v += *reinterpret_cast<const f4*>(p);
      *reinterpret_cast<f4*>(p) = v;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < cols) p[e] = add ? p[e] + v[e] : v[e];
  }
}

// A tile of dh (rows of the piece): K = V in CHUNKS chunks of KC slices.
template <class S>
__device__ __forceinline__ void loss_dh(const Loss<S>& L, float* out, char* lds, uint32_t block) {
  const LossState* st = L.state();
  const uint32_t piece = st->current;
  constexpr uint32_t TILES = S::NP / 128 * (S::DP / 128);
  const uint32_t chunk = block / TILES;
  const TileAt tile = tile_at(block % TILES, S::NP / 128, S::DP / 128);
  f4 acc[4][4];
  const uint32_t first = chunk * S::HK, left = S::VP / 32 - first;
  gemm_f16x2_sum<2, 2, 4, 4, true, true>(L.g_planes(), L.w_planes(), tile.row * 128, tile.col * 128, first * 32, left < S::HK ? left : S::HK, lds, acc);
  const int back = -(st->g + st->w);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t col0 = tile.col * 128 + wave % 2 * 64 + 4 * (lane >> 4), row0 = tile.row * 128 + wave / 2 * 64 + (lane & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t row = row0 + i * 16, col = col0 + j * 16;
      f4 v = acc[i][j];
      if constexpr (S::HCHUNKS > 1) {
        *reinterpret_cast<f4*>(L.at(S::HPART) + ((size_t)chunk * S::NP + row) * S::DP + col) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], back);
        put_four<S::VECD>(out, (size_t)piece * S::NP + row, S::N, col, S::D, v, false);
      }
    }
}
// The chunks of dh added in order.
template <class S>
__device__ __forceinline__ void loss_dh_sum(const Loss<S>& L, float* out, uint32_t block) {
  const LossState* st = L.state();
  const uint32_t i = block * 256 + threadIdx.x, row = i / (S::DP / 4), col = i % (S::DP / 4) * 4;
  if (row >= S::NP) return;
  const int back = -(st->g + st->w);
  f4 v = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t c = 0; c < S::HCHUNKS; ++c) v += *reinterpret_cast<const f4*>(L.at(S::HPART) + ((size_t)c * S::NP + row) * S::DP + col);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], back);
  put_four<S::VECD>(out, (size_t)st->current * S::NP + row, S::N, col, S::D, v, false);
}

// A tile of dW: K = the piece's rows in CHUNKS chunks of WK slices.
template <class S>
__device__ __forceinline__ void loss_dw(const Loss<S>& L, float* out, char* lds, uint32_t block) {
  const LossState* st = L.state();
  const uint32_t piece = st->current;
  constexpr uint32_t TILES = S::DP / 128 * (S::VP / 128);
  const uint32_t chunk = block / TILES;
  const TileAt tile = tile_at(block % TILES, S::DP / 128, S::VP / 128);
  Pairs a = L.h_planes();
  a.hi += (size_t)piece * S::NP * a.ld;
  f4 acc[4][4];
  const uint32_t first = chunk * S::WK, left = S::NP / 32 - first;
  gemm_f16x2_sum<2, 2, 4, 4, false, false>(a, L.g_planes(), tile.row * 128, tile.col * 128, first * 32, left < S::WK ? left : S::WK, lds, acc);
  const int back = -(st->g + st->h);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t col0 = tile.col * 128 + wave % 2 * 64 + 4 * (lane >> 4), row0 = tile.row * 128 + wave / 2 * 64 + (lane & 15);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t row = row0 + i * 16, col = col0 + j * 16;
      f4 v = acc[i][j];
      if constexpr (S::WCHUNKS > 1) {
        *reinterpret_cast<f4*>(L.at(S::WPART) + ((size_t)chunk * S::DP + row) * S::VP + col) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], back);
        put_four<S::VECV>(out, row, S::D, col, S::V, v, piece > 0);
      }
    }
}
template <class S>
__device__ __forceinline__ void loss_dw_sum(const Loss<S>& L, float* out, uint32_t block) {
  const LossState* st = L.state();
  const size_t i = (size_t)block * 256 + threadIdx.x;
  const size_t row = i / (S::VP / 4);
  const uint32_t col = i % (S::VP / 4) * 4;
  if (row >= S::D) return;
  const int back = -(st->g + st->h);
  f4 v = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t c = 0; c < S::WCHUNKS; ++c) v += *reinterpret_cast<const f4*>(L.at(S::WPART) + ((size_t)c * S::DP + row) * S::VP + col);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], back);
  put_four<S::VECV>(out, row, S::D, col, S::V, v, st->current > 0);
}

// dbias from the column sums of each RB rows, added in order: 16 threads a column, then theirs. Counts the piece as done.
template <class S, bool BIAS>
__device__ __forceinline__ void loss_end(const Loss<S>& L, float* out, float* scratch, uint32_t block) {
  LossState* st = L.state();
  const uint32_t piece = st->current;
  if constexpr (BIAS) {
    const uint32_t col = block * 16 + threadIdx.x % 16, k0 = threadIdx.x / 16;
    float sum = 0.f;
    for (uint32_t k = k0; k < S::NP / S::RB; k += 16) sum += L.at(S::SUMS)[(size_t)k * S::VP + col];
    scratch[threadIdx.x] = sum;
    __syncthreads();
    if (k0 == 0 && col < S::V) {
      for (uint32_t k = 1; k < 16; ++k) sum += scratch[k * 16 + threadIdx.x];
      const float v = ldexpf(sum, -st->g);
      out[col] = piece > 0 ? out[col] + v : v;
    }
  }
  if (block == 0 && threadIdx.x == 0) st->piece = piece + 1;
}

}  // namespace tcmi
