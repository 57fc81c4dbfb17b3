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
// All products are of pairs of halves (tcmi_gemm_f16x2.h), each operand split once, times a power of two that brings
// its largest finite magnitude below 2^15: h's rows each their own, G's rows each its cotangent's, so that a row's
// loss and dh hang on nothing that other rows hold; W one for all. dW sums over the rows: it takes a split of h of its own, each
// row times what G's row lacks of one scale for all, that of the largest |w|·|h|. What a pair loses below 2^-36 is then at most
// 2^-50 of |h row|·|W| a term of z, of |w|·|W| one of dh and of the largest |w|·|h| one of dW, these magnitudes the largest in each.
//
//   maxima   h's row exponents, the least exponent of |w|·|h|, partial maxima of |W|
//   split    h (for dW again, times w's scale) and W as pairs, padded with zeros to whole tiles
//   logits   z tile by tile; each wavefront's 64 columns of a row leave (maximum, sum of
//            exponentials), and z itself where G will be formed
//   join     a row's pairs joined in order; the losses; (M, 1/s) a row
//   spread   G as pairs, and the column sums of a few rows each (with few pairs a row it joins them itself)
//   grads    the tiles of dh and dW, and dbias, side by side in one launch; K split over
//            workgroups where tiles are few; dW and dbias are added up over the pieces
//   sums     the parts of a split K added in order
// The piece that a kernel works on is counted in the workspace (two slots, so that no kernel
// reads the one it writes), which keeps one kernel text and one argument block for all pieces.
//
// Bound: the matrix cores (6·N·d·V flops with gradients, 2·N·d·V without). 8192 rows of d 1024 against 65 536 classes, us: maxima
// 59 (5.1 TB/s), split 114 (5.6 TB/s), and each of 4 pieces logits 747 (368 TFLOP/s), join 9, spread 214 (4.9 TB/s), grads 1311
// (419), sums 9. Fewer passes would need W's scale before it is read, and a row's sum before its logits are left.

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
  int w, g;                        // exponents of W's scale, and of dW's operands' (the row's of G and of its h together)
};

// S: the sizes of one launch as constants of its text: N, D, V; NP rows a piece, PIECES of them; DP, VP: d and V padded to
// whole tiles; BIAS; HBLOCKS, WBLOCKS workgroups of `maxima` over h's rows (HLANES lanes each) and W; PER groups of four a thread of `split` takes; LKIND, HKIND and
// WKIND of tiles for the logits, dh and dW; RB rows a workgroup of `spread`, CT threads across columns there;
// JOINED: `join` runs; VECD, VECV: d, V multiples of 4; HCHUNKS, HK, WCHUNKS, WK: chunks of K of dh and dW, their slices.
// WS: byte offsets in the workspace.
template <class S>
struct Loss {
  const float *h, *W, *t, *bias, *w;
  char* ws;
  __device__ __forceinline__ LossState* state() const { return reinterpret_cast<LossState*>(ws); }
  __device__ __forceinline__ float* at(size_t off) const { return reinterpret_cast<float*>(ws + off); }
  __device__ __forceinline__ Pairs h_pairs() const { return {ws + S::HP, S::DP * 4}; }
  __device__ __forceinline__ Pairs x_pairs() const { return {ws + S::XP, S::DP * 4}; }       // h for dW
  __device__ __forceinline__ int* exponents() const { return reinterpret_cast<int*>(ws + S::EXPS); }
  __device__ __forceinline__ Pairs w_pairs() const { return {ws + S::WP, S::VP * 4}; }
  __device__ __forceinline__ Pairs g_pairs() const { return {ws + S::GP, S::VP * 4}; }
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

__device__ __forceinline__ float top_of(const f4& v, float top) {
  return fmaxf(fmaxf(fmaxf(finite_abs(v[0]), finite_abs(v[1])), fmaxf(finite_abs(v[2]), finite_abs(v[3]))), top);
}

// That of a row's cotangent.
__device__ __forceinline__ int weight_scale(float w) { return scale_of(finite_abs(w)); }

constexpr int NO_SCALE = 252;      // at most: two of scale_of's

template <class S, bool DW>
__device__ __forceinline__ void loss_maxima(const Loss<S>& L, float* scratch, uint32_t block) {
  if (block < S::HBLOCKS) {
    // HLANES lanes a row. Rows left out are loaded all the same, so that no load waits for a target.
    const uint32_t lane = threadIdx.x % S::HLANES;
    int least = NO_SCALE;
    for (uint32_t r = block * (256 / S::HLANES) + threadIdx.x / S::HLANES; r < S::N; r += S::HBLOCKS * (256 / S::HLANES)) {
      const float* h = L.h + (size_t)r * S::D;
      float top = 0.f;
      if constexpr (S::VECD) {
#pragma unroll 4
        for (uint32_t i = lane; i < S::D / 4; i += S::HLANES) top = top_of(reinterpret_cast<const f4*>(h)[i], top);
      } else {
#pragma unroll 8
        for (uint32_t i = lane; i < S::D; i += S::HLANES) top = fmaxf(top, finite_abs(h[i]));
      }
#pragma unroll
      for (int off = S::HLANES / 2; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
      const bool kept = L.kept(r);
      const int e = scale_of(kept ? top : 0.f);
      if (lane == 0) L.exponents()[r] = e;
      if constexpr (DW) {
        const float w = finite_abs(L.w[r]);
        if (kept && top > 0.f && w > 0.f) least = min(least, e + weight_scale(w));
      }
    }
    if constexpr (DW) {
      int* const leasts = reinterpret_cast<int*>(scratch);
#pragma unroll
      for (int off = 32; off >= S::HLANES; off >>= 1) least = min(least, __shfl_xor(least, off, 64));
      if (threadIdx.x % 64 == 0) leasts[threadIdx.x / 64] = least;
      __syncthreads();
      if (threadIdx.x == 0) reinterpret_cast<int*>(L.at(S::MAXIMA))[block] = min(min(leasts[0], leasts[1]), min(leasts[2], leasts[3]));
    }
    return;
  }
  float top = 0.f;
  {
    // Four loads in flight a thread.
    constexpr size_t n = (size_t)S::D * S::V, n4 = n / 4, step = (size_t)S::WBLOCKS * 256;
    const size_t i0 = (size_t)(block - S::HBLOCKS) * 256 + threadIdx.x;
    const f4* w = reinterpret_cast<const f4*>(L.W);
    size_t i = i0;
    for (; i + 3 * step < n4; i += 4 * step) {
      const f4 a = w[i], b = w[i + step], c = w[i + 2 * step], d = w[i + 3 * step];
      top = top_of(a, top_of(b, top_of(c, top_of(d, top))));
    }
    for (; i < n4; i += step) top = top_of(w[i], top);
    if (i0 < n % 4) top = fmaxf(top, finite_abs(L.W[4 * n4 + i0]));
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
// The largest of maxima[0 .. count).
__device__ __forceinline__ float top_of_blocks(const float* maxima, uint32_t count, float* scratch) {
  float top = 0.f;
  for (uint32_t i = threadIdx.x; i < count; i += 256) top = fmaxf(top, maxima[i]);
  return block_reduce<true, 256>(top, scratch);
}

// The least of leasts[0 .. count).
__device__ __forceinline__ int least_of_blocks(const int* leasts, uint32_t count, int* scratch) {
  int least = NO_SCALE;
  for (uint32_t i = threadIdx.x; i < count; i += 256) least = min(least, leasts[i]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) least = min(least, __shfl_xor(least, off, 64));
  if (threadIdx.x % 64 == 0) scratch[threadIdx.x / 64] = least;
  __syncthreads();
  return min(min(scratch[0], scratch[1]), min(scratch[2], scratch[3]));
}
__device__ __forceinline__ f4 scaled(f4 v, int by) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = ldexpf(v[e], by);
  return v;
}

template <class S, bool DW>
__device__ __forceinline__ void loss_split(const Loss<S>& L, float* scratch, uint32_t block) {
  constexpr size_t HG = (size_t)S::NP * S::PIECES * S::DP / 4, WG = (size_t)S::DP * S::VP / 4;
  constexpr uint32_t HB = (HG + 256 * S::PER - 1) / (256 * S::PER);
  const float* maxima = L.at(S::MAXIMA);
  LossState* st = L.state();
  if (block >= HB) {
    const int s = scale_of(top_of_blocks(maxima + S::HBLOCKS, S::WBLOCKS, scratch));
    if (block == HB && threadIdx.x == 0) st->w = s;
    for (uint32_t u = 0; u < S::PER; ++u) {
      const size_t i = ((size_t)(block - HB) * S::PER + u) * 256 + threadIdx.x;
      if (i >= WG) return;
      const size_t row = i / (S::VP / 4);
      const uint32_t col = i % (S::VP / 4) * 4;
      put_pairs(L.w_pairs(), row, col, scaled(four<S::VECV>(L.W, row, S::D, col, S::V), s));
    }
    return;
  }
  const int least = DW ? least_of_blocks(reinterpret_cast<const int*>(maxima), S::HBLOCKS, reinterpret_cast<int*>(scratch)) : 0;
  if (block == 0 && threadIdx.x == 0) {
    st->piece = 0u;
    st->g = least;
  }
  for (uint32_t u = 0; u < S::PER; ++u) {
    const size_t i = ((size_t)block * S::PER + u) * 256 + threadIdx.x;
    if (i >= HG) return;
    const size_t row = i / (S::DP / 4);
    const uint32_t col = i % (S::DP / 4) * 4;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    const bool kept = L.kept(row);
    if (kept) v = four<S::VECD>(L.h, row, S::N, col, S::D);
    put_pairs(L.h_pairs(), row, col, scaled(v, kept ? L.exponents()[row] : 0));
    if constexpr (DW) {
      // A row of weight 0 (whose G is 0) has none of the least exponents.
      const float w = kept ? finite_abs(L.w[row]) : 0.f;
      put_pairs(L.x_pairs(), row, col, w > 0.f ? scaled(v, least - weight_scale(w)) : f4{0.f, 0.f, 0.f, 0.f});
    }
  }
}

// One tile of the piece's logits.
template <class S, bool KEEP>
__device__ __forceinline__ void loss_logits(const Loss<S>& L, char* lds, uint32_t block) {
  using P = Tile<S::LKIND>;
  LossState* st = L.state();
  const uint32_t piece = st->piece;
  if (block == 0 && threadIdx.x == 0) st->current = piece;
  const TileAt tile = tile_at<P::GROUP>(block, S::NP / P::ROWS, S::VP / P::COLS);
  Pairs a = L.h_pairs();
  a.at += (size_t)piece * S::NP * a.ld;
  typename P::Sums acc;
  P::template sum<true, false>(a, L.w_pairs(), tile, 0, (S::D + 31) / 32, lds, acc);
  const int back_w = -st->w;
  const uint32_t col0 = P::col(tile), row0 = P::row(tile);
  float m[P::TI];
  int back[P::TI];             // exponents of a row's sums
  uint32_t ahead[P::TI];       // the columns from col0 on to a row's target, where that is a class
#pragma unroll
  for (int i = 0; i < P::TI; ++i) {
    const uint32_t r = piece * S::NP + row0 + i * 16;
    const float target = r < S::N ? L.t[r] : -1.f;
    back[i] = r < S::N ? back_w - L.exponents()[r] : 0;
    ahead[i] = L.is_class(target) ? static_cast<uint32_t>(target) - col0 : ~0u;
    m[i] = -TCMI_INF;
  }
#pragma unroll
  for (int j = 0; j < P::TJ; ++j) {
    const uint32_t col = col0 + j * 16;
    const f4 b = S::BIAS ? four<S::VECV>(L.bias, 0, 1, col, S::V) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < P::TI; ++i) {
      f4& z = acc[i][j];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        z[e] = ldexpf(z[e], back[i]) + b[e];
        if (S::V != S::VP && col + e >= S::V) z[e] = -TCMI_INF;
        m[i] = fmaxf(m[i], z[e]);
      }
      const uint32_t e = ahead[i] - 16u * j;
      if (e < 4u) L.at(S::PICKED)[row0 + i * 16] = e < 2u ? (e ? z[1] : z[0]) : e == 2u ? z[2] : z[3];
      if constexpr (KEEP) *reinterpret_cast<f4*>(L.at(S::Z) + (size_t)(row0 + i * 16) * S::VP + col) = z;
    }
  }
  // Sums of a wavefront's columns by op_exp: its error, |x|·2^-24 of an e^x, is least where e^x counts.
#pragma unroll
  for (int i = 0; i < P::TI; ++i) {
    const float top = quad16_reduce<true>(m[i]), shift = top == -TCMI_INF ? 0.f : top;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < P::TJ; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s += op_exp(acc[i][j][e] - shift);
    s = quad16_reduce<false>(s);
    if (threadIdx.x % 64 < 16) {
      reinterpret_cast<float2*>(L.at(S::STATS))[(size_t)(tile.col * P::WN + threadIdx.x / 64 % P::WN) * S::NP + row0 + i * 16] = make_float2(top, s);
    }
  }
}

// A row's statistics (maximum, sum of exponentials) joined with some columns' more.
struct RowSum {
  float m = -TCMI_INF, s = 0.f;
  __device__ __forceinline__ void add(const float2 x) {
    const float top = red_max(m, x.x), shift = top == -TCMI_INF ? 0.f : top;
    s = s * exp_full(m - shift) + x.y * exp_full(x.x - shift);
    m = top;
  }
};
template <class S>
constexpr uint32_t loss_parts() { return S::VP / (16 * Tile<S::LKIND>::T); }

// The statistics of 16 rows, 64 threads a row.
template <class S, bool LOSS, bool LAST>
__device__ __forceinline__ void loss_join(const Loss<S>& L, float* out, float2* scratch, uint32_t block) {
  LossState* st = L.state();
  const uint32_t piece = S::PIECES > 1 ? st->current : 0u;
  const uint32_t row = block * 16 + threadIdx.x % 16, k0 = threadIdx.x / 16;
  const float2* stats = reinterpret_cast<const float2*>(L.at(S::STATS)) + row;
  RowSum sum;
#pragma unroll 4
  for (uint32_t k = k0; k < loss_parts<S>(); k += 64) sum.add(stats[(size_t)k * S::NP]);
  scratch[threadIdx.x] = make_float2(sum.m, sum.s);
  __syncthreads();
  if (k0 < 8) {
    for (uint32_t k = k0 + 8; k < 64; k += 8) sum.add(scratch[k * 16 + threadIdx.x % 16]);
  }
  __syncthreads();
  if (k0 < 8) scratch[threadIdx.x] = make_float2(sum.m, sum.s);
  __syncthreads();
  if (k0 == 0) {
    for (uint32_t k = 1; k < 8; ++k) sum.add(scratch[k * 16 + threadIdx.x]);
    reinterpret_cast<float2*>(L.at(S::ROWS))[row] = make_float2(sum.m, 1.f / sum.s);
    const uint32_t r = piece * S::NP + row;
    if constexpr (LOSS) {
      if (r < S::N) out[r] = L.kept(r) ? (sum.m - L.at(S::PICKED)[row]) + op_log(sum.s) : 0.f;
    }
  }
  if constexpr (LAST) {
    if (block == 0 && threadIdx.x == 0) st->piece = piece + 1;
  }
}

// RB rows of 8·CT columns of G: 256 / CT threads a column group, each its own rows in turn. rows: of LDS, and 512 more for
// the sums, and RB / 4 for the rows' scales back. out: the losses, where this kernel joins the statistics (not JOINED).
template <class S, bool PAIRS, bool SUMS, bool LOSS>
__device__ __forceinline__ void loss_spread(const Loss<S>& L, float* out, f4* rows, uint32_t bx, uint32_t by) {
  const LossState* st = L.state();
  const uint32_t piece = st->current;
  const uint32_t row0 = by * S::RB;
  float* const unscale = reinterpret_cast<float*>(rows + S::RB + 512);
  if (threadIdx.x < S::RB) {
    const uint32_t row = row0 + threadIdx.x, r = piece * S::NP + row;
    f4 c = {0.f, 0.f, 0.f, -1.f};       // M, w/s and w in the row's scale, the target (-1: the row is left out)
    float one = 1.f;
    const bool kept = L.kept(r);
    if (kept) {
      float2 x;
      if constexpr (S::JOINED) {
        x = reinterpret_cast<const float2*>(L.at(S::ROWS))[row];
      } else {
        // As `join` adds them: every eighth in turn, then those eight.
        RowSum sum;
        for (uint32_t p = 0; p < 8 && p < loss_parts<S>(); ++p) {
          RowSum part;
          for (uint32_t k = p; k < loss_parts<S>(); k += 8) part.add(reinterpret_cast<const float2*>(L.at(S::STATS))[(size_t)k * S::NP + row]);
          sum.add(make_float2(part.m, part.s));
        }
        x = make_float2(sum.m, 1.f / sum.s);
        if constexpr (LOSS) {
          if (bx == 0) out[r] = (sum.m - L.at(S::PICKED)[row]) + op_log(sum.s);
        }
      }
      const int scale = weight_scale(L.w[r]);
      const float w = ldexpf(L.w[r], scale);
      one = ldexpf(1.f, -scale);
      c = f4{x.x, w * x.y, w, L.t[r]};
    } else if constexpr (LOSS && !S::JOINED) {
      if (bx == 0 && r < S::N) out[r] = 0.f;
    }
    rows[threadIdx.x] = c;
    if constexpr (SUMS) unscale[threadIdx.x] = one;
  }
  __syncthreads();
  constexpr uint32_t RG = 256 / S::CT;
  const uint32_t col = (bx * S::CT + threadIdx.x % S::CT) * 8, group = threadIdx.x / S::CT;
  const Pairs p = L.g_pairs();
  f4 sum[2] = {};
  if (col < S::VP) {
#pragma unroll 2
    for (uint32_t k = group; k < S::RB; k += RG) {
      const f4 c = rows[k];
      const f4* z = reinterpret_cast<const f4*>(L.at(S::Z) + (size_t)(row0 + k) * S::VP + col);
      const f4 y[2] = {z[0], z[1]};
      f4 g[2] = {};
      if (c[3] >= 0.f) {
        const uint32_t ahead = static_cast<uint32_t>(c[3]) - col;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // exp(-inf) of a column that is no class is 0.
          g[e / 4][e % 4] = exp_full(y[e / 4][e % 4] - c[0]) * c[1] - (ahead == e ? c[2] : 0.f);
        }
        if (S::V % 8 != 0 && col + 8 > S::V) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e >= S::V) g[e / 4][e % 4] = 0.f;      // also where M is not finite
        }
      }
      if constexpr (SUMS) {
        sum[0] += g[0] * unscale[k];
        sum[1] += g[1] * unscale[k];
      }
      if constexpr (PAIRS) {
        h8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          _Float16 a, b;
          split_pair(g[e / 4][e % 4], a, b);
          hi[e] = a;
          lo[e] = b;
        }
        char* at = pair_at(p, row0 + k, col);
        *reinterpret_cast<h8*>(at) = hi;
        *reinterpret_cast<h8*>(at + 64) = lo;
      }
    }
  }
  if constexpr (SUMS) {
    f4* const parts = rows + S::RB;
    if constexpr (RG > 1) {
      parts[2 * threadIdx.x] = sum[0];
      parts[2 * threadIdx.x + 1] = sum[1];
      __syncthreads();
      if (group == 0) {
        for (uint32_t k = 1; k < RG; ++k) {
          sum[0] += parts[2 * (k * S::CT + threadIdx.x)];
          sum[1] += parts[2 * (k * S::CT + threadIdx.x) + 1];
        }
      }
    }
    if (group == 0 && col < S::VP) {
      f4* to = reinterpret_cast<f4*>(L.at(S::SUMS) + (size_t)by * S::VP + col);
      to[0] = sum[0];
      to[1] = sum[1];
    }
  }
}

// Four columns of C [rows, cols] = v, or added to what is there.
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
// Workgroups of `grads`: dh's tiles by chunks of K, dW's, then dbias.
template <class S>
struct GradTiles {
  using H = Tile<S::HKIND>;
  using W = Tile<S::WKIND>;
  static_assert(H::THREADS == W::THREADS, "one launch");
  static constexpr uint32_t HR = S::NP / H::ROWS, HC = S::DP / H::COLS, WR = S::DP / W::ROWS, WC = S::VP / W::COLS;
  static constexpr int LDS = H::LDS > W::LDS ? H::LDS : W::LDS;
};

// The exponent that row r's sums of dh lack.
template <class S>
__device__ __forceinline__ int dh_back(const Loss<S>& L, uint32_t r) {
  return r < S::N ? -(weight_scale(L.w[r]) + L.state()->w) : 0;
}

template <class S, bool DH, bool DW, bool DB>
__device__ __forceinline__ void loss_grads(const Loss<S>& L, float* dh, float* dw, float* db, char* lds, uint32_t block) {
  using G = GradTiles<S>;
  constexpr uint32_t HB = DH ? G::HR * G::HC * S::HCHUNKS : 0, WB = DW ? G::WR * G::WC * S::WCHUNKS : 0;
  LossState* st = L.state();
  const uint32_t piece = st->current;
  if (block == 0 && threadIdx.x == 0) st->piece = piece + 1;     // this piece is done with the next kernel
  if (DH && block < HB) {
    using P = typename G::H;
    // A chunk's tiles, which read the same columns of G and W, on one XCD.
    const uint32_t at = xcd_run(block, HB), chunk = at / (G::HR * G::HC), in = at % (G::HR * G::HC), first = chunk * S::HK, left = S::VP / 32 - first;
    const TileAt tile = {in % G::HR, in / G::HR};
    typename P::Sums acc;
    P::template sum<true, true>(L.g_pairs(), L.w_pairs(), tile, first * 32, left < S::HK ? left : S::HK, lds, acc);
    const uint32_t row0 = P::row(tile);
    int back[P::TI];
    if constexpr (S::HCHUNKS == 1) {
#pragma unroll
      for (int i = 0; i < P::TI; ++i) back[i] = dh_back(L, piece * S::NP + row0 + i * 16);
    }
    P::each(tile, acc, [&](uint32_t row, uint32_t col, const f4& v) {
      if constexpr (S::HCHUNKS > 1) *reinterpret_cast<f4*>(L.at(S::HPART) + ((size_t)chunk * S::NP + row) * S::DP + col) = v;
      else put_four<S::VECD>(dh, (size_t)piece * S::NP + row, S::N, col, S::D, scaled(v, back[(row - row0) / 16]), false);
    });
  } else if (DW && block - HB < WB) {
    using P = typename G::W;
    const uint32_t id = block - HB, chunk = id / (G::WR * G::WC), first = chunk * S::WK, left = S::NP / 32 - first;
    const TileAt tile = tile_at<P::GROUP>(id % (G::WR * G::WC), G::WR, G::WC);
    Pairs a = L.x_pairs();
    a.at += (size_t)piece * S::NP * a.ld;
    typename P::Sums acc;
    P::template sum<false, false>(a, L.g_pairs(), tile, first * 32, left < S::WK ? left : S::WK, lds, acc);
    const int back = -st->g;
    P::each(tile, acc, [&](uint32_t row, uint32_t col, const f4& v) {
      if constexpr (S::WCHUNKS > 1) *reinterpret_cast<f4*>(L.at(S::WPART) + ((size_t)chunk * S::DP + row) * S::VP + col) = v;
      else put_four<S::VECV>(dw, row, S::D, col, S::V, scaled(v, back), piece > 0);
    });
  } else if constexpr (DB) {
    // The column sums of each RB rows in order: PER threads a column, then theirs.
    constexpr uint32_t PER = G::H::THREADS / 16;
    float* const scratch = reinterpret_cast<float*>(lds);
    const uint32_t col = (block - HB - WB) * 16 + threadIdx.x % 16, k0 = threadIdx.x / 16;
    float sum = 0.f;
    for (uint32_t k = k0; k < S::NP / S::RB; k += PER) sum += L.at(S::SUMS)[(size_t)k * S::VP + col];
    scratch[threadIdx.x] = sum;
    __syncthreads();
    if (k0 == 0 && col < S::V) {
      for (uint32_t k = 1; k < PER; ++k) sum += scratch[k * 16 + threadIdx.x];
      db[col] = piece > 0 ? db[col] + sum : sum;
    }
  }
}

// The chunks of dh (HB workgroups) and of dW added in order, four columns a thread.
template <class S, bool DH, bool DW>
__device__ __forceinline__ void loss_sums(const Loss<S>& L, float* dh, float* dw, uint32_t block) {
  constexpr uint32_t HB = DH ? (S::NP * (S::DP / 4) + 255) / 256 : 0;
  const LossState* st = L.state();
  if (DH && block < HB) {
    const uint32_t i = block * 256 + threadIdx.x, row = i / (S::DP / 4), col = i % (S::DP / 4) * 4;
    if (row >= S::NP) return;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t c = 0; c < S::HCHUNKS; ++c) v += *reinterpret_cast<const f4*>(L.at(S::HPART) + ((size_t)c * S::NP + row) * S::DP + col);
    put_four<S::VECD>(dh, (size_t)st->current * S::NP + row, S::N, col, S::D, scaled(v, dh_back(L, st->current * S::NP + row)), false);
  } else if constexpr (DW) {
    const size_t i = (size_t)(block - HB) * 256 + threadIdx.x, row = i / (S::VP / 4);
    const uint32_t col = i % (S::VP / 4) * 4;
    if (row >= S::D) return;
    f4 v = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t c = 0; c < S::WCHUNKS; ++c) v += *reinterpret_cast<const f4*>(L.at(S::WPART) + ((size_t)c * S::DP + row) * S::VP + col);
    put_four<S::VECV>(dw, row, S::D, col, S::V, scaled(v, -st->g), st->current > 0);
  }
}

}  // namespace tcmi
