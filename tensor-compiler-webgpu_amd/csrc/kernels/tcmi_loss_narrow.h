// Softmax cross entropy (tcmi_loss.h: the formulas, the rows that are left out) over few classes, at most 128: a workgroup
// holds whole rows of logits, so one pass over h makes losses, G and dh.
//
//   rows     16·RT rows a workgroup: z = h·W + bias, K over its wavefronts; the losses; G in LDS, and in memory where dW or
//            dbias follow; dh = G·Wᵀ
//   dw       dW = hᵀ·G, 64 rows of dW a workgroup, K over its wavefronts and over workgroups; dbias
//   sums     the parts of dW and dbias added in order
//
// All products are of float32 (16 x 16 x 4), operands read as they are: for so few classes the products of pairs spend longer
// on looking for their scales and splitting. Which k and which columns a matrix instruction takes is chosen so that lanes load
// neighbours and results come out in whole groups of four.
//
// Bound: the latency of launches and loads up to some thousand rows; then memory, 12·N·d bytes with gradients and 4·N·d without, up to
// about 32 classes, and the matrix cores beyond (65 536 rows, d 512: 117 us of 32 classes, 226 of 96, 80 TFLOP/s).

#pragma once

#include "tcmi_loss_few.h"

namespace tcmi {

typedef float f2 __attribute__((ext_vector_type(2)));
typedef float run2 __attribute__((ext_vector_type(2), aligned(4)));

// Two floats of a row from column c on, as raw_four and placed.
__device__ __forceinline__ f2 raw_two(const float* p, uint32_t c, uint32_t cols) {
  if (cols < 2) return f2{p[0], 0.f};
  const run2 x = *reinterpret_cast<const run2*>(p + min(c, cols - 2));
  return f2{x[0], x[1]};
}
__device__ __forceinline__ f2 placed_two(f2 v, uint32_t c, uint32_t cols) {
  if (cols < 2) return f2{c == 0 ? v[0] : 0.f, 0.f};
  if (c + 2 <= cols) return v;
  return f2{c + 1 == cols ? v[1] : 0.f, 0.f};
}

// S, beside the sizes: RT; CG groups of 32 columns, VP = 32·CG; `dw`: RC rows a chunk, CHUNKS chunks, DG groups of 64 rows of W.
template <class S>
constexpr int narrow_ld() { return S::VP + 4; }

template <class S, bool LOSS, bool DH, bool KEEP>
__device__ __forceinline__ void narrow_rows(const Loss<S>& L, float* out, float* dh, float* lds, uint32_t block) {
  constexpr uint32_t ROWS = 16 * S::RT, LD = narrow_ld<S>(), CG = S::CG;
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row0 = block * ROWS;
  {
    f4 acc[S::RT][2 * CG];
#pragma unroll
    for (int r = 0; r < S::RT; ++r)
#pragma unroll
      for (int c = 0; c < 2 * CG; ++c) acc[r][c] = f4{0.f, 0.f, 0.f, 0.f};
    const float* h[S::RT];
#pragma unroll
    for (int r = 0; r < S::RT; ++r) h[r] = L.h + (size_t)min(row0 + 16 * r + t, S::N - 1) * S::D;
    // 16 k at a time, this lane's 4q ... 4q + 3, its columns 2t and 2t + 1 of each 32; the next ones' loads in flight.
    f2 w[4][CG];
    f4 x[S::RT];
    auto load = [&](uint32_t k, f2 (&w)[4][CG], f4 (&x)[S::RT]) __attribute__((always_inline)) {
#pragma unroll
      for (int r = 0; r < S::RT; ++r) x[r] = raw_four<S::VECD>(h[r], k + 4 * q, S::D);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g) w[i][g] = raw_two(L.W + (size_t)(k + 4 * q + i < S::D ? k + 4 * q + i : 0u) * S::V, 32 * g + 2 * t, S::V);
    };
    load(16 * wave, w, x);
    for (uint32_t k = 16 * wave; k < S::D; k += 64) {
      f2 nw[4][CG];
      f4 nx[S::RT];
      load(k + 64, nw, nx);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int r = 0; r < S::RT; ++r) x[r] = placed<S::VECD>(x[r], k + 4 * q, S::D);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g) {
          f2 v = placed_two(w[i][g], 32 * g + 2 * t, S::V);
          if (S::D % 16 != 0 && k + 4 * q + i >= S::D) v = f2{0.f, 0.f};
#pragma unroll
          for (int r = 0; r < S::RT; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) acc[r][2 * g + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e], x[r][i], acc[r][2 * g + e], 0, 0, 0);
        }
#pragma unroll
      for (int r = 0; r < S::RT; ++r) x[r] = nx[r];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < CG; ++g) w[i][g] = nw[i][g];
    }
    // Row 16r + t, columns 32g + 8q ... + 7.
#pragma unroll
    for (int r = 0; r < S::RT; ++r)
#pragma unroll
      for (int g = 0; g < CG; ++g) {
        f4* to = reinterpret_cast<f4*>(lds + (wave * ROWS + 16 * r + t) * LD + 32 * g + 8 * q);
        const f4 &a = acc[r][2 * g], &b = acc[r][2 * g + 1];
        to[0] = f4{a[0], b[0], a[1], b[1]};
        to[1] = f4{a[2], b[2], a[3], b[3]};
      }
  }
  __syncthreads();
  // LANES lanes a row, a lane's groups of four LANES apart.
  constexpr uint32_t LANES = 256 / ROWS, OWN = (S::VP / 4 + LANES - 1) / LANES;
  const uint32_t row = threadIdx.x / LANES, r = row0 + row, c0 = 4 * (threadIdx.x % LANES);
  const float target = r < S::N ? L.t[r] : -1.f;
  const bool kept = L.is_class(target);
  const uint32_t hot = kept ? static_cast<uint32_t>(target) : ~0u;
  f4 z[OWN];
  float top = -TCMI_INF, picked = 0.f, sum = 0.f;
#pragma unroll
  for (uint32_t u = 0; u < OWN; ++u) {
    const uint32_t c = c0 + 4 * LANES * u;
    z[u] = f4{0.f, 0.f, 0.f, 0.f};
    if (c < S::VP) {
#pragma unroll
      for (uint32_t g = 0; g < 4; ++g) z[u] += *reinterpret_cast<const f4*>(lds + (g * ROWS + row) * LD + c);
    }
    const f4 b = S::BIAS ? four_of<false>(L.bias, c, S::V) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      z[u][e] = c + e < S::V ? z[u][e] + b[e] : -TCMI_INF;
      top = fmaxf(top, z[u][e]);
      picked += c + e == hot ? z[u][e] : 0.f;
    }
  }
#pragma unroll
  for (int off = 1; off < LANES; off *= 2) top = fmaxf(top, __shfl_xor(top, off, 64));
  const float shift = top == -TCMI_INF ? 0.f : top;
#pragma unroll
  for (uint32_t u = 0; u < OWN; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += op_exp(z[u][e] - shift);
#pragma unroll
  for (int off = 1; off < LANES; off *= 2) {
    sum += __shfl_xor(sum, off, 64);
    picked += __shfl_xor(picked, off, 64);
  }
  if constexpr (LOSS) {
    if (c0 == 0 && r < S::N) out[r] = kept ? (top - picked) + op_log(sum) : 0.f;
  }
  if constexpr (DH || KEEP) {
    __syncthreads();
    const float w = kept ? L.w[r] : 0.f, by = w * (1.f / sum);
#pragma unroll
    for (uint32_t u = 0; u < OWN; ++u) {
      const uint32_t c = c0 + 4 * LANES * u;
      f4 g = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (kept && c + e < S::V) g[e] = exp_full(z[u][e] - top) * by - (c + e == hot ? w : 0.f);
      if (c < S::VP) {
        *reinterpret_cast<f4*>(lds + row * LD + c) = g;
        if constexpr (KEEP) *reinterpret_cast<f4*>(L.at(S::GP) + (size_t)r * S::VP + c) = g;
      }
    }
    __syncthreads();
  }
  if constexpr (DH) {
    constexpr uint32_t TILES = (S::D + 15) / 16;
    // The next tile's loads in flight.
    f4 x[S::VP / 16];
    auto load = [&](uint32_t tile, f4 (&x)[S::VP / 16]) __attribute__((always_inline)) {
      const float* w = L.W + (size_t)min(16 * tile + t, S::D - 1) * S::V;
#pragma unroll
      for (uint32_t v = 0; v < S::VP / 16; ++v) x[v] = raw_four<S::VECV>(w, 16 * v + 4 * q, S::V);
    };
    load(wave, x);
    for (uint32_t tile = wave; tile < TILES; tile += 4) {
      const uint32_t d0 = 16 * tile;
      f4 acc[S::RT], nx[S::VP / 16];
      load(tile + 4, nx);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int k = 0; k < S::RT; ++k) acc[k] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (uint32_t v = 0; v < S::VP / 16; ++v) {
        x[v] = placed<S::VECV>(x[v], 16 * v + 4 * q, S::V);
        f4 g[S::RT];
#pragma unroll
        for (int k = 0; k < S::RT; ++k) g[k] = *reinterpret_cast<const f4*>(lds + (16 * k + t) * LD + 16 * v + 4 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int k = 0; k < S::RT; ++k) acc[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[v][i], g[k][i], acc[k], 0, 0, 0);
        x[v] = nx[v];
      }
#pragma unroll
      for (int k = 0; k < S::RT; ++k) {
        const uint32_t n = row0 + 16 * k + t;
        if (n < S::N) put_four_of<S::VECD>(dh + (size_t)n * S::D, d0 + 4 * q, S::D, acc[k]);
      }
    }
  }
}

// Rows 64·dg on of dW, over the rows of a chunk; with dg = 0 the chunk's part of dbias.
template <class S, bool DW, bool DB>
__device__ __forceinline__ void narrow_dw(const Loss<S>& L, float* lds, uint32_t chunk, uint32_t dg) {
  constexpr uint32_t CG = S::CG, COLS = S::VP, LD = narrow_ld<S>();
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t d0 = 64 * dg, first = chunk * S::RC + wave * (S::RC / 4);
  f4 acc[4][2 * CG];
  f2 sums[CG];
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int c = 0; c < 2 * CG; ++c) acc[d][c] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < CG; ++g) sums[g] = f2{0.f, 0.f};
  // Row first + 4u + q: this lane's 4 of h's columns, 2 of each 32 of G's; two steps ahead in flight.
  f4 x, x1;
  f2 y[CG], y1[CG];
  float target, target1;
  auto load = [&](uint32_t u, f4& x, f2 (&y)[CG], float& target) __attribute__((always_inline)) {
    const uint32_t n = first + 4 * u + q, at = min(n, S::N - 1);
    target = n < S::N ? L.t[at] : -1.f;
    if constexpr (DW) x = raw_four<S::VECD>(L.h + (size_t)at * S::D, d0 + 4 * t, S::D);
#pragma unroll
    for (int g = 0; g < CG; ++g) y[g] = *reinterpret_cast<const f2*>(L.at(S::GP) + (size_t)at * S::VP + 32 * g + 2 * t);
  };
  load(0, x, y, target);
  load(1, x1, y1, target1);
  for (uint32_t u = 0; u < S::RC / 16; ++u) {
    f4 x2;
    f2 y2[CG];
    float target2;
    load(u + 2, x2, y2, target2);
    __builtin_amdgcn_sched_barrier(0);
    const bool kept = L.is_class(target);
    if constexpr (DW) x = kept ? placed<S::VECD>(x, d0 + 4 * t, S::D) : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < CG; ++g) {
      if (!kept) y[g] = f2{0.f, 0.f};
      if constexpr (DB) sums[g] += y[g];
      if constexpr (DW) {
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) acc[d][2 * g + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[g][e], x[d], acc[d][2 * g + e], 0, 0, 0);
      }
    }
    if constexpr (DW) {
      x = x1;
      x1 = x2;
    }
    target = target1;
    target1 = target2;
#pragma unroll
    for (int g = 0; g < CG; ++g) {
      y[g] = y1[g];
      y1[g] = y2[g];
    }
  }
  if constexpr (DW) {
    // Row 4t + d, columns 32g + 8q ... + 7, of each wavefront; then the four added in order.
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int g = 0; g < CG; ++g) {
        f4* to = reinterpret_cast<f4*>(lds + (wave * 64 + 4 * t + d) * LD + 32 * g + 8 * q);
        const f4 &a = acc[d][2 * g], &b = acc[d][2 * g + 1];
        to[0] = f4{a[0], b[0], a[1], b[1]};
        to[1] = f4{a[2], b[2], a[3], b[3]};
      }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 64 * COLS / 4; i += 256) {
      const uint32_t d = i / (COLS / 4), c = i % (COLS / 4) * 4;
      f4 v = *reinterpret_cast<const f4*>(lds + d * LD + c);
#pragma unroll
      for (uint32_t g = 1; g < 4; ++g) v += *reinterpret_cast<const f4*>(lds + (g * 64 + d) * LD + c);
      if (d0 + d < S::D) *reinterpret_cast<f4*>(L.at(S::WPART) + ((size_t)chunk * S::D + d0 + d) * S::VP + c) = v;
    }
  }
  if constexpr (DB) {
    if (dg == 0) {
      if constexpr (DW) __syncthreads();
#pragma unroll
      for (int g = 0; g < CG; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float s = sums[g][e];
          s += __shfl_xor(s, 16, 64);
          s += __shfl_xor(s, 32, 64);
          if (q == 0) lds[wave * COLS + 32 * g + 2 * t + e] = s;
        }
      __syncthreads();
      if (threadIdx.x < COLS) {
        float s = lds[threadIdx.x];
#pragma unroll
        for (uint32_t g = 1; g < 4; ++g) s += lds[g * COLS + threadIdx.x];
        L.at(S::SUMS)[(size_t)chunk * S::VP + threadIdx.x] = s;
      }
    }
  }
}

// The chunks of dW, then of dbias, added up: 32 groups of four columns a workgroup, every eighth chunk a thread, then those eight.
template <class S, bool DW, bool DB>
__device__ __forceinline__ void narrow_sums(const Loss<S>& L, float* dw, float* db, f4* scratch, uint32_t block) {
  constexpr uint32_t ALL = DW ? S::D * (S::VP / 4) : 0;
  const uint32_t i = block * 32 + threadIdx.x % 32, p = threadIdx.x / 32;
  const bool of_w = i < ALL, any = of_w || (DB && i < ALL + S::VP / 4);
  const float* at = of_w ? L.at(S::WPART) + 4 * (size_t)i : L.at(S::SUMS) + 4 * (size_t)(i - ALL);
  const size_t step = of_w ? (size_t)S::D * S::VP : S::VP;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (any) {
#pragma unroll 4
    for (uint32_t c = p; c < S::CHUNKS; c += 8) v += *reinterpret_cast<const f4*>(at + c * step);
  }
  scratch[threadIdx.x] = v;
  __syncthreads();
  if (p == 0 && any) {
    for (uint32_t k = 1; k < 8; ++k) v += scratch[32 * k + threadIdx.x];
    const uint32_t col = (of_w ? i % (S::VP / 4) : i - ALL) * 4;
    float* const to = of_w ? dw + (size_t)(i / (S::VP / 4)) * S::V : db;
    if (of_w) put_four_of<S::VECV>(to, col, S::V, v);
    else put_four_of<false>(to, col, S::V, v);
  }
}

}  // namespace tcmi
