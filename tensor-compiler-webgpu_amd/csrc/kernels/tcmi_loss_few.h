// Softmax cross entropy (tcmi_loss.h: the formulas, the rows that are left out) of few rows, at most 64, against
// many classes: W is read as it is, once for the losses and once more for the gradients, where the products of
// pairs first look for its largest value, split it and read the pairs.
//
//   logits   64 columns a workgroup, K over its wavefronts; the statistics of those columns, and z where G will be formed
//   join     as there
//   grads    256 columns of G in LDS; from them the columns' part of dh, and their dW and dbias
//   sums     the columns' parts of dh added in order
//
// All products are of float32 (16 x 16 x 4). A lane loads four neighbours of W, and four of the k or of the columns that
// one matrix instruction takes are 4 apart: sums take their terms in an order of their own, the result comes out in whole
// groups of four columns.
//
// Bound: memory, 4·d·V bytes for the losses and 8·d·V more for the gradients; past 32 rows the matrix cores. Of d 1024 and
// 131 072 classes 103 us for one row, 107 for 16 (5.0 TB/s), 178 for 64 (96 TFLOP/s); with gradients, which read W again, 384, 388 and 552.

#pragma once

#include "tcmi_loss.h"

namespace tcmi {

typedef float run4 __attribute__((ext_vector_type(4), aligned(4)));

// Four floats of a row from column c on, those from `cols` on 0. Not VEC: the row starts anywhere. Without a branch, so that
// loads of several iterations are in flight: a group past the row's end is read inside it (raw_four), and moved into place
// where it is used (placed).
template <bool VEC>
__device__ __forceinline__ f4 raw_four(const float* p, uint32_t c, uint32_t cols) {
  if (cols < 4) return f4{p[min(c, cols - 1)], p[min(c + 1, cols - 1)], p[min(c + 2, cols - 1)], 0.f};
  p += min(c, cols - 4);
  if (VEC) return *reinterpret_cast<const f4*>(p);
  const run4 x = *reinterpret_cast<const run4*>(p);
  return f4{x[0], x[1], x[2], x[3]};
}
template <bool VEC>
__device__ __forceinline__ f4 placed(f4 v, uint32_t c, uint32_t cols) {
  if (cols < 4) {
#pragma unroll
    for (int e = 0; e < 3; ++e) v[e] = c + e < cols ? v[e] : 0.f;
    return v;
  }
  const uint32_t over = c + 4 > cols ? c + 4 - cols : 0u;
  if (!VEC) {
    if (over & 1u) v = f4{v[1], v[2], v[3], 0.f};
    if (over & 2u) v = f4{v[2], v[3], 0.f, 0.f};
  }
  return over < 4u ? v : f4{0.f, 0.f, 0.f, 0.f};
}
template <bool VEC>
__device__ __forceinline__ f4 four_of(const float* p, uint32_t c, uint32_t cols) {
  return placed<VEC>(raw_four<VEC>(p, c, cols), c, cols);
}
template <bool VEC>
__device__ __forceinline__ void put_four_of(float* p, uint32_t c, uint32_t cols, const f4& v) {
  if (VEC) {
    if (c < cols) *reinterpret_cast<f4*>(p + c) = v;
  } else if (c + 4 <= cols) {
    *reinterpret_cast<run4*>(p + c) = run4{v[0], v[1], v[2], v[3]};
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (c + e < cols) p[c + e] = v[e];
  }
}

// S, beside what `join` takes: RT = NP / 16; WAVES of `logits`; COLS columns a workgroup of `grads`, CHUNKS such; DTILES 16-row
// tiles of W a workgroup takes there.
constexpr int FEW_LD = 68;        // floats of a row of 64 logits in LDS

template <class S, bool KEEP>
__device__ __forceinline__ void few_logits(const Loss<S>& L, float* lds, uint32_t block) {
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col0 = block * 64;
  f4 acc[S::RT][4];
#pragma unroll
  for (int r = 0; r < S::RT; ++r)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] = f4{0.f, 0.f, 0.f, 0.f};
  const float* h[S::RT];
#pragma unroll
  for (int r = 0; r < S::RT; ++r) h[r] = L.h + (size_t)min(16u * r + t, S::N - 1) * S::D;
  // 16 k at a time: this lane's are 4q ... 4q + 3 of them. The next ones' loads (past the last: of row 0, not used) in flight.
  f4 w[4], x[S::RT];
  auto load = [&](uint32_t k, f4 (&w)[4], f4 (&x)[S::RT]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = raw_four<S::VECV>(L.W + (size_t)(k + 4 * q + i < S::D ? k + 4 * q + i : 0u) * S::V, col0 + 4 * t, S::V);
#pragma unroll
    for (int r = 0; r < S::RT; ++r) x[r] = raw_four<S::VECD>(h[r], k + 4 * q, S::D);
  };
  load(16 * wave, w, x);
  for (uint32_t k = 16 * wave; k < S::D; k += 16 * S::WAVES) {
    f4 nw[4], nx[S::RT];
    load(k + 16 * S::WAVES, nw, nx);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = placed<S::VECV>(w[i], col0 + 4 * t, S::V);
      if (S::D % 16 != 0 && k + 4 * q + i >= S::D) w[i] = f4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int r = 0; r < S::RT; ++r) x[r] = placed<S::VECD>(x[r], k + 4 * q, S::D);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < S::RT; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i][e], x[r][i], acc[r][e], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = nw[i];
#pragma unroll
    for (int r = 0; r < S::RT; ++r) x[r] = nx[r];
  }
#pragma unroll
  for (int r = 0; r < S::RT; ++r)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<f4*>(lds + (wave * S::NP + 16 * r + t) * FEW_LD + 16 * q + 4 * i) = f4{acc[r][0][i], acc[r][1][i], acc[r][2][i], acc[r][3][i]};
    }
  __syncthreads();
  const uint32_t c = 4 * (threadIdx.x % 16), col = col0 + c;
  const f4 b = S::BIAS ? four_of<false>(L.bias, col, S::V) : f4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t row = threadIdx.x / 16; row < S::NP; row += 4 * S::WAVES) {
    f4 z = *reinterpret_cast<const f4*>(lds + row * FEW_LD + c);
#pragma unroll
    for (uint32_t g = 1; g < S::WAVES; ++g) z += *reinterpret_cast<const f4*>(lds + (g * S::NP + row) * FEW_LD + c);
    float top = -TCMI_INF, sum = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      z[e] = col + e < S::V ? z[e] + b[e] : -TCMI_INF;
      top = fmaxf(top, z[e]);
    }
#pragma unroll
    for (int off = 1; off < 16; off *= 2) top = fmaxf(top, __shfl_xor(top, off, 64));
    const float shift = top == -TCMI_INF ? 0.f : top;
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += op_exp(z[e] - shift);
#pragma unroll
    for (int off = 1; off < 16; off *= 2) sum += __shfl_xor(sum, off, 64);
    if (c == 0) reinterpret_cast<float2*>(L.at(S::STATS))[(size_t)block * S::NP + row] = make_float2(top, sum);
    const float target = row < S::N ? L.t[row] : -1.f;
    const uint32_t e = L.is_class(target) ? static_cast<uint32_t>(target) - col : ~0u;
    if (e < 4u) L.at(S::PICKED)[row] = e < 2u ? (e ? z[1] : z[0]) : e == 2u ? z[2] : z[3];
    if constexpr (KEEP) *reinterpret_cast<f4*>(L.at(S::Z) + (size_t)row * S::VP + col) = z;
  }
}

// Columns `chunk`·COLS on of G, and rows `part`·DTILES·16 on of W.
template <class S, bool DH, bool DW, bool DB>
__device__ __forceinline__ void few_grads(const Loss<S>& L, float* dh, float* dw, float* db, float* lds, uint32_t chunk, uint32_t part) {
  constexpr uint32_t LD = S::COLS + 4, THREADS = 256, WAVES = THREADS / 64;
  const uint32_t lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col0 = chunk * S::COLS;
  for (uint32_t i = threadIdx.x; i < S::NP * (S::COLS / 4); i += THREADS) {
    const uint32_t row = i / (S::COLS / 4), c = i % (S::COLS / 4) * 4, col = col0 + c;
    f4 g = {0.f, 0.f, 0.f, 0.f};
    if (L.kept(row) && col < S::V) {
      const float2 x = reinterpret_cast<const float2*>(L.at(S::ROWS))[row];
      const float w = L.w[row], by = w * x.y;
      const uint32_t ahead = static_cast<uint32_t>(L.t[row]) - col;
      const f4 z = *reinterpret_cast<const f4*>(L.at(S::Z) + (size_t)row * S::VP + col);
#pragma unroll
      for (uint32_t e = 0; e < 4; ++e)
        if (col + e < S::V) g[e] = exp_full(z[e] - x.x) * by - (ahead == e ? w : 0.f);
    }
    *reinterpret_cast<f4*>(lds + row * LD + c) = g;
  }
  __syncthreads();
  if constexpr (DB) {
    if (part == 0) {
      for (uint32_t c = threadIdx.x; c < S::COLS; c += THREADS) {
        if (col0 + c >= S::V) break;
        float sum = 0.f;
        for (uint32_t r = 0; r < S::N; ++r) sum += lds[r * LD + c];
        db[col0 + c] = sum;
      }
    }
  }
  if constexpr (!DH && !DW) return;
  constexpr uint32_t TILES = (S::D + 15) / 16;
  const uint32_t end = min(TILES, (part + 1) * S::DTILES);
  // The group of four columns (of 16) that a lane's operand is of, so that four lanes' results are neighbours.
  const uint32_t turned = (t >> 2) + 4 * (t & 3);
  uint32_t kept = 0;        // rows 4s + q, bit s
  if constexpr (DW) {
#pragma unroll
    for (uint32_t s = 0; s < 4 * S::RT; ++s) kept |= (L.kept(4 * s + q) ? 1u : 0u) << s;
  }
  for (uint32_t tile = part * S::DTILES + wave; tile < end; tile += WAVES) {
    const uint32_t d0 = 16 * tile;
    if constexpr (DH) {
      const bool in = S::D % 16 == 0 || d0 + t < S::D;
      const float* w = L.W + (size_t)(in ? d0 + t : 0u) * S::V;
      f4 acc[S::RT];
#pragma unroll
      for (int r = 0; r < S::RT; ++r) acc[r] = f4{0.f, 0.f, 0.f, 0.f};
      // Eight loads in flight, 128 columns.
      constexpr uint32_t AT_ONCE = S::COLS / 16 < 8 ? S::COLS / 16 : 8;
#pragma unroll
      for (uint32_t v0 = 0; v0 < S::COLS; v0 += 16 * AT_ONCE) {
        f4 x[AT_ONCE];
#pragma unroll
        for (uint32_t u = 0; u < AT_ONCE; ++u) x[u] = raw_four<S::VECV>(w, col0 + v0 + 16 * u + 4 * q, S::V);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (uint32_t u = 0; u < AT_ONCE; ++u) {
          x[u] = placed<S::VECV>(x[u], col0 + v0 + 16 * u + 4 * q, S::V);
          f4 g[S::RT];
#pragma unroll
          for (int r = 0; r < S::RT; ++r) g[r] = *reinterpret_cast<const f4*>(lds + (16 * r + t) * LD + v0 + 16 * u + 4 * q);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < S::RT; ++r) acc[r] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[u][i], g[r][i], acc[r], 0, 0, 0);
        }
      }
#pragma unroll
      for (int r = 0; r < S::RT; ++r) {
        const uint32_t row = 16 * r + t, d = d0 + 4 * q;
        if constexpr (S::CHUNKS > 1) *reinterpret_cast<f4*>(L.at(S::HPART) + ((size_t)chunk * S::NP + row) * S::DP + d) = acc[r];
        else if (row < S::N) put_four_of<S::VECD>(dh + (size_t)row * S::D, d, S::D, acc[r]);
      }
    }
    if constexpr (DW) {
      float x[4 * S::RT];       // h[4s + q][d0 + t]
#pragma unroll
      for (uint32_t s = 0; s < 4 * S::RT; ++s) {
        const float v = L.h[(size_t)min(4 * s + q, S::N - 1) * S::D + min(d0 + t, S::D - 1)];
        x[s] = kept >> s & 1u ? v : 0.f;
      }
      for (uint32_t v0 = 0; v0 < S::COLS; v0 += 64) {
        f4 acc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t s = 0; s < 4 * S::RT; ++s) {
          const f4 g = *reinterpret_cast<const f4*>(lds + (4 * s + q) * LD + v0 + 4 * turned);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[e], x[s], acc[e], 0, 0, 0);
        }
        if (d0 + t < S::D) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            put_four_of<S::VECV>(dw + (size_t)(d0 + t) * S::V, col0 + v0 + 16 * i + 4 * q, S::V, f4{acc[0][i], acc[1][i], acc[2][i], acc[3][i]});
          }
        }
      }
    }
  }
}

// The parts of dh added up: 32 groups of four columns a workgroup, every eighth part a thread, then those eight.
template <class S>
__device__ __forceinline__ void few_sums(const Loss<S>& L, float* dh, f4* scratch, uint32_t block) {
  const uint32_t i = block * 32 + threadIdx.x % 32, p = threadIdx.x / 32;
  const uint32_t row = i / (S::DP / 4), col = i % (S::DP / 4) * 4;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  if (row < S::NP) {
    const float* at = L.at(S::HPART) + (size_t)row * S::DP + col;
#pragma unroll 4
    for (uint32_t c = p; c < S::CHUNKS; c += 8) v += *reinterpret_cast<const f4*>(at + (size_t)c * S::NP * S::DP);
  }
  scratch[threadIdx.x] = v;
  __syncthreads();
  if (p == 0 && row < S::N) {
    for (uint32_t k = 1; k < 8; ++k) v += scratch[32 * k + threadIdx.x];
    put_four_of<S::VECD>(dh + (size_t)row * S::D, col, S::D, v);
  }
}

}  // namespace tcmi
