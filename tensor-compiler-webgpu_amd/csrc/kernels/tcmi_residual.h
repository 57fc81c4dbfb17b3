// A block's branch y joined to its stream x, with the norms on both sides of the block in the same pass:
//
//   h = residual·x + gate·N(y),   n = N(h),   N(v) = (v - mean)·r·gain + bias,  r = (mean((v - mean)²) + eps)^-1/2
// (mean 0 and no bias for the root mean square; N(y) = y without a norm), and the gradient of both, with ^ for
// (v - mean)·r:
//   dH = dh + N'(dn·gain; h),   N'(g; v) = r·(g - mean(g) - v^·mean(g·v^)),
//   dx = residual·dH,   dp = dH·gate,   dy = N'(dp·postGain; y),
//   dgain = sum dn·h^, dbias = sum dn, dgate = sum dH·p (or each row's own), dpostGain = sum dp·y^, dpostBias = sum dp.
//
// LANES lanes share a row, at most 16 floats of it each, in registers: a row is read once and what the
// gradient needs of the forward pass is formed again. Means are of the row itself, squares of what is left. A workgroup walks
// its rows and keeps the vectors' sums in registers; its rows side by side are then added in LDS, and the
// workgroups' sums by a second launch, always in the same order.
//
// Bound: HBM. 8189 rows of 4095, root mean squares with a branch's norm and a gate: 98 us (537 MB, 5.5 TB/s), their gradients 162 (805 MB, 5.0 TB/s) and
// 8.5 for the vectors' sums; 8192 rows of 256 with mean and bias 7, 9.5 and 4 (34 and 50 MB, from the caches in part); 32 rows of 1024 3.2, a launch's time.

#pragma once

#include "tcmi_device.h"

namespace tcmi {

struct ResidualArgs {
  const float *x, *y, *gain, *bias, *postGain, *postBias, *gate, *dh, *dn;
};

// Four floats at any address of a float: one 128-bit access each.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// A row's floats of one lane: UNITS groups of four, LANES groups apart; past the row's end 0. (Rows of 4095 floats start at any
// float's address: by a float a lane their gradients take 193 us, by four 180.)
template <class S>
struct ResidualLane {
  static constexpr int F = S::UNITS * 4;
  typedef float Row[F];
  uint32_t lane;
  float* lds;

  __device__ __forceinline__ uint32_t dim(int i) const { return (i / 4 * S::LANES + lane) * 4u + i % 4; }
  __device__ __forceinline__ bool in(int i) const { return S::D % (S::LANES * 4u) == 0u || dim(i) < S::D; }
  __device__ __forceinline__ void load(const float* __restrict__ p, Row& v) const {
#pragma unroll
    for (int u = 0; u < F; u += 4) {
      f4u q = {0.f, 0.f, 0.f, 0.f};
      if (in(u + 3)) {
        q = *reinterpret_cast<const f4u*>(p + dim(u));
      } else if (S::D % 4u != 0u) {
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          if (in(u + e)) q[e] = p[dim(u + e)];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[u + e] = q[e];
    }
  }
  __device__ __forceinline__ void store(float* __restrict__ p, const Row& v) const {
#pragma unroll
    for (int u = 0; u < F; u += 4) {
      if (in(u + 3)) {
        *reinterpret_cast<f4u*>(p + dim(u)) = f4u{v[u], v[u + 1], v[u + 2], v[u + 3]};
      } else if (S::D % 4u != 0u) {
#pragma unroll
        for (int e = 0; e < 3; ++e) {
          if (in(u + e)) p[dim(u + e)] = v[u + e];
        }
      }
    }
  }
  // A vector of a row's floats, kept in LDS as the lanes hold it (STAGED), or read from memory.
  static constexpr uint32_t PAD = S::UNITS * 4 * S::LANES;
  __device__ __forceinline__ void keep(const float* __restrict__ p, float* to) const {
    Row v;
    load(p, v);
#pragma unroll
    for (int u = 0; u < F; u += 4) *reinterpret_cast<f4*>(to + dim(u)) = f4{v[u], v[u + 1], v[u + 2], v[u + 3]};
  }
  __device__ __forceinline__ void kept(const float* __restrict__ p, const float* from, Row& v) const {
    if constexpr (S::STAGED) {
#pragma unroll
      for (int u = 0; u < F; u += 4) {
        const f4 q = *reinterpret_cast<const f4*>(from + dim(u));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[u + e] = q[e];
      }
    } else {
      load(p, v);
    }
  }
  // Sums over the row's lanes, every lane getting them; over several wavefronts through LDS.
  template <int N>
  __device__ __forceinline__ void total(float (&v)[N]) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
      for (uint32_t off = min(S::LANES, 64u) / 2u; off >= 1u; off >>= 1) v[k] += __shfl_xor(v[k], off, 64);
    }
    if constexpr (S::LANES > 64u) {
      // A row's wavefronts are the workgroup's (LANES = THREADS) or a part of them.
      constexpr uint32_t WAVES = S::LANES / 64u;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        __syncthreads();
        if (threadIdx.x % 64u == 0u) lds[threadIdx.x / 64u] = v[k];
        __syncthreads();
        const uint32_t first = threadIdx.x / S::LANES * WAVES;
        float sum = lds[first];
#pragma unroll
        for (uint32_t w = 1; w < WAVES; ++w) sum += lds[first + w];
        v[k] = sum;
      }
    }
  }
  // v to its normalised row, without gain and bias; r.
  __device__ __forceinline__ float normalise(Row& v) const {
    if constexpr (S::LAYER) {
      float m[1] = {0.f};
#pragma unroll
      for (int i = 0; i < F; ++i) m[0] += v[i];
      total(m);
      const float mean = m[0] * (1.f / S::D);
#pragma unroll
      for (int i = 0; i < F; ++i) v[i] = in(i) ? v[i] - mean : 0.f;
    }
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < F; ++i) s[0] = fmaf(v[i], v[i], s[0]);
    total(s);
    // (The instruction takes what is below the normal numbers as 0.)
    const float square = s[0] * (1.f / S::D) + S::eps();
    float r = __builtin_amdgcn_rsqf(square);
    if (square < 0x1p-126f) r = __builtin_amdgcn_rsqf(square * 0x1p48f) * 0x1p24f;
#pragma unroll
    for (int i = 0; i < F; ++i) v[i] *= r;
    return r;
  }
  // g, a gradient of a normalised row v, to that of the row: r·(g - mean(g) - v·mean(g·v)).
  __device__ __forceinline__ void back(Row& g, const Row& v, float r) const {
    float s[S::LAYER ? 2 : 1] = {};
#pragma unroll
    for (int i = 0; i < F; ++i) {
      s[0] = fmaf(g[i], v[i], s[0]);
      if constexpr (S::LAYER) s[1] += g[i];
    }
    total(s);
    const float gv = s[0] * (1.f / S::D);
    float m = 0.f;
    if constexpr (S::LAYER) m = s[1] * (1.f / S::D);
#pragma unroll
    for (int i = 0; i < F; ++i) g[i] = r * (g[i] - m - v[i] * gv);
  }
};

// A gate's floats of row `row`.
template <class S>
__device__ __forceinline__ void residual_gate(const ResidualLane<S>& l, const ResidualArgs& a, uint32_t row, const float* vectors, typename ResidualLane<S>::Row& g) {
  if constexpr (S::GATE == 2) l.load(a.gate + (size_t)row * S::D, g);
  else l.kept(a.gate, vectors + 3 * ResidualLane<S>::PAD, g);
}

// p = N(y) and h of one row; yh: y, then y normalised (where it has a norm), whose r is returned; h: x, then h.
template <class S>
__device__ __forceinline__ float residual_join(const ResidualLane<S>& l, const ResidualArgs& a, uint32_t row, typename ResidualLane<S>::Row& yh,
                                               typename ResidualLane<S>::Row& p, typename ResidualLane<S>::Row& h, const float* vectors) {
  using L = ResidualLane<S>;
  float r = 1.f;
  if constexpr (S::POST) {
    r = l.normalise(yh);
    typename L::Row g;
    l.kept(a.postGain, vectors + L::PAD, g);
#pragma unroll
    for (int i = 0; i < L::F; ++i) p[i] = yh[i] * g[i];
    if (a.postBias != nullptr) {
      l.kept(a.postBias, vectors + 2 * L::PAD, g);
#pragma unroll
      for (int i = 0; i < L::F; ++i) p[i] += g[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < L::F; ++i) p[i] = yh[i];
  }
  if constexpr (S::GATE != 0) {
    typename L::Row g;
    residual_gate(l, a, row, vectors, g);
#pragma unroll
    for (int i = 0; i < L::F; ++i) h[i] = fmaf(S::residual(), h[i], g[i] * p[i]);
  } else {
#pragma unroll
    for (int i = 0; i < L::F; ++i) h[i] = fmaf(S::residual(), h[i], p[i]);
  }
  return r;
}

// H and NORM: which of h and n are written.
template <class S>
__device__ __forceinline__ void residual(const ResidualArgs& a, float* __restrict__ hout, float* __restrict__ nout, float* lds, uint32_t block, uint32_t blocks) {
  using L = ResidualLane<S>;
  constexpr uint32_t ROWS = S::THREADS / S::LANES;
  const L l{threadIdx.x % S::LANES, lds};
  for (uint32_t row0 = block * ROWS; row0 < S::N; row0 += blocks * ROWS) {
    // (Every lane takes part in the sums: a row past the last is the last again, and not written.)
    const uint32_t at = row0 + threadIdx.x / S::LANES, row = min(at, S::N - 1u);
    typename L::Row yh, p, h;
    l.load(a.y + (size_t)row * S::D, yh);
    l.load(a.x + (size_t)row * S::D, h);
    residual_join<S>(l, a, row, yh, p, h, nullptr);
    if (S::H && at < S::N) l.store(hout + (size_t)row * S::D, h);
    if constexpr (S::NORM) {
      l.normalise(h);
      typename L::Row g;
      l.load(a.gain, g);
#pragma unroll
      for (int i = 0; i < L::F; ++i) h[i] *= g[i];
      if (a.bias != nullptr) {
        l.load(a.bias, g);
#pragma unroll
        for (int i = 0; i < L::F; ++i) h[i] += g[i];
      }
      if (at < S::N) l.store(nout + (size_t)row * S::D, h);
    }
  }
}

// DX ... DGATE: the gradients to form; DH, DN: which cotangents there are; STAGED: gain, postGain, postBias and a gate of one
// vector are kept in LDS, from lds + SCRATCH on. partial: the SUMS vectors' sums of each
// workgroup, [SUMS][blocks][D]; lds: ROWS·D floats where rows stand side by side.
template <class S>
__device__ __forceinline__ void residual_grad(const ResidualArgs& a, float* __restrict__ dx, float* __restrict__ dy, float* __restrict__ dgate,
                                              float* __restrict__ partial, float* lds, uint32_t block, uint32_t blocks) {
  using L = ResidualLane<S>;
  constexpr uint32_t ROWS = S::THREADS / S::LANES;
  constexpr bool BRANCH = S::DY || S::DPOSTGAIN || S::DPOSTBIAS || S::DGATE;
  const L l{threadIdx.x % S::LANES, lds};
  // The vectors, which every row waits for (8189 rows of 4095 floats 180 us where they come from memory for each, 162 so).
  float* const vectors = lds + S::SCRATCH;
  if constexpr (S::STAGED) {
    const float* from[4] = {a.gain, a.postGain, a.postBias, S::GATE == 1 ? a.gate : nullptr};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (from[k] != nullptr && threadIdx.x < S::LANES) l.keep(from[k], vectors + k * L::PAD);
    }
    __syncthreads();
  }
  float sums[S::SUMS > 0 ? S::SUMS : 1][L::F];
#pragma unroll
  for (int k = 0; k < S::SUMS; ++k) {
#pragma unroll
    for (int i = 0; i < L::F; ++i) sums[k][i] = 0.f;
  }
  for (uint32_t row0 = block * ROWS; row0 < S::N; row0 += blocks * ROWS) {
    const uint32_t at = row0 + threadIdx.x / S::LANES, row = min(at, S::N - 1u);
    const bool on = at < S::N;
    // All that is read of the row, before any of it is used.
    typename L::Row yh, p, h, d, dh;
    l.load(a.y + (size_t)row * S::D, yh);
    l.load(a.x + (size_t)row * S::D, h);
    if constexpr (S::DN) l.load(a.dn + (size_t)row * S::D, d);
    if constexpr (S::DH && (S::DX || BRANCH)) l.load(a.dh + (size_t)row * S::D, dh);
    __builtin_amdgcn_sched_barrier(0);
    const float ry = residual_join<S>(l, a, row, yh, p, h, vectors);
    int k = 0;
    // What a sum adds of a row past the last: nothing.
    auto add = [&](float (&sum)[L::F], auto f) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < L::F; ++i) sum[i] += on ? f(i) : 0.f;
    };
    if constexpr (S::DN) {
      const float rh = l.normalise(h);
      if constexpr (S::DGAIN) add(sums[k++], [&](int i) { return d[i] * h[i]; });
      if constexpr (S::DBIAS) add(sums[k++], [&](int i) { return d[i]; });
      if constexpr (S::DX || BRANCH) {
        typename L::Row g;
        l.kept(a.gain, vectors, g);
#pragma unroll
        for (int i = 0; i < L::F; ++i) d[i] *= g[i];
        l.back(d, h, rh);
      }
    } else {
#pragma unroll
      for (int i = 0; i < L::F; ++i) d[i] = 0.f;
    }
    if constexpr (S::DH && (S::DX || BRANCH)) {
#pragma unroll
      for (int i = 0; i < L::F; ++i) d[i] += dh[i];
    }
    if constexpr (S::DX) {
      typename L::Row g;
#pragma unroll
      for (int i = 0; i < L::F; ++i) g[i] = S::residual() * d[i];
      if (on) l.store(dx + (size_t)row * S::D, g);
    }
    if constexpr (BRANCH) {
      if constexpr (S::GATE != 0) {
        if constexpr (S::DGATE) {
#pragma unroll
          for (int i = 0; i < L::F; ++i) p[i] *= d[i];
          if constexpr (S::GATE == 2) {
            if (on) l.store(dgate + (size_t)row * S::D, p);
          }
        }
        typename L::Row g;
        residual_gate(l, a, row, vectors, g);
#pragma unroll
        for (int i = 0; i < L::F; ++i) d[i] *= g[i];
      }
      if constexpr (S::DPOSTGAIN) add(sums[k++], [&](int i) { return d[i] * yh[i]; });
      if constexpr (S::DPOSTBIAS) add(sums[k++], [&](int i) { return d[i]; });
      if constexpr (S::DGATE && S::GATE == 1) add(sums[k++], [&](int i) { return p[i]; });
      if constexpr (S::DY) {
        if constexpr (S::POST) {
          typename L::Row g;
          l.kept(a.postGain, vectors + L::PAD, g);
#pragma unroll
          for (int i = 0; i < L::F; ++i) d[i] *= g[i];
          l.back(d, yh, ry);
        }
        if (on) l.store(dy + (size_t)row * S::D, d);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < S::SUMS; ++k) {
    float* to = partial + ((size_t)k * blocks + block) * S::D;
    if constexpr (ROWS == 1u) {
      l.store(to, sums[k]);
    } else {
      __syncthreads();
      l.store(lds + threadIdx.x / S::LANES * S::D, sums[k]);
      __syncthreads();
      for (uint32_t e = threadIdx.x; e < S::D; e += S::THREADS) {
        float sum = lds[e];
#pragma unroll
        for (uint32_t g = 1; g < ROWS; ++g) sum += lds[g * S::D + e];
        to[e] = sum;
      }
    }
  }
}

// out[e] = the sum of vector `which`'s `blocks` partial rows: a workgroup of 1024 takes 32 columns, 32 threads a
// column, each its own rows in turn, their sums added in order by fours.
template <uint32_t D>
__device__ __forceinline__ void residual_sum(const float* __restrict__ partial, float* __restrict__ out, uint32_t blocks, float* scratch, uint32_t block, uint32_t which) {
  const uint32_t e = block * 32u + threadIdx.x % 32u, part = threadIdx.x / 32u;
  const float* from = partial + (size_t)which * blocks * D;
  float sum = 0.f;
  if (e < D) {
#pragma unroll 8
    for (uint32_t k = part; k < blocks; k += 32u) sum += from[(size_t)k * D + e];
  }
  scratch[threadIdx.x] = sum;
  __syncthreads();
  if (part < 4u) {
#pragma unroll
    for (uint32_t q = part + 4u; q < 32u; q += 4u) sum += scratch[q * 32u + threadIdx.x % 32u];
  }
  __syncthreads();
  if (part < 4u) scratch[threadIdx.x] = sum;
  __syncthreads();
  if (part == 0u && e < D) {
#pragma unroll
    for (uint32_t q = 1; q < 4u; ++q) sum += scratch[q * 32u + threadIdx.x];
    out[e] = sum;
  }
}

}  // namespace tcmi
