// Rows normalised by their root mean square and rotated by their tokens' positions, and
// the gradient of that, one pass over the rows each.
//
// A row x (one head of one token, DH floats) gives n = x·r·gain, r = (mean(x²) + eps)^-1/2
// (n = x without a gain), and each of its R pairs of dims (a, b) turns by the token's
// angle t = position·frequency: (n_a cos t - n_b sin t, n_b cos t + n_a sin t). Its
// gradient turns dy back (dn), then with h = x·r and g = dn·gain
//   dx = r·(g - h·mean(g·h)),   dgain = sum over rows of dn·h.
//
// Angles: a position of a million and a frequency of 1 leave float32 no digit of the
// angle's sine, so the turns position·(frequency / 2 pi) are formed and reduced in
// float64 (to an eighth of a turn around a multiple of a quarter), and the sine and cosine
// of what is left are Taylor polynomials in float32 (to t^11, t^12: below 2^-28 at pi/4).
//
// Layout: G = LANES lanes share a row, a lane holding its own pairs whole (E floats from
// each half, or E whole pairs where pairs are adjacent), so the rotation needs no
// exchange; the sums over a row are butterflies over its lanes. A token's angles are formed once by each
// group of lanes that holds some of its heads (SLOTS groups, a power of two) and used for
// all of them.
//
// Bound: HBM (x read and y written; x, dy read and dx written). 65 536 tokens of 32 heads of 128: 365 us (5.9 TB/s); gradients of 8191 tokens of 16
// heads, the gain's among them, 32.4 us (6.2 TB/s) and 4.6 for the gain's last sums.

#pragma once

#include "tcmi_device.h"

namespace tcmi {

// Sine and cosine of `turns` whole turns.
__device__ __forceinline__ void sincos_turns(double turns, float& s, float& c) {
  const double quarters = 4.0 * (turns - __builtin_rint(turns));   // [-2, 2]
  const double k = __builtin_rint(quarters);
  const float t = static_cast<float>((quarters - k) * 1.5707963267948966);   // [-pi/4, pi/4]
  const float t2 = t * t;
  const float sn = fmaf(t * t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, -1.f / 39916800.f, 1.f / 362880.f), -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), t);
  const float cs = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, 1.f / 479001600.f, -1.f / 3628800.f), 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const int q = static_cast<int>(k) & 3;
  const float a = q & 1 ? cs : sn, b = q & 1 ? sn : cs;
  s = q & 2 ? -a : a;
  c = (q + 1) & 2 ? -b : b;
}

// Sum over aligned groups of LANES lanes (a power of two up to 64), every lane getting it.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int off = LANES / 2; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// S: the sizes of one launch, as constants of its text:
//   DH, R, ADJ (adjacent pairs), GAIN, DX and DGAIN (which gradients; neither: forward)
//   E        floats of each half that a lane holds together (4: 128-bit loads, 1: any size)
//   LANES    lanes of a row; UNITS: groups of E pairs that a lane holds, TAILS: its groups
//            of E floats that are not rotated
//   B, M1, T, M2   x as [B, M1, T, M2, DH]: T tokens, M1·M2 heads; SHARED: one position a
//            token for all of B; AXES position axes
//   SLOTS    groups of lanes that a token's heads are dealt to
//   THREADS, and eps(), turns(j), axis(j)
template <class S>
struct RotaryLane {
  static constexpr int PAIRS = S::UNITS * S::E;     // pairs of this lane
  static constexpr int REST = S::TAILS * S::E;
  static constexpr int A = PAIRS > 0 ? PAIRS : 1, N = REST > 0 ? REST : 1;
  int lane;                                          // in the row

  // The pair that this lane's pair p is, or -1 past the row's.
  __device__ __forceinline__ int pair(int p) const {
    const int j = ((p / S::E) * S::LANES + lane) * S::E + p % S::E;
    return j < S::R ? j : -1;
  }
  // The dims of pair j, and of this lane's unrotated float p.
  static __device__ __forceinline__ int dim_a(int j) { return S::ADJ ? 2 * j : j; }
  static __device__ __forceinline__ int dim_b(int j) { return S::ADJ ? 2 * j + 1 : j + S::R; }
  __device__ __forceinline__ int rest(int p) const {
    const int e = 2 * S::R + ((p / S::E) * S::LANES + lane) * S::E + p % S::E;
    return e < S::DH ? e : -1;
  }

  // A row's floats: its pairs' a and b, then the rest.
  struct Row { float a[A], b[A], n[N]; };

  template <class F>
  static __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) f(p);
  }

  __device__ __forceinline__ void load(const float* __restrict__ x, Row& v) const {
    if constexpr (S::E == 4) {
#pragma unroll
      for (int u = 0; u < S::UNITS; ++u) {
        const int j = pair(u * 4);
        f4 p = {0.f, 0.f, 0.f, 0.f}, q = {0.f, 0.f, 0.f, 0.f};
        if (j >= 0) {
          p = *reinterpret_cast<const f4*>(x + (S::ADJ ? 2 * j : j));
          q = *reinterpret_cast<const f4*>(x + (S::ADJ ? 2 * j + 4 : j + S::R));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v.a[u * 4 + e] = S::ADJ ? (e < 2 ? p[2 * e] : q[2 * e - 4]) : p[e];
          v.b[u * 4 + e] = S::ADJ ? (e < 2 ? p[2 * e + 1] : q[2 * e - 3]) : q[e];
        }
      }
#pragma unroll
      for (int u = 0; u < S::TAILS; ++u) {
        const int e0 = rest(u * 4);
        f4 p = {0.f, 0.f, 0.f, 0.f};
        if (e0 >= 0) p = *reinterpret_cast<const f4*>(x + e0);
#pragma unroll
        for (int e = 0; e < 4; ++e) v.n[u * 4 + e] = p[e];
      }
    } else {
#pragma unroll
      for (int p = 0; p < PAIRS; ++p) {
        const int j = pair(p);
        v.a[p] = j >= 0 ? x[dim_a(j)] : 0.f;
        v.b[p] = j >= 0 ? x[dim_b(j)] : 0.f;
      }
#pragma unroll
      for (int p = 0; p < REST; ++p) {
        const int e = rest(p);
        v.n[p] = e >= 0 ? x[e] : 0.f;
      }
    }
  }

  __device__ __forceinline__ void store(float* __restrict__ y, const Row& v) const {
    if constexpr (S::E == 4) {
#pragma unroll
      for (int u = 0; u < S::UNITS; ++u) {
        const int j = pair(u * 4);
        f4 p, q;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = S::ADJ ? (e & 1 ? v.b[u * 4 + e / 2] : v.a[u * 4 + e / 2]) : v.a[u * 4 + e];
          q[e] = S::ADJ ? (e & 1 ? v.b[u * 4 + 2 + e / 2] : v.a[u * 4 + 2 + e / 2]) : v.b[u * 4 + e];
        }
        if (j >= 0) {
          *reinterpret_cast<f4*>(y + (S::ADJ ? 2 * j : j)) = p;
          *reinterpret_cast<f4*>(y + (S::ADJ ? 2 * j + 4 : j + S::R)) = q;
        }
      }
#pragma unroll
      for (int u = 0; u < S::TAILS; ++u) {
        const int e0 = rest(u * 4);
        if (e0 >= 0) *reinterpret_cast<f4*>(y + e0) = f4{v.n[u * 4], v.n[u * 4 + 1], v.n[u * 4 + 2], v.n[u * 4 + 3]};
      }
    } else {
#pragma unroll
      for (int p = 0; p < PAIRS; ++p) {
        const int j = pair(p);
        if (j >= 0) {
          y[dim_a(j)] = v.a[p];
          y[dim_b(j)] = v.b[p];
        }
      }
#pragma unroll
      for (int p = 0; p < REST; ++p) {
        const int e = rest(p);
        if (e >= 0) y[e] = v.n[p];
      }
    }
  }

  // f(i) over every float of a row that the lane holds, as (a, b, n)[i] of the rows given.
  template <class F, class... Rows>
  static __device__ __forceinline__ void zip(F f, Rows&... rows) {
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) f(rows.a[p]...);
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) f(rows.b[p]...);
#pragma unroll
    for (int p = 0; p < REST; ++p) f(rows.n[p]...);
  }
};

// The groups of SLOTS lane groups walk the tokens `first`, `first + step`, ...: one token a
// step, workgroup `block` of `blocks`. partial: S::DGAIN's sums of each workgroup [blocks][DH]; scratch: its lanes' sums in LDS.
template <class S>
__device__ __forceinline__ void rotary(const float* __restrict__ x, const float* __restrict__ pos, const float* __restrict__ gain,
                                       const float* __restrict__ dy, float* __restrict__ out, float* __restrict__ partial, float* scratch,
                                       const uint32_t block, const uint32_t blocks) {
  using L = RotaryLane<S>;
  constexpr bool GRAD = S::DX || S::DGAIN;
  constexpr uint32_t HEADS = S::M1 * S::M2, TOKENS = S::B * S::T;
  const uint32_t group = threadIdx.x / S::LANES;              // of this workgroup
  constexpr uint32_t GROUPS = S::THREADS / S::LANES;
  const L l{static_cast<int>(threadIdx.x % S::LANES)};
  const uint32_t slot = group % S::SLOTS;
  typename L::Row gn, dg;
  if constexpr (S::GAIN) l.load(gain, gn);
  L::zip([](float& d) { d = 0.f; }, dg);
  // This lane's pairs: turns a position, and the position's axis.
  double turns[L::A];
  uint32_t axis[L::A];
#pragma unroll
  for (int p = 0; p < L::PAIRS; ++p) {
    const int j = l.pair(p) < 0 ? 0 : l.pair(p);
    turns[p] = S::turns(j);
    axis[p] = S::axis(j);
  }
  const uint32_t step = blocks * (GROUPS / S::SLOTS);
  for (uint32_t token = block * (GROUPS / S::SLOTS) + group / S::SLOTS; token < TOKENS; token += step) {
    const uint32_t b = token / S::T, t = token % S::T;
    const float* at = pos + (size_t)(S::SHARED ? t : token) * S::AXES;
    float cs[L::A], sn[L::A];
#pragma unroll
    for (int p = 0; p < L::PAIRS; ++p) sincos_turns(static_cast<double>(at[S::AXES > 1 ? axis[p] : 0u]) * turns[p], sn[p], cs[p]);
    for (uint32_t h = slot; h < HEADS; h += S::SLOTS) {
      const size_t row = (((size_t)b * S::M1 + h / S::M2) * S::T + t) * S::M2 + h % S::M2;
      typename L::Row v, d;
      if constexpr (S::GAIN || !GRAD) l.load(x + row * S::DH, v);
      if constexpr (GRAD) l.load(dy + row * S::DH, d);
      float r = 1.f;
      if constexpr (S::GAIN) {
        float ss = 0.f;
        L::zip([&](float& e) { ss = fmaf(e, e, ss); }, v);
        // 1 ulp; a Newton step on it leaves every error as it is (outputs 6.5e-8, dx 7e-8, dgain 1.2e-7 - 2e-7 of their norms).
        r = __builtin_amdgcn_rsqf(lanes_sum<S::LANES>(ss) * (1.f / S::DH) + S::eps());
      }
      if constexpr (!GRAD) {
        if constexpr (S::GAIN) L::zip([&](float& e, float& g) { e = e * r * g; }, v, gn);
#pragma unroll
        for (int p = 0; p < L::PAIRS; ++p) {
          const float a = v.a[p], c = v.b[p];
          v.a[p] = fmaf(a, cs[p], -(c * sn[p]));
          v.b[p] = fmaf(c, cs[p], a * sn[p]);
        }
        l.store(out + row * S::DH, v);
      } else {
#pragma unroll
        for (int p = 0; p < L::PAIRS; ++p) {
          const float a = d.a[p], c = d.b[p];
          d.a[p] = fmaf(a, cs[p], c * sn[p]);
          d.b[p] = fmaf(c, cs[p], -(a * sn[p]));
        }
        if constexpr (S::GAIN) {
          float gh = 0.f;
          L::zip([&](float& e, float& dn, float& g, float& sum) {
            e *= r;
            if constexpr (S::DGAIN) sum = fmaf(dn, e, sum);
            dn *= g;
            gh = fmaf(dn, e, gh);
          }, v, d, gn, dg);
          if constexpr (S::DX) {
            const float mean = lanes_sum<S::LANES>(gh) * (1.f / S::DH);
            L::zip([&](float& e, float& dn) { dn = r * (dn - e * mean); }, v, d);
          }
        }
        if constexpr (S::DX) l.store(out + row * S::DH, d);
      }
    }
  }
  if constexpr (S::DGAIN) {
    // The workgroup's lane groups in turn: scratch[group][DH].
    l.store(scratch + group * S::DH, dg);
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < S::DH; e += S::THREADS) {
      float sum = 0.f;
      for (uint32_t g = 0; g < GROUPS; ++g) sum += scratch[g * S::DH + e];
      partial[(size_t)block * S::DH + e] = sum;
    }
  }
}

// out[e] = the sum of `blocks` partial rows: a workgroup of 1024 takes 16 columns, 64 threads a
// column, each its own rows in turn, their sums added in order by eights.
template <int DH>
__device__ __forceinline__ void rotary_gain_sum(const float* __restrict__ partial, float* __restrict__ out, uint32_t blocks, float* scratch, uint32_t block) {
  const uint32_t e = block * 16u + threadIdx.x % 16u, part = threadIdx.x / 16u;
  float sum = 0.f;
  if (e < DH) {
#pragma unroll 4
    for (uint32_t k = part; k < blocks; k += 64u) sum += partial[(size_t)k * DH + e];
  }
  scratch[threadIdx.x] = sum;
  __syncthreads();
  if (part < 8u) {
    for (uint32_t p = part + 8u; p < 64u; p += 8u) sum += scratch[p * 16u + threadIdx.x % 16u];
  }
  __syncthreads();
  if (part < 8u) scratch[threadIdx.x] = sum;
  __syncthreads();
  if (part == 0u && e < DH) {
    for (uint32_t p = 1; p < 8u; ++p) sum += scratch[p * 16u + threadIdx.x];
    out[e] = sum;
  }
}

}  // namespace tcmi
