// Softmax attention over a sliding window with sinks, and its gradient, on the fp32 matrix cores.
//
// A query at position p of a sequence of L keys sees the keys j <= p with p - WINDOW < j or j < SINKS. With
// s_j = scale·q·k_j over those:
//   o = sum_j P_j v_j,  P_j = exp(s_j - lse),  lse = log(sum_j exp(s_j));
//   dS_j = P_j·(dy·v_j - dy·o),  dq = scale·sum_j dS_j k_j,  dk_j = scale·sum dS_j q,  dv_j = sum P_j dy (over the queries that see j).
// A query that sees nothing has o = 0, lse = -inf and no gradients. A key whose key or value holds a number that is not finite makes
// NaN of o and lse of the queries that see it, and a query's row with one (dy's too) of the gradients of the keys it sees; what does not
// see them, or is not seen, is as without them: 0 times them is taken as 0 (they are read as 0 where a sum runs over them). (What bf16 rounds to
// infinity counts as that wherever operands are split into parts, tcmi_window_wide.h: everywhere but in the forward pass here.)
//
// Rows: the queries of the R = H/HK heads that share a key head, query t's heads side by side. Here up to 16 of them, single tokens over a cache,
// on the fp32 matrix cores; more are tcmi_window_wide.h's, and all gradients. Keys 16 a
// tile. With lane = 16·q + t (t in 0..15) of a 16x16x4 product:
//   scores   mfma(key value, row value): lane (t, q) holds row t, keys 4q ... 4q + 3, which is
//   output   mfma(V value, P value): the second product's operand for those keys; lane (t, q) gets row t, dims 16g + 4q ....
// So scores never leave the registers, and keys and values are read
// from memory as the products take them. The four wavefronts of a workgroup deal the tiles among them and join at the
// end through LDS, always in the same order; several workgroups do (SPLITS), whose sums are joined by a launch.
//
// Bound: HBM (the keys and values that are seen, read once). 8 heads of 64 by 2 over caches of 131072 keys, 4 sequences: 101 us (5.3 TB/s) with 5 of them to
// join 128 splits; over 1024 keys and 4 of 32 sequences (34 MB) 12 and 4: the loads' time of a few tiles a wavefront, and the second launch's.

#pragma once

#include "tcmi_device.h"

namespace tcmi {

constexpr float LOG2E = 1.4426950408889634f;

// What a sequence's queries see.
template <class S>
struct WindowSpan {
  static constexpr uint32_t R = S::H / S::HK, ROWS = S::T * R;
  static constexpr bool FEW = ROWS <= 16u;      // whose forward pass is window_rows
  int32_t length, first;       // keys, and the position of query 0

  __device__ __forceinline__ WindowSpan(const float* lengths, uint32_t b) {
    length = static_cast<int32_t>(S::KEYS);
    if constexpr (S::LENGTHS) {
      const float l = lengths[b];
      // (Neither NaN nor what lies outside reaches the conversion.)
      if (!(l < static_cast<float>(S::KEYS))) length = l >= static_cast<float>(S::KEYS) ? length : 0;
      else length = l > 0.f ? static_cast<int32_t>(l) : 0;
    }
    first = S::LAST ? length - static_cast<int32_t>(S::T) : 0;
  }
  // The first key of the window of position p.
  __device__ __forceinline__ int32_t from(int32_t p) const { return S::WINDOW == 0u || p < static_cast<int32_t>(S::WINDOW) ? 0 : p - static_cast<int32_t>(S::WINDOW) + 1; }
  __device__ __forceinline__ bool stands(int32_t p) const { return p >= 0 && p < length; }
  // Whether position p (in 0 .. length-1) sees key j.
  __device__ __forceinline__ bool sees(int32_t p, int32_t j) const { return j <= p && (j >= from(p) || j < static_cast<int32_t>(S::SINKS)); }
};

// Tiles of 16 in order: `sinks` of them from 0, then from `main` up to `all` in number. Their keys that any of the rows sees: lo ... hi
// and the sinks before.
struct WindowTiles {
  int32_t sinks, main, all, lo, hi;
  __device__ __forceinline__ int32_t at(int32_t i) const { return i < sinks ? i : main + i - sinks; }
};

// The tiles of keys that rows row0 .. row1 see, of those that stand in their sequence.
template <class S>
__device__ __forceinline__ WindowTiles window_keys(const WindowSpan<S>& w, uint32_t row0, uint32_t row1) {
  constexpr int32_t R = WindowSpan<S>::R;
  int32_t p0 = w.first + static_cast<int32_t>(row0) / R, p1 = w.first + static_cast<int32_t>(row1) / R;
  p0 = max(p0, 0);
  p1 = min(p1, w.length - 1);
  if (p0 > p1) return {0, 0, 0, 0, -1};
  const int32_t lo = w.from(p0), sinks = (min(static_cast<int32_t>(S::SINKS), lo) + 15) / 16, main = max(lo / 16, sinks);
  return {sinks, main, sinks + p1 / 16 + 1 - main, lo, p1};
}

// Floats d ... d + 3 of the head at p, 0 where not `on` or past its end. The load is made in any case, of the head's last floats where d is
// past them (so p is a head that may be read): a branch around it would make the next one wait for it. INSIDE: of a head of whole 32 floats,
// d is within it.
template <class S, bool INSIDE = false>
__device__ __forceinline__ f4 window_load(const float* __restrict__ p, uint32_t d, bool on) {
  f4 v;
  if constexpr (S::VEC) {
    constexpr bool WHOLE = INSIDE && S::DH % 32u == 0u;
    v = *reinterpret_cast<const f4*>(p + (WHOLE ? d : min(d, S::DH - 4u)));
    const bool in = on && (WHOLE || d < S::DH);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = in ? v[i] : 0.f;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = p[min(d + i, S::DH - 1u)];
      v[i] = on && d + i < S::DH ? x : 0.f;
    }
  }
  return v;
}
template <class S>
__device__ __forceinline__ void window_store(float* __restrict__ p, uint32_t d, const f4& v) {
  if constexpr (S::VEC) {
    if (d < S::DH) *reinterpret_cast<f4*>(p + d) = v;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (d + i < S::DH) p[d + i] = v[i];
    }
  }
}

// Lane (t, q)'s part of a 16 x DH tile along its rows: dims 16g + 4q ... of row t.
template <class S, int G>
__device__ __forceinline__ void window_along(f4 (&v)[G], const float* __restrict__ row, bool on) {
#pragma unroll
  for (int g = 0; g < G; ++g) v[g] = window_load<S, true>(row, 16 * g + 4 * ((threadIdx.x >> 4) & 3u), on);
}
// And across them: dim 16g + t of the tile's key 4q + s, of the keys from j0 on. Every load is made, of the last key that one of the rows
// sees where its own is past it.
template <class S, int G>
__device__ __forceinline__ void window_read(f4 (&v)[G], const float* __restrict__ base, size_t step, int32_t j0, const WindowTiles& tiles) {
  const int t = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const float* at = base + (size_t)min(j0 + 4 * q + s, tiles.hi) * step + t;
#pragma unroll
    for (int g = 0; g < G; ++g) v[g][s] = at[16 * g + 16 <= static_cast<int>(S::DH) || 16 * g + t < static_cast<int>(S::DH) ? 16 * g : 0 - t];
  }
}
// What was read, 0 where it is not finite or of a key that none of the rows sees. Bit s: key 4q + s held a number that is not finite.
template <class S, int G>
__device__ __forceinline__ uint32_t window_clean(f4 (&v)[G], int32_t j0, const WindowTiles& tiles) {
  const int t = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
  uint32_t bad = 0u;
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int32_t j = j0 + 4 * q + s;
    const bool on = j <= tiles.hi && (j >= tiles.lo || j < static_cast<int32_t>(S::SINKS));
    bool all = true;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const bool in = on && (16 * g + 16 <= static_cast<int>(S::DH) || 16 * g + t < static_cast<int>(S::DH)), finite = __builtin_isfinite(v[g][s]);
      all = all && (finite || !in);
      v[g][s] = in && finite ? v[g][s] : 0.f;
    }
    if ((__ballot(!all) >> (threadIdx.x & 48u)) & 0xffffu) bad |= 1u << s;
  }
  return bad;
}
// Bit t: row t of a tile read along its rows holds a number that is not finite.
template <int G>
__device__ __forceinline__ uint32_t window_infinite(const f4 (&v)[G]) {
  bool all = true;
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int i = 0; i < 4; ++i) all = all && __builtin_isfinite(v[g][i]);
  }
  uint64_t bad = __ballot(!all);
  bad |= bad >> 32;
  bad |= bad >> 16;
  return static_cast<uint32_t>(bad) & 0xffffu;
}
// acc[k of a][t of b] += the products of two tiles along their rows.
template <int G>
__device__ __forceinline__ f4 window_scores(const f4 (&a)[G], const f4 (&b)[G]) {
  f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[g][s], b[g][s], acc, 0, 0, 0);
  }
  return acc;
}
template <int G>
__device__ __forceinline__ void window_sum(f4 (&acc)[G], const f4 (&across)[G], const f4& p) {
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int s = 0; s < 4; ++s) acc[g] = __builtin_amdgcn_mfma_f32_16x16x4f32(across[g][s], p[s], acc[g], 0, 0, 0);
  }
}

template <int DH>
constexpr int window_lds() { return 4 * 64 * ((DH + 15) / 16) * 4 + 4 * 32; }

// The four wavefronts' acc added into the first's, each times its factor f.
template <int G>
__device__ __forceinline__ void window_gather(f4 (&acc)[G], float f, float* lds) {
  f4* at = reinterpret_cast<f4*>(lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
#pragma unroll
  for (int g = 0; g < G; ++g) at[(wave * G + g) * 64 + lane] = acc[g] * f;
  __syncthreads();
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = at[g * 64 + lane] + at[(G + g) * 64 + lane] + at[(2 * G + g) * 64 + lane] + at[(3 * G + g) * 64 + lane];
}

// Workgroup: a sequence's key head, a split of the keys that its rows see.
template <class S>
__device__ __forceinline__ void window_rows(const float* __restrict__ qp, const float* __restrict__ kp, const float* __restrict__ vp, const float* __restrict__ lengths,
                                            float* __restrict__ out, float* __restrict__ lse, char* ws, float* lds, uint32_t wg) {
  constexpr int G = (S::DH + 15) / 16;
  using Span = WindowSpan<S>;
  constexpr uint32_t R = Span::R, ROWS = Span::ROWS;
  const uint32_t split = wg % S::SPLITS, head = wg / S::SPLITS, b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = threadIdx.x >> 6;
  const Span w(lengths, b);
  const uint32_t row = t, at = min(row, ROWS - 1u);
  const size_t line = ((size_t)b * S::T + at / R) * S::H + hk * R + at % R;
  const int32_t p = w.first + static_cast<int32_t>(at / R);
  const bool on = row < ROWS && w.stands(p);
  f4 qf[G], acc[G];
  window_along<S>(qf, qp + line * S::DH, on);
  // Scores in powers of two.
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
#pragma unroll
  for (int g = 0; g < G; ++g) acc[g] = f4{0.f, 0.f, 0.f, 0.f};
  const WindowTiles tiles = window_keys(w, 0u, ROWS - 1u);
  const int32_t each = (tiles.all + static_cast<int32_t>(S::SPLITS) - 1) / static_cast<int32_t>(S::SPLITS);
  const int32_t begin = min(tiles.all, static_cast<int32_t>(split) * each), end = min(tiles.all, begin + each);
  const size_t step = (size_t)S::HK * S::DH;
  const float* kb = kp + ((size_t)b * S::KEYS * S::HK + hk) * S::DH;
  const float* vb = vp + ((size_t)b * S::KEYS * S::HK + hk) * S::DH;
  float m = -TCMI_INF, l = 0.f, lowest = 0.f;
  // (Of a key past the last, the last again: its scores are not taken.) All loads of a tile are made before the tile before it is used.
  auto load = [&](int32_t i, f4 (&kf)[G], f4 (&vf)[G]) __attribute__((always_inline)) {
    const int32_t j0 = tiles.at(i) * 16;
    window_along<S>(kf, kb + (size_t)min(j0 + t, tiles.hi) * step, true);
    window_read<S>(vf, vb, step, j0, tiles);
  };
  f4 kf[G], vf[G], kn[G], vn[G];
  if (begin + wave < end) load(begin + wave, kn, vn);
  for (int32_t i = begin + wave; i < end; i += 4) {
    const int32_t j0 = tiles.at(i) * 16;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      kf[g] = kn[g];
      vf[g] = vn[g];
    }
    if (G <= 8 && i + 4 < end) load(i + 4, kn, vn);
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t bad = window_clean<S>(vf, j0, tiles);
    f4 s = window_scores(kf, qf);
    float top = -TCMI_INF;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      lowest = fminf(lowest, s[r]);
      s[r] = on && w.sees(p, j0 + 4 * q + r) ? (bad >> r & 1u ? __builtin_nanf("") : s[r] * scale) : -TCMI_INF;
      top = fmaxf(top, s[r]);
    }
    top = fmaxf(m, quad16_reduce<true>(top));
    const float base = top == -TCMI_INF ? 0.f : top, alpha = __builtin_amdgcn_exp2f(m - base);
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s[r] = __builtin_amdgcn_exp2f(s[r] - base);
      sum += s[r];
    }
    l = l * alpha + sum;
    m = top;
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] *= alpha;
    window_sum(acc, vf, s);
    if (G > 8 && i + 4 < end) load(i + 4, kn, vn);
  }
  // A key or a query that is infinite gives scores of NaN or of infinities, and of -infinity, which has no weight, makes NaN like the
  // others: where there was one, keys and queries are looked at again. (Read again, not kept,
  // for the registers.)
  if (__ballot(lowest == -TCMI_INF) != 0ull) {
    const float* again = qp;
    asm volatile("" : "+s"(again));
    window_along<S>(kf, again + line * S::DH, on);
    if (window_infinite(kf) >> t & 1u) l = __builtin_nanf("");
    for (int32_t i = begin + wave; i < end; i += 4) {
      const int32_t j0 = tiles.at(i) * 16;
      window_along<S>(kf, kb + (size_t)min(j0 + t, tiles.hi) * step, true);
      const uint32_t bad = window_infinite(kf) >> 4 * q;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if (bad >> r & 1u && on && w.sees(p, j0 + 4 * q + r)) l = __builtin_nanf("");
      }
    }
  }
  // (Each lane has added its own keys.)
  l = quad16_reduce<false>(l);
  float* stats = lds + 4 * 64 * G * 4;
  if (q == 0) {
    stats[wave * 32 + t] = m;
    stats[wave * 32 + 16 + t] = l;
  }
  __syncthreads();
  float top = -TCMI_INF, total = 0.f;
#pragma unroll
  for (int v = 0; v < 4; ++v) top = fmaxf(top, stats[v * 32 + t]);
  const float base = top == -TCMI_INF ? 0.f : top;
#pragma unroll
  for (int v = 0; v < 4; ++v) total += stats[v * 32 + 16 + t] * __builtin_amdgcn_exp2f(stats[v * 32 + t] - base);
  window_gather(acc, __builtin_amdgcn_exp2f(m - base), lds);
  if (wave != 0 || row >= ROWS) return;
  if constexpr (S::SPLITS == 1u) {
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
    if (out != nullptr) {
#pragma unroll
      for (int g = 0; g < G; ++g) window_store<S>(out + line * S::DH, 16 * g + 4 * q, acc[g] * inv);
    }
    if (lse != nullptr && q == 0) lse[line] = total > 0.f || total != total ? (base + __builtin_amdgcn_logf(total)) * 0.69314718055994531f : -TCMI_INF;
  } else {
    const size_t place = ((size_t)split * S::B * S::HK + head) * 16u + row;
#pragma unroll
    for (int g = 0; g < G; ++g) window_store<S>(reinterpret_cast<float*>(ws + S::OUT) + place * S::DH, 16 * g + 4 * q, acc[g]);
    if (q == 0) reinterpret_cast<float2*>(ws + S::STATS)[place] = make_float2(top, total);
  }
}

// Row `at` of all key heads' rows: its splits' sums. LANES lanes hold its floats; of many splits a
// workgroup's PARTS groups of them take some each (lds: PARTS·4·LANES floats).
template <class S, uint32_t LANES, uint32_t PARTS>
__device__ __forceinline__ void window_join(float* __restrict__ out, float* __restrict__ lse, const char* __restrict__ ws, float* lds, uint32_t at) {
  using Span = WindowSpan<S>;
  constexpr uint32_t R = Span::R, HEADS = S::B * S::HK;
  const uint32_t head = at / (S::TILES * 16u), row = at % (S::TILES * 16u), lane = threadIdx.x % LANES, part = PARTS > 1u ? threadIdx.x / LANES : 0u;
  if (head >= HEADS || row >= Span::ROWS) return;
  const float2* stats = reinterpret_cast<const float2*>(ws + S::STATS) + at;
  const float* sums = reinterpret_cast<const float*>(ws + S::OUT) + (size_t)at * S::DH;
  const size_t step = (size_t)HEADS * S::TILES * 16u;
  float top = -TCMI_INF, total = 0.f, base;
  if constexpr (PARTS > 1u) {
    // (A wavefront's lanes look at a split each.)
    for (uint32_t k = threadIdx.x & 63u; k < S::SPLITS; k += 64u) top = fmaxf(top, stats[k * step].x);
    top = wave_reduce<true>(top);
    base = top == -TCMI_INF ? 0.f : top;
    for (uint32_t k = threadIdx.x & 63u; k < S::SPLITS; k += 64u) total = fmaf(stats[k * step].y, __builtin_amdgcn_exp2f(stats[k * step].x - base), total);
    total = wave_reduce<false>(total);
  } else {
#pragma unroll 8
    for (uint32_t k = 0; k < S::SPLITS; ++k) top = fmaxf(top, stats[k * step].x);
    base = top == -TCMI_INF ? 0.f : top;
#pragma unroll 8
    for (uint32_t k = 0; k < S::SPLITS; ++k) total = fmaf(stats[k * step].y, __builtin_amdgcn_exp2f(stats[k * step].x - base), total);
  }
  const bool some = total > 0.f || total != total;
  const size_t line = ((size_t)(head / S::HK) * S::T + row / R) * S::H + head % S::HK * R + row % R;
  if (lse != nullptr && lane == 0u && part == 0u) lse[line] = some ? (base + __builtin_amdgcn_logf(total)) * 0.69314718055994531f : -TCMI_INF;
  if (out == nullptr) return;
  const float inv = some ? 1.f / total : 0.f;
  f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (uint32_t k = part; k < S::SPLITS; k += PARTS) {
    const f4 x = window_load<S>(sums + k * step * S::DH, 4u * lane, true);
    const float f = __builtin_amdgcn_exp2f(stats[k * step].x - base);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = fmaf(x[i], f, sum[i]);
  }
  if constexpr (PARTS > 1u) {
    f4* all = reinterpret_cast<f4*>(lds);
    all[threadIdx.x] = sum;
    __syncthreads();
    if (part != 0u) return;
#pragma unroll
    for (uint32_t p = 1; p < PARTS; ++p) sum += all[p * LANES + lane];
  }
  window_store<S>(out + line * S::DH, 4u * lane, sum * inv);
}

}  // namespace tcmi
