// Attention over a sliding window (tcmi_window.h's formulas) for many rows, on the bf16 matrix cores: every operand as three
// bf16 parts, x = x0 + x1 + x2, and every product as the six of a_i·b_j with i + j <= 2, in float32 (what is left
// out: 2^-24 of a product at most). No operand needs a scale, so a key or value of any size is what it is to the queries that see it and
// nothing to the others; parts below bf16's least normal number, of values below 2^-102, are lost, and values from 2^128 - 2^119 on, which
// bf16 rounds to infinity, count as infinite.
//
// A workgroup's four wavefronts take 16 rows each (tcmi_window.h's rows: the queries of the heads that share a key head) and walk
// the tiles of NB keys that one of the 64 sees. A tile is loaded one ahead into registers, split by the thread that loaded it and
// kept in LDS as three planes. With lane = 16·q + t of a 16 x 16 x 32 product, whose operands are lines of 32 along the
// sum (8q ... of line t) and whose result is (lines 4q ... of the first, line t of the second):
//   scores   first operand K (lines: keys; the sum: dims), second Q: lane (t, q) holds row t, keys 4q ... of each 16;
//   output   first V transposed (lines: dims; the sum: 32 keys), second P: lane (t, q) gives row t, keys 4q ... of the first 16
//            and of the second 16 as its eight, as it holds them; V's lines are read in the same order of keys by
//            ds_read_b64_tr_b16, 4 keys of each lane's dim at a time.
// A tile's output is summed from 0 and joined to the rows' by one multiplication and addition with their change of maximum, so an
// accumulator is rounded once a tile.
//
// The gradients: tiles of 32 rows or keys; a gradient of queries walks the keys that its rows see, one of keys the rows that see its keys, in chunks, and
// each forms the scores again (seven products in all where five would do, but no sum is left to be joined over workgroups that
// do not share its lines). Both run side by side in one launch.
//
// Bound: few tiles a workgroup, with each its loads' time, its split into parts and two barriers; of longer sequences the matrix cores (tcmi_window_packed.h).
// 64 sequences of 128 tokens, 4 heads of 64: 11.5 us, with the gradients' 27; six bf16 products at the rate of a large one would take 2 and 5, the bytes 3 and 9.

#pragma once

#include "tcmi_window.h"
#include "tcmi_gemm_bf16x3.h"

namespace tcmi {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// What counts as a number here: what is below 2^128 - 2^119. The rest as NaN.
__device__ __forceinline__ bool window_finite(float x) { return fabsf(x) < 0x1.ffp127f; }
__device__ __forceinline__ f4 window_number(f4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = window_finite(v[i]) ? v[i] : __builtin_nanf("");
  return v;
}
// Of eight floats the first four, the first NaN where one of them is no number.
__device__ __forceinline__ f4 window_row(f4 a, const f4& b) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) most = fmaxf(fmaxf(most, fabsf(a[i])), fabsf(b[i]));
  a[0] = window_finite(most) ? a[0] : __builtin_nanf("");
  return a;
}

// Eight floats as three parts each.
struct Parts {
  bf16x8 p[3];
};
__device__ __forceinline__ void window_parts(const f4& a, const f4& b, const Minus& minus, Parts& out) {
  u4 w[3];
  float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float u = x[2 * i], v = x[2 * i + 1];
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const bf16x2 h = bf16_pair(u, v);
      w[p][i] = __builtin_bit_cast(uint32_t, h);
      if (p < 2) {
        u = minus.less_lo(u, h);
        v = minus.less_hi(v, h);
      }
    }
  }
#pragma unroll
  for (int p = 0; p < 3; ++p) out.p[p] = __builtin_bit_cast(bf16x8, w[p]);
}

// acc += a·b.
__device__ __forceinline__ void window_mfma(f4& acc, const Parts& a, const Parts& b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[2], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[2], b.p[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[1], b.p[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[0], b.p[0], acc, 0, 0, 0);
}

// A tile of NB lines of DP floats in LDS, three planes of LD bytes a line; 256 threads load and split it. A line's 16-byte chunk c is at
// place c ^ swap(line), so that the lanes that meet in a cycle of 256 bytes read all banks both ways: 16 lines of one chunk each, and 8
// lines of two chunks each.
template <class S, int NB>
struct WindowTile {
  static constexpr int DP = (S::DH + 31) / 32 * 32, LD = DP <= 32 ? 64 : DP <= 64 ? 128 : DP <= 128 ? 256 : 512, PLANE = NB * LD, BYTES = 3 * PLANE;
  static constexpr int CHUNKS = NB * DP / 4 / 256;             // of four floats, a thread's
  static_assert(NB * DP / 4 % 256 == 0, "whole chunks a thread");
  f4 x[CHUNKS];

  static __device__ __forceinline__ int swap(int line) {
    const int low = LD == 64 ? (line >> 2) & 1 : LD == 128 ? (line >> 1) & 3 : line & 7;
    return 2 * low + ((line >> 3) & 1);
  }
  static __device__ __forceinline__ int line(int i) { return (threadIdx.x + i * 256) / (DP / 4); }
  static __device__ __forceinline__ int dim(int i) { return (threadIdx.x + i * 256) % (DP / 4) * 4; }
  // at(line, on): where line `line`'s floats are (in any case somewhere that may be read); on = false for zeros.
  template <class F>
  __device__ __forceinline__ void load(F at) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      bool on = true;
      const float* p = at(line(i), on);
      x[i] = window_load<S, true>(p, dim(i), on);
    }
  }
  // CLEAN: what is not finite as 0, with bad[line] (if there is one) and *some set for its line.
  template <bool CLEAN>
  __device__ __forceinline__ void store(char* tile, const Minus& minus, uint32_t* bad = nullptr, uint32_t* some = nullptr) const {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      float u[4] = {x[i][0], x[i][1], x[i][2], x[i][3]};
      if constexpr (CLEAN) {
        bool all = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool finite = window_finite(u[e]);
          all = all && finite;
          u[e] = finite ? u[e] : 0.f;
        }
        if (bad != nullptr && !all) {
          bad[line(i)] = 1u;
          *some = 1u;
        }
      }
      char* to = tile + line(i) * LD + (((dim(i) >> 3) ^ swap(line(i))) << 4) + (dim(i) & 4) * 2;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const bf16x2 a = bf16_pair(u[0], u[1]), b = bf16_pair(u[2], u[3]);
        *reinterpret_cast<uint2*>(to + p * PLANE) = make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
        if (p < 2) {
          u[0] = minus.less_lo(u[0], a);
          u[1] = minus.less_hi(u[1], a);
          u[2] = minus.less_lo(u[2], b);
          u[3] = minus.less_hi(u[3], b);
        }
      }
    }
  }
  // This lane's part of a first operand: lines line0 + t, floats 32·slice + 8q .... (line0: a multiple of 16)
  static __device__ __forceinline__ void lines(const char* tile, int line0, int slice, Parts& f) {
    const int t = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3, at = t * LD + ((q ^ swap(t)) << 4);
#pragma unroll
    for (int p = 0; p < 3; ++p) f.p[p] = *reinterpret_cast<const bf16x8*>(tile + p * PLANE + line0 * LD + (at ^ (slice << 6)));
  }
  // Transposed: line dim0 + t, the sum over tile lines line0 + 4q ... and line0 + 16 + 4q ....
  static __device__ __forceinline__ void across(const char* tile, int line0, int dim0, Parts& f, int lane = threadIdx.x) {
    const int t = lane & 15, q = (lane >> 4) & 3, line = 4 * q + (t >> 2);
    const int at = (line * LD + ((((t >> 1) & 1) ^ swap(line)) << 4) + (t & 1) * 8) ^ (dim0 << 1);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      const char* from = tile + p * PLANE + line0 * LD + at;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(from));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(from + 16 * LD));
      f.p[p] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// Tiles of `size` keys that rows row0 .. row1 see, as window_keys gives those of 16.
template <int NB>
__device__ __forceinline__ WindowTiles window_wider(const WindowTiles& k) {
  if (k.hi < k.lo) return {0, 0, 0, 0, -1};
  const int32_t sinks = (k.sinks * 16 + NB - 1) / NB, main = max(k.lo / NB, sinks);
  return {sinks, main, sinks + k.hi / NB + 1 - main, k.lo, k.hi};
}

template <class S>
struct WindowWide {
  static constexpr int DP = (S::DH + 31) / 32 * 32, SLICES = DP / 32, G = DP / 16;
  static constexpr int NB = DP <= 64 ? 64 : 32;        // keys of a tile: as many floats whatever the head
  static constexpr int BLOCKS = NB / 16;
  static constexpr uint32_t ROWS = 64;                 // of a workgroup
  using T = WindowTile<S, NB>;
  static constexpr int LDS = 2 * T::BYTES + (NB + 4) * 4;
};

// The `split`-th of SPLITS runs of n.
template <class S>
__device__ __forceinline__ void window_run(int32_t n, uint32_t split, int32_t& begin, int32_t& end) {
  const int32_t each = (n + static_cast<int32_t>(S::SPLITS) - 1) / static_cast<int32_t>(S::SPLITS);
  begin = min(n, static_cast<int32_t>(split) * each);
  end = min(n, begin + each);
}

// Dot products of this lane's row with a tile's lines: acc[k] = lines 16k ... of `tile` by f.
template <class T, int BLOCKS, int SLICES>
__device__ __forceinline__ void window_dots(f4 (&acc)[BLOCKS], const char* tile, const Parts (&f)[SLICES]) {
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {
    acc[k] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < SLICES; ++d) {
      Parts x;
      T::lines(tile, 16 * k, d, x);
      window_mfma(acc[k], x, f[d]);
    }
  }
}

// Workgroup: W::ROWS rows of a sequence's key head, a split of the keys they see.
template <class S>
__device__ __forceinline__ void window_wide(const float* __restrict__ qp, const float* __restrict__ kp, const float* __restrict__ vp, const float* __restrict__ lengths,
                                            float* __restrict__ out, float* __restrict__ lse, char* ws, char* lds, uint32_t head, uint32_t tile, uint32_t split) {
  using W = WindowWide<S>;
  using Span = WindowSpan<S>;
  constexpr uint32_t R = Span::R, ROWS = Span::ROWS;
  constexpr int NB = W::NB, BLOCKS = W::BLOCKS, SLICES = W::SLICES, G = W::G;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span w(lengths, b);
  const Minus minus;
  const uint32_t row0 = tile * W::ROWS;
  const WindowTiles keys = window_keys(w, min(row0, ROWS - 1u), min(row0 + W::ROWS - 1u, ROWS - 1u)), tiles = window_wider<NB>(keys);
  // The wavefront's rows, scores in powers of two.
  const uint32_t mine = row0 + 16u * wave, row = mine + t, at = min(row, ROWS - 1u);
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
  const size_t line = ((size_t)b * S::T + at / R) * S::H + hk * R + at % R;
  const int32_t pos = w.first + static_cast<int32_t>(at / R);
  const bool on = row < ROWS && w.stands(pos);
  Parts qf[SLICES];
#pragma unroll
  for (int s = 0; s < SLICES; ++s) {
    const f4 x = window_load<S, true>(qp + line * S::DH, 32 * s + 8 * q, on), y = window_load<S, true>(qp + line * S::DH, 32 * s + 8 * q + 4, on);
    window_parts(window_row(x, y) * scale, y * scale, minus, qf[s]);
  }
  // Positions of the wavefront's first and last row: tiles between them need no look at each pair.
  const bool full = mine + 16u <= ROWS && w.stands(w.first + static_cast<int32_t>(mine / R)) && w.stands(w.first + static_cast<int32_t>((mine + 15u) / R));
  const int32_t p0 = w.first + static_cast<int32_t>(min(mine, ROWS - 1u) / R), p1 = w.first + static_cast<int32_t>(min(mine + 15u, ROWS - 1u) / R);
  f4 o[G];
  float m = -TCMI_INF, l = 0.f;
#pragma unroll
  for (int g = 0; g < G; ++g) o[g] = f4{0.f, 0.f, 0.f, 0.f};
  const size_t step = (size_t)S::HK * S::DH, base = ((size_t)b * S::KEYS * S::HK + hk) * S::DH;
  using T = typename W::T;
  T x;                                   // K's next tile, or V's: never both at once
  char *klds = lds, *vlds = lds + T::BYTES;
  uint32_t *bad = reinterpret_cast<uint32_t*>(lds + 2 * T::BYTES), *some_bad = bad + NB;      // values of the tile that are not finite
  auto load = [&](const float* p, int32_t i) __attribute__((always_inline)) {
    const int32_t j0 = tiles.at(i) * NB;
    x.load([&](int line, bool& on) {
      const int32_t j = j0 + line;
      on = j <= keys.hi && (j >= keys.lo || j < static_cast<int32_t>(S::SINKS));
      return p + base + (size_t)min(j, keys.hi) * step;
    });
  };
  int32_t begin, end;
  window_run<S>(tiles.all, split, begin, end);
  auto scores = [&](int32_t j0, bool whole, float& alpha, Parts (&pf)[BLOCKS / 2]) __attribute__((always_inline)) {
    f4 s[BLOCKS];
    window_dots<T>(s, klds, qf);
    if (!whole) {
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[k][r] = on && w.sees(pos, j0 + 16 * k + 4 * q + r) ? s[k][r] : -TCMI_INF;
      }
    }
    float top = -TCMI_INF;
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
      for (int r = 0; r < 4; ++r) top = fmaxf(top, s[k][r]);
    }
    top = fmaxf(m, quad16_reduce<true>(top));
    const float zero = top == -TCMI_INF ? 0.f : top;
    alpha = __builtin_amdgcn_exp2f(m - zero);
    m = top;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[k][r] = __builtin_amdgcn_exp2f(s[k][r] - zero);
        sum += s[k][r];
      }
    }
    l = fmaf(l, alpha, sum);
#pragma unroll
    for (int k = 0; k < BLOCKS; k += 2) window_parts(s[k], s[k + 1], minus, pf[k / 2]);
  };
  if (begin < end) load(kp, begin);
  for (int32_t i = begin; i < end; ++i) {
    const int32_t j0 = tiles.at(i) * NB;
    __syncthreads();
    x.template store<false>(klds, minus);
    if (threadIdx.x <= NB) bad[threadIdx.x] = 0u;
    load(vp, i);
    __syncthreads();
    // (What none of the wavefront's rows sees: past its last position, or between its sinks and its windows.)
    const bool some = j0 <= p1 && (j0 + NB > w.from(p0) || j0 < static_cast<int32_t>(S::SINKS));
    const bool whole = full && j0 + NB - 1 <= p0 && (j0 >= w.from(p1) || j0 + NB <= static_cast<int32_t>(S::SINKS));
    float alpha;
    Parts pf[BLOCKS / 2];
    if (some) scores(j0, whole, alpha, pf);
    x.template store<true>(vlds, minus, bad, some_bad);
    __syncthreads();
    if (i + 1 < end) load(kp, i + 1);
    if (!some) continue;
    if (*some_bad) {
      for (int k = 0; k < BLOCKS * 4; ++k) {
        const int at = k / 4 * 16 + 4 * q + k % 4;
        if (bad[at] && on && w.sees(pos, j0 + at)) l = __builtin_nanf("");
      }
    }
#pragma unroll
    for (int g = 0; g < G; g += 2) {
      f4 sum[2] = {f4{0.f, 0.f, 0.f, 0.f}, f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < BLOCKS / 2; ++k) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          Parts f;
          T::across(vlds, 32 * k, 16 * (g + e), f);
          window_mfma(sum[e], f, pf[k]);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[g + e][r] = fmaf(o[g + e][r], alpha, sum[e][r]);
      }
    }
  }
  const float total = quad16_reduce<false>(l);
  const bool some = total > 0.f || total != total;
  if (row >= ROWS) return;
  if constexpr (S::SPLITS > 1u) {
    const size_t place = ((size_t)split * S::B * S::HK + head) * S::TILES * 16u + row;
#pragma unroll
    for (int g = 0; g < G; ++g) window_store<S>(reinterpret_cast<float*>(ws + S::OUT) + place * S::DH, 16 * g + 4 * q, o[g]);
    if (q == 0) reinterpret_cast<float2*>(ws + S::STATS)[place] = make_float2(m, total);
    return;
  }
  const float inv = some ? 1.f / total : 0.f;
  if (out != nullptr) {
#pragma unroll
    for (int g = 0; g < G; ++g) window_store<S>(out + line * S::DH, 16 * g + 4 * q, o[g] * inv);
  }
  if (lse != nullptr && q == 0) lse[line] = some ? (m + __builtin_amdgcn_logf(total)) * 0.69314718055994531f : -TCMI_INF;
}

// acc[h][g] += the sums over a tile's lines of its floats 16g ... times f[h].
template <class T, int HB, int G, int PAIRS>
__device__ __forceinline__ void window_sums(f4 (&acc)[HB][G], const char* tile, const Parts (&f)[HB][PAIRS]) {
  // (The wavefront that multiplies goes before one that loads or forms parts.)
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int g = 0; g < G; g += 2) {
    f4 sum[HB][2];
#pragma unroll
    for (int h = 0; h < HB; ++h) sum[h][0] = sum[h][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < PAIRS; ++k) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        Parts x;
        T::across(tile, 32 * k, 16 * (g + e), x);
#pragma unroll
        for (int h = 0; h < HB; ++h) window_mfma(sum[h][e], x, f[h][k]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int h = 0; h < HB; ++h) acc[h][g + e] += sum[h][e];
    }
  }
  __builtin_amdgcn_s_setprio(0);
}
// A line's parts, as a second operand.
template <class S, int SLICES>
__device__ __forceinline__ void window_line(Parts (&f)[SLICES], const float* __restrict__ p, bool on, float scale, const Minus& minus) {
  const int q = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int s = 0; s < SLICES; ++s) {
    const f4 x = window_load<S, true>(p, 32 * s + 8 * q, on), y = window_load<S, true>(p, 32 * s + 8 * q + 4, on);
    window_parts(x * scale, y * scale, minus, f[s]);
  }
}

struct WindowGradArgs {
  const float *q, *k, *v, *lengths, *o, *lse, *dy, *mass;
};

// The bits of the largest magnitude so far (of NaN above all others), and whether all are numbers.
__device__ __forceinline__ uint32_t window_most(uint32_t most, float x) { return max(most, __float_as_uint(x) & 0x7fffffffu); }
__device__ __forceinline__ bool window_numbers(uint32_t most) { return most < __float_as_uint(0x1.ffp127f); }
// A lane's share of dy·o, to be added to others': 2^-8 of it, so that up to 128 of them stay in float32, infinity where it has left that itself, and NaN
// only where an operand is no number: P, which dv is made of, does not hang on dy·o.
__device__ __forceinline__ float window_share(float sum, uint32_t most) {
  sum = fabsf(sum) < TCMI_INF ? sum * 0x1p-8f : TCMI_INF;
  return window_numbers(most) ? sum : __builtin_nanf("");
}
// dy·o of a row, whose floats 32·s + 8q ... lane (t, q) adds up; every lane of the row gets it. NaN where dy holds what is no number.
template <class S>
__device__ __forceinline__ float window_row_mass(const float* __restrict__ o, const float* __restrict__ dy, bool on) {
  const int q = (threadIdx.x >> 4) & 3;
  float sum = 0.f;
  uint32_t most = 0u;
#pragma unroll
  for (int s = 0; s < (static_cast<int>(S::DH) + 31) / 32; ++s) {
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      const f4 x = window_load<S, true>(o, 32 * s + 8 * q + h, on), y = window_load<S, true>(dy, 32 * s + 8 * q + h, on);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum = fmaf(x[i], y[i], sum);
        most = window_most(most, y[i]);
      }
    }
  }
  return quad16_reduce<false>(window_share(sum, most)) * 0x1p8f;
}
// Of 16 lines a wavefront from `line` on, for heads above 128. (NaN also of a query that is no number here and was one to tcmi_window.h.)
template <class S>
__device__ __forceinline__ void window_wide_mass(const float* __restrict__ qp, const float* __restrict__ o, const float* __restrict__ dy, float* __restrict__ mass, size_t line) {
  constexpr size_t LINES = (size_t)S::B * S::T * S::H;
  const size_t at = line + (threadIdx.x & 15u), row = min(at, LINES - 1u) * S::DH;
  float sum = window_row_mass<S>(o + row, dy + row, true);
  if constexpr (WindowSpan<S>::FEW) {
    bool all = true;
    for (uint32_t d = threadIdx.x >> 4 & 3u; d < S::DH; d += 4u) all = all && window_finite(qp[row + d]);
    const uint64_t bad = __ballot(!all);
    if ((bad | bad >> 16 | bad >> 32 | bad >> 48) >> (threadIdx.x & 15u) & 1u) sum = __builtin_nanf("");
  }
  if ((threadIdx.x & 48u) == 0u && at < LINES) mass[at] = sum;
}

// The gradients: tiles of 32 lines, 16 lines a wavefront's own.
template <class S>
struct WindowBack {
  static constexpr int DP = (S::DH + 31) / 32 * 32, SLICES = DP / 32, G = DP / 16, NB = 32;
  static constexpr uint32_t ROWS = 64;
  using T = WindowTile<S, NB>;
  static constexpr int LDS = 2 * T::BYTES + (2 + SLICES) * NB * 4;
};

// Workgroup: W::ROWS rows of a sequence's key head, a split of the keys they see. parts: the splits' sums, [SPLITS][lines][DH].
template <class S>
__device__ __forceinline__ void window_wide_dq(const WindowGradArgs a, float* __restrict__ dq, float* __restrict__ parts, char* lds, uint32_t head, uint32_t tile, uint32_t split) {
  using W = WindowBack<S>;
  using T = typename W::T;
  using Span = WindowSpan<S>;
  constexpr uint32_t R = Span::R, ROWS = Span::ROWS;
  constexpr int NB = W::NB, SLICES = W::SLICES, G = W::G;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span w(a.lengths, b);
  const Minus minus;
  const uint32_t row0 = tile * W::ROWS, mine = row0 + 16u * wave, row = mine + t, own = min(row, ROWS - 1u);
  const WindowTiles keys = window_keys(w, min(row0, ROWS - 1u), min(row0 + W::ROWS - 1u, ROWS - 1u)), tiles = window_wider<NB>(keys);
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
  const size_t line = ((size_t)b * S::T + own / R) * S::H + hk * R + own % R;
  const int32_t pos = w.first + static_cast<int32_t>(own / R);
  const bool on = row < ROWS && w.stands(pos);
  Parts qf[SLICES], df[SLICES];
  window_line<S>(qf, a.q + line * S::DH, on, scale, minus);
  window_line<S>(df, a.dy + line * S::DH, on, 1.f, minus);
  const float lse = on ? a.lse[line] * LOG2E : 0.f, mass = window_row_mass<S>(a.o + line * S::DH, a.dy + line * S::DH, on);
  f4 acc[1][G];
#pragma unroll
  for (int g = 0; g < G; ++g) acc[0][g] = f4{0.f, 0.f, 0.f, 0.f};
  const bool full = mine + 16u <= ROWS && w.stands(w.first + static_cast<int32_t>(mine / R)) && w.stands(w.first + static_cast<int32_t>((mine + 15u) / R));
  const int32_t p0 = w.first + static_cast<int32_t>(min(mine, ROWS - 1u) / R), p1 = w.first + static_cast<int32_t>(min(mine + 15u, ROWS - 1u) / R);
  const size_t step = (size_t)S::HK * S::DH, base = ((size_t)b * S::KEYS * S::HK + hk) * S::DH;
  T kt, vt;
  char *klds = lds, *vlds = lds + T::BYTES;
  auto load = [&](int32_t i) __attribute__((always_inline)) {
    const int32_t j0 = tiles.at(i) * NB;
    auto at = [&](const float* p) {
      return [=, &keys](int line, bool& on) {
        const int32_t j = j0 + line;
        on = j <= keys.hi && (j >= keys.lo || j < static_cast<int32_t>(S::SINKS));
        return p + base + (size_t)min(j, keys.hi) * step;
      };
    };
    kt.load(at(a.k));
    vt.load(at(a.v));
  };
  int32_t begin, end;
  window_run<S>(tiles.all, split, begin, end);
  if (begin < end) load(begin);
  for (int32_t i = begin; i < end; ++i) {
    const int32_t j0 = tiles.at(i) * NB;
    __syncthreads();
    // (Of a key that is no number the scores here are of zeros, whose row's lse is NaN. Where tcmi_window.h took it for a number its value's line is.)
#pragma unroll
    for (int c = 0; c < T::CHUNKS && Span::FEW; ++c) {
      const f4 x = kt.x[c];
      if (!window_finite(fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fabsf(x[2])), fabsf(x[3])))) vt.x[c][0] = __builtin_nanf("");
    }
    kt.template store<true>(klds, minus);
    vt.template store<false>(vlds, minus);
    __syncthreads();
    if (i + 1 < end) load(i + 1);
    if (j0 > p1 || (j0 + NB <= w.from(p0) && j0 >= static_cast<int32_t>(S::SINKS))) continue;
    const bool whole = full && j0 + NB - 1 <= p0 && (j0 >= w.from(p1) || j0 + NB <= static_cast<int32_t>(S::SINKS));
    f4 s[2], dp[2];
    window_dots<T>(s, klds, qf);
    window_dots<T>(dp, vlds, df);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float d = __builtin_amdgcn_exp2f(s[k][r] - lse) * (dp[k][r] - mass);
        s[k][r] = whole || (on && w.sees(pos, j0 + 16 * k + 4 * q + r)) ? d : 0.f;
      }
    }
    Parts ds[1][1];
    window_parts(s[0], s[1], minus, ds[0][0]);
    window_sums<T>(acc, klds, ds);
  }
  if (row >= ROWS) return;
  float* to = S::SPLITS > 1u ? parts + ((size_t)split * S::B * S::T * S::H + line) * S::DH : dq + line * S::DH;
  const float by = S::SPLITS > 1u ? 1.f : static_cast<float>(S::scale());
#pragma unroll
  for (int g = 0; g < G; ++g) window_store<S>(to, 16 * g + 4 * q, acc[0][g] * by);
}

// The positions that see one of `keys` keys from `first` on: from the first key on, up to the last one's window or the sequence's
// end; and their tiles of 32 rows.
template <class S>
struct WindowSeen {
  int32_t p0, p1, begin, end;
  __device__ __forceinline__ WindowSeen(const WindowSpan<S>& w, int32_t first, int32_t keys) {
    constexpr int32_t R = WindowSpan<S>::R;
    const int32_t last = min(first + keys, w.length) - 1;
    p0 = max(first, w.first);
    p1 = w.length - 1;
    if (S::WINDOW != 0u && first >= static_cast<int32_t>(S::SINKS) && p1 - last >= static_cast<int32_t>(S::WINDOW)) p1 = last + static_cast<int32_t>(S::WINDOW) - 1;
    p1 = min(p1, w.first + static_cast<int32_t>(S::T) - 1);
    if (first >= w.length) p1 = p0 - 1;
    begin = end = 0;
    if (p0 <= p1) {
      begin = (p0 - w.first) * R / 32;
      end = ((p1 - w.first + 1) * R + 31) / 32;
    }
  }
  // Their chunks of CHUNK tiles: of a window's counted from the first tile, or of all rows', which the chunks of other keys share.
  static constexpr bool SHARED = S::WINDOW == 0u;
  __device__ __forceinline__ uint32_t start() const { return SHARED ? begin / S::CHUNK : 0u; }
  __device__ __forceinline__ uint32_t chunks() const { return (end - (SHARED ? begin / S::CHUNK * S::CHUNK : begin) + S::CHUNK - 1u) / S::CHUNK; }
  __device__ __forceinline__ int32_t from(uint32_t chunk) const { return SHARED ? max(begin, static_cast<int32_t>((start() + chunk) * S::CHUNK)) : begin + static_cast<int32_t>(chunk * S::CHUNK); }
  __device__ __forceinline__ int32_t to(uint32_t chunk) const { return min(end, static_cast<int32_t>(SHARED ? (start() + chunk + 1u) * S::CHUNK : begin + (chunk + 1u) * S::CHUNK)); }
};

// The sums of a lane's keys to dk and dv, or to chunk `chunk` of their parts: [c][keys][DH] for c < CHUNKS, and for more (keys below
// SINKS alone have them) the FEW first keys' [c - CHUNKS][B][FEW][HK][DH].
template <class S, bool DK, bool DV, int HB, int G>
__device__ __forceinline__ void window_key_sums(float* __restrict__ dk, float* __restrict__ dv, char* ws, uint32_t b, uint32_t hk, uint32_t chunk, const int32_t (&key)[HB],
                                                const f4 (&dka)[HB][G], const f4 (&dva)[HB][G]) {
  const int q = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    if (key[h] >= static_cast<int32_t>(S::KEYS)) continue;
    const size_t line = ((size_t)b * S::KEYS + key[h]) * S::HK + hk;
    float *tk = dk + line * S::DH, *tv = dv + line * S::DH;
    float by = static_cast<float>(S::scale());
    if constexpr (S::CHUNKS_MOST > 1u) {
      if (chunk >= S::CHUNKS && key[h] >= static_cast<int32_t>(S::FEW)) continue;
      constexpr size_t ALL = (size_t)S::B * S::KEYS * S::HK, SOME = (size_t)S::B * S::FEW * S::HK;
      const size_t at = (chunk < S::CHUNKS ? chunk * ALL + line : S::CHUNKS * ALL + (chunk - S::CHUNKS) * SOME + ((size_t)b * S::FEW + key[h]) * S::HK + hk) * S::DH;
      tk = reinterpret_cast<float*>(ws + S::DKPARTS) + at;
      tv = reinterpret_cast<float*>(ws + S::DVPARTS) + at;
      by = 1.f;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if constexpr (DK) window_store<S>(tk, 16 * g + 4 * q, dka[h][g] * by);
      if constexpr (DV) window_store<S>(tv, 16 * g + 4 * q, dva[h][g]);
    }
  }
}

// Workgroup: W::ROWS keys of a sequence's key head, the `chunk`-th CHUNK tiles of 32 rows of those that see one of them.
template <class S, bool DK, bool DV>
__device__ __forceinline__ void window_wide_dkv(const WindowGradArgs a, float* __restrict__ dk, float* __restrict__ dv, char* ws, char* lds, uint32_t head, uint32_t tile, uint32_t chunk) {
  using W = WindowBack<S>;
  using T = typename W::T;
  using Span = WindowSpan<S>;
  constexpr int32_t R = Span::R, ROWS = Span::ROWS;
  constexpr int NB = W::NB, SLICES = W::SLICES, G = W::G;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span w(a.lengths, b);
  const Minus minus;
  const int32_t j0 = tile * W::ROWS, mine = j0 + 16 * wave, key = mine + t;
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
  Parts kf[SLICES], vf[SLICES];
  f4 dka[1][G], dva[1][G];
  const WindowSeen<S> all(w, j0, W::ROWS), own(w, mine, 16);
  if (chunk < all.start()) return;
  chunk -= all.start();
  if (chunk > 0u && chunk >= all.chunks()) return;
  const int32_t p0 = all.p0, p1 = all.p1, m0 = own.p0, m1 = own.p1;
  const int32_t begin = all.from(chunk), end = all.to(chunk);
  const size_t line = ((size_t)b * S::KEYS + min(key, static_cast<int32_t>(S::KEYS) - 1)) * S::HK + hk;
  const bool on = begin < end && key < w.length;
  window_line<S>(kf, a.k + line * S::DH, on, scale, minus);
  if constexpr (DK) window_line<S>(vf, a.v + line * S::DH, on, 1.f, minus);
#pragma unroll
  for (int g = 0; g < G; ++g) dka[0][g] = dva[0][g] = f4{0.f, 0.f, 0.f, 0.f};
  const size_t top = ((size_t)b * S::T) * S::H + hk * R;
  auto place = [&](int32_t r) { return top + (size_t)(r / R) * S::H + r % R; };
  T qt, dt, ot;
  float lse = 0.f, before = 0.f;
  char *qlds = lds, *dlds = lds + T::BYTES;
  float* const row_lse = reinterpret_cast<float*>(lds + 2 * T::BYTES);
  float* const row_mass = row_lse + NB;
  int32_t* const row_pos = reinterpret_cast<int32_t*>(row_mass + SLICES * NB);
  int32_t row_at = 0;
  auto at = [&](const float* p, int32_t r0) {
    return [=, &place, &w](int l, bool& on) {
      const int32_t r = r0 + l, pos = w.first + r / R;
      on = r < ROWS && pos >= p0 && pos <= p1;
      return p + place(min(r, ROWS - 1)) * S::DH;
    };
  };
  // dy·o is formed of the tiles here; of heads above 128, whose products leave no registers for o, by a launch before.
  constexpr bool OWN = SLICES <= 4;
  auto load = [&](int32_t i) __attribute__((always_inline)) {
    const int32_t r0 = i * NB;
    qt.load(at(a.q, r0));
    dt.load(at(a.dy, r0));
    if constexpr (DK && OWN) ot.load(at(a.o, r0));
    if (threadIdx.x < NB) {
      const int32_t r = r0 + threadIdx.x;
      row_at = w.first + r / R;
      const bool on = r < ROWS && row_at >= p0 && row_at <= p1;
      if (!on) row_at = -1;
      lse = on ? a.lse[place(r)] * LOG2E : 0.f;
      if constexpr (!OWN) before = on ? a.mass[place(r)] : 0.f;
    }
  };
  auto mass = [&](int k) __attribute__((always_inline)) {
    f4 sum = *reinterpret_cast<const f4*>(row_mass + 16 * k + 4 * q);
#pragma unroll
    for (int s = 1; OWN && s < SLICES; ++s) sum += *reinterpret_cast<const f4*>(row_mass + s * NB + 16 * k + 4 * q);
    return sum;
  };
  if (begin < end) load(begin);
  for (int32_t i = begin; i < end; ++i) {
    __syncthreads();
    qt.template store<true>(qlds, minus);
    dt.template store<true>(dlds, minus);
    // dy·o of 32 floats of a row by its eight threads; NaN where dy holds what is no number, or q does that tcmi_window.h took for one (of the
    // others' lse is NaN).
    if constexpr (OWN) {
#pragma unroll
      for (int c = 0; c < T::CHUNKS; ++c) {
        float sum = 0.f;
        uint32_t most = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sum = fmaf(dt.x[c][e], DK ? ot.x[c][e] : 0.f, sum);
          most = window_most(Span::FEW ? window_most(most, qt.x[c][e]) : most, dt.x[c][e]);
        }
        sum = window_share(sum, most);
#pragma unroll
        for (int off = 1; off < 8; off *= 2) sum += __shfl_xor(sum, off, 64);
        if (threadIdx.x % 8u == 0u) row_mass[T::dim(c) / 32 * NB + T::line(c)] = sum;
      }
    } else if (threadIdx.x < NB) {
      row_mass[threadIdx.x] = before;
    }
    if (threadIdx.x < NB) {
      row_lse[threadIdx.x] = lse;
      row_pos[threadIdx.x] = row_at;
    }
    __syncthreads();
    if (i + 1 < end) load(i + 1);
    const int32_t r0 = i * NB, a0 = w.first + r0 / R, a1 = w.first + min(r0 + NB - 1, ROWS - 1) / R;
    if (m0 > m1 || a1 < m0 || a0 > m1) continue;
    const bool whole = r0 + NB <= ROWS && a0 >= max(p0, mine + 15) && a1 <= p1 && mine + 16 <= w.length && (w.from(a1) <= mine || mine + 16 <= static_cast<int32_t>(S::SINKS));
    f4 s[2];
    window_dots<T>(s, qlds, kf);
    Parts f[1][1];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      // (NaN where the row's numbers are not finite.)
      f4 ls = *reinterpret_cast<const f4*>(row_lse + 16 * k + 4 * q);
      const f4 marks = mass(k);
      const int4 ps = *reinterpret_cast<const int4*>(row_pos + 16 * k + 4 * q);
      const int32_t pos[4] = {ps.x, ps.y, ps.z, ps.w};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ls[r] = marks[r] == marks[r] ? ls[r] : marks[r];
        s[k][r] = whole || (pos[r] >= 0 && w.sees(pos[r], key)) ? __builtin_amdgcn_exp2f(s[k][r] - ls[r]) : 0.f;
      }
    }
    if constexpr (DV) {
      window_parts(s[0], s[1], minus, f[0][0]);
      window_sums<T>(dva, dlds, f);
    }
    if constexpr (DK) {
      f4 dp[2];
      window_dots<T>(dp, dlds, vf);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const f4 ms = mass(k);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[k][r] = whole || s[k][r] != 0.f ? s[k][r] * fmaf(ms[r], OWN ? -0x1p8f : -1.f, dp[k][r]) : 0.f;
      }
      window_parts(s[0], s[1], minus, f[0][0]);
      window_sums<T>(dka, qlds, f);
    }
  }
  window_key_sums<S, DK, DV>(dk, dv, ws, b, hk, chunk, {key}, dka, dva);
}

// dq from its splits' sums: thread `at`, four floats.
template <class S>
__device__ __forceinline__ void window_wide_add(float* __restrict__ dq, const float* __restrict__ parts, size_t at) {
  constexpr size_t N = (size_t)S::B * S::T * S::H * S::DH, E = S::VEC ? 4 : 1;
  if (at * E >= N) return;
  f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t k = 0; k < S::SPLITS; ++k) {
    if constexpr (S::VEC) sum += *reinterpret_cast<const f4*>(parts + k * N + at * E);
    else sum[0] += parts[k * N + at];
  }
  sum *= static_cast<float>(S::scale());
  if constexpr (S::VEC) *reinterpret_cast<f4*>(dq + at * E) = sum;
  else dq[at] = sum[0];
}
// dk (scaled) or dv from their chunks' sums.
template <class S>
__device__ __forceinline__ void window_wide_join(float* __restrict__ out, const float* __restrict__ parts, const float* __restrict__ lengths, float by, size_t at) {
  constexpr size_t ROW = (size_t)S::HK * S::DH, N = (size_t)S::B * S::KEYS * ROW, E = S::VEC ? 4 : 1;
  if (at * E >= N) return;
  const uint32_t b = at * E / (S::KEYS * ROW), key = at * E / ROW % S::KEYS;
  const WindowSpan<S> w(lengths, b);
  // (A chunk without rows was not written, but the first.)
  const uint32_t chunks = max(1u, WindowSeen<S>(w, key / S::ROWS_EACH * S::ROWS_EACH, S::ROWS_EACH).chunks());
  f4 sum = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const float* p) __attribute__((always_inline)) {
    if constexpr (S::VEC) sum += *reinterpret_cast<const f4*>(p);
    else sum[0] += *p;
  };
#pragma unroll 4
  for (uint32_t k = 0; k < min(chunks, S::CHUNKS + 0u); ++k) add(parts + k * N + at * E);
  if (key < S::FEW) {
    const float* more = parts + S::CHUNKS * N + ((size_t)b * S::FEW + key) * ROW + at * E % ROW;
#pragma unroll 4
    for (uint32_t k = S::CHUNKS; k < chunks; ++k) add(more + (size_t)(k - S::CHUNKS) * S::B * S::FEW * ROW);
  }
  sum *= by;
  if constexpr (S::VEC) *reinterpret_cast<f4*>(out + at * E) = sum;
  else out[at] = sum[0];
}

}  // namespace tcmi
