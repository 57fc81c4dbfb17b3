// Attention over a sliding window (tcmi_window.h's formulas) where several workgroups read each key: a launch before splits keys and
// values (and for the gradients queries and dy) once into the parts that the matrix cores take, laid out as their tiles stand in LDS, so
// that the products' kernels copy tiles to LDS without touching them.
//
// Two forms of an operand:
//   dots   for sums over a head (q·k, dy·v): pairs of halves, hi = half(x·2^e), lo = half(x·2^e - hi), e a row's own so that its
//          largest |x|·2^e is in 2^14 ... 2^15: 22 bits of every entry from 2^-17 of the row's largest on, an absolute 2^-39 of it below. The product is
//          hi·hi + hi·lo + lo·hi (2^-22 of it left out) times 2^-e of both rows. Neither of the two steps leaves float32 where the
//          result does not (WindowFactor).
//   sums   for sums over keys or queries: three bf16 parts and the six products of tcmi_window_wide.h, since such a sum has no
//          scale of its own: a key may be any size where another query sees it alone.
// A row that holds a number that is not finite is zeros in both forms, and its 2^-e is NaN (a key's where its value
// has one, and a query's where dy has): what sees it, or it sees, becomes NaN, and nothing else: a score that a query does not see is
// taken for none before anything is summed.
//
// The kernels' layout is tcmi_window_wide.h's. A tile's dots are copied while the sums before them are multiplied, and its sums while the
// dots are: each form has one place in LDS, and a barrier after each of the two halves of a tile.
//
// Bound: the matrix cores. A library's bf16 product of 8192 x 8192 x 8192 reaches 1310 TFLOP/s here, which is 291 of these forward products (three of halves and
// six of bf16 for two), and 218 of the gradients' (30 for five, as scores and dy·v are formed for queries and for keys).
//   two sequences of 16384 tokens, 16 heads of 128 by 4, a window of 1024    1085 us (254 TFLOP/s), 49 to split keys and values
//   8192 tokens, 8 heads of 64 by 2: 267 us (257 TFLOP/s) and 9 to join two splits; its gradients 911 (189) and 27 to split, 21 to join
// (Medians of 60 passes; the first ten or twenty after the card was idle take up to a third longer.) Plain heads of 128 without a window keep 10 registers in
// memory, one operand of four of them read again a tile: 8 sequences of 1024 tokens, 8 heads 141 us (58 at the rate above).
// Of the cycles the matrix cores are busy in 49 %: the rest are the softmax, the split of P and dS into parts and the barriers, which two wavefronts a
// SIMD do not hide whole. Taking the next tile's scores beside this one's softmax needs their registers twice: 313 us of 320 at heads of 64, and spilled at 128.

#pragma once

#include "tcmi_window_wide.h"
#include "tcmi_gemm_f16x2.h"

namespace tcmi {

// Eight floats as a pair of halves each.
struct Pair8 {
  h8 p[2];
};
__device__ __forceinline__ void window_pair(const f4& a, const f4& b, float by, Pair8& out) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = (i < 4 ? a[i & 3] : b[i & 3]) * by;
    const _Float16 h = static_cast<_Float16>(x);
    out.p[0][i] = h;
    out.p[1][i] = static_cast<_Float16>(x - static_cast<float>(h));
  }
}
__device__ __forceinline__ void window_mfma(f4& acc, const Pair8& a, const Pair8& b) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[0], b.p[1], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[1], b.p[0], acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[0], b.p[0], acc, 0, 0, 0);
}
// 2^e for a row whose largest magnitude is `top`, and 2^-e. (e at most 126: both are normal numbers.) Packed is `word`, 2^-23 of the second: a dot
// of 128 products below 2^30 times it stays in float32 whatever e is, and a dot of that size keeps 30 bits where the word is
// below the normal numbers, all of which the multiplication takes.
struct RowScale {
  float up, down;
  __device__ __forceinline__ RowScale(float top) {
    const int e = top > 0.f ? min(126, 14 - static_cast<int>((__float_as_uint(top) >> 23) - 127u)) : 0;
    up = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  }
  __device__ __forceinline__ float word() const { return down * 0x1p-23f; }
};
// What a lane's rows multiply dots by that were multiplied by the other operand's words: 2^23 of their own 2^-e. Of the rows for which that
// leaves float32 (their largest entry is 2^118 or more) 2^14 of it, and `far` has the dots multiplied by the other 2^9 before: 2^9 times
// dots that leave float32 leave it once more by such a row's scale.
template <int HB>
struct WindowFactor {
  float by[HB];
  bool far[HB];
  __device__ __forceinline__ void set(int h, float down) {
    far[h] = !(down <= 0x1p104f);
    by[h] = down * (far[h] ? 0x1p14f : 0x1p23f);
  }
  __device__ __forceinline__ float more(int h) const { return far[h] ? 0x1p9f : 1.f; }
  // Whether a row of the wavefront's is.
  __device__ __forceinline__ bool some() const {
    bool any = false;
#pragma unroll
    for (int h = 0; h < HB; ++h) any = any || far[h];
    return __ballot(any) != 0ull;
  }
  template <int BLOCKS>
  __device__ __forceinline__ void reach(f4 (&s)[HB][BLOCKS]) const {
    if (!some()) return;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) s[h][k] *= more(h);
    }
  }
};
// The largest magnitude; NaN where one of the eight is not finite (a sum of zeros and what is not).
__device__ __forceinline__ float window_top(const f4& a, const f4& b, float top) {
  float bad = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    top = fmaxf(top, fmaxf(fabsf(a[i]), fabsf(b[i])));
    bad = fmaf(a[i], 0.f, fmaf(b[i], 0.f, bad));
  }
  return top + bad;
}
// The larger, NaN where either is.
__device__ __forceinline__ float window_larger(float a, float b) { return a != a ? a : b != b ? b : fmaxf(a, b); }

// Where a form of an operand is: [heads][planes][lines][LD] bytes, a line's chunks as in WindowTile.
template <class S>
struct Packed {
  using T = WindowTile<S, 64>;
  static constexpr int DP = T::DP, LD = T::LD, LANES = LD / 16;     // lanes of a row, eight floats each
  static constexpr size_t KP = (S::KEYS + 63u) / 64u * 64u, RP = (S::T * (S::H / S::HK) + 63u) / 64u * 64u, HEADS = S::B * S::HK;

  template <int PLANES>
  static __device__ __forceinline__ char* at(char* form, size_t lines, uint32_t head, size_t line) { return form + ((size_t)head * PLANES * lines + line) * LD; }

  static __device__ __forceinline__ int place(int line, int c) { return (c ^ T::swap(line)) << 4; }
  static __device__ __forceinline__ void dots(char* form, size_t lines, uint32_t head, uint32_t line, int c, const f4& x, const f4& y, float up) {
    Pair8 f;
    window_pair(x, y, up, f);
    char* to = at<2>(form, lines, head, line) + place(line & 15, c);
#pragma unroll
    for (int p = 0; p < 2; ++p) *reinterpret_cast<h8*>(to + p * lines * LD) = f.p[p];
  }
  static __device__ __forceinline__ void sums(char* form, size_t lines, uint32_t head, uint32_t line, int c, const f4& x, const f4& y, const Minus& minus) {
    Parts f;
    window_parts(x, y, minus, f);
    char* to = at<3>(form, lines, head, line) + place(line & 15, c);
#pragma unroll
    for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(to + p * lines * LD) = f.p[p];
  }
  static __device__ __forceinline__ float row_top(float top) {
#pragma unroll
    for (int off = LANES / 2; off >= 1; off >>= 1) top = window_larger(top, __shfl_xor(top, off, 64));
    return top;
  }
};

// Line `id` of the heads' keys: K's dots and V's sums, or of the gradients (BACK) K's and V's dots and (DQ) K's sums; their scales.
template <class S, bool BACK, bool DQ>
__device__ __forceinline__ void window_pack_keys(const float* __restrict__ kp, const float* __restrict__ vp, const float* __restrict__ lengths, char* ws, uint32_t id) {
  using P = Packed<S>;
  const uint32_t head = id / P::KP, j = id % P::KP;
  const int c = threadIdx.x % P::LANES;
  if (head >= P::HEADS) return;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const WindowSpan<S> w(lengths, b);
  const WindowTiles keys = window_keys(w, 0u, WindowSpan<S>::ROWS - 1u);
  const int32_t key = static_cast<int32_t>(j);
  const auto seen = [&](int32_t i) { return i <= keys.hi && (i >= keys.lo || i < static_cast<int32_t>(S::SINKS)); };
  // (A tile of 64 that no query sees a key of is never read.)
  const int32_t first = key & ~63;
  if (first > keys.hi || (first + 63 < keys.lo && first >= static_cast<int32_t>(S::SINKS))) return;
  const bool on = seen(key);
  const size_t row = (((size_t)b * S::KEYS + (on ? j : 0u)) * S::HK + hk) * S::DH;
  const auto load = [&](const float* p, int d) { return window_number(window_load<S>(p + row, 8 * c + d, on)); };
  f4 k0 = load(kp, 0), k1 = load(kp, 4), v0 = load(vp, 0), v1 = load(vp, 4);
  const float kt = P::row_top(window_top(k0, k1, 0.f)), vt = P::row_top(window_top(v0, v1, 0.f));
  const bool bad = kt != kt || vt != vt;
  if (bad) k0 = k1 = v0 = v1 = f4{0.f, 0.f, 0.f, 0.f};
  const RowScale ks(bad ? 0.f : kt), vs(bad ? 0.f : vt);
  if (c == 0) {
    reinterpret_cast<float*>(ws + S::KSCALE)[id] = bad ? __builtin_nanf("") : ks.word();
    if constexpr (BACK) reinterpret_cast<float*>(ws + S::VSCALE)[id] = bad ? __builtin_nanf("") : vs.word();
  }
  if (c >= P::DP / 8) return;
  const Minus minus;
  P::dots(ws + S::KDOTS, P::KP, head, j, c, k0, k1, ks.up);
  if constexpr (BACK) {
    if constexpr (DQ) P::sums(ws + S::KSUMS, P::KP, head, j, c, k0, k1, minus);
    P::dots(ws + S::VDOTS, P::KP, head, j, c, v0, v1, vs.up);
  } else {
    P::sums(ws + S::VSUMS, P::KP, head, j, c, v0, v1, minus);
  }
}

// Line `id` of the heads' rows: q's (times scale·log2 e) and dy's dots and q's and dy's sums, their scales, lse in powers of two and dy·o.
template <class S, bool DOTS>
__device__ __forceinline__ void window_pack_rows(const WindowGradArgs a, char* ws, uint32_t id) {
  using P = Packed<S>;
  using Span = WindowSpan<S>;
  constexpr uint32_t R = Span::R;
  const uint32_t head = id / P::RP, r = id % P::RP;
  const int c = threadIdx.x % P::LANES;
  if (head >= P::HEADS) return;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const Span w(a.lengths, b);
  const bool on = r < Span::ROWS && w.stands(w.first + static_cast<int32_t>(r / R));
  const uint32_t at = on ? r : 0u;
  const size_t line = ((size_t)b * S::T + at / R) * S::H + hk * R + at % R;
  const auto load = [&](const float* p, int d) { return window_number(window_load<S>(p + line * S::DH, 8 * c + d, on)); };
  f4 q0 = load(a.q, 0), q1 = load(a.q, 4), d0 = load(a.dy, 0), d1 = load(a.dy, 4);
  const f4 o0 = window_load<S>(a.o + line * S::DH, 8 * c, on), o1 = window_load<S>(a.o + line * S::DH, 8 * c + 4, on);
  float mass = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) mass = fmaf(d0[i], o0[i], fmaf(d1[i], o1[i], mass));
#pragma unroll
  for (int off = P::LANES / 2; off >= 1; off >>= 1) mass += __shfl_xor(mass, off, 64);
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
  const f4 s0 = q0 * scale, s1 = q1 * scale;
  const float qt = P::row_top(window_top(s0, s1, 0.f)), dt = P::row_top(window_top(d0, d1, 0.f));
  const bool bad = qt != qt || dt != dt;
  const f4 zero = {0.f, 0.f, 0.f, 0.f};
  if (bad) q0 = q1 = d0 = d1 = zero;
  const RowScale qs(bad ? 0.f : qt), ds(bad ? 0.f : dt);
  if (c == 0) {
    reinterpret_cast<float4*>(ws + S::ROWSTATS)[id] = make_float4(bad ? __builtin_nanf("") : qs.word(), ds.word(), on ? a.lse[line] * LOG2E : 0.f, mass);
  }
  if (!DOTS || c >= P::DP / 8) return;
  const Minus minus;
  P::dots(ws + S::QDOTS, P::RP, head, r, c, bad ? zero : s0, bad ? zero : s1, qs.up);
  P::dots(ws + S::DDOTS, P::RP, head, r, c, d0, d1, ds.up);
  P::sums(ws + S::QSUMS, P::RP, head, r, c, q0, q1, minus);
  P::sums(ws + S::DSUMS, P::RP, head, r, c, d0, d1, minus);
}

// The first KEYBLOCKS workgroups: keys, the rest: rows.
template <class S, bool DQ, bool DKV, uint32_t KEYBLOCKS>
__device__ __forceinline__ void window_pack_both(const WindowGradArgs a, char* ws, uint32_t block, uint32_t key, uint32_t row) {
  if (block < KEYBLOCKS) window_pack_keys<S, true, DQ>(a.k, a.v, a.lengths, ws, key);
  else window_pack_rows<S, DKV>(a, ws, row);
}

// Copies of 16 bytes (4: one word) a lane from `from` on to LDS from `to` on (both uniform), in flight until vmcnt reaches 0. Written as
// instructions: of the compiler's own it takes every later read of LDS to depend on them, and waits for them there (of a gradient of keys
// twice a tile: 950 us, 908 so). They have no register results, and a wait that the compiler counts without them is only
// longer for them; barrier_ahead() is what the tiles' readers wait at.
__device__ __forceinline__ void window_copy16(uint32_t to, const char* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"((threadIdx.x & 63u) * 16u), "s"(from) : "memory", "m0");
}
__device__ __forceinline__ void window_copy4(uint32_t to, const char* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"((threadIdx.x & 63u) * 4u), "s"(from) : "memory", "m0");
}
__device__ __forceinline__ uint32_t window_lds(char* p) { return static_cast<uint32_t>(reinterpret_cast<size_t>((__attribute__((address_space(3))) char*)p)); }

// The copy of PLANES planes of NB lines of a form to LDS, by THREADS threads.
template <int NB, int LD, int PLANES, int THREADS>
__device__ __forceinline__ void window_fetch(char* to, const char* from, size_t plane) {
  constexpr int BYTES = NB * LD, ALL = PLANES * BYTES;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  static_assert(BYTES % 1024 == 0, "a wavefront's 1 KiB is of one plane");
#pragma unroll
  for (int u = 0; u < (ALL + THREADS * 16 - 1) / (THREADS * 16); ++u) {
    const int byte = (u * (THREADS / 64) + wave) * 1024;
    if (ALL % (THREADS * 16) != 0 && byte >= ALL) break;
    window_copy16(window_lds(to) + byte, from + byte / BYTES * plane + byte % BYTES);
  }
}
// And of 64 words by wavefront `by`.
__device__ __forceinline__ void window_fetch_words(char* to, const void* from, int by) {
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) == by) window_copy4(window_lds(to), static_cast<const char*>(from));
}

// This lane's part of a first operand of dots: lines line0 + t, floats 32·slice + 8q ....
template <class T>
__device__ __forceinline__ void window_pair_lines(const char* tile, int line0, int slice, Pair8& f) {
  const int t = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3, at = t * T::LD + ((q ^ T::swap(t)) << 4);
#pragma unroll
  for (int p = 0; p < 2; ++p) f.p[p] = *reinterpret_cast<const h8*>(tile + p * T::PLANE + line0 * T::LD + (at ^ (slice << 6)));
}
template <class T, int HB, int BLOCKS, int SLICES>
__device__ __forceinline__ void window_pair_dots(f4 (&acc)[HB][BLOCKS], const char* tile, const Pair8 (&f)[HB][SLICES]) {
  // (The wavefront that multiplies goes before the one beside it: forward 349 -> 320 us of 8192 tokens.)
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
    for (int h = 0; h < HB; ++h) acc[h][k] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < SLICES; ++d) {
      Pair8 x;
      window_pair_lines<T>(tile, 16 * k, d, x);
#pragma unroll
      for (int h = 0; h < HB; ++h) window_mfma(acc[h][k], x, f[h][d]);
    }
  }
  __builtin_amdgcn_s_setprio(0);
}
// A row's dots as a second operand, from memory: `up` times it. Its scale comes back in `down`.
template <class S, int SLICES>
__device__ __forceinline__ void window_pair_row(Pair8 (&f)[SLICES], const float* __restrict__ p, bool on, float by, float& down) {
  const int q = (threadIdx.x >> 4) & 3;
  f4 x[SLICES], y[SLICES];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < SLICES; ++s) {
    x[s] = window_number(window_load<S, true>(p, 32 * s + 8 * q, on)) * by;
    y[s] = window_number(window_load<S, true>(p, 32 * s + 8 * q + 4, on)) * by;
    top = window_larger(top, window_top(x[s], y[s], 0.f));
  }
  top = window_larger(top, __shfl_xor(top, 16, 64));
  top = window_larger(top, __shfl_xor(top, 32, 64));
  const bool bad = top != top;
  const RowScale r(bad ? 0.f : top);
  down = bad ? __builtin_nanf("") : r.down;
#pragma unroll
  for (int s = 0; s < SLICES; ++s) window_pair(bad ? f4{0.f, 0.f, 0.f, 0.f} : x[s], bad ? f4{0.f, 0.f, 0.f, 0.f} : y[s], r.up, f[s]);
}
// The same, already packed.
template <class S, int SLICES>
__device__ __forceinline__ void window_packed_row(Pair8 (&f)[SLICES], const char* form, size_t lines, uint32_t head, uint32_t line) {
  using P = Packed<S>;
  const int q = (threadIdx.x >> 4) & 3;
  const char* from = P::template at<2>(const_cast<char*>(form), lines, head, line);
#pragma unroll
  for (int s = 0; s < SLICES; ++s) {
#pragma unroll
    for (int p = 0; p < 2; ++p) f[s].p[p] = *reinterpret_cast<const h8*>(from + p * lines * P::LD + P::place(line & 15, 4 * s + q));
  }
}

// What the kernels of packed operands share. S::WAVES wavefronts of 16·HB lines each.
template <class S>
struct WindowPacked {
  static constexpr int DP = (S::DH + 31) / 32 * 32, SLICES = DP / 32, G = DP / 16, HB = S::HB;
  static constexpr int NB = DP <= 64 ? 64 : 32, BLOCKS = NB / 16;
  using T = WindowTile<S, NB>;
  static constexpr uint32_t THREADS = 64 * S::WAVES, ROWS = 16 * HB * S::WAVES;
  static constexpr int DOTS = 2 * T::PLANE, SUMS = 3 * T::PLANE, WORDS = 256;
  static constexpr int FORWARD = DOTS + SUMS + WORDS, DQ = 2 * DOTS + SUMS + 2 * WORDS;
};
// And those over tiles of 32 rows.
template <class S>
struct WindowPackedRows {
  static constexpr int NB = 32, BLOCKS = 2;
  using T = WindowTile<S, NB>;
  static constexpr int DOTS = 2 * T::PLANE, SUMS = 3 * T::PLANE, LDS = 2 * DOTS + 2 * SUMS + 32 * 16;
};

// The rows of a lane: lines, positions and whether they stand; and of its wavefront.
template <class S, int HB>
struct WindowLines {
  size_t line[HB];
  int32_t pos[HB], p0, p1;
  bool on[HB], full;
  __device__ __forceinline__ WindowLines(const WindowSpan<S>& w, uint32_t b, uint32_t hk, uint32_t mine) {
    constexpr uint32_t R = WindowSpan<S>::R, ROWS = WindowSpan<S>::ROWS;
    const uint32_t t = threadIdx.x & 15u;
#pragma unroll
    for (int h = 0; h < HB; ++h) {
      const uint32_t row = mine + 16u * h + t, at = min(row, ROWS - 1u);
      line[h] = ((size_t)b * S::T + at / R) * S::H + hk * R + at % R;
      pos[h] = w.first + static_cast<int32_t>(at / R);
      on[h] = row < ROWS && w.stands(pos[h]);
    }
    p0 = w.first + static_cast<int32_t>(min(mine, ROWS - 1u) / R);
    p1 = w.first + static_cast<int32_t>(min(mine + 16u * HB - 1u, ROWS - 1u) / R);
    full = mine + 16u * HB <= ROWS && w.stands(p0) && w.stands(p1);
  }
  // Whether one of the rows sees a key of NB from j0 on, and whether all see all of them.
  __device__ __forceinline__ bool some(const WindowSpan<S>& w, int32_t j0, int NB) const { return j0 <= p1 && (j0 + NB > w.from(p0) || j0 < static_cast<int32_t>(S::SINKS)); }
  __device__ __forceinline__ bool whole(const WindowSpan<S>& w, int32_t j0, int NB) const {
    return full && j0 + NB - 1 <= p0 && (j0 >= w.from(p1) || j0 + NB <= static_cast<int32_t>(S::SINKS));
  }
};

// Workgroup: W::ROWS rows of a sequence's key head, a split of the keys they see.
template <class S>
__device__ __forceinline__ void window_packed(const float* __restrict__ qp, const float* __restrict__ lengths, float* __restrict__ out, float* __restrict__ lse,
                                              char* ws, char* lds, uint32_t head, uint32_t tile, uint32_t split) {
  using W = WindowPacked<S>;
  using T = typename W::T;
  using P = Packed<S>;
  using Span = WindowSpan<S>;
  constexpr uint32_t ROWS = Span::ROWS;
  constexpr int NB = W::NB, HB = W::HB, BLOCKS = W::BLOCKS, SLICES = W::SLICES, G = W::G;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span w(lengths, b);
  const Minus minus;
  const uint32_t row0 = tile * W::ROWS, mine = row0 + 16u * HB * wave;
  const WindowTiles tiles = window_wider<NB>(window_keys(w, min(row0, ROWS - 1u), min(row0 + W::ROWS - 1u, ROWS - 1u)));
  int32_t begin, end;
  window_run<S>(tiles.all, split, begin, end);
  char *kd = lds, *vs = lds + W::DOTS, *words = vs + W::SUMS;
  auto keys = [&](int32_t i) __attribute__((always_inline)) {
    const size_t j0 = (size_t)tiles.at(i) * NB;
    window_fetch<NB, T::LD, 2, W::THREADS>(kd, P::template at<2>(ws + S::KDOTS, P::KP, head, j0), P::KP * T::LD);
    window_fetch_words(words, reinterpret_cast<const float*>(ws + S::KSCALE) + head * P::KP + (NB == 64 ? j0 : j0 & ~(size_t)63), 0);
  };
  if (begin < end) keys(begin);
  const WindowLines<S, HB> rows(w, b, hk, mine);
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
  Pair8 qf[HB][SLICES];
  f4 o[HB][G];
  float m[HB], l[HB];
  WindowFactor<HB> qs;
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    float down;
    window_pair_row<S>(qf[h], qp + rows.line[h] * S::DH, rows.on[h], scale, down);
    qs.set(h, down);
    m[h] = -TCMI_INF;
    l[h] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) o[h][g] = f4{0.f, 0.f, 0.f, 0.f};
  }
  barrier_ahead<0>();
  for (int32_t i = begin; i < end; ++i) {
    const int32_t j0 = tiles.at(i) * NB;
    window_fetch<NB, T::LD, 3, W::THREADS>(vs, P::template at<3>(ws + S::VSUMS, P::KP, head, (size_t)j0), P::KP * T::LD);
    const bool some = rows.some(w, j0, NB);
    f4 s[HB][BLOCKS];
    if (some) {
      window_pair_dots<T>(s, kd, qf);
      const float* by = reinterpret_cast<const float*>(words) + (NB == 64 ? 0 : j0 & 63);
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
        const f4 ks = *reinterpret_cast<const f4*>(by + 16 * k + 4 * q);
#pragma unroll
        for (int h = 0; h < HB; ++h) s[h][k] *= ks;
      }
    }
    barrier_ahead<0>();
    if (i + 1 < end) keys(i + 1);
    if (some) {
      if (!rows.whole(w, j0, NB) || qs.some()) {
        // (The rows' positions are found again here: kept, they spill more registers.)
        int own = lane;
        asm volatile("" : "+v"(own));
#pragma unroll
        for (int h = 0; h < HB; ++h) {
          const uint32_t row = mine + 16u * h + (own & 15);
          const int32_t pos = w.first + static_cast<int32_t>(min(row, ROWS - 1u) / Span::R);
          const bool on = row < ROWS && w.stands(pos);
#pragma unroll
          for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[h][k][r] = on && w.sees(pos, j0 + 16 * k + 4 * (own >> 4) + r) ? s[h][k][r] * qs.more(h) : -TCMI_INF;
          }
        }
      }
      float alpha[HB];
      Parts pf[HB][BLOCKS / 2];
#pragma unroll
      for (int h = 0; h < HB; ++h) {
        float top = -TCMI_INF;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, s[h][k][r]);
        }
        // (A row's scale is positive, or NaN: its scores' order is theirs before it.)
        top = fmaxf(m[h], quad16_reduce<true>(top) * qs.by[h]);
        const float zero = top == -TCMI_INF ? 0.f : top;
        alpha[h] = __builtin_amdgcn_exp2f(m[h] - zero);
        m[h] = top;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[h][k][r] = __builtin_amdgcn_exp2f(fmaf(s[h][k][r], qs.by[h], -zero));
            sum += s[h][k][r];
          }
        }
        l[h] = fmaf(l[h], alpha[h], sum);
#pragma unroll
        for (int k = 0; k < BLOCKS; k += 2) window_parts(s[h][k], s[h][k + 1], minus, pf[h][k / 2]);
      }
      // (The places of heads above 64 are found again for each tile: kept, they spill more registers, whose reloads wait for the copies.)
      int own = lane;
      if constexpr (G > 4) asm volatile("" : "+v"(own));
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int g = 0; g < G; g += 2) {
        f4 sum[HB][2];
#pragma unroll
        for (int h = 0; h < HB; ++h) sum[h][0] = sum[h][1] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < BLOCKS / 2; ++k) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            Parts f;
            T::across(vs, 32 * k, 16 * (g + e), f, own);
#pragma unroll
            for (int h = 0; h < HB; ++h) window_mfma(sum[h][e], f, pf[h][k]);
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int h = 0; h < HB; ++h) {
#pragma unroll
            for (int r = 0; r < 4; ++r) o[h][g + e][r] = fmaf(o[h][g + e][r], alpha[h], sum[h][e][r]);
          }
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    barrier_ahead<0>();
  }
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    const float total = quad16_reduce<false>(l[h]);
    const bool some = total > 0.f || total != total;
    uint32_t row = mine + 16u * h + t;
    if (row >= ROWS) continue;
    // (Its line is found again too.)
    asm("" : "+v"(row));
    const size_t line = ((size_t)b * S::T + row / Span::R) * S::H + hk * Span::R + row % Span::R;
    if constexpr (S::SPLITS > 1u) {
      const size_t place = ((size_t)split * S::B * S::HK + head) * S::TILES * 16u + row;
#pragma unroll
      for (int g = 0; g < G; ++g) window_store<S>(reinterpret_cast<float*>(ws + S::OUT) + place * S::DH, 16 * g + 4 * q, o[h][g]);
      if (q == 0) reinterpret_cast<float2*>(ws + S::STATS)[place] = make_float2(m[h], total);
      continue;
    }
    const float inv = some ? 1.f / total : 0.f;
    if (out != nullptr) {
#pragma unroll
      for (int g = 0; g < G; ++g) window_store<S>(out + line * S::DH, 16 * g + 4 * q, o[h][g] * inv);
    }
    if (lse != nullptr && q == 0) lse[line] = some ? (m[h] + __builtin_amdgcn_logf(total)) * 0.69314718055994531f : -TCMI_INF;
  }
}

// Workgroup: W::ROWS rows of a sequence's key head, a split of the keys they see. parts: as window_wide_dq's.
template <class S>
__device__ __forceinline__ void window_packed_dq(const WindowGradArgs a, float* __restrict__ dq, float* __restrict__ parts, char* ws, char* lds, uint32_t head, uint32_t tile, uint32_t split) {
  using W = WindowPacked<S>;
  using T = typename W::T;
  using P = Packed<S>;
  using Span = WindowSpan<S>;
  constexpr uint32_t ROWS = Span::ROWS;
  constexpr int NB = W::NB, HB = W::HB, BLOCKS = W::BLOCKS, SLICES = W::SLICES, G = W::G;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span w(a.lengths, b);
  const Minus minus;
  const uint32_t row0 = tile * W::ROWS, mine = row0 + 16u * HB * wave;
  const WindowTiles tiles = window_wider<NB>(window_keys(w, min(row0, ROWS - 1u), min(row0 + W::ROWS - 1u, ROWS - 1u)));
  int32_t begin, end;
  window_run<S>(tiles.all, split, begin, end);
  char *kd = lds, *vd = lds + W::DOTS, *ksums = vd + W::DOTS, *words = ksums + W::SUMS;
  auto dots = [&](int32_t i) __attribute__((always_inline)) {
    const size_t j0 = (size_t)tiles.at(i) * NB, word = head * P::KP + (NB == 64 ? j0 : j0 & ~(size_t)63);
    window_fetch<NB, T::LD, 2, W::THREADS>(kd, P::template at<2>(ws + S::KDOTS, P::KP, head, j0), P::KP * T::LD);
    window_fetch<NB, T::LD, 2, W::THREADS>(vd, P::template at<2>(ws + S::VDOTS, P::KP, head, j0), P::KP * T::LD);
    window_fetch_words(words, reinterpret_cast<const float*>(ws + S::KSCALE) + word, 0);
    window_fetch_words(words + W::WORDS, reinterpret_cast<const float*>(ws + S::VSCALE) + word, 1);
  };
  if (begin < end) dots(begin);
  const WindowLines<S, HB> rows(w, b, hk, mine);
  Pair8 qf[HB][SLICES], df[HB][SLICES];
  f4 acc[HB][G];
  WindowFactor<HB> qby, dby;
  float lse[HB], mass[HB];
  const float scale = static_cast<float>(S::scale() * 1.4426950408889634);
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    const uint32_t at = min(mine + 16u * h + t, ROWS - 1u);
    const float4 stats = reinterpret_cast<const float4*>(ws + S::ROWSTATS)[head * P::RP + at];
    qby.set(h, stats.x * 0x1p23f);
    dby.set(h, stats.y * 0x1p23f);
    lse[h] = stats.z;
    mass[h] = stats.w;
    float down;
    window_pair_row<S>(qf[h], a.q + rows.line[h] * S::DH, rows.on[h], scale, down);
    window_pair_row<S>(df[h], a.dy + rows.line[h] * S::DH, rows.on[h], 1.f, down);
#pragma unroll
    for (int g = 0; g < G; ++g) acc[h][g] = f4{0.f, 0.f, 0.f, 0.f};
  }
  barrier_ahead<0>();
  for (int32_t i = begin; i < end; ++i) {
    const int32_t j0 = tiles.at(i) * NB;
    window_fetch<NB, T::LD, 3, W::THREADS>(ksums, P::template at<3>(ws + S::KSUMS, P::KP, head, (size_t)j0), P::KP * T::LD);
    const bool some = rows.some(w, j0, NB);
    Parts ds[HB][BLOCKS / 2];
    if (some) {
      const bool whole = rows.whole(w, j0, NB);
      f4 s[HB][BLOCKS], dp[HB][BLOCKS];
      window_pair_dots<T>(s, kd, qf);
      window_pair_dots<T>(dp, vd, df);
      qby.reach(s);
      dby.reach(dp);
      const float* by = reinterpret_cast<const float*>(words) + (NB == 64 ? 0 : j0 & 63);
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
        const f4 ks = *reinterpret_cast<const f4*>(by + 16 * k + 4 * q), vs = *reinterpret_cast<const f4*>(by + W::WORDS / 4 + 16 * k + 4 * q);
#pragma unroll
        for (int h = 0; h < HB; ++h) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[h][k][r] * ks[r], qby.by[h], -lse[h]));
            const float d = p * fmaf(dp[h][k][r] * vs[r], dby.by[h], -mass[h]);
            s[h][k][r] = whole || (rows.on[h] && w.sees(rows.pos[h], j0 + 16 * k + 4 * q + r)) ? d : 0.f;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < HB; ++h) {
#pragma unroll
        for (int k = 0; k < BLOCKS; k += 2) window_parts(s[h][k], s[h][k + 1], minus, ds[h][k / 2]);
      }
    }
    barrier_ahead<0>();
    if (i + 1 < end) dots(i + 1);
    if (some) window_sums<T>(acc, ksums, ds);
    barrier_ahead<0>();
  }
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    if (mine + 16u * h + t >= ROWS) continue;
    float* to = S::SPLITS > 1u ? parts + ((size_t)split * S::B * S::T * S::H + rows.line[h]) * S::DH : dq + rows.line[h] * S::DH;
    const float by = S::SPLITS > 1u ? 1.f : static_cast<float>(S::scale());
#pragma unroll
    for (int g = 0; g < G; ++g) window_store<S>(to, 16 * g + 4 * q, acc[h][g] * by);
  }
}

// Workgroup: W::ROWS keys of a sequence's key head, a chunk of the rows that see one of them. parts: as window_wide_dkv's.
template <class S, bool DK, bool DV>
__device__ __forceinline__ void window_packed_dkv(const WindowGradArgs a, float* __restrict__ dk, float* __restrict__ dv, char* ws, char* lds, uint32_t head, uint32_t tile, uint32_t chunk) {
  using W = WindowPacked<S>;
  using X = WindowPackedRows<S>;
  using T = typename X::T;
  using P = Packed<S>;
  using Span = WindowSpan<S>;
  constexpr int32_t R = Span::R, ROWS = Span::ROWS;
  constexpr int NB = X::NB, HB = W::HB, BLOCKS = X::BLOCKS, SLICES = W::SLICES, G = W::G;
  const uint32_t b = head / S::HK, hk = head % S::HK;
  const int lane = threadIdx.x & 63, t = lane & 15, q = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Span w(a.lengths, b);
  const Minus minus;
  const int32_t mine = tile * W::ROWS + 16 * HB * wave;
  const WindowSeen<S> all(w, tile * W::ROWS, W::ROWS), own(w, mine, 16 * HB);
  if (chunk < all.start()) return;
  chunk -= all.start();
  if (chunk > 0u && chunk >= all.chunks()) return;
  const int32_t begin = all.from(chunk), end = all.to(chunk);
  char *qd = lds, *dd = qd + X::DOTS, *qs = dd + X::DOTS, *ds = qs + X::SUMS, *stats = ds + X::SUMS;
  auto dots = [&](int32_t i) __attribute__((always_inline)) {
    const size_t r0 = (size_t)i * NB;
    window_fetch<NB, T::LD, 2, W::THREADS>(qd, P::template at<2>(ws + S::QDOTS, P::RP, head, r0), P::RP * T::LD);
    if constexpr (DK) window_fetch<NB, T::LD, 2, W::THREADS>(dd, P::template at<2>(ws + S::DDOTS, P::RP, head, r0), P::RP * T::LD);
    // Their statistics, 128 words.
    const char* from = ws + S::ROWSTATS + (head * P::RP + r0) * 16u;
    window_fetch_words(stats, from, 0);
    window_fetch_words(stats + 256, from + 256, 1);
  };
  auto sums = [&](int32_t i) __attribute__((always_inline)) {
    const size_t r0 = (size_t)i * NB;
    if constexpr (DK) window_fetch<NB, T::LD, 3, W::THREADS>(qs, P::template at<3>(ws + S::QSUMS, P::RP, head, r0), P::RP * T::LD);
    if constexpr (DV) window_fetch<NB, T::LD, 3, W::THREADS>(ds, P::template at<3>(ws + S::DSUMS, P::RP, head, r0), P::RP * T::LD);
  };
  if (begin < end) dots(begin);
  int32_t key[HB];
  WindowFactor<HB> kby, vby;
  Pair8 kf[HB][SLICES], vf[HB][SLICES];
  f4 dka[HB][G], dva[HB][G];
#pragma unroll
  for (int h = 0; h < HB; ++h) {
    key[h] = mine + 16 * h + t;
    // (Of keys past the sequence, which have no rows to see them, whatever the workspace holds.)
    const uint32_t at = min(key[h], static_cast<int32_t>(P::KP) - 1);
    window_packed_row<S>(kf[h], ws + S::KDOTS, P::KP, head, at);
    if constexpr (DK) window_packed_row<S>(vf[h], ws + S::VDOTS, P::KP, head, at);
    kby.set(h, reinterpret_cast<const float*>(ws + S::KSCALE)[head * P::KP + at] * 0x1p23f);
    vby.set(h, reinterpret_cast<const float*>(ws + S::VSCALE)[head * P::KP + at] * 0x1p23f);
#pragma unroll
    for (int g = 0; g < G; ++g) dka[h][g] = dva[h][g] = f4{0.f, 0.f, 0.f, 0.f};
  }
  barrier_ahead<0>();
  for (int32_t i = begin; i < end; ++i) {
    sums(i);
    const int32_t r0 = i * NB, a0 = w.first + r0 / R, a1 = w.first + min(r0 + NB - 1, ROWS - 1) / R;
    const bool some = own.p0 <= own.p1 && a1 >= own.p0 && a0 <= own.p1;
    Parts pf[HB][1], df[HB][1];
    if (some) {
      const bool whole = r0 + NB <= ROWS && a0 >= max(own.p0, mine + 16 * HB - 1) && a1 <= own.p1 && mine + 16 * HB <= w.length && (w.from(a1) <= mine || mine + 16 * HB <= static_cast<int32_t>(S::SINKS));
      f4 s[HB][BLOCKS], dp[HB][BLOCKS];
      window_pair_dots<T>(s, qd, kf);
      kby.reach(s);
      if constexpr (DK) {
        window_pair_dots<T>(dp, dd, vf);
        vby.reach(dp);
      }
#pragma unroll
      for (int k = 0; k < BLOCKS; ++k) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * k + 4 * q + r;
          const f4 st = *reinterpret_cast<const f4*>(stats + row * 16);
          const int32_t at = r0 + row, pos = at < ROWS ? w.first + at / R : -1;
#pragma unroll
          for (int h = 0; h < HB; ++h) {
            const bool sees = whole || (w.stands(pos) && key[h] < w.length && w.sees(pos, key[h]));
            s[h][k][r] = sees ? __builtin_amdgcn_exp2f(fmaf(s[h][k][r] * st[0], kby.by[h], -st[2])) : 0.f;
            if constexpr (DK) dp[h][k][r] = sees ? s[h][k][r] * fmaf(dp[h][k][r] * st[1], vby.by[h], -st[3]) : 0.f;
          }
        }
      }
#pragma unroll
      for (int h = 0; h < HB; ++h) {
        if constexpr (DV) window_parts(s[h][0], s[h][1], minus, pf[h][0]);
        if constexpr (DK) window_parts(dp[h][0], dp[h][1], minus, df[h][0]);
      }
    }
    barrier_ahead<0>();
    if (i + 1 < end) dots(i + 1);
    if (some) {
      if constexpr (DV) window_sums<T>(dva, ds, pf);
      if constexpr (DK) window_sums<T>(dka, qs, df);
    }
    barrier_ahead<0>();
  }
  window_key_sums<S, DK, DV>(dk, dv, ws, b, hk, chunk, key, dka, dva);
}

}  // namespace tcmi
