// Products of float32 matrices on CDNA4's fp16 matrix cores, each operand a pair of halves.
//
// x (scaled by a power of two into half's range) is split once, by the kernel that
// produces it, into hi = half(x) and lo = half((x - hi)·2^11): 11 + 11 significant bits,
// the remainder brought back to hi's range, so a pair holds 22 bits or more of every |x| from
// 2^-14 up to 2^16, and an absolute 2^-36 below. The product keeps three of the four terms,
//   a·b = hi_a·hi_b + 2^-11·(hi_a·lo_b + lo_a·hi_b) + (lo_a·lo_b·2^-22 left out),
// each exact in float32, in two float32 accumulators joined at the end. A product is off by
// at most 2^-22 + 2·2^-23 of |a·b| (the term left out, and the two remainders' roundings), one
// in the root mean square by 2^-23.5: less than a float32 sum's own roundings from 16 terms on.
// Half the matrix-core work of six products of bf16 parts (tcmi_gemm_bf16x3.h).
//
// Operands are read from memory as matrices of pairs: row r takes `ld` = 4·columns bytes, in blocks of 32
// columns of 128 bytes, 32 hi halves and then their 32 lo halves, so a row's slice of 32 is one cache
// line. An operand's lines (A: rows of C, B: columns of C) are the matrix's rows (KC: k runs along the
// row) or its columns (k runs down): neither has to be transposed. The matrices are padded with zeros to
// whole tiles (lines to the tile's, k to 32), so the loop has no bounds. Loads go straight to LDS (16
// bytes a lane); a slice of 32 k of L lines there:
//   KC       128 bytes a line, its eight 16-byte chunks c at slot c ^ (line % 8): the 16 lanes of a
//            256-byte LDS cycle (16 lines, one chunk) meet all banks. A lane's fragment, 8 k of one line, is
//            one ds_read_b128.
//   not KC   4·L bytes a k row; its 32-byte groups g (16 lines of one half of the pairs) at g ^ (k % 4), its
//            128-byte blocks at block ^ (k / 8 % 2). Fragments are read by ds_read_b64_tr_b16, which transposes: of
//            16 lanes each gives the address of 4 lines of one of 4 rows, and gets its own line's 4 k; two reads
//            make a fragment, and the 32 lanes of a cycle (4 rows k and 4 rows k + 8) meet all banks.
//
// Bound: power. 4096^3 by 128 x 128 tiles takes 314 us with pauses between launches and 370 us without
// (438 and 371 TFLOP/s), the matrix cores busy for 67 % of the cycles at 1.86 GHz; and the same launches on zeros, which toggle no
// operand, are a fifth faster (4096 rows of d 512 against 32 768 classes 431 and 340 us, two orthogonalized 4096^2 7420 and 5840, on one card); reading the next
// slice's fragments beside a column of products (one barrier a slice, as tcmi_gemm_bf16x3.h) is as fast, products of
// 32 x 32 are slower (412 us). With planes of hi and of lo apart, a line's slice half a cache line: KC 417 us.

#pragma once

#include "tcmi_device.h"

namespace tcmi {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float PAIR_LO = 0x1p11f;   // what a remainder is multiplied by

// x as a pair. A value that is not finite is its own hi.
__device__ __forceinline__ void split_pair(float x, _Float16& hi, _Float16& lo) {
  hi = static_cast<_Float16>(x);
  const float r = x - static_cast<float>(hi);
  lo = __builtin_isfinite(r) ? static_cast<_Float16>(r * PAIR_LO) : static_cast<_Float16>(0.f);
}
__device__ __forceinline__ void split_pair(const f4& x, h4& hi, h4& lo) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    _Float16 a, b;
    split_pair(x[i], a, b);
    hi[i] = a;
    lo[i] = b;
  }
}
__device__ __forceinline__ f4 join_pair(const h4& hi, const h4& lo) {
  f4 x;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(hi[i]) + static_cast<float>(lo[i]) * (1.f / PAIR_LO);
  return x;
}

// A matrix of pairs: its first byte, and bytes a row.
struct Pairs {
  const char* at;
  uint32_t ld;
};

// Where four floats of a row from column c on (a multiple of 4) keep their hi halves; the lo ones 64 bytes on.
__device__ __forceinline__ char* pair_at(const Pairs& p, size_t row, uint32_t c) {
  return const_cast<char*>(p.at) + row * p.ld + (c >> 5) * 128u + (c & 31u) * 2u;
}
__device__ __forceinline__ void put_pairs(const Pairs& p, size_t row, uint32_t c, const f4& v) {
  h4 hi, lo;
  split_pair(v, hi, lo);
  char* at = pair_at(p, row, c);
  *reinterpret_cast<h4*>(at) = hi;
  *reinterpret_cast<h4*>(at + 64) = lo;
}
__device__ __forceinline__ f4 get_pairs(const Pairs& p, size_t row, uint32_t c) {
  const char* at = pair_at(p, row, c);
  return join_pair(*reinterpret_cast<const h4*>(at), *reinterpret_cast<const h4*>(at + 64));
}

// The tile of L lines x 32 k of one operand in LDS, filled by WAVES wavefronts.
template <bool KC, int L, int WAVES>
struct PairStage {
  static constexpr int BYTES = L * 128;
  static constexpr int LOADS = L / 8 / WAVES;                // of 1 KiB, of each wavefront
  static_assert(L % (8 * WAVES) == 0 && L >= 64, "each wavefront fills as much of the tile");
  static constexpr int CPR = L / 4;                          // 16-byte chunks of a k row

  const char* base;        // of the tile at its k (uniform)
  size_t step;             // bytes of 32 k
  uint32_t off[LOADS];     // of this lane's 16 bytes
  uint32_t at;             // of this lane in a fragment of the wavefront's first lines

  // line0, k0: the tile's; first: the wavefront's own first line in it.
  __device__ __forceinline__ void begin(const Pairs& p, uint32_t line0, uint32_t k0, int first, int wave, int lane) {
    base = p.at + (KC ? (size_t)line0 * p.ld + 4u * (size_t)k0 : (size_t)k0 * p.ld + 4u * (size_t)line0);
    step = KC ? 128u : (size_t)32u * p.ld;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int i = (u * WAVES + wave) * 64 + lane;
      if constexpr (KC) {
        const int line = i / 8, c = (i % 8) ^ (line % 8);
        off[u] = line * p.ld + c * 16u;
      } else {
        const int row = i / CPR, c = (i % CPR) ^ (row % 4 * 2) ^ (row / 8 % 2 * 8);
        off[u] = row * p.ld + c * 16u;
      }
    }
    const int t = lane & 15, q = lane >> 4;
    if constexpr (KC) {
      at = (first + t) * 128 + ((q ^ (t & 7)) << 4);
    } else {
      const int k = 8 * q + (t >> 2);
      at = k * 4 * L + (((first >> 5) ^ (q & 1)) << 7) + ((((first >> 4) & 1) ^ (k & 3)) << 5) + (t & 3) * 8;
    }
  }
  // The next slice's loads, in flight until vmcnt reaches 0.
  __device__ __forceinline__ void load(char* tile, int wave) {
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(base + off[u]),
                                       (__attribute__((address_space(3))) uint32_t*)(tile + (u * WAVES + wave) * 1024), 16, 0, 0);
    }
    base += step;
  }
  // The wavefront's fragment i (16 lines) of hi (p 0) or lo (1) halves. At most 4 fragments, the
  // first line a multiple of 16 times as many (1, 2 or 4).
  __device__ __forceinline__ h8 frag(const char* tile, int i, int p) const {
    if constexpr (KC) {
      return *reinterpret_cast<const h8*>(tile + (at ^ (p << 6)) + i * 2048);
    } else {
      const char* x = tile + (at ^ (p << 6) ^ ((i & 1) << 5) ^ ((i >> 1) << 7));
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(x));
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(x + 16 * L));
      return __builtin_bit_cast(h8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// LDS bytes of a tile's product: STAGES slices of both operands.
template <int BM, int BN, int STAGES = 2>
constexpr int f16x2_lds() { return STAGES * 128 * (BM + BN); }

template <int N>
struct Ahead { static constexpr int value = N; };

// Waits until at most N of this wavefront's loads to LDS are in flight and all its reads of LDS are done.
template <int N>
__device__ __forceinline__ void arrived() {
  static_assert(N < 64, "vmcnt");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 << 14) | 0x0070);   // vmcnt(N) lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// That of every wavefront (__syncthreads() would wait for every load).
template <int N>
__device__ __forceinline__ void barrier_ahead() {
  arrived<N>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The slices that nothing is loaded beside, A after the first of them and fewer after each.
template <int A, class F>
__device__ __forceinline__ void last_slices(uint32_t s, const uint32_t slices, F& slice) {
  if (s + A < slices) {
    slice(Ahead<A>(), false);
    ++s;
  }
  if constexpr (A > 0) last_slices<A - 1>(s, slices, slice);
}

// The BM x BN = (WM·TM·16) x (WN·TN·16) tile of A·B at (m0, n0), summed over `slices` (1 or more) slices of 32 k
// from k0: lane (t, q) = (lane % 16, lane / 16) of wavefront (wm, wn) holds in acc[i][j] row
// m0 + (wm·TM + i)·16 + t, columns n0 + (wn·TN + j)·16 + 4q ... + 3. STAGES - 1 slices are loaded ahead. lds: f16x2_lds() bytes.
template <int WM, int WN, int TM, int TN, bool AKC, bool BKC, int STAGES = 2>
__device__ __forceinline__ void gemm_f16x2_sum(const Pairs& a, const Pairs& b, const uint32_t m0, const uint32_t n0, const uint32_t k0,
                                               const uint32_t slices, char* lds, f4 (&acc)[TM][TN]) {
  constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  using SA = PairStage<AKC, BM, WAVES>;
  using SB = PairStage<BKC, BN, WAVES>;
  constexpr int BUF = SA::BYTES + SB::BYTES, LOADS = SA::LOADS + SB::LOADS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  SA sa;
  SB sb;
  sa.begin(a, m0, k0, wave / WN * TM * 16, wave, lane);
  sb.begin(b, n0, k0, wave % WN * TN * 16, wave, lane);
  f4 low[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = low[i][j] = f4{0.f, 0.f, 0.f, 0.f};

  uint32_t buf = 0, fill = 0;      // of the slice multiplied next, and of the slice loaded next
  auto load = [&](char* to) {
    sa.load(to, wave);
    sb.load(to + SA::BYTES, wave);
    fill = fill + 1 == STAGES ? 0 : fill + 1;
  };
  // The slice in `from` multiplied, and (more) the next one loaded into `to`. The pointers are restrict so that
  // the compiler does not make the reads wait for every load to LDS: they wait at the barrier, for their own.
  auto multiply = [&](const char* __restrict__ from, char* __restrict__ to, const bool more) __attribute__((always_inline)) {
    h8 x[TM][2], y[TN][2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int j = 0; j < TN; ++j) y[j][p] = sb.frag(from + SA::BYTES, j, p);
#pragma unroll
      for (int i = 0; i < TM; ++i) x[i][p] = sa.frag(from, i, p);
    }
    if (more) load(to);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[j][0], x[i][0], acc[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) low[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[j][1], x[i][0], low[i][j], 0, 0, 0);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) low[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[j][0], x[i][1], low[i][j], 0, 0, 0);
  };
  // One slice, once its loads (all but those of the `ahead` slices after it) have arrived and every wavefront has read
  // the slice before, whose buffer is filled next.
  auto slice = [&](auto ahead, const bool more) __attribute__((always_inline)) {
    barrier_ahead<decltype(ahead)::value * LOADS>();
    const char* from = lds + buf * BUF;
    buf = buf + 1 == STAGES ? 0 : buf + 1;
    multiply(from, lds + fill * BUF, more);
  };
  uint32_t s = 0;
  for (uint32_t k = 0; k < STAGES - 1 && k < slices; ++k) load(lds + fill * BUF);
  for (; s + STAGES - 1 < slices; ++s) slice(Ahead<STAGES - 2>(), true);
  last_slices<STAGES - 2>(s, slices, slice);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] += low[i][j] * (1.f / PAIR_LO);
}

// The place of workgroup `id` of n in an order whose runs stay on one XCD: the 8 XCDs take workgroups in turn, and each gets a run of
// its own, so that neighbours in the order, which share operand panels, share an L2.
__device__ __forceinline__ uint32_t xcd_run(uint32_t id, uint32_t n) {
  const uint32_t per = n / 8u, left = n % 8u, x = id % 8u;
  return x * per + min(x, left) + id / 8u;
}
// The tile of workgroup `id` of rows x cols of them: down GROUP tile rows before the next column.
struct TileAt {
  uint32_t row, col;
};
template <uint32_t GROUP>
__device__ __forceinline__ TileAt tile_at(uint32_t id, uint32_t rows, uint32_t cols) {
  const uint32_t t = xcd_run(id, rows * cols);
  const uint32_t band = t / (GROUP * cols), first = band * GROUP, tall = min(rows - first, GROUP), in = t - band * GROUP * cols;
  return {first + in % tall, in / tall};
}

// The tiles that kernels take: 64 x 64 by four wavefronts of 32 x 32 (SMALL); 128 x 128 by four of 64 x 64 (SQUARE); 128 x 256 (WIDE)
// and 256 x 128 (TALL) by eight. At 4096^3 SQUARE takes 370 us, WIDE and TALL 352 - 365; 1024 x 1024 x 65536 448 and 417 - 425. SMALL is
// for products whose larger tiles would leave CUs idle: its wavefronts read 8 KiB of LDS for 192 cycles of products, the others' 16 KiB for 768, so
// that a full chip of them runs at 245 TFLOP/s; one a CU takes 0.3 us a slice, whose 16 KiB come at that rate. Neither loads further
// ahead nor a slice's fragments read while the one before is multiplied shorten that (25 slices 10.5 and 9.5 us, 8 slices 7.6 and 7.7).
enum { SMALL = 0, SQUARE = 1, WIDE = 2, TALL = 3 };
template <int KIND>
struct Tile {
  static constexpr int T = KIND == SMALL ? 2 : 4;
  static constexpr int WM = KIND == TALL ? 4 : 2, WN = KIND == WIDE ? 4 : 2;
  static constexpr int ROWS = WM * T * 16, COLS = WN * T * 16, THREADS = 64 * WM * WN;
  static constexpr int STAGES = KIND == SQUARE ? 2 : 3;
  static constexpr int LDS = f16x2_lds<ROWS, COLS, STAGES>();
  // Tile rows of a band: what the tiles that run at once on an XCD read is least where they form a square.
  static constexpr uint32_t GROUP = KIND == TALL ? 4 : 8;
  // The fragments of 16 rows and of 16 columns that a wavefront holds.
  static constexpr int TI = T, TJ = T;
  typedef f4 Sums[TI][TJ];

  // The tile's sums over `slices` slices from k0.
  template <bool AKC, bool BKC>
  static __device__ __forceinline__ void sum(const Pairs& a, const Pairs& b, const TileAt& at, uint32_t k0, uint32_t slices, char* lds, Sums& acc) {
    gemm_f16x2_sum<WM, WN, T, T, AKC, BKC, STAGES>(a, b, at.row * ROWS, at.col * COLS, k0, slices, lds, acc);
  }
  // The row, and the first column, of this lane's first four sums: fragment (i, j)'s 16·i rows and 16·j columns on.
  static __device__ __forceinline__ uint32_t row(const TileAt& at) { return at.row * ROWS + threadIdx.x / 64 / WN * TI * 16 + threadIdx.x % 16; }
  static __device__ __forceinline__ uint32_t col(const TileAt& at) { return at.col * COLS + threadIdx.x / 64 % WN * TJ * 16 + threadIdx.x % 64 / 16 * 4; }
  // f(row, col, v) of each four columns that this lane holds, 16 rows at a time: what f loads for all of them does not fit the
  // registers beside the sums.
  template <class F>
  static __device__ __forceinline__ void each(const TileAt& at, Sums& acc, F f) {
    const uint32_t row0 = row(at), col0 = col(at);
#pragma unroll
    for (int i = 0; i < TI; ++i) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < TJ; ++j) f(row0 + i * 16, col0 + j * 16, acc[i][j]);
    }
  }
};

}  // namespace tcmi
