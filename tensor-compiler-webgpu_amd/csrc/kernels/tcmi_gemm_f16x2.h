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
// Operands are planes in memory: element (line, k) of an operand (A: row of C, B: column
// of C) at line·ld + k (KC: k contiguous) or k·ld + line, hi and lo planes of one layout.
// They are padded with zeros to whole tiles (lines to the tile's, k to 32), so the loop has
// no bounds. Loads go straight to LDS (16 bytes a lane). A slice of 32 k of L lines:
//   KC       64 bytes a line, its four 16-byte chunks q rotated: chunk q of line l at
//            slot q ^ (l / 2 % 4), so the 8 lanes of a 128-byte LDS cycle (8 lines, one q) meet
//            all banks. A lane's fragment, 8 k of one line, is one ds_read_b128.
//   not KC   2·L bytes a k, its 32-byte groups of 16 lines rotated: group g of row k at
//            g ^ (k % 4). Fragments are read by ds_read_b64_tr_b16, which
//            transposes: lanes of 16 each give the address of 4 lines of one of 4 rows of k, and
//            each gets its own line's 4 k; two reads make a fragment.
// Either way neither layout is materialised transposed.

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

// An operand: its hi plane, the lo plane `plane` bytes after it, and bytes a line (or k).
struct Pairs {
  const char* hi;
  size_t plane;
  uint32_t ld;
};

// The tile of L lines x 32 k of one operand in LDS, filled by WAVES wavefronts.
template <bool KC, int L, int WAVES>
struct PairStage {
  static constexpr int PLANE = L * 64, BYTES = 2 * PLANE;
  static constexpr int UNITS = L / 16;                       // loads of 1 KiB a plane
  static constexpr int LOADS = UNITS / WAVES;                // of each wavefront
  static_assert(UNITS % WAVES == 0, "each wavefront fills as much of a plane");
  static constexpr int CPR = L / 8;                          // 16-byte chunks of a k row

  const char* base;        // of the tile at k = 0 (uniform)
  size_t plane;
  size_t step;             // bytes of 32 k
  uint32_t off[LOADS];     // of this lane's 16 bytes

  __device__ __forceinline__ void begin(const Pairs& p, uint32_t line0, uint32_t k0, int wave, int lane) {
    base = p.hi + (KC ? (size_t)line0 * p.ld + 2u * (size_t)k0 : (size_t)k0 * p.ld + 2u * (size_t)line0);
    plane = p.plane;
    step = KC ? 64u : (size_t)32u * p.ld;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      const int unit = u * WAVES + wave;
      if constexpr (KC) {
        const int line = unit * 16 + (lane >> 2), q = (lane & 3) ^ ((line >> 1) & 3);
        off[u] = line * p.ld + q * 16u;
      } else {
        const int row = unit * (64 / CPR) + lane / CPR, c = (lane % CPR) ^ ((row & 3) << 1);
        off[u] = row * p.ld + c * 16u;
      }
    }
  }
  // The next slice's loads, in flight until vmcnt reaches 0.
  __device__ __forceinline__ void load(char* tile, int wave) {
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int u = 0; u < LOADS; ++u) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(base + p * plane + off[u]),
                                         (__attribute__((address_space(3))) uint32_t*)(tile + p * PLANE + (u * WAVES + wave) * 1024), 16, 0, 0);
      }
    base += step;
  }
  // This lane's address in a plane: of fragment i of the lines from `line0` (a multiple of 32), at + i·FRAG (KC) or at ^ i·32.
  static __device__ __forceinline__ uint32_t frag_at(int line0, int lane) {
    const int t = lane & 15, q = lane >> 4;
    if constexpr (KC) return (line0 + t) * 64 + ((q ^ ((t >> 1) & 3)) << 4);
    const int k = 8 * q + (t >> 2);
    return k * 2 * L + (((line0 >> 4) ^ (k & 3)) << 5) + (t & 3) * 8;
  }
  static __device__ __forceinline__ h8 frag(const char* plane, uint32_t at, int i) {
    if constexpr (KC) {
      return *reinterpret_cast<const h8*>(plane + at + i * 1024);
    } else {
      const char* p = plane + (at ^ (i << 5));
      const s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p));
      const s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(p + 8 * L));
      return __builtin_bit_cast(h8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  }
};

// LDS bytes of gemm_f16x2_sum: two buffers of both operands' slices.
template <int BM, int BN>
constexpr int f16x2_lds() { return 2 * 128 * (BM + BN); }

// The BM x BN = (WM·TM·16) x (WN·TN·16) tile of A·B at (m0, n0), summed over `slices` slices of 32 k
// from k0: lane (t, q) = (lane % 16, lane / 16) of wavefront (wm, wn) holds in acc[i][j] row
// m0 + (wm·TM + i)·16 + t, columns n0 + (wn·TN + j)·16 + 4q ... + 3. lds: f16x2_lds() bytes.
template <int WM, int WN, int TM, int TN, bool AKC, bool BKC>
__device__ __forceinline__ void gemm_f16x2_sum(const Pairs& a, const Pairs& b, const uint32_t m0, const uint32_t n0, const uint32_t k0,
                                               const uint32_t slices, char* lds, f4 (&acc)[TM][TN]) {
  constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
  using SA = PairStage<AKC, BM, WAVES>;
  using SB = PairStage<BKC, BN, WAVES>;
  constexpr int BUF = SA::BYTES + SB::BYTES;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN;
  SA sa;
  SB sb;
  sa.begin(a, m0, k0, wave, lane);
  sb.begin(b, n0, k0, wave, lane);
  const uint32_t fa = SA::frag_at(wm * TM * 16, lane), fb = SB::frag_at(wn * TN * 16, lane);
  f4 low[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = low[i][j] = f4{0.f, 0.f, 0.f, 0.f};

  sa.load(lds, wave);
  sb.load(lds + SA::BYTES, wave);
  for (uint32_t s = 0; s < slices; ++s) {
    // This slice's loads have arrived, and every wavefront has read the other buffer's slice.
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
    const char* from = lds + (s & 1) * BUF;
    h8 x[TM][2], y[TN][2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int j = 0; j < TN; ++j) y[j][p] = SB::frag(from + SA::BYTES + p * SB::PLANE, fb, j);
#pragma unroll
      for (int i = 0; i < TM; ++i) x[i][p] = SA::frag(from + p * SA::PLANE, fa, i);
    }
    if (s + 1 < slices) {
      char* to = lds + ((s + 1) & 1) * BUF;
      sa.load(to, wave);
      sb.load(to + SA::BYTES, wave);
    }
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
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] += low[i][j] * (1.f / PAIR_LO);
}

// The tile of workgroup `id` of rows x cols of them, so that the 8 XCDs (which take workgroups in
// turn) each walk a run of tiles of their own, down `GROUP` tile rows before the next column:
// neighbours in time share operand panels in one L2.
struct TileAt {
  uint32_t row, col;
};
__device__ __forceinline__ TileAt tile_at(uint32_t id, uint32_t rows, uint32_t cols) {
  constexpr uint32_t GROUP = 8;
  const uint32_t n = rows * cols, per = n / 8u, left = n % 8u, x = id % 8u;
  const uint32_t t = x * per + min(x, left) + id / 8u;
  const uint32_t band = t / (GROUP * cols), first = band * GROUP, tall = min(rows - first, GROUP), in = t - band * GROUP * cols;
  return {first + in % tall, in / tall};
}

}  // namespace tcmi
