// Rows of a table by token, and the table's gradient: for each row the sum of its tokens' rows.
//
//   e[i] = scale·table[t_i],   dtable[v] = scale·(sum over i with t_i = v of dy[i]),
// a token that is no whole number in 0 .. V - 1 left out of both (its e is 0).
//
// The sums are of sorted tokens: (token, place) pairs are sorted by token, equal ones in their
// places' order, by a radix sort of BITS bits a pass, and CH sorted pairs after the other are summed by the lanes of a
// group, which hold a block of columns of one row of dy each. A token whose pairs lie in one chunk is written there; of a
// token that goes on in the next chunk, its first pairs' sum and those of the chunks after it are written apart and added in order by the
// chunk that it starts in. So the order of a sum is given by the tokens alone. Rows without a token are found by a
// search for each and written as zeros.
//
// A table of few rows takes no sort: a wavefront adds its rows of dy in their order into a table of its own in LDS, a lane a column, and the
// wavefronts' and then the workgroups' tables are added in order.
//
// A pass of the sort, a tile of keys a workgroup: a key's place is the count of smaller digits, of
// its digit in the tiles before, in the wavefronts before and among the lanes before it (found by comparing digits bit by bit
// over the wavefront). The tiles are counted by a launch before each pass; a few keys are one tile, and one launch makes all passes.
//
// Bound: HBM (rows read and written; dy read, the table's gradient written). 32768 tokens of 1024 floats over 65536 rows: rows 42 us (268 MB, 6.4 TB/s), the
// gradient 23 to sort by two digits of eight bits, 83 for the sums (403 MB, 4.9 TB/s) and 7 to join them; 8192 tokens of 256 over 96 rows 3.8, and 8.2 and 3.7
// for the gradient's tables and their sum; 32 tokens of 1024 3.1, a launch's time.

#pragma once

#include "tcmi_device.h"

namespace tcmi {

// A row's token as a key, or -1.
__device__ __forceinline__ int32_t embed_key(float t, uint32_t rows) {
  return t >= 0.f && t < static_cast<float>(rows) && t == __builtin_truncf(t) ? static_cast<int32_t>(t) : -1;
}

// E floats at p (128 bits of them where E is 4).
template <int E>
__device__ __forceinline__ f4 embed_load(const float* __restrict__ p) {
  if constexpr (E == 4) return *reinterpret_cast<const f4*>(p);
  return f4{*p, 0.f, 0.f, 0.f};
}
template <int E>
__device__ __forceinline__ void embed_store(float* __restrict__ p, const f4& v) {
  if constexpr (E == 4) {
    *reinterpret_cast<f4*>(p) = v;
  } else {
    *p = v[0];
  }
}

// Token `row`, its lanes' groups of E floats from group `block`·UNITS·LANES on.
template <class S>
__device__ __forceinline__ void embed(const float* __restrict__ tokens, const float* __restrict__ table, float* __restrict__ out, uint32_t row, uint32_t block) {
  if (row >= S::N) return;
  const int32_t key = embed_key(tokens[row], S::V);
  const float* from = table + (size_t)(key < 0 ? 0 : key) * S::D;
  float* to = out + (size_t)row * S::D;
  const uint32_t first = (block * S::UNITS * S::LANES + threadIdx.x % S::LANES) * S::E;
  f4 v[S::UNITS];
#pragma unroll
  for (uint32_t u = 0; u < S::UNITS; ++u) {
    const uint32_t c = first + u * S::LANES * S::E;
    v[u] = key >= 0 && c < S::D ? embed_load<S::E>(from + c) * S::scale() : f4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (uint32_t u = 0; u < S::UNITS; ++u) {
    const uint32_t c = first + u * S::LANES * S::E;
    if (c < S::D) embed_store<S::E>(to + c, v[u]);
  }
}

// The pairs before pass PASS (0: the tokens themselves), and those after it.
template <class S, int PASS>
struct EmbedPairs {
  const float* tokens;
  char* ws;
  __device__ __forceinline__ uint32_t count() const { return PASS == 0 ? static_cast<uint32_t>(S::N) : *reinterpret_cast<const uint32_t*>(ws + S::COUNT); }
  __device__ __forceinline__ int32_t key(uint32_t i) const {
    return PASS == 0 ? embed_key(tokens[i], S::V) : reinterpret_cast<const int32_t*>(ws + (PASS % 2 ? S::KEYS0 : S::KEYS1))[i];
  }
  __device__ __forceinline__ uint32_t place(uint32_t i) const {
    return PASS == 0 ? i : reinterpret_cast<const uint32_t*>(ws + (PASS % 2 ? S::PLACES0 : S::PLACES1))[i];
  }
  __device__ __forceinline__ void put(uint32_t i, int32_t key, uint32_t place) const {
    reinterpret_cast<int32_t*>(ws + (PASS % 2 ? S::KEYS1 : S::KEYS0))[i] = key;
    reinterpret_cast<uint32_t*>(ws + (PASS % 2 ? S::PLACES1 : S::PLACES0))[i] = place;
  }
  static __device__ __forceinline__ uint32_t digit(int32_t key) { return (static_cast<uint32_t>(key) >> (PASS * S::BITS)) & ((1u << S::BITS) - 1u); }
};

// The lanes that have a key of this lane's digit.
template <int BITS>
__device__ __forceinline__ uint64_t embed_same(bool has, uint32_t digit) {
  uint64_t same = __ballot(has);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const uint64_t ones = __ballot((digit >> b) & 1u);
    same &= (digit >> b) & 1u ? ones : ~ones;
  }
  return same;
}

// One step of a wavefront's lanes on LDS that only it uses: what a lane wrote before is read after, and nothing earlier.
__device__ __forceinline__ void embed_step() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Keys that a wavefront of the sort holds at a time, 64 each: their loads are in flight together.
constexpr uint32_t EMBED_HELD = 8;

// Counts tile `tile`'s digits.
template <class S, int PASS>
__device__ __forceinline__ void embed_count(const float* __restrict__ tokens, char* ws, uint32_t* bins, uint32_t tile) {
  const EmbedPairs<S, PASS> in{tokens, ws};
  constexpr uint32_t BINS = 1u << S::BITS;
  const uint32_t n = in.count(), begin = tile * S::TILE, end = min(n, begin + S::TILE), lane = threadIdx.x % 64u;
  for (uint32_t b = threadIdx.x; b < BINS; b += S::SORT) bins[b] = 0u;
  __syncthreads();
  for (uint32_t base = begin + threadIdx.x - lane; base < end; base += S::SORT * EMBED_HELD) {
    int32_t key[EMBED_HELD];
#pragma unroll
    for (uint32_t u = 0; u < EMBED_HELD; ++u) {
      const uint32_t i = base + u * S::SORT + lane;
      key[u] = i < end ? in.key(i) : -1;
    }
#pragma unroll
    for (uint32_t u = 0; u < EMBED_HELD; ++u) {
      if (key[u] >= 0) atomicAdd(bins + in.digit(key[u]), 1u);
    }
  }
  __syncthreads();
  uint32_t* hist = reinterpret_cast<uint32_t*>(ws + S::HIST) + (size_t)tile * BINS;
  for (uint32_t b = threadIdx.x; b < BINS; b += S::SORT) hist[b] = bins[b];
}

// Tile `tile`'s pairs to their places, by SORT threads. lds: (1 + SORT / 64)·BINS + SORT / 64 words.
template <class S, int PASS>
__device__ __forceinline__ void embed_sort(const float* __restrict__ tokens, char* ws, uint32_t* lds, uint32_t tile) {
  const EmbedPairs<S, PASS> in{tokens, ws};
  constexpr uint32_t BINS = 1u << S::BITS, WAVES = S::SORT / 64u;
  const uint32_t n = in.count(), begin = tile * S::TILE, end = min(n, begin + S::TILE);
  const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u;
  uint32_t *own = lds, *before = lds + WAVES * BINS, *part = before + BINS;    // own: of each wavefront; before: of smaller digits, and of the tiles before
  for (uint32_t b = threadIdx.x; b < WAVES * BINS; b += S::SORT) own[b] = 0u;
  // Each wavefront's keys of the tile are a run of their own.
  constexpr uint32_t RUN = S::TILE / WAVES;
  static_assert(RUN % 64u == 0u, "runs of whole wavefronts");
  const uint32_t mine = min(end, begin + wave * RUN), mine_end = min(end, mine + RUN);
  __syncthreads();
  for (uint32_t base = mine; base < mine_end; base += 64u * EMBED_HELD) {
    int32_t key[EMBED_HELD];
#pragma unroll
    for (uint32_t u = 0; u < EMBED_HELD; ++u) {
      const uint32_t i = base + u * 64u + lane;
      key[u] = i < mine_end ? in.key(i) : -1;
    }
#pragma unroll
    for (uint32_t u = 0; u < EMBED_HELD; ++u) {
      if (key[u] >= 0) atomicAdd(own + wave * BINS + in.digit(key[u]), 1u);
    }
  }
  __syncthreads();
  // Thread t's PER digits: how many there are of each, and of them in the tiles before.
  constexpr uint32_t PER = (BINS + S::SORT - 1u) / S::SORT;
  uint32_t sum = 0u, smaller[PER], prior[PER];
#pragma unroll
  for (uint32_t k = 0; k < PER; ++k) {
    const uint32_t b = threadIdx.x * PER + k;
    smaller[k] = sum;
    prior[k] = 0u;
    if (b < BINS) {
      uint32_t all = 0u;
      if constexpr (S::TILES == 1u) {
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) all += own[w * BINS + b];
      } else {
        const uint32_t* hist = reinterpret_cast<const uint32_t*>(ws + S::HIST) + b;
#pragma unroll 8
        for (uint32_t t = 0; t < S::TILES; ++t) {
          const uint32_t c = hist[(size_t)t * BINS];
          all += c;
          prior[k] += t < tile ? c : 0u;
        }
      }
      sum += all;
    }
  }
  // The sums of the threads before it come by wavefront.
  uint32_t scan = sum;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) {
    const uint32_t v = __shfl_up(scan, off, 64);
    if (lane >= static_cast<uint32_t>(off)) scan += v;
  }
  if (lane == 63u) part[wave] = scan;
  __syncthreads();
  uint32_t first = scan - sum;
  for (uint32_t w = 0; w < wave; ++w) first += part[w];
#pragma unroll
  for (uint32_t k = 0; k < PER; ++k) {
    const uint32_t b = threadIdx.x * PER + k;
    if (b < BINS) {
      uint32_t at = first + smaller[k] + prior[k];
#pragma unroll
      for (uint32_t w = 0; w < WAVES; ++w) {
        const uint32_t c = own[w * BINS + b];
        own[w * BINS + b] = at;
        at += c;
      }
    }
  }
  if (PASS == 0 && tile == 0 && threadIdx.x == S::SORT - 1u) *reinterpret_cast<uint32_t*>(ws + S::COUNT) = first + sum;
  __syncthreads();
  for (uint32_t base = mine; base < mine_end; base += 64u * EMBED_HELD) {
    int32_t key[EMBED_HELD];
    uint32_t from[EMBED_HELD];
#pragma unroll
    for (uint32_t u = 0; u < EMBED_HELD; ++u) {
      const uint32_t i = base + u * 64u + lane;
      key[u] = i < mine_end ? in.key(i) : -1;
      from[u] = i < mine_end ? in.place(i) : 0u;
    }
#pragma unroll
    for (uint32_t u = 0; u < EMBED_HELD; ++u) {
      const uint32_t d = in.digit(key[u]);
      const uint64_t same = embed_same<S::BITS>(key[u] >= 0, d);
      if (key[u] >= 0) {
        const uint32_t at = own[wave * BINS + d];
        embed_step();
        in.put(at + static_cast<uint32_t>(__popcll(same & ((1ull << lane) - 1ull))), key[u], from[u]);
        if (__builtin_ctzll(same) == static_cast<int>(lane)) own[wave * BINS + d] = at + static_cast<uint32_t>(__popcll(same));
      }
      embed_step();
    }
  }
}

// All passes by one workgroup, whose tile all keys are: a pass reads what the one before wrote.
template <class S, int PASS = 0>
__device__ __forceinline__ void embed_sort_all(const float* __restrict__ tokens, char* ws, uint32_t* lds) {
  embed_sort<S, PASS>(tokens, ws, lds, 0u);
  if constexpr (PASS + 1 < S::PASSES) {
    __threadfence();
    __syncthreads();
    embed_sort_all<S, PASS + 1>(tokens, ws, lds);
  }
}

// The sorted pairs, after the last pass.
template <class S, int LAST>
struct EmbedSorted {
  char* ws;
  __device__ __forceinline__ uint32_t count() const { return *reinterpret_cast<const uint32_t*>(ws + S::COUNT); }
  __device__ __forceinline__ const int32_t* keys() const { return reinterpret_cast<const int32_t*>(ws + (LAST ? S::KEYS1 : S::KEYS0)); }
  __device__ __forceinline__ const uint32_t* places() const { return reinterpret_cast<const uint32_t*>(ws + (LAST ? S::PLACES1 : S::PLACES0)); }
  // A chunk's sum of the token that goes on from the chunk before (0) or goes on in the next alone (1).
  __device__ __forceinline__ float* part(uint32_t chunk, uint32_t which) const { return reinterpret_cast<float*>(ws + S::PARTS) + ((size_t)chunk * 2u + which) * S::D; }
};

// Workgroups: the chunks' sums, all groups of one block of columns after the other, then the rows without a token. lds: ROWS words.
template <class S, int LAST>
__device__ __forceinline__ void embed_sums(const float* __restrict__ dy, float* __restrict__ out, char* ws, uint32_t* lds, uint32_t wg) {
  const EmbedSorted<S, LAST> in{ws};
  const uint32_t n = in.count();
  const int32_t* __restrict__ keys = in.keys();
  constexpr uint32_t GROUPS = 256u / S::LANES, COLUMNS = (S::D + S::E * S::LANES - 1u) / (S::E * S::LANES), SUMS = (S::CHUNKS + GROUPS - 1u) / GROUPS * COLUMNS;
  if (wg < SUMS) {
    const uint32_t chunk = wg / COLUMNS * GROUPS + threadIdx.x / S::LANES, c = (wg % COLUMNS * S::LANES + threadIdx.x % S::LANES) * S::E;
    const uint32_t begin = chunk * S::CH, end = min(n, begin + S::CH);
    if (begin >= end || c >= S::D) return;
    const uint32_t* __restrict__ places = in.places();
    const int32_t earlier = begin > 0u ? keys[begin - 1u] : -1, later = end < n ? keys[end] : -1;
    f4 sum = {0.f, 0.f, 0.f, 0.f};
    constexpr uint32_t AHEAD = 8u;
    uint32_t i = begin;
    bool whole = keys[begin] != earlier;          // the token's first pair is in this chunk
    for (; i < end; i += AHEAD) {
      f4 v[AHEAD];
      int32_t key[AHEAD + 1u];
#pragma unroll
      for (uint32_t u = 0; u < AHEAD; ++u) {
        const uint32_t j = min(i + u, end - 1u);
        key[u] = keys[j];
        v[u] = embed_load<S::E>(dy + (size_t)places[j] * S::D + c);
      }
      key[AHEAD] = i + AHEAD < end ? keys[i + AHEAD] : later;
#pragma unroll
      for (uint32_t u = 0; u < AHEAD; ++u) {
        if (i + u >= end) break;
        sum += v[u];
        const int32_t next = i + u + 1u < end ? key[u + 1u] : later;
        if (next != key[u]) {
          // (A token that no chunk shares is whole here.)
          if (whole) embed_store<S::E>(out + (size_t)key[u] * S::D + c, sum * S::scale());
          else embed_store<S::E>(in.part(chunk, 0u) + c, sum);
          sum = f4{0.f, 0.f, 0.f, 0.f};
          whole = true;
        } else if (i + u + 1u == end) {
          embed_store<S::E>(in.part(chunk, whole ? 1u : 0u) + c, sum);
        }
      }
    }
    return;
  }
  const uint32_t row0 = (wg - SUMS) * S::ROWS;
  if (threadIdx.x < S::ROWS) {
    const int32_t row = static_cast<int32_t>(row0 + threadIdx.x);
    uint32_t lo = 0u, hi = n;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2u;
      if (keys[mid] < row) lo = mid + 1u;
      else hi = mid;
    }
    lds[threadIdx.x] = lo < n && keys[lo] == row;
  }
  __syncthreads();
  constexpr uint32_t C = S::D / S::E;
  for (uint32_t r = threadIdx.x / S::LANES; r < S::ROWS && row0 + r < S::V; r += GROUPS) {
    if (lds[r]) continue;
    for (uint32_t g = threadIdx.x % S::LANES; g < C; g += S::LANES) embed_store<S::E>(out + (size_t)(row0 + r) * S::D + g * S::E, f4{0.f, 0.f, 0.f, 0.f});
  }
}

// The sum of a token that starts in chunk `chunk` and goes on: eight wavefronts take its chunks in turn, their sums in
// order. lds: 8·64·E floats.
template <class S, int LAST>
__device__ __forceinline__ void embed_join(float* __restrict__ out, char* ws, float* lds, uint32_t chunk, uint32_t block) {
  const EmbedSorted<S, LAST> in{ws};
  const uint32_t n = in.count(), begin = chunk * S::CH, end = begin + S::CH;
  if (end >= n) return;
  const int32_t* __restrict__ keys = in.keys();
  const int32_t key = keys[end - 1u];
  if (keys[end] != key || (begin > 0u && keys[begin] == key && keys[begin - 1u] == key)) return;
  const uint32_t lane = threadIdx.x % 64u, wave = threadIdx.x / 64u, c = (block * 64u + lane) * S::E;
  // The chunks after this one that begin with the token: a wavefront looks at 64 of them at a time.
  uint32_t more = 0u;
  for (;;) {
    const uint64_t i = (uint64_t)(chunk + 1u + more + lane) * S::CH;
    const uint64_t on = __ballot(i < n && keys[i < n ? i : 0u] == key);
    const uint32_t run = on == ~0ull ? 64u : static_cast<uint32_t>(__builtin_ctzll(~on));
    more += run;
    if (run < 64u) break;
  }
  f4 sum = {0.f, 0.f, 0.f, 0.f};
  if (c < S::D) {
    if (wave == 0u) sum = embed_load<S::E>(in.part(chunk, 1u) + c);
#pragma unroll 4
    for (uint32_t k = wave; k < more; k += 8u) sum += embed_load<S::E>(in.part(chunk + 1u + k, 0u) + c);
  }
#pragma unroll
  for (uint32_t e = 0; e < S::E; ++e) lds[(wave * S::E + e) * 64u + lane] = sum[e];
  __syncthreads();
  if (wave != 0u || c >= S::D) return;
  for (uint32_t w = 1; w < 8u; ++w) {
#pragma unroll
    for (uint32_t e = 0; e < S::E; ++e) sum[e] += lds[(w * S::E + e) * 64u + lane];
  }
  embed_store<S::E>(out + (size_t)key * S::D + c, sum * S::scale());
}

// A table of few rows: workgroup `chunk` of CHUNKS adds CH rows of dy, a quarter a wavefront, 64 columns from 64·`block` on. lds: 4·V·64 floats.
template <class S>
__device__ __forceinline__ void embed_few(const float* __restrict__ tokens, const float* __restrict__ dy, float* __restrict__ out, float* __restrict__ parts, float* lds, uint32_t chunk, uint32_t block) {
  const uint32_t lane = threadIdx.x % 64u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u), c = block * 64u + lane;
  float* const own = lds + wave * S::V * 64u;
  constexpr uint32_t RUN = S::CH / 4u, HELD = 32u;
  const uint32_t begin = min(static_cast<uint32_t>(S::N), chunk * S::CH + wave * RUN), end = min(static_cast<uint32_t>(S::N), begin + RUN);
  for (uint32_t i = begin; i < end; i += HELD) {
    // (Every load is made, of the run's last row and the table's last column where its own is past them.)
    float x[HELD];
    const float token = tokens[min(i + lane % HELD, end - 1u)];
#pragma unroll
    for (uint32_t u = 0; u < HELD; ++u) x[u] = dy[(size_t)min(i + u, end - 1u) * S::D + min(c, S::D - 1u)];
    const int32_t mine = i + lane % HELD < end ? embed_key(token, S::V) : -1;
    if (i == begin) {
      // (While the first rows are on their way.)
      for (uint32_t v = lane; v < S::V * 16u; v += 64u) reinterpret_cast<f4*>(own)[v] = f4{0.f, 0.f, 0.f, 0.f};
      embed_step();
    }
#pragma unroll
    for (uint32_t u = 0; u < HELD; ++u) {
      const int32_t key = __builtin_amdgcn_readlane(mine, u);
      if (key >= 0) own[key * 64 + lane] += x[u];
    }
  }
  if (begin >= end) {
    for (uint32_t v = lane; v < S::V * 16u; v += 64u) reinterpret_cast<f4*>(own)[v] = f4{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();
  float* const to = S::CHUNKS > 1u ? parts + (size_t)chunk * S::V * S::D : out;
#pragma unroll 8
  for (uint32_t v = wave; v < S::V; v += 4u) {
    float sum = lds[v * 64u + lane];
#pragma unroll
    for (uint32_t w = 1; w < 4u; ++w) sum += lds[(w * S::V + v) * 64u + lane];
    if (c < S::D) to[(size_t)v * S::D + c] = S::CHUNKS > 1u ? sum : sum * S::scale();
  }
}

// Its chunks' tables: a workgroup takes 16 groups of four floats, 16 threads a group, each its own chunks in turn. lds: 1024 floats.
template <class S>
__device__ __forceinline__ void embed_fold(float* __restrict__ out, const float* __restrict__ parts, float* lds, uint32_t block) {
  constexpr size_t ALL = (size_t)S::V * S::D;
  const uint32_t part = threadIdx.x / 16u;
  const size_t at = ((size_t)block * 16u + threadIdx.x % 16u) * 4u;
  f4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (uint32_t k = part; k < S::CHUNKS; k += 16u) {
    if constexpr (ALL % 4u == 0u) {
      if (at < ALL) sum += *reinterpret_cast<const f4*>(parts + k * ALL + at);
    } else {
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e) sum[e] += at + e < ALL ? parts[k * ALL + at + e] : 0.f;
    }
  }
  f4* all = reinterpret_cast<f4*>(lds);
  all[threadIdx.x] = sum;
  __syncthreads();
  if (part != 0u) return;
#pragma unroll
  for (uint32_t p = 1; p < 16u; ++p) sum += all[p * 16u + threadIdx.x];
  sum *= S::scale();
#pragma unroll
  for (uint32_t e = 0; e < 4u; ++e) {
    if (at + e < ALL) out[at + e] = sum[e];
  }
}

}  // namespace tcmi
