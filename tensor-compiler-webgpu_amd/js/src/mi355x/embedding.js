'use strict';
// Launches of embedding and its gradient (tcmi_embedding.h).

const { size } = require('../ir/shapes');
const { ceil, align, double, constants, kernel } = require('./operator_parts');

// Tokens at most: they are counted in 32 bits, and a column of 16 threads a token in a grid.
const MOST_TOKENS = 2 ** 28;
const S = '__KERNEL___s';

function make(z, scale, types) {
  return (kind, grid, threads, lds, call) => kernel(kind, `#include "tcmi_embedding.h"
struct ${S} {
${constants(z, types)}
  static __device__ __forceinline__ float scale() { return static_cast<float>(${double(scale)}); }
};
extern "C" __global__ void __launch_bounds__(${threads}) __KERNEL__(const TcmiArgs A) {
${lds ? `  __shared__ __attribute__((aligned(16))) ${lds};\n` : ''}  tcmi::${call};
}
`, grid, threads);
}

/** Lanes of a row of d floats, each with E of them, and blocks of columns that those lanes take at a time. */
function rowLanes(d) {
  const E = d % 4 === 0 ? 4 : 1, groups = d / E;
  let lanes = 1;
  while (lanes < 64 && lanes < groups) lanes *= 2;
  return { E, lanes, columns: ceil(groups, lanes) };
}

function lowerEmbedding(graph, node) {
  const [V, D] = graph.nodes[node.inputs[1]].shape, N = size(graph.nodes[node.inputs[0]].shape);
  if (N > MOST_TOKENS) throw new Error(`embedding: ${N} tokens (at most ${MOST_TOKENS})`);
  const { E, lanes, columns } = rowLanes(D);
  // A lane takes up to four groups of a row; more of them are other workgroups'.
  const z = { N, V, D, E, LANES: lanes, UNITS: Math.min(4, columns) };
  const blocks = ceil(columns, z.UNITS);
  if (ceil(N, 256 / lanes) * 256 >= 2 ** 32) throw new Error(`embedding: ${N} tokens of ${D} floats (a grid has 2^32 threads, ${lanes} a token)`);
  if (blocks > 65535) throw new Error(`embedding: rows of ${D} floats (at most ${65535 * 64 * 4 * E})`);
  const k = make(z, node.attrs.scale)('emb', [ceil(N, 256 / lanes), blocks, 1], 256, null,
    `embed<${S}>(A.in[0], A.in[1], A.out, blockIdx.x * (256u / ${S}::LANES) + threadIdx.x / ${S}::LANES, blockIdx.y)`);
  return { kind: 'embedding', kernels: [k], workspace: 0 };
}

// Keys that one workgroup sorts, of 1024 threads; beyond, tiles of them are sorted by 256. (Gradients of 2000 tokens over 1000 rows 22.7 us by one, 26.7 by
// tiles; of 4096 27.0 and 25.2; of 16384 57.7 and 32.9.)
const ONE_TILE = 2048;

/**
 * Rows of a table that a wavefront keeps for itself, four wavefronts' in LDS, which holds no more: with rows and gradients, 8192 tokens of 256 floats over 96 rows
 * 23.8 us by sorted tokens, 14.0 so, over 128 23.6 and 15.3; 65536 tokens of 1024 over 128 149 and 153.
 */
const FEW_ROWS = 128;

function fewRows(node, N, V, D) {
  const columns = ceil(D, 64);
  // A workgroup a CU, of no fewer rows than the table that it writes has.
  const CH = align(Math.max(V, ceil(N * columns, 256), 64), 64), CHUNKS = ceil(N, CH);
  if (columns > 65535) throw new Error(`embedding: rows of ${D} floats (at most ${65535 * 64})`);
  const m = make({ N, V, D, CH, CHUNKS }, node.attrs.scale, {});
  const kernels = [m('embfew', [CHUNKS, columns, 1], 256, `float lds[${4 * V * 64}]`, `embed_few<${S}>(A.in[0], A.in[1], A.out, A.ws, lds, blockIdx.x, blockIdx.y)`)];
  if (CHUNKS > 1) kernels.push(m('embfold', [ceil(V * D, 64), 1, 1], 256, 'float lds[1024]', `embed_fold<${S}>(A.out, A.ws, lds, blockIdx.x)`));
  return { kind: 'embedding-grad', kernels, workspace: CHUNKS > 1 ? 4 * CHUNKS * V * D : 0 };
}

function lowerEmbeddingGrad(graph, node) {
  const N = size(graph.nodes[node.inputs[0]].shape), [V, D] = node.shape;
  if (N > MOST_TOKENS) throw new Error(`embedding: ${N} tokens (at most ${MOST_TOKENS})`);
  if (V <= FEW_ROWS) return fewRows(node, N, V, D);
  const { E, lanes, columns } = rowLanes(D);
  if (columns > 65535) throw new Error(`embedding: rows of ${D} floats (at most ${65535 * 64 * E})`);
  // Digits of at most nine bits of the token; a tile of keys a workgroup, at most 128 of them.
  const bits = Math.max(1, Math.ceil(Math.log2(V))), PASSES = ceil(bits, 9), BITS = ceil(bits, PASSES);
  const one = N <= ONE_TILE, SORT = one ? Math.min(1024, align(N, 64)) : 256;
  const TILE = one ? align(N, SORT) : Math.max(1024, align(ceil(N, 128), 256)), TILES = ceil(N, TILE);
  // Keys of a sum: few enough that 4096 wavefronts walk them. (32768 tokens of 1024 floats, in all: by 8 169 us, 16 161, 32, which this takes, 154, 64 160; 8192 of 256
  // by 8, which this takes, 27.1, 16 28.4, 64 43.)
  const waves = N * columns * lanes / 64;
  let CH = 8;
  while (CH < 64 && waves / CH > 4096) CH *= 2;
  const CHUNKS = ceil(N, CH), split = CHUNKS > 1;
  // Rows of the table that a workgroup looks for: a wavefront's worth where there are enough of them.
  const ROWS = Math.max(4, Math.min(64, ceil(V, 2048)));
  const z = { N, V, D, E, LANES: lanes, BITS, PASSES, TILE, TILES, SORT, CH, CHUNKS, ROWS };
  const types = {};
  let at = 0;
  const place = (name, bytes) => { z[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  place('COUNT', 256);
  place('HIST', one ? 0 : 4 * TILES * 2 ** BITS);
  for (const i of [0, 1]) {
    const used = i < PASSES;
    place(`KEYS${i}`, used ? 4 * N : 0);
    place(`PLACES${i}`, used ? 4 * N : 0);
  }
  place('PARTS', split ? 8 * CHUNKS * D : 0);
  const m = make(z, node.attrs.scale, types);
  const kernels = [];
  const ws = 'reinterpret_cast<char*>(A.ws)', lds = `uint32_t lds[${(1 + SORT / 64) * 2 ** BITS + SORT / 64}]`;
  if (one) kernels.push(m('embsort', [1, 1, 1], SORT, lds, `embed_sort_all<${S}>(A.in[0], ${ws}, lds)`));
  for (let p = 0; p < PASSES && !one; p++) {
    kernels.push(m('embcount', [TILES, 1, 1], SORT, `uint32_t lds[${2 ** BITS}]`, `embed_count<${S}, ${p}>(A.in[0], ${ws}, lds, blockIdx.x)`));
    kernels.push(m('embsort', [TILES, 1, 1], SORT, lds, `embed_sort<${S}, ${p}>(A.in[0], ${ws}, lds, blockIdx.x)`));
  }
  const last = (PASSES - 1) % 2, sums = ceil(CHUNKS, 256 / lanes) * columns, rows = ceil(V, ROWS);
  kernels.push(m('embsums', [sums + rows, 1, 1], 256, `uint32_t lds[${ROWS}]`, `embed_sums<${S}, ${last}>(A.in[1], A.out, reinterpret_cast<char*>(A.ws), lds, blockIdx.x)`));
  if (split) {
    kernels.push(m('embjoin', [CHUNKS, ceil(D, 64 * E), 1], 512, `float lds[${8 * 64 * E}]`, `embed_join<${S}, ${last}>(A.out, reinterpret_cast<char*>(A.ws), lds, blockIdx.x, blockIdx.y)`));
  }
  return { kind: 'embedding-grad', kernels, workspace: at };
}

module.exports = { lowerEmbedding, lowerEmbeddingGrad };
