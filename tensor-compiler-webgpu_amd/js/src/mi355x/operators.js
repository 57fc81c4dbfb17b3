'use strict';
// Launches of the operators that are one node each (ir/operators.js): the kernels of
// tcmi_rotary.h, tcmi_loss.h and tcmi_orthogonalize.h (embedding.js, residual.js and window.js: of the
// other operators'), their sizes written as constants of
// each text, and the workspace they share between the kernels of one launch.
//
// A gradient's parts (`dx`, `dgain`; `dh`, `dW`, `dbias`, and with them the losses) are nodes
// of their own and lower to launches of their own. The perf lowering runs the parts that
// it keeps as one launch (lower.js batchPlan): `joint` on a part's first kernel names the
// node's parts and forms the kernels of any set of them. Every part is computed by the same code in either form.

const { size } = require('../ir/shapes');
const { singularBound } = require('../ir/operators');
const { XCD_GROUPED, MAX_BATCH } = require('./codegen');
const { ceil, align, double, kernel, entry, joint } = require('./operator_parts');
const { lowerEmbedding, lowerEmbeddingGrad } = require('./embedding');
const { lowerResidual } = require('./residual');
const { lowerWindow } = require('./window');

const OPERATORS = new Set(['rotary', 'rotaryGrad', 'linearCrossEntropy', 'linearCrossEntropyGrad', 'orthogonalize', 'embedding', 'embeddingGrad',
  'residualNorm', 'residualNormGrad', 'windowAttention', 'windowAttentionGrad']);

// ---- rotary -------------------------------------------------------------------------------

const ROTARY_THREADS = 256;
const ROTARY_HEAD = 4096;       // floats of a head at most: 32 pairs a lane

function rotarySizes(graph, node) {
  const x = graph.nodes[node.inputs[0]].shape, pos = graph.nodes[node.inputs[1]].shape, a = node.attrs;
  const DH = x[x.length - 1], R = a.frequencies.length, T = x[a.axis];
  if (DH > ROTARY_HEAD) throw new Error(`rotary: heads of ${DH} floats (at most ${ROTARY_HEAD})`);
  const B = a.axis > 0 ? x[0] : 1, M1 = size(x.slice(1, Math.max(1, a.axis))), M2 = size(x.slice(a.axis + 1, -1));
  if (B * T >= 2 ** 31 || M1 * M2 >= 2 ** 31) throw new Error('rotary: tokens and heads are counted in 32 bits (at most 2^31 - 1)');
  const axes = a.positionAxes;
  const shared = size(pos) === T * axes && B > 1;
  // 128-bit loads where a group of four pairs (and of four floats that are not rotated) is whole and aligned.
  const E = DH % 4 === 0 && R % 4 === 0 ? 4 : 1;
  const groups = Math.max(R, DH - 2 * R) / E;
  let lanes = 1;
  while (lanes < 64 && lanes < groups) lanes *= 2;
  const slots = (() => { let s = 1; while (2 * s <= Math.min(M1 * M2, ROTARY_THREADS / lanes)) s *= 2; return s; })();
  return { DH, R, B, M1, T, M2, axes, shared, E, lanes, units: ceil(R / E, lanes), tails: ceil((DH - 2 * R) / E, lanes), slots };
}

function rotaryText(z, attrs, gain, grads, e) {
  const dx = grads.includes('dx'), dgain = grads.includes('dgain');
  const table = z.R ? `  static __device__ __forceinline__ double turns(int j) {
    static constexpr double t[${z.R}] = {${attrs.frequencies.map((f) => double(f / (2 * Math.PI))).join(', ')}};
    return t[j];
  }
  static __device__ __forceinline__ uint32_t axis(int j) {
    static constexpr unsigned char t[${z.R}] = {${attrs.axes.join(', ')}};
    return t[j];
  }` : `  static __device__ __forceinline__ double turns(int) { return 0.0; }
  static __device__ __forceinline__ uint32_t axis(int) { return 0u; }`;
  const last = gain ? 3 : 2;
  return `#include "tcmi_rotary.h"
struct __KERNEL___s {
  static constexpr int DH = ${z.DH}, R = ${z.R}, E = ${z.E}, LANES = ${z.lanes}, UNITS = ${z.units}, TAILS = ${z.tails}, THREADS = ${ROTARY_THREADS};
  static constexpr bool ADJ = ${attrs.pairs === 'adjacent'}, GAIN = ${gain}, DX = ${dx}, DGAIN = ${dgain}, SHARED = ${z.shared};
  static constexpr uint32_t B = ${z.B}u, M1 = ${z.M1}u, T = ${z.T}u, M2 = ${z.M2}u, AXES = ${z.axes}u, SLOTS = ${z.slots}u;
  static __device__ __forceinline__ float eps() { return static_cast<float>(${double(gain ? attrs.eps : 0)}); }
${table}
};
extern "C" __global__ void __launch_bounds__(${ROTARY_THREADS}) __KERNEL__(${e.sig}) {
${e.open}${dgain ? `  __shared__ __attribute__((aligned(16))) float scratch[${ROTARY_THREADS / z.lanes * z.DH}];\n` : ''}  tcmi::rotary<__KERNEL___s>(A.in[0], A.in[1], ${gain ? 'A.in[2]' : 'nullptr'}, ${grads.length ? `A.in[${last}]` : 'nullptr'}, ${
  dx || !grads.length ? e.out('dx') : 'nullptr'}, ${dgain ? `${e.ws}, scratch` : 'nullptr, nullptr'}, blockIdx.x, gridDim.x);
}
`;
}

function rotaryKernels(z, attrs, gain, grads, parts, groups) {
  // A few tokens to a workgroup. The gradient of the gain walks them in at most 1024 workgroups, whose sums are then added.
  const perBlock = ROTARY_THREADS / z.lanes / z.slots;
  const want = ceil(z.B * z.T, perBlock), dgain = grads.includes('dgain'), Z = groups || 1;
  const blocks = Math.min(want, dgain ? 1024 : 65536), floats = dgain ? align(blocks * z.DH, 64) : 0;
  const e = entry(parts, Z, floats);
  const kernels = [kernel('rot', rotaryText(z, attrs, gain, grads, e), [blocks, 1, Z], ROTARY_THREADS)];
  if (dgain) {
    kernels.push(kernel('rotsum', `#include "tcmi_rotary.h"
extern "C" __global__ void __launch_bounds__(1024) __KERNEL__(${e.sig}) {
${e.open}  __shared__ float scratch[1024];
  tcmi::rotary_gain_sum<${z.DH}>(${e.ws}, ${e.out('dgain')}, ${blocks}u, scratch, blockIdx.x);
}
`, [ceil(z.DH, 16), 1, Z], 1024));
  }
  return { kernels, workspace: 4 * floats * Z };
}

function lowerRotary(graph, node) {
  const grad = node.op === 'rotaryGrad';
  const gain = node.inputs.length - (grad ? 1 : 0) === 3;
  const z = rotarySizes(graph, node);
  const k = rotaryKernels(z, node.attrs, gain, grad ? [node.attrs.part] : [], null);
  if (grad && gain) {
    const { part, ...rest } = node.attrs;
    joint(k.kernels[0], part, ['dx', 'dgain'], ['rotary', rest, z], (parts, groups) => rotaryKernels(z, node.attrs, gain, parts, parts, groups), undefined, true);
  }
  return { kind: grad ? 'rotary-grad' : 'rotary', kernels: k.kernels, workspace: k.workspace };
}

// ---- linearCrossEntropy --------------------------------------------------------------------

// Bytes of a piece's logits at most (a piece is 128 rows or more): each piece reads W and adds to dW. 8192 rows of d 1024 against 65 536 classes
// 10.08 ms by 2^28, 9.53 by 2^29, 9.52 by 2^30.
const LOSS_PIECE = 2 ** 29;
// Rows at most: they are counted in 32 bits, and 16 of them take 256 threads of a grid of 2^32 at most.
const LOSS_ROWS = 2 ** 28;
const LOSS_PARTS = ['dh', 'dW', 'dbias', 'loss'];
const CUS = 256;
/**
 * Rows up to which W is read as it is (tcmi_loss_few.h): those its kernels are laid out for, four tiles of rows in registers, not where both
 * forms take as long. Without and with gradients, of d 1024, V 131072 (us): 16 rows 107 and 388, 64 rows 178 and 552, by products of
 * pairs 504 and 1019; the next row, by pairs, 484 and 962, and 128 rows 500 and 973: more tiles of rows would carry it to some 130 rows
 * without gradients, 100 with them.
 */
const FEW_ROWS = 64;
/**
 * Whether losses over V classes take whole rows (tcmi_loss_narrow.h), by time, with gradients and by products of pairs (us): 8192 rows of d 256
 * 29 and 42 (V 96), 35 and 42 (V 128); of d 1024 70 and 71, 85 and 72; 65 536 of d 512 226 and 287, 288 and 284. Without
 * gradients: 8 and 22, 10 and 22; 23 and 37, 28 and 37; 75 and 135, 99 and 134. Of few rows (64 of d 64, V 96) 5 and 14, where
 * few rows' own launches take 10 and 19. One workgroup walks a row's d.
 */
const fewClasses = (D, V) => D <= 65536 && (V <= 96 || (V <= 128 && D <= 512));
// tcmi_gemm_f16x2.h's tiles: rows, columns and threads of each kind.
const SMALL = 0, SQUARE = 1, WIDE = 2, TALL = 3;
const TILES = [[64, 64, 256], [128, 128, 256], [128, 256, 512], [256, 128, 512]];
/**
 * The time (us) of a product of `tiles` tiles of `slices` slices of 32 k, K in chunks of `each` slices. 64 x 64 tiles: a slice of one a CU 0.3, of a
 * full chip 0.275 a CU; larger ones (256 x 128, one a CU) 1.3. Starting and ending a tile: 3.4 and 6.
 */
function productTime(large, tiles, slices, each) {
  const all = tiles * ceil(slices, each), rounds = all / CUS;
  return large ? Math.max(1, rounds < 4 ? Math.ceil(rounds) : rounds) * (1.3 * each + 6) : 3.4 + each * Math.max(0.3, 0.275 * rounds);
}
/**
 * How K is split for the least time: { chunks, each, time }. Partial sums (of tiles of so many elements) are written and read by one more
 * launch, at 8 TB/s up to 32 MB, at 4 beyond.
 */
function splitK(large, tiles, slices, elements, least) {
  let best = null;
  for (let c = 1; c <= Math.min(64, Math.max(1, Math.floor(slices / least))); c++) {
    const each = ceil(slices, c), chunks = ceil(slices, each);
    const bytes = 8 * chunks * tiles * elements;
    const time = productTime(large, tiles, slices, each) + (chunks > 1 ? bytes / (bytes > 2 ** 25 ? 4e6 : 8e6) + 3.5 : 0);
    if (!best || time < best.time) best = { chunks, each, time };
  }
  return best;
}

/** A product's kernel keeps two wavefronts a SIMD, 256 registers each. */
const bounds = (threads, lds) => (/Tile/.test(lds || '') ? ', 2' : '');

// Columns of a matrix of pairs at most: an offset among 256 of its rows has 32 bits.
const PAIR_COLS = 2 ** 22;

/** The sizes of a loss's launch forming `parts`, and its workspace's layout. */
function lossSizes(N, D, V, bias, parts, piece) {
  const grad = parts.some((p) => p !== 'loss');
  // The large tiles are 128 x 256; padding of up to 256 columns and rows is little beside 2048 and 512.
  const VP = align(V, V > 2048 ? 256 : 128), rows = N > 512 ? 256 : 128;
  // The rows of a piece: its logits, or without gradients a row's pair of statistics for each 64 columns.
  const row = grad ? 4 * VP : VP / 8;
  // (At most 2^20 rows of logits: `spread` counts them by 32 in its grid's second extent.)
  const most = Math.max(rows, Math.min(grad ? 2 ** 20 : Infinity, Math.floor((piece || LOSS_PIECE) / row / rows) * rows));
  const PIECES = ceil(align(N, rows), most), NP = align(ceil(N, PIECES), rows);
  const RB = NP * VP >= 2 ** 20 ? 32 : 16;
  const clamp = (n, most) => Math.max(1, Math.min(Math.ceil(n), most));
  // Large tiles (1024 x 65536 of K 1024: 256 x 128 395 us, 128 x 256 426, 128 x 128 460) or 64 x 64, by time and by all rows: a
  // loss has the same bits whatever its pieces.
  const slices = ceil(D, 32), rowsAll = align(N, 256);
  const large = VP % 256 === 0 && rows === 256 && productTime(true, rowsAll / 256 * (VP / 128), slices, slices) < productTime(false, rowsAll / 64 * (VP / 64), slices, slices);
  const LT = large ? 4 : 2;
  // The gradients' tiles and the chunks of K by time.
  const g = gradTiles(NP, D, VP), DP = grad ? g.DP : align(D, 64);
  // Threads across columns: fewer, and rows side by side, where workgroups would be fewer than two a CU.
  const CT = (() => { let t = 16; while (2 * t <= Math.min(256, VP / 8) && ceil(VP, 16 * t) * NP / RB >= 2 * CUS) t *= 2; return t; })();
  const lanes = (() => { let n = 1; while (n < 64 && n < (D % 4 === 0 ? D / 4 : D)) n *= 2; return n; })();
  const z = { N, D, V, DP, VP, NP, PIECES, RB, CT, BIAS: bias, HLANES: lanes, HBLOCKS: clamp(N * lanes / 256, 1024), WBLOCKS: clamp(D * V / 16384, 1024),
    PER: clamp((NP * PIECES * DP + DP * VP) / 4 / 256 / 1024, 16), LKIND: large ? TALL : SMALL, HKIND: g.large ? TALL : SMALL, WKIND: g.large ? WIDE : SMALL, JOINED: !grad || VP / (16 * LT) > 32, VECD: D % 4 === 0, VECV: V % 4 === 0,
    HCHUNKS: g.h.chunks, HK: g.h.each, WCHUNKS: g.w.chunks, WK: g.w.each };
  let at = 0;
  const place = (name, bytes) => { z[name] = at; at = align(at + bytes, 256); };
  place('STATE', 256);
  place('MAXIMA', (z.HBLOCKS + z.WBLOCKS) * 4);
  place('EXPS', 4 * N);
  place('HP', 4 * NP * PIECES * DP);
  if (parts.includes('dW')) place('XP', 4 * NP * PIECES * DP); else z.XP = 0;
  place('WP', 4 * DP * VP);
  place('STATS', 8 * NP * (VP / (16 * LT)));
  place('PICKED', 4 * NP);
  place('ROWS', 8 * NP);
  if (grad) place('Z', 4 * NP * VP); else z.Z = 0;
  if (parts.includes('dh') || parts.includes('dW')) place('GP', 4 * NP * VP); else z.GP = 0;
  if (parts.includes('dbias')) place('SUMS', 4 * NP / RB * VP); else z.SUMS = 0;
  if (parts.includes('dh') && g.h.chunks > 1) place('HPART', 4 * g.h.chunks * NP * DP); else z.HPART = 0;
  if (parts.includes('dW') && g.w.chunks > 1) place('WPART', 4 * g.w.chunks * DP * VP); else z.WPART = 0;
  return { z, workspace: at, grad };
}

/**
 * The tiles of dh [NP, d] over V and of dW [d, V] over NP, and the chunks their K is split into: those of the least estimated time, by
 * the sizes alone, not by which gradients a launch forms. 1808 rows of d 907, 15 840 classes: 546 us by 64 x 64 tiles, 374 by 256 x 128.
 */
function gradTiles(NP, D, VP) {
  const of = (large) => {
    const [hr, hc, wr, wc] = large ? [256, 128, 128, 256] : [64, 64, 64, 64], DP = align(D, large ? 128 : 64);
    const h = splitK(large, NP / hr * (DP / hc), VP / 32, hr * hc, 4), w = splitK(large, DP / wr * (VP / wc), NP / 32, wr * wc, 4);
    return { large, DP, h, w, time: h.time + w.time };
  };
  const small = of(false);
  if (NP % 256 || VP % 256) return small;
  const large = of(true);
  return small.time < large.time ? small : large;
}

/** The sizes of a loss's launch over few rows (tcmi_loss_few.h), and its workspace's layout. */
function fewSizes(N, D, V, bias, parts) {
  const grad = parts.some((p) => p !== 'loss');
  const NP = align(N, 16), DP = align(D, 16), VP = align(V, 64), RT = NP / 16;
  // Enough workgroups for every CU: fewer columns of G, then fewer rows of W to each. LKIND: `join` finds a pair of
  // statistics for each 64 columns, as of the large tiles.
  const COLS = V >= 256 * CUS / 2 ? 256 : 64, CHUNKS = ceil(V, COLS), tiles = DP / 16;
  const z = { N, D, V, DP, VP, NP, RT, PIECES: 1, BIAS: bias, LKIND: TALL, WAVES: RT > 2 ? 4 : 8, COLS, CHUNKS,
    DTILES: Math.max(4, ceil(tiles, ceil(2 * CUS, CHUNKS))), VECD: D % 4 === 0, VECV: V % 4 === 0 };
  let at = 0;
  const place = (name, bytes) => { z[name] = at; at = align(at + bytes, 256); };
  place('STATS', 8 * NP * (VP / 64));
  place('PICKED', 4 * NP);
  place('ROWS', 8 * NP);
  if (grad) place('Z', 4 * NP * VP); else z.Z = 0;
  if (parts.includes('dh') && CHUNKS > 1) place('HPART', 4 * CHUNKS * NP * DP); else z.HPART = 0;
  return { z, workspace: at, grad };
}

function lossMaker(z, e, bias, grad) {
  const counts = /^([NDV]P?|NP|RT|PIECES|RB|CT|HLANES|[HW]BLOCKS|PER|[HW]CHUNKS|[HW]K|WAVES|COLS|CHUNKS|DTILES|CG|RC|DG)$/;
  const sizes = Object.keys(z).map((k) => (typeof z[k] === 'boolean' ? `  static constexpr bool ${k} = ${z[k]};`
    : k.endsWith('KIND') ? `  static constexpr int ${k} = ${z[k]};`
      : `  static constexpr ${counts.test(k) ? 'uint32_t' : 'size_t'} ${k} = ${z[k]}u;`)).join('\n');
  return (kind, grid, threads, lds, call) => kernel(kind, `#include "${/narrow_/.test(call) ? 'tcmi_loss_narrow.h' : /few_/.test(call) ? 'tcmi_loss_few.h' : 'tcmi_loss.h'}"
struct __KERNEL___s {
${sizes}
};
extern "C" __global__ void __launch_bounds__(${threads}${bounds(threads, lds)}) __KERNEL__(${e.sig}) {
${e.open}  const tcmi::Loss<__KERNEL___s> L{A.in[0], A.in[1], A.in[2], ${bias ? 'A.in[3]' : 'nullptr'}, ${grad ? `A.in[${bias ? 4 : 3}]` : 'nullptr'}, reinterpret_cast<char*>(A.ws)};
${lds ? `  __shared__ __attribute__((aligned(1024))) ${lds};\n` : ''}  tcmi::${call};
}
`, grid, threads);
}

function fewKernels(N, D, V, bias, parts, joined) {
  const { z, workspace, grad } = fewSizes(N, D, V, bias, parts);
  const e = entry(joined ? parts : null);
  const has = (p) => parts.includes(p);
  const make = lossMaker(z, e, bias, grad);
  const S = '__KERNEL___s';
  const outs = (...names) => names.map((p) => (has(p) ? e.out(p) : 'nullptr')).join(', ');
  const kernels = [make('losslogits', [z.VP / 64, 1, 1], 64 * z.WAVES, `float lds[${z.WAVES * z.NP} * tcmi::FEW_LD]`, `few_logits<${S}, ${grad}>(L, lds, blockIdx.x)`),
    make('lossjoin', [z.NP / 16, 1, 1], 1024, 'float2 scratch[1024]', `loss_join<${S}, ${has('loss')}, false>(L, ${outs('loss')}, scratch, blockIdx.x)`)];
  const [dh, dW, db] = ['dh', 'dW', 'dbias'].map(has);
  if (dh || dW || db) {
    kernels.push(make('lossgrads', [z.CHUNKS, dh || dW ? ceil(z.DP / 16, z.DTILES) : 1, 1], 256, `float lds[${z.NP * (z.COLS + 4)}]`,
      `few_grads<${S}, ${dh}, ${dW}, ${db}>(L, ${outs('dh', 'dW', 'dbias')}, lds, blockIdx.x, blockIdx.y)`));
    if (dh && z.CHUNKS > 1) {
      kernels.push(make('losssums', [ceil(z.NP * z.DP / 4, 32), 1, 1], 256, 'tcmi::f4 scratch[256]', `few_sums<${S}>(L, ${outs('dh')}, scratch, blockIdx.x)`));
    }
  }
  return { kernels, workspace };
}

/** The sizes of a loss's launch over few classes (tcmi_loss_narrow.h), and its workspace's layout. */
function narrowSizes(N, D, V, bias, parts) {
  const VP = align(V, 32), CG = VP / 32, DG = ceil(D, 64);
  // 16 rows a workgroup, 32 where that leaves enough of them: 8192 rows 29.3 us by 32, 30.9 by 16; 1001 rows of d 515 33.6 and 27.7.
  const RT = N >= 4096 ? 2 : 1;
  // A workgroup of dw a CU.
  const RC = align(ceil(N, Math.max(1, Math.min(ceil(N, 64), Math.floor(CUS / DG)))), 64), CHUNKS = ceil(N, RC);
  const z = { N, D, V, VP, NP: align(N, 16 * RT), RT, CG, RC, CHUNKS, DG, BIAS: bias, VECD: D % 4 === 0, VECV: V % 4 === 0 };
  const dw = parts.includes('dW'), db = parts.includes('dbias');
  let at = 0;
  const place = (name, bytes) => { z[name] = at; at = align(at + bytes, 256); };
  place('GP', dw || db ? 4 * z.NP * VP : 0);
  place('WPART', dw ? 4 * CHUNKS * D * VP : 0);
  place('SUMS', db ? 4 * CHUNKS * VP : 0);
  return { z, workspace: at };
}

function narrowKernels(N, D, V, bias, parts, joined) {
  const { z, workspace } = narrowSizes(N, D, V, bias, parts);
  const e = entry(joined ? parts : null);
  const has = (p) => parts.includes(p);
  const make = lossMaker(z, e, bias, parts.some((p) => p !== 'loss'));
  const S = '__KERNEL___s';
  const outs = (...names) => names.map((p) => (has(p) ? e.out(p) : 'nullptr')).join(', ');
  const [dh, dW, db] = ['dh', 'dW', 'dbias'].map(has);
  const kernels = [make('lossrows', [z.NP / (16 * z.RT), 1, 1], 256, `float lds[${64 * z.RT} * tcmi::narrow_ld<${S}>()]`,
    `narrow_rows<${S}, ${has('loss')}, ${dh}, ${dW || db}>(L, ${outs('loss', 'dh')}, lds, blockIdx.x)`)];
  if (dW || db) {
    kernels.push(make('lossdw', [z.CHUNKS, dW ? z.DG : 1, 1], 256, `float lds[${dW ? 4 * 64 * (z.VP + 4) : 4 * z.VP}]`,
      `narrow_dw<${S}, ${dW}, ${db}>(L, lds, blockIdx.x, blockIdx.y)`));
    kernels.push(make('losssums', [ceil((dW ? D * z.VP / 4 : 0) + (db ? z.VP / 4 : 0), 32), 1, 1], 256, 'tcmi::f4 scratch[256]',
      `narrow_sums<${S}, ${dW}, ${db}>(L, ${outs('dW', 'dbias')}, scratch, blockIdx.x)`));
  }
  return { kernels, workspace };
}

function lossKernels(N, D, V, bias, parts, joined, bytes) {
  if (fewClasses(D, V)) return narrowKernels(N, D, V, bias, parts, joined);
  if (N <= FEW_ROWS) return fewKernels(N, D, V, bias, parts, joined);
  const { z, workspace, grad } = lossSizes(N, D, V, bias, parts, bytes);
  if (Math.max(z.DP, z.VP) > PAIR_COLS) throw new Error(`linearCrossEntropy: ${Math.max(D, V)} columns (at most ${PAIR_COLS} for more than ${FEW_ROWS} rows)`);
  const e = entry(joined ? parts : null);
  const has = (p) => parts.includes(p);
  const make = lossMaker(z, e, bias, grad);
  const S = '__KERNEL___s';
  const [lr, lc, lt] = TILES[z.LKIND], [hr, hc, gt] = TILES[z.HKIND], [wr, wc] = TILES[z.WKIND];
  const outs = (...names) => names.map((p) => (has(p) ? e.out(p) : 'nullptr')).join(', ');
  const HG = z.NP * z.PIECES * z.DP / 4, WG = z.DP * z.VP / 4;
  const once = [make('lossmax', [z.HBLOCKS + z.WBLOCKS, 1, 1], 256, 'float scratch[4]', `loss_maxima<${S}, ${has('dW')}>(L, scratch, blockIdx.x)`),
    make('losssplit', [ceil(HG, 256 * z.PER) + ceil(WG, 256 * z.PER), 1, 1], 256, 'float scratch[4]', `loss_split<${S}, ${has('dW')}>(L, scratch, blockIdx.x)`)];
  const piece = [make('losslogits', [z.NP / lr * (z.VP / lc), 1, 1], lt, `char lds[tcmi::Tile<${z.LKIND}>::LDS]`, `loss_logits<${S}, ${grad}>(L, lds, blockIdx.x)`)];
  if (z.JOINED) {
    piece.push(make('lossjoin', [z.NP / 16, 1, 1], 1024, 'float2 scratch[1024]',
      `loss_join<${S}, ${has('loss')}, ${!grad}>(L, ${outs('loss')}, scratch, blockIdx.x)`));
  }
  if (grad) {
    const [dh, dW, db] = ['dh', 'dW', 'dbias'].map(has);
    piece.push(make('lossspread', [ceil(z.VP, 8 * z.CT), z.NP / z.RB, 1], 256, `tcmi::f4 rows[${z.RB + 512 + z.RB / 4}]`,
      `loss_spread<${S}, ${dh || dW}, ${db}, ${has('loss')}>(L, ${outs('loss')}, rows, blockIdx.x, blockIdx.y)`));
    const blocks = (dh ? z.NP / hr * (z.DP / hc) * z.HCHUNKS : 0) + (dW ? z.DP / wr * (z.VP / wc) * z.WCHUNKS : 0) + (db ? z.VP / 16 : 0);
    piece.push(make('lossgrads', [blocks, 1, 1], gt, `char lds[tcmi::GradTiles<${S}>::LDS]`, `loss_grads<${S}, ${dh}, ${dW}, ${db}>(L, ${outs('dh', 'dW', 'dbias')}, lds, blockIdx.x)`));
    const sh = dh && z.HCHUNKS > 1, sw = dW && z.WCHUNKS > 1;
    if (sh || sw) {
      piece.push(make('losssums', [(sh ? ceil(z.NP * z.DP / 4, 256) : 0) + (sw ? ceil(z.D * z.VP / 4, 256) : 0), 1, 1], 256, null,
        `loss_sums<${S}, ${sh}, ${sw}>(L, ${outs('dh', 'dW')}, blockIdx.x)`));
    }
  }
  const kernels = once.slice();
  for (let p = 0; p < z.PIECES; p++) kernels.push(...piece);
  return { kernels, workspace };
}

function lowerLoss(graph, node, tuning) {
  const { piece } = (tuning || {}).loss || {};
  const grad = node.op === 'linearCrossEntropyGrad';
  const [N, D] = graph.nodes[node.inputs[0]].shape, V = graph.nodes[node.inputs[1]].shape[1];
  if (N > LOSS_ROWS) throw new Error(`linearCrossEntropy: ${N} rows (at most ${LOSS_ROWS})`);
  const operands = node.inputs.length - (grad ? 1 : 0);
  const bias = operands === 4;
  const part = grad ? node.attrs.part : 'loss';
  const k = lossKernels(N, D, V, bias, [part], false, piece);
  joint(k.kernels[0], part, LOSS_PARTS, ['loss', N, D, V, bias], (parts) => lossKernels(N, D, V, bias, parts, true, piece), operands);
  return { kind: grad ? 'linear-cross-entropy-grad' : 'linear-cross-entropy', kernels: k.kernels, workspace: k.workspace,
    flops: part === 'dbias' ? 0 : 2 * N * D * V };
}

// ---- orthogonalize -------------------------------------------------------------------------

/**
 * Which of a symmetric product's tiles are split along K, of each of `count` matrices: by 128 x 128 tiles those left over when the rest fill the
 * chip (two workgroups a CU) a whole number of times, into as many chunks of 8 slices or more as fill it once more; by 64 x 64 tiles all or none,
 * by time (25 tiles of 114 slices: 38 us whole, 11 in chunks with their sums).
 */
function splitTiles(kind, tiles, slices, count) {
  const none = { split: 0, chunks: 1, each: slices };
  if (kind === SMALL) {
    const s = splitK(false, tiles * count, slices, 64 * 64, 4);
    return s.chunks > 1 ? { split: tiles, chunks: s.chunks, each: s.each, time: s.time } : Object.assign(none, { time: s.time });
  }
  const split = Math.floor(tiles * count % (2 * CUS) / count), chunks = split ? Math.min(Math.floor(2 * CUS / (split * count)), Math.floor(slices / 8)) : 1;
  if (chunks < 2) return none;
  const each = ceil(slices, chunks);
  return { split, chunks: ceil(slices, each), each };
}

/** The largest exponent that keeps values up to `top` within half's range. */
const fits = (top) => Math.floor(Math.log2(60000 / top));

/**
 * The side up to which all steps are made on one small matrix in float64 (tcmi_orthogonalize_thin.h), what its LDS holds; by time, and by
 * products of pairs (us, 5 steps): 8 x 8 10.9 and 51.5, 16 of 32 x 2416 24 and 144, 64 x 64 47 and 56, 64 x 4096 54 and 160, 16 of
 * 64 x 1024 55 and 97.
 */
const THIN_SIDE = 64;

/** Matrices with a side of at most THIN_SIDE. */
function thinKernels(node, M, N, count) {
  const { steps, eps, coefficients: [a, b, c] } = node.attrs;
  const s = Math.min(M, N), l = Math.max(M, N), T = s <= 16 ? 1 : s <= 32 ? 2 : 4, SP = 16 * T, entries = T * (T + 1) / 2 * 256;
  // A wavefront takes 16 of the long side at a time; 32 chunks are enough of them for any length that stays small beside a launch.
  const KC = align(ceil(l, 32), 64), CHUNKS = ceil(l, KC), summed = CHUNKS > 4;
  const z = { M, N, T, KC, CHUNKS, STEPS: steps, TALL: M > N, VEC: N % 4 === 0, SUMMED: summed };
  let at = 0;
  const put = (name, bytes) => { z[name] = at; at = align(at + bytes, 256); };
  put('PART', 8 * CHUNKS * entries);
  put('SUM', 8 * entries);
  put('Q', 8 * SP * SP);
  z.PER = at;
  const sizes = Object.keys(z).map((k) => (typeof z[k] === 'boolean' ? `  static constexpr bool ${k} = ${z[k]};`
    : k === 'T' ? `  static constexpr int T = ${T};` : `  static constexpr ${/^(PART|SUM|Q|PER)$/.test(k) ? 'size_t' : 'uint32_t'} ${k} = ${z[k]}u;`)).join('\n');
  const S = '__KERNEL___s';
  const make = (kind, blocks, threads, lds, call) => kernel(kind, `#include "tcmi_orthogonalize_thin.h"
struct __KERNEL___s {
${sizes}
  static __device__ __forceinline__ double a() { return ${double(a)}; }
  static __device__ __forceinline__ double b() { return ${double(b)}; }
  static __device__ __forceinline__ double c() { return ${double(c)}; }
  static __device__ __forceinline__ double eps() { return ${double(eps)}; }
};
extern "C" __global__ void __launch_bounds__(${threads}) __KERNEL__(const TcmiArgs A) {
  const tcmi::Thin<__KERNEL___s> o(A.in[0], A.out, A.ws, blockIdx.z);
${lds ? `  __shared__ __attribute__((aligned(1024))) double lds[${lds}];\n` : ''}  tcmi::${call};
}
`, [blocks, 1, count], threads);
  const kernels = [make('orththingram', CHUNKS, 256, 4 * entries, `thin_gram<${S}>(o, lds, blockIdx.x)`)];
  if (summed) kernels.push(make('orththinsum', entries / 32, 256, 256, `thin_sum<${S}>(o, lds, blockIdx.x)`));
  kernels.push(make('orththiniterate', 1, 512, 4 * SP * (SP + 2), `thin_iterate<${S}>(o, lds)`));
  kernels.push(make('orththinapply', M > N ? ceil(M, 64) : ceil(ceil(N, 64) * T, 4), 256, null, `thin_apply<${S}>(o, blockIdx.x)`));
  return { kind: 'orthogonalize', kernels, workspace: count * z.PER, flops: count * steps * (3 * s * s * l + s ** 3) };
}

/** How many other nodes are equal to `node` (op, shape, attributes) and neither depend on it nor it on them. */
function equalBeside(graph, node) {
  const same = (n) => n !== node && n.op === node.op && n.shape.join() === node.shape.join() && JSON.stringify(n.attrs) === JSON.stringify(node.attrs);
  if (!graph.nodes.some(same)) return 0;
  const before = new Set([node.id]), after = new Set([node.id]);
  for (let id = node.id; id >= 0; id--) if (before.has(id)) for (const i of graph.nodes[id].inputs) before.add(i);
  for (const n of graph.nodes) if (n.inputs.some((i) => after.has(i))) after.add(n.id);
  return graph.nodes.filter((n) => same(n) && !before.has(n.id) && !after.has(n.id)).length;
}

function lowerOrthogonalize(graph, node) {
  const x = node.shape, M = x[x.length - 2], N = x[x.length - 1], count = size(x.slice(0, -2));
  const { steps, eps, coefficients: [a, b, c] } = node.attrs;
  if (count > 65535) throw new Error(`orthogonalize: ${count} matrices (at most 65535)`);
  if (Math.max(M, N) > PAIR_COLS) throw new Error(`orthogonalize: a matrix of ${M} x ${N} (at most ${PAIR_COLS} on a side)`);
  const tall = M > N, s = Math.min(M, N), l = Math.max(M, N);
  if (s <= THIN_SIDE && steps > 0) return thinKernels(node, M, N, count);
  // Tiles of 128, or of 64 where those leave much of the chip idle, counting the equal nodes that run side by side with it.
  const alike = count * Math.min(1 + equalBeside(graph, node), MAX_BATCH);
  const square = ceil(s, 128) * ceil(l, 128) * alike >= 2 * CUS;
  const pad = square ? 128 : 64, MP = align(M, pad), NP = align(N, pad), SP = Math.min(MP, NP);
  const n = SP / pad, kind = square ? SQUARE : SMALL, upper = n * (n + 1) / 2;
  const AKIND = square && MP % 256 === 0 ? TALL : square && NP % 256 === 0 ? WIDE : kind;
  const ablocks = MP / TILES[AKIND][0] * (NP / TILES[AKIND][1]);
  const splits = (t) => [splitTiles(kind, t, ceil(l, 32), alike), splitTiles(kind, t, ceil(s, 32), alike)];
  // All tiles where that costs no time (a mirrored tile's scattered writes take 1.5 us).
  const time = (t) => splits(t).reduce((q, x) => q + x.time, 0);
  const half = square || time(upper) + 3 < time(n * n), tilesOf = half ? upper : n * n;
  const [G, B] = splits(tilesOf);
  const top = singularBound(node.attrs);
  const z = { M, N, MP, NP, SP, KIND: kind, AKIND, HALF: half, TALL: tall, VEC: N % 4 === 0, BLOCKS: Math.min(256, ceil(M * N, 4096)),
    GSPLIT: G.split, GCHUNKS: G.chunks, GEACH: G.each, BSPLIT: B.split, BCHUNKS: B.chunks, BEACH: B.each,
    SX: fits(top), SA: fits(top ** 2), SB: Math.max(-60, Math.min(60, fits(Math.max(Math.abs(b) * top ** 2 + Math.abs(c) * top ** 4, 2 ** -40)))) };
  let at = 0;
  const put = (name, bytes) => { z[name] = at; at = align(at + bytes, 256); };
  put('NORM', 8 * z.BLOCKS);
  put('X0', steps > 0 ? 4 * MP * NP : 0);
  put('X1', steps > 1 ? 4 * MP * NP : 0);
  put('A', steps > 0 ? 4 * SP * SP : 0);
  put('B', steps > 0 ? 4 * SP * SP : 0);
  put('PART', steps > 0 ? 4 * pad * pad * Math.max(G.split * G.chunks, B.split * B.chunks) : 0);
  z.PER = at;
  const sizes = Object.keys(z).map((k) => (typeof z[k] === 'boolean' ? `  static constexpr bool ${k} = ${z[k]};`
    : ['KIND', 'AKIND', 'SX', 'SA', 'SB'].includes(k) ? `  static constexpr int ${k} = ${z[k]};`
      : `  static constexpr ${/^([MNS]P?|BLOCKS|[GB](SPLIT|CHUNKS|EACH))$/.test(k) ? 'uint32_t' : 'size_t'} ${k} = ${z[k]}u;`)).join('\n');
  const S = '__KERNEL___s', place = square ? 'blockIdx' : 'wg';
  const make = (kind, blocks, threads, lds, call) => kernel(kind, `#include "tcmi_orthogonalize.h"
struct __KERNEL___s {
${sizes}
  static __device__ __forceinline__ float a() { return static_cast<float>(${double(a)}); }
  static __device__ __forceinline__ float b() { return static_cast<float>(${double(b)}); }
  static __device__ __forceinline__ float c() { return static_cast<float>(${double(c)}); }
  static __device__ __forceinline__ double eps() { return ${double(eps)}; }
};
extern "C" __global__ void __launch_bounds__(${threads}${bounds(threads, lds)}) __KERNEL__(const TcmiArgs A) {
${square ? '' : `  ${XCD_GROUPED}\n`}  const tcmi::Orth<__KERNEL___s> o(A.in[0], A.out, A.ws, ${place}.z);
${lds ? `  __shared__ __attribute__((aligned(1024))) ${lds};\n` : ''}  tcmi::${call};
}
`, [blocks, 1, count], threads);
  const pool = (k) => `char lds[tcmi::Tile<${k}>::LDS]`;
  const kernels = [make('orthnorm', z.BLOCKS, 256, 'double scratch[4]', `orth_norm<${S}>(o, scratch, ${place}.x)`),
    make('orthsplit', ceil(MP * NP, 4096), 256, 'double scratch[4]', `orth_split<${S}, ${steps === 0}>(o, scratch, ${place}.x)`)];
  for (let k = 0; k < steps; k++) {
    for (const [poly, t] of [[false, G], [true, B]]) {
      const from = poly ? 0 : k % 2, name = poly ? 'poly' : 'gram';
      kernels.push(make(`orth${name}`, tilesOf + t.split * (t.chunks - 1), TILES[kind][2], pool(kind), `orth_symmetric<${S}, ${poly}, ${from}>(o, lds, ${place}.x)`));
      if (t.split) kernels.push(make(`orthjoin${name}`, t.split * (square ? 4 : 2), TILES[kind][2], null, `orth_join<${S}, ${poly}>(o, ${place}.x)`));
    }
    kernels.push(make('orthapply', ablocks, TILES[AKIND][2], pool(AKIND), `orth_apply<${S}, ${k % 2}, ${k === steps - 1}>(o, lds, ${place}.x)`));
  }
  return { kind: 'orthogonalize', kernels, workspace: count * z.PER, flops: count * steps * (3 * s * s * l + s ** 3) };
}

/** The launch of an operator's node: { kind, kernels, params, workspace, flops }. tuning.loss.piece: bytes of a piece's logits. */
function lowerOperator(graph, node, tuning) {
  let k;
  if (node.op === 'rotary' || node.op === 'rotaryGrad') k = lowerRotary(graph, node);
  else if (node.op === 'linearCrossEntropy' || node.op === 'linearCrossEntropyGrad') k = lowerLoss(graph, node, tuning);
  else if (node.op === 'orthogonalize') k = lowerOrthogonalize(graph, node);
  else if (node.op === 'embedding') k = lowerEmbedding(graph, node);
  else if (node.op === 'embeddingGrad') k = lowerEmbeddingGrad(graph, node);
  else if (node.op === 'residualNorm' || node.op === 'residualNormGrad') k = lowerResidual(graph, node);
  else if (node.op === 'windowAttention' || node.op === 'windowAttentionGrad') k = lowerWindow(graph, node);
  else throw new Error(`no MI355X lowering for '${node.op}'`);
  return Object.assign({ params: new Uint32Array(0), flops: 0 }, k);
}

module.exports = { OPERATORS, lowerOperator };
