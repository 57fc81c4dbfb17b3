'use strict';
// Launches of residualNorm and its gradient (tcmi_residual.h).

const { size } = require('../ir/shapes');
const { ceil, align, double, constants, kernel, entry, joint } = require('./operator_parts');

const MOST_ROW = 16384;         // floats of a row at most: 1024 threads of 16
const FORWARD = ['h', 'n'], BACKWARD = ['dx', 'dy', 'dgain', 'dbias', 'dpostGain', 'dpostBias', 'dgate'];
const GATE = { none: 0, vector: 1, full: 2 };

function residualSizes(graph, node) {
  const x = graph.nodes[node.inputs[0]].shape, D = x[x.length - 1], N = size(x) / D, a = node.attrs;
  if (D > MOST_ROW) throw new Error(`residualNorm: rows of ${D} floats (at most ${MOST_ROW})`);
  if (N >= 2 ** 31) throw new Error(`residualNorm: ${N} rows (at most 2^31 - 1)`);
  const grad = node.op === 'residualNormGrad';
  const names = ['x', 'y', a.pre && 'gain', a.bias && !grad && 'bias', a.post && 'postGain', a.postBias && 'postBias', a.gate && 'gate'].filter(Boolean).concat(grad ? a.has : []);
  const gated = names.indexOf('gate');
  const full = gated >= 0 && size(graph.nodes[node.inputs[gated]].shape) !== D;
  // Lanes of a row, a power of two, with at most 16 floats each.
  let lanes = 16;
  while (lanes * 16 < D) lanes *= 2;
  const threads = Math.max(256, lanes), units = ceil(D, lanes * 4);
  return { z: { N, D, LANES: lanes, UNITS: units, THREADS: threads, LAYER: a.norm === 'layer', POST: a.post, GATE: gated < 0 ? GATE.none : full ? GATE.full : GATE.vector },
    names, grad };
}

function residualKernels(node, sizes, parts, joined) {
  const { z, names, grad } = sizes, a = node.attrs;
  const e = entry(joined ? parts : null);
  const rows = z.THREADS / z.LANES;
  // The gradients of vectors: sums of each workgroup's rows, added by a second launch.
  const sums = ['dgain', 'dbias', 'dpostGain', 'dpostBias'].concat(z.GATE === GATE.vector ? ['dgate'] : []).filter((p) => parts.includes(p));
  // (8189 rows of 4095, forward and back: by 256 workgroups 300 us, 512 268, 1024 283; 8192 of 256 19.2, 17.9 and 17.9; 4096 of 1024 35.8, 36.8 and 39.2.)
  const blocks = Math.min(ceil(z.N, rows), sums.length ? 512 : 65536);
  const floats = blocks * sums.length * z.D;
  const at = (name) => (names.includes(name) ? `A.in[${names.indexOf(name)}]` : 'nullptr');
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const text = (includes, call, threads, lds) => `#include "tcmi_residual.h"
struct __KERNEL___s {
${constants(Object.assign({}, z, includes), { GATE: 'int', UNITS: 'int', SUMS: 'int' })}
  static __device__ __forceinline__ float eps() { return static_cast<float>(${double(a.eps)}); }
  static __device__ __forceinline__ float residual() { return static_cast<float>(${double(a.residual)}); }
};
extern "C" __global__ void __launch_bounds__(${threads}) __KERNEL__(${e.sig}) {
${e.open}  __shared__ __attribute__((aligned(16))) float lds[${lds}];
  const tcmi::ResidualArgs R{${['x', 'y', 'gain', 'bias', 'postGain', 'postBias', 'gate', 'dh', 'dn'].map(at).join(', ')}};
  tcmi::${call};
}
`;
  if (!grad) {
    const k = kernel('res', text({ H: parts.includes('h'), NORM: parts.includes('n'), STAGED: false }, `residual<__KERNEL___s>(R, ${out('h')}, ${out('n')}, lds, blockIdx.x, gridDim.x)`, z.THREADS, z.THREADS / 64), [blocks, 1, 1], z.THREADS);
    return { kernels: [k], workspace: 0 };
  }
  const has = (p) => parts.includes(p);
  const flags = { DX: has('dx'), DY: has('dy'), DGAIN: has('dgain'), DBIAS: has('dbias'), DPOSTGAIN: has('dpostGain'), DPOSTBIAS: has('dpostBias'), DGATE: has('dgate'),
    DH: a.has.includes('dh'), DN: a.has.includes('dn'), SUMS: sums.length };
  // Vectors in LDS where four of them, for two workgroups a CU, fit.
  const pad = z.UNITS * 4 * z.LANES, STAGED = pad <= 4096, SCRATCH = align(Math.max(z.THREADS / 64, sums.length && rows > 1 ? z.THREADS / z.LANES * z.D : 0), 4);
  Object.assign(flags, { STAGED, SCRATCH });
  const lds = SCRATCH + (STAGED ? 4 * pad : 0);
  const kernels = [kernel('resgrad', text(flags, `residual_grad<__KERNEL___s>(R, ${out('dx')}, ${out('dy')}, ${out('dgate')}, ${e.ws}, lds, blockIdx.x, gridDim.x)`, z.THREADS, lds), [blocks, 1, 1], z.THREADS)];
  if (sums.length) {
    kernels.push(kernel('ressum', `#include "tcmi_residual.h"
extern "C" __global__ void __launch_bounds__(1024) __KERNEL__(${e.sig}) {
${e.open}  __shared__ float scratch[1024];
  float* const out[] = {${sums.map(e.out).join(', ')}};
  tcmi::residual_sum<${z.D}>(${e.ws}, out[blockIdx.y], ${blocks}u, scratch, blockIdx.x, blockIdx.y);
}
`, [ceil(z.D, 32), sums.length, 1], 1024));
  }
  return { kernels, workspace: align(4 * floats, 256) };
}

function lowerResidual(graph, node) {
  const sizes = residualSizes(graph, node);
  const { part, ...rest } = node.attrs;
  const k = residualKernels(node, sizes, [part], false);
  joint(k.kernels[0], part, sizes.grad ? BACKWARD : FORWARD, [node.op, rest, sizes.z], (parts) => residualKernels(node, sizes, parts, true));
  return { kind: sizes.grad ? 'residual-norm-grad' : 'residual-norm', kernels: k.kernels, workspace: k.workspace };
}

module.exports = { lowerResidual };
