'use strict';
// Launches of windowAttention and its gradient (tcmi_window.h).

const { ceil, align, double, constants, kernel, entry, joint } = require('./operator_parts');

const MOST_HEAD = 256;          // floats of a head at most
const CUS = 256;
const S = '__KERNEL___s';

function windowSizes(graph, node) {
  const [B, T, H, DH] = graph.nodes[node.inputs[0]].shape, [, KEYS, HK] = graph.nodes[node.inputs[1]].shape, a = node.attrs;
  const grad = node.op === 'windowAttentionGrad';
  if (DH > MOST_HEAD) throw new Error(`windowAttention: heads of ${DH} floats (at most ${MOST_HEAD})`);
  if (T * H >= 2 ** 31 || KEYS * HK >= 2 ** 31) throw new Error('windowAttention: a sequence\'s rows are counted in 32 bits (at most 2^31 - 1)');
  const lengths = node.inputs.length - (grad ? 3 : 0) === 4;
  return { z: { B, T, H, DH, KEYS, HK, WINDOW: a.window, SINKS: a.sinks, LAST: a.queries === 'last', LENGTHS: lengths, VEC: DH % 4 === 0 }, scale: a.scale, lengths, grad };
}

function maker(s, e, types) {
  return (kind, grid, threads, lds, call, more) => kernel(kind, `#include "tcmi_window.h"
struct ${S} {
${constants(Object.assign({}, s.z, more || {}), types)}
  static __device__ __forceinline__ double scale() { return ${double(s.scale)}; }
};
extern "C" __global__ void __launch_bounds__(${threads}) __KERNEL__(${e.sig}) {
${e.open}${lds ? `  __shared__ __attribute__((aligned(16))) ${lds};\n` : ''}  tcmi::${call};
}
`, grid, threads);
}

/** Workgroups of `rows` x `heads`, along the first axis of a grid. */
function grid(n) {
  if (n >= 2 ** 24) throw new Error(`windowAttention: ${n} workgroups (at most 2^24)`);
  return [n, 1, 1];
}

function forwardKernels(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null);
  const R = z.H / z.HK, TILES = ceil(z.T * R, 16), heads = z.B * z.HK;
  // The keys that one tile sees at most, in tiles of 16, dealt to as many workgroups as fill the chip four times, eight tiles each or more.
  const most = ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW + ceil(16, R) + 32 + z.SINKS) : z.KEYS, 16);
  const SPLITS = Math.max(1, Math.min(256, Math.floor(most / 8), ceil(4 * CUS, TILES * heads)));
  const types = { SUMS: 'size_t' };
  let at = 0;
  const more = { TILES, SPLITS };
  const place = (name, bytes) => { more[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  place('OUT', SPLITS > 1 ? 4 * SPLITS * heads * TILES * 16 * z.DH : 0);
  place('STATS', SPLITS > 1 ? 8 * SPLITS * heads * TILES * 16 : 0);
  const m = maker(s, e, types);
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', ws = `reinterpret_cast<char*>(${e.ws})`;
  const kernels = [m('win', grid(TILES * heads * SPLITS), 256, `float lds[tcmi::window_lds<${z.DH}>()]`,
    `window_rows<${S}>(A.in[0], A.in[1], A.in[2], ${L}, ${out('o')}, ${out('lse')}, ${ws}, lds, blockIdx.x)`, more)];
  if (SPLITS > 1) {
    kernels.push(m('winjoin', grid(ceil(heads * TILES * 16, 4)), 256, null, `window_join<${S}>(${out('o')}, ${out('lse')}, ${ws}, blockIdx.x * 4u + threadIdx.x / 64u)`, more));
  }
  return { kernels, workspace: at };
}

function backwardKernels(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null);
  const R = z.H / z.HK, TILES = ceil(z.T * R, 16), heads = z.B * z.HK, KTILES = ceil(z.KEYS, 16);
  const m = maker(s, e, {});
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', at = s.lengths ? 4 : 3;
  const operands = `A.in[0], A.in[1], A.in[2], ${L}, A.in[${at}], A.in[${at + 1}], A.in[${at + 2}]`;
  const dk = parts.includes('dk'), dv = parts.includes('dv');
  const kernels = [];
  if (dk || parts.includes('dq')) kernels.push(m('winmass', grid(ceil(z.B * z.T * z.H, 16)), 256, null, `window_mass<${S}>(A.in[${at}], A.in[${at + 2}], ${e.ws}, blockIdx.x * 16u + threadIdx.x / 16u)`));
  if (parts.includes('dq')) {
    kernels.push(m('windq', grid(TILES * heads), 256, `float lds[tcmi::window_lds<${z.DH}>()]`,
      `window_dq<${S}>({${operands}, ${e.ws}}, ${out('dq')}, lds, blockIdx.x)`, { TILES }));
  }
  if (dk || dv) {
    kernels.push(m('windkv', grid(KTILES * heads), 256, `float lds[tcmi::window_lds<${z.DH}>()]`,
      `window_dkv<${S}, ${dk}, ${dv}>({${operands}, ${e.ws}}, ${out('dk')}, ${out('dv')}, lds, blockIdx.x)`, { KTILES }));
  }
  return { kernels, workspace: align(4 * z.B * z.T * z.H, 256) };
}

/** Products of one head's pairs of a query and a key that it sees, were its sequence full: the flops of one product. */
function seen(z) {
  const first = z.LAST ? z.KEYS - z.T : 0;
  let pairs = 0;
  for (let t = 0; t < z.T; t++) {
    const at = first + t;
    if (at < 0 || at >= z.KEYS) continue;
    const from = z.WINDOW ? Math.max(0, at - z.WINDOW + 1) : 0;
    pairs += at + 1 - from + Math.min(from, z.SINKS);
  }
  return 2 * z.B * z.H * z.DH * pairs;
}

function lowerWindow(graph, node) {
  const s = windowSizes(graph, node), { part, ...rest } = node.attrs;
  const build = s.grad ? backwardKernels : forwardKernels;
  const k = build(s, [part], false);
  joint(k.kernels[0], part, s.grad ? ['dq', 'dk', 'dv'] : ['o', 'lse'], [node.op, rest, s.z], (parts) => build(s, parts, true));
  return { kind: s.grad ? 'window-attention-grad' : 'window-attention', kernels: k.kernels, workspace: k.workspace,
    flops: seen(s.z) * { o: 2, lse: 1, dq: 1, dk: 1, dv: 1 }[part] };
}

module.exports = { lowerWindow };
