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
  return (kind, grid, threads, lds, call, more) => kernel(kind, `#include "${/_wide/.test(call) ? 'tcmi_window_wide.h' : 'tcmi_window.h'}"
struct ${S} {
${constants(Object.assign({}, s.z, more || {}), types)}
  static __device__ __forceinline__ double scale() { return ${double(s.scale)}; }
};
extern "C" __global__ void __launch_bounds__(${threads}${/_wide(_dq|_dkv)?</.test(call) && s.z.DH <= 128 ? ', 2' : ''}) __KERNEL__(${e.sig}) {
${e.open}${lds ? `  __shared__ __attribute__((aligned(16))) ${lds};\n` : ''}  tcmi::${call};
}
`, grid, threads);
}

/** Workgroups of `rows` x `heads`, along the first axis of a grid. */
function grid(n) {
  if (n >= 2 ** 24) throw new Error(`windowAttention: ${n} workgroups (at most 2^24)`);
  return [n, 1, 1];
}

/** Rows of a key head from which 128 of them are a workgroup's (tcmi_window_wide.h). */
const WIDE_ROWS = 64;

/**
 * Workgroups that a chip's worth is: two a CU run at once, and as many wait, so that those that see many keys leave no CU idle
 * at the end.
 */
const FILL = 4 * CUS;

/** Splits of the tiles of NB keys that `rows` rows of one head see, of `blocks` workgroups otherwise: eight tiles each or more. */
function keySplits(z, rows, NB, blocks) {
  const R = z.H / z.HK;
  const most = ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW + ceil(rows, R) + z.SINKS) : z.KEYS, NB);
  return Math.max(1, Math.min(64, Math.floor(most / 8), ceil(FILL, blocks)));
}

function wideForward(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null), heads = z.B * z.HK, R = z.H / z.HK;
  const rows = z.DH <= 128 ? 128 : 64, tiles = ceil(z.T * R, rows), SPLITS = keySplits(z, rows, z.DH <= 64 ? 64 : 32, tiles * heads);
  const more = { TILES: ceil(z.T * R, 16), SPLITS }, types = {};
  let at = 0;
  const place = (name, bytes) => { more[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  place('OUT', SPLITS > 1 ? 4 * SPLITS * heads * more.TILES * 16 * z.DH : 0);
  place('STATS', SPLITS > 1 ? 8 * SPLITS * heads * more.TILES * 16 : 0);
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', ws = `reinterpret_cast<char*>(${e.ws})`, m = maker(s, e, types);
  // The last rows, which see most, first; a head's on one XCD, whose L2 its keys share, where heads are a multiple of eight.
  const kernels = [m('winwide', grid(tiles * heads * SPLITS), 256, `char lds[tcmi::WindowWide<${S}>::LDS]`,
    `window_wide<${S}>(A.in[0], A.in[1], A.in[2], ${L}, ${out('o')}, ${out('lse')}, ${ws}, lds, blockIdx.x % ${heads}u, ${tiles - 1}u - blockIdx.x / ${heads * SPLITS}u, blockIdx.x / ${heads}u % ${SPLITS}u)`, more)];
  if (SPLITS > 1) kernels.push(joinKernel(m, z, out, ws, more, heads));
  return { kernels, workspace: at };
}

/** The launch that joins the splits of rows. */
function joinKernel(m, z, out, ws, more, heads) {
  return m('winjoin', grid(ceil(heads * more.TILES * 16, 4)), 256, null, `window_join<${S}>(${out('o')}, ${out('lse')}, ${ws}, blockIdx.x * 4u + threadIdx.x / 64u)`, more);
}

function forwardKernels(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null);
  if (z.T * (z.H / z.HK) >= WIDE_ROWS) return wideForward(s, parts, joined);
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
  if (SPLITS > 1) kernels.push(joinKernel(m, z, out, ws, more, heads));
  return { kernels, workspace: at };
}

function backwardKernels(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null);
  const R = z.H / z.HK, heads = z.B * z.HK, wide = z.T * R >= WIDE_ROWS;
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', first = s.lengths ? 4 : 3;
  const args = `{A.in[0], A.in[1], A.in[2], ${L}, A.in[${first}], A.in[${first + 1}], A.in[${first + 2}], ${e.ws}}`;
  const dq = parts.includes('dq'), dk = parts.includes('dk'), dv = parts.includes('dv');
  const types = {}, more = {};
  let at = align(4 * z.B * z.T * z.H, 256);
  const place = (name, bytes) => { more[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  const m = maker(s, e, types), ws = `reinterpret_cast<char*>(${e.ws})`;
  const kernels = [];
  if (dk || dq) kernels.push(m('winmass', grid(ceil(z.B * z.T * z.H, 16)), 256, null, `window_mass<${S}>(A.in[${first}], A.in[${first + 2}], ${e.ws}, blockIdx.x * 16u + threadIdx.x / 16u)`));
  if (!wide) {
    const TILES = ceil(z.T * R, 16), KTILES = ceil(z.KEYS, 16), lds = `float lds[tcmi::window_lds<${z.DH}>()]`;
    if (dq) kernels.push(m('windq', grid(TILES * heads), 256, lds, `window_dq<${S}>(${args}, ${out('dq')}, lds, blockIdx.x)`, { TILES }));
    if (dk || dv) kernels.push(m('windkv', grid(KTILES * heads), 256, lds, `window_dkv<${S}, ${dk}, ${dv}>(${args}, ${out('dk')}, ${out('dv')}, lds, blockIdx.x)`, { KTILES }));
    return { kernels, workspace: at };
  }
  const rows = z.DH <= 64 ? 128 : 64, lds = `char lds[tcmi::WindowBack<${S}>::LDS]`, add = (n) => grid(ceil(z.DH % 4 ? n : n / 4, 256));
  if (dq) {
    const tiles = ceil(z.T * R, rows), SPLITS = keySplits(z, rows, 32, tiles * heads), lines = z.B * z.T * z.H;
    more.SPLITS = SPLITS;
    place('DQPARTS', SPLITS > 1 ? 4 * SPLITS * lines * z.DH : 0);
    const sums = `reinterpret_cast<float*>(${ws} + ${S}::DQPARTS)`;
    kernels.push(m('winwidedq', grid(tiles * heads * SPLITS), 256, lds,
      `window_wide_dq<${S}>(${args}, ${out('dq')}, ${sums}, lds, blockIdx.x % ${heads}u, ${tiles - 1}u - blockIdx.x / ${heads * SPLITS}u, blockIdx.x / ${heads}u % ${SPLITS}u)`, more));
    if (SPLITS > 1) kernels.push(m('winadd', add(lines * z.DH), 256, null, `window_wide_add<${S}>(${out('dq')}, ${sums}, blockIdx.x * 256u + threadIdx.x)`, more));
  }
  if (dk || dv) {
    // Tiles of 32 rows that see a key of one workgroup's at most: of any key by the window, of a sink all.
    const tiles = ceil(z.KEYS, rows), all = ceil(z.T * R, 32), most = z.WINDOW ? Math.min(all, ceil((z.WINDOW + rows) * R, 32) + 1) : all;
    const sinks = z.WINDOW ? Math.min(tiles, ceil(Math.min(z.SINKS, z.KEYS), rows)) : 0;
    const CHUNK = Math.max(8, ceil(most, Math.max(1, ceil(FILL, tiles * heads))));
    const CHUNKS = ceil(most, CHUNK), CHUNKS_MOST = sinks ? Math.max(CHUNKS, ceil(all, CHUNK)) : CHUNKS, FEW = Math.min(z.KEYS, sinks * rows);
    Object.assign(more, { CHUNK, CHUNKS, CHUNKS_MOST, FEW });
    const floats = CHUNKS_MOST > 1 ? (CHUNKS * z.KEYS + (CHUNKS_MOST - CHUNKS) * FEW) * z.B * z.HK * z.DH : 0;
    place('DKPARTS', dk ? 4 * floats : 0);
    place('DVPARTS', dv ? 4 * floats : 0);
    // The sinks' chunks, then the other tiles', the keys that most queries see first.
    const few = sinks * CHUNKS_MOST, id = `(blockIdx.x / ${heads}u)`;
    const where = `blockIdx.x % ${heads}u, ${id} < ${few}u ? ${id} / ${CHUNKS_MOST}u : ${sinks}u + (${id} - ${few}u) / ${CHUNKS}u, ${id} < ${few}u ? ${id} % ${CHUNKS_MOST}u : (${id} - ${few}u) % ${CHUNKS}u`;
    kernels.push(m('winwidedkv', grid((few + (tiles - sinks) * CHUNKS) * heads), 256, lds,
      `window_wide_dkv<${S}, ${dk}, ${dv}>(${args}, ${out('dk')}, ${out('dv')}, ${ws}, lds, ${where})`, more));
    if (CHUNKS_MOST > 1) {
      const n = z.B * z.KEYS * z.HK * z.DH;
      for (const [p, name, by] of [['dk', 'DKPARTS', `static_cast<float>(${S}::scale())`], ['dv', 'DVPARTS', '1.f']]) {
        if (parts.includes(p)) kernels.push(m('winadd', add(n), 256, null, `window_wide_join<${S}>(${out(p)}, reinterpret_cast<const float*>(${ws} + ${S}::${name}), ${by}, blockIdx.x * 256u + threadIdx.x)`, more));
      }
    }
  }
  return { kernels, workspace: at };
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
