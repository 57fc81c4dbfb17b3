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
  // (Positions of a tile or a window past the last stay below 2^31.)
  if (T * H > 2 ** 30 || KEYS * HK > 2 ** 30) throw new Error('windowAttention: a sequence\'s rows are counted in 32 bits (at most 2^30)');
  const lengths = node.inputs.length - (grad ? 3 : 0) === 4;
  return { z: { B, T, H, DH, KEYS, HK, WINDOW: a.window, SINKS: a.sinks, LAST: a.queries === 'last', LENGTHS: lengths, VEC: DH % 4 === 0 }, scale: a.scale, lengths, grad };
}

function maker(s, e, types) {
  const text = (kind, blocks, threads, structs, calls, lds, body) => {
    const header = calls.some((c) => /_pack/.test(c)) ? 'tcmi_window_packed.h' : calls.some((c) => /_wide/.test(c)) ? 'tcmi_window_wide.h' : 'tcmi_window.h';
    // Two workgroups of four wavefronts a CU, or one of eight: 256 registers each. (Few rows, heads of 128 over 50000 keys: 106 us by one, 86 by two.)
    const two = calls.some((c) => /_packed(_dq|_dkv)?</.test(c) || (/_wide(_dq|_dkv)?</.test(c) && s.z.DH <= 64) || (/window_rows</.test(c) && s.z.DH > 64 && s.z.DH <= 128));
    return kernel(kind, `#include "${header}"
${structs.map(([name, more]) => `struct ${name} {
${constants(Object.assign({}, s.z, more || {}), types)}
  static __device__ __forceinline__ double scale() { return ${double(s.scale)}; }
};`).join('\n')}
extern "C" __global__ void __launch_bounds__(${threads}${two ? ', 2' : ''}) __KERNEL__(${e.sig}) {
${e.open}${lds ? `  __shared__ __attribute__((aligned(16))) ${lds};\n` : ''}${body}}
`, blocks, threads);
  };
  const m = (kind, blocks, threads, lds, call, more) => text(kind, blocks, threads, [[S, more]], [call], lds, `  tcmi::${call};\n`);
  /**
   * Several jobs in one launch, a run of workgroups each. A job: { blocks, more, lds, call }, its LDS in bytes and its call given its struct of
   * sizes' name, the call also its workgroup's number.
   */
  m.jobs = (kind, threads, jobs) => {
    if (jobs.length === 1) {
      const [j] = jobs;
      return m(kind, grid(j.blocks), threads, j.lds && `char lds[${j.lds(S)}]`, j.call(S, 'blockIdx.x'), j.more);
    }
    const structs = jobs.map((j, k) => [k ? `${S}${k}` : S, j.more]), calls = jobs.map((j, k) => j.call(structs[k][0], 'block'));
    const bytes = jobs.map((j, k) => j.lds && j.lds(structs[k][0])).filter(Boolean);
    let first = 0, body = '';
    jobs.forEach((j, k) => {
      body += `  ${k ? '} else ' : ''}${k < jobs.length - 1 ? `if (blockIdx.x < ${first + j.blocks}u) ` : ''}{\n    const uint32_t block = blockIdx.x - ${first}u;\n    tcmi::${calls[k]};\n`;
      first += j.blocks;
    });
    return text(kind, grid(first), threads, structs, calls, bytes.length ? `char lds[${bytes.reduce((x, y) => `(${x} > ${y} ? ${x} : ${y})`)}]` : null, `${body}  }\n`);
  };
  return m;
}

/** n workgroups along the first axis of a grid, whose threads are counted in 32 bits: up to 512 each. */
function grid(n) {
  if (n >= 2 ** 23) throw new Error(`windowAttention: ${n} workgroups (at most 2^23)`);
  return [n, 1, 1];
}

/**
 * Rows of a key head that tcmi_window.h takes, a tile of it: more of them are a workgroup's of tcmi_window_wide.h, which reads the keys once for all. (16
 * rows over 4096 keys, heads of 64: 32.6 us by the first, 43.6 by the second; 20 rows, heads of 128: 71 and 45. The gradients are the second's for any
 * rows: 8 tokens of 64 sequences, heads of 64, 16.4 us by the first's way, 9.1 by the second's; 1 over 8000 keys 460 and 64.)
 */
const FEW_ROWS = 16;

/**
 * Workgroups that a chip's worth is: two a CU run at once, and as many wait, so that those that see many keys leave no CU idle
 * at the end.
 */
const FILL = 4 * CUS;

/**
 * Blocks of 16 lines of a wavefront's own, of `lines` of a head over `tiles` tiles of the other side: two where its registers `hold` them and two
 * workgroups a CU are left, of which several may deal the tiles among them, eight each or more. Of packed operands alone: where a workgroup splits
 * what it reads, one is faster (4 sequences of 4000 tokens, 8 heads of 64, a window of 100 62 us by two, 53 by one; gradients of 2000 tokens 152 and 134).
 */
function blocksOf(hold, lines, heads, tiles) { return hold && ceil(lines, 128) * heads * Math.max(1, Math.min(8, Math.floor(tiles / 8))) >= 2 * CUS ? 2 : 1; }

/**
 * Whether operands are split by a launch of their own (tcmi_window_packed.h), not by each workgroup that reads them (tcmi_window_wide.h): where
 * four workgroups or more read a key, by its registers for heads up to 128. (With gradients, heads of 64: windows of 512 266 us packed, 298 otherwise, 4
 * sequences of 512 tokens without one 67 and 64, of 768 111 and 119; heads of 128, 2 of 896 tokens: 153 and 190.)
 */
const packs = (z) => z.DH <= 128 && ceil(Math.min(z.T, z.WINDOW || z.T) * (z.H / z.HK), 128) >= 4;

/** Floats of a line, eight a lane, as they stand in LDS (WindowTile::LD). */
const lanesOf = (DH) => (DH <= 32 ? 4 : DH <= 64 ? 8 : DH <= 128 ? 16 : 32);

/** Workspace of `planes` planes of `lines` lines a head of two bytes a float. */
const formBytes = (z, lines, planes) => z.B * z.HK * lines * lanesOf(z.DH) * 16 * planes;

/**
 * Splits of the tiles of NB keys that `rows` rows of one head see, of `blocks` workgroups otherwise: eight tiles each or more, four where there would be
 * fewer than two workgroups a CU (288 workgroups of ten tiles, each with its loads' time: 22 us, by halves 15 and 5 to join them; by fifths 30 in all), two
 * where there would be fewer than one (80 workgroups of ten tiles: by halves 20 us in all, by fifths 15, by tenths 18).
 */
function keySplits(z, rows, NB, blocks) {
  const R = z.H / z.HK;
  const most = ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW + ceil(rows, R) + z.SINKS) : z.KEYS, NB);
  return Math.max(1, Math.min(64, Math.floor(most / (blocks < CUS ? 2 : blocks < 2 * CUS ? 4 : 8)), ceil(FILL, blocks)));
}

function wideForward(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null), heads = z.B * z.HK, R = z.H / z.HK;
  const packed = packs(z), HB = blocksOf(packed, z.T * R, heads, ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW) : z.KEYS, 64)), rows = 64 * HB, tiles = ceil(z.T * R, rows), SPLITS = keySplits(z, rows, z.DH <= 64 ? 64 : 32, tiles * heads);
  const more = { TILES: ceil(z.T * R, 16), SPLITS }, types = { HB: 'int', WAVES: 'int' };
  let at = 0;
  const place = (name, bytes) => { more[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  place('OUT', SPLITS > 1 ? 4 * SPLITS * heads * more.TILES * 16 * z.DH : 0);
  place('STATS', SPLITS > 1 ? 8 * SPLITS * heads * more.TILES * 16 : 0);
  const KP = align(z.KEYS, 64);
  if (packed) {
    Object.assign(more, { WAVES: 4, HB });
    place('KSCALE', 4 * heads * KP);
    place('KDOTS', formBytes(z, KP, 2));
    place('VSUMS', formBytes(z, KP, 3));
  }
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', ws = `reinterpret_cast<char*>(${e.ws})`, m = maker(s, e, types);
  // The last rows, which see most, first; a head's on one XCD, whose L2 its keys share, where heads are a multiple of eight.
  const kernels = [], where = `blockIdx.x % ${heads}u, ${tiles - 1}u - blockIdx.x / ${heads * SPLITS}u, blockIdx.x / ${heads}u % ${SPLITS}u`;
  if (packed) {
    kernels.push(packKeys(m, z, L, ws, more, heads, KP));
    kernels.push(m('winpacked', grid(tiles * heads * SPLITS), 256, `char lds[tcmi::WindowPacked<${S}>::FORWARD]`,
      `window_packed<${S}>(A.in[0], ${L}, ${out('o')}, ${out('lse')}, ${ws}, lds, ${where})`, more));
  } else {
    kernels.push(m('winwide', grid(tiles * heads * SPLITS), 256, `char lds[tcmi::WindowWide<${S}>::LDS]`,
      `window_wide<${S}>(A.in[0], A.in[1], A.in[2], ${L}, ${out('o')}, ${out('lse')}, ${ws}, lds, ${where})`, more));
  }
  if (SPLITS > 1) kernels.push(joinKernel(m, z, out, ws, more, heads));
  return { kernels, workspace: at };
}

/** The launch that splits keys and values. */
function packKeys(m, z, L, ws, more, heads, KP) {
  const each = 256 / lanesOf(z.DH);
  return m('winpack', grid(ceil(heads * KP, each)), 256, null,
    `window_pack_keys<${S}, false, false>(A.in[1], A.in[2], ${L}, ${ws}, blockIdx.x * ${each}u + threadIdx.x / ${lanesOf(z.DH)}u)`, more);
}

/**
 * How the gradients are dealt out: CHUNK tiles of 32 rows of those that see one of `keyRows` keys a workgroup's, and SPLITS of the tiles of 32 keys
 * that `rows` rows see, the gradients of keys before those of queries on the `slots` workgroups that run at once. A tile of the
 * first is four products and about 3 us of heads of 64, one of the second three; a workgroup starts in the time of four tiles; the last ones end a
 * sixth of one apart; a byte of sums is written and read at 5 TB/s in all. (9 heads of 1001 tokens in a window of 257: chunks of 8 tiles 105 us, of 12 (this takes
 * 13) 92, of 16 102; 8192 tokens of 8 heads: chunks of 50 tiles 1271, of 94 1220, of 128 1208, by no splits 1360, by two 1245, by four 1256; two
 * sequences of 1024 tokens, 16 heads of 128: by no splits 298, by two 300, by four 317.)
 */
function deal(z, heads, slots, keyRows, rows) {
  const R = z.H / z.HK, first = z.LAST ? z.KEYS - z.T : 0, counts = [], us = 3 * z.DH / 64;
  for (let j = 0; j < z.KEYS; j += keyRows) {
    const p0 = Math.max(j, first), last = Math.min(j + keyRows, z.KEYS) - 1;
    const p1 = Math.min(z.WINDOW && j >= z.SINKS ? Math.min(z.KEYS - 1, last + z.WINDOW - 1) : z.KEYS - 1, first + z.T - 1);
    counts.push(p0 <= p1 ? ceil((p1 - first + 1) * R, 32) - Math.floor((p0 - first) * R / 32) : 0);
  }
  const most = counts.reduce((a, c) => Math.max(a, c), 1), work = 1.75 * heads * counts.reduce((a, c) => a + c, 0);
  const time = (block, starts) => us * Math.max(block, (work + starts) / slots + block / 6);
  let best = { time: Infinity };
  for (let CHUNK = Math.min(most, 8); ; CHUNK = Math.min(most, Math.floor(CHUNK * 1.05) + 1)) {
    const n = heads * counts.reduce((q, c) => q + Math.max(1, ceil(c, CHUNK)), 0);
    const t = time(CHUNK + 4, 4 * n) + (n > heads * counts.length ? n * keyRows * z.DH * 16 / 5e6 : 0);
    if (t < best.time) best = { CHUNK, time: t };
    if (CHUNK >= most) break;
  }
  const { CHUNK } = best, keys = ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW + ceil(rows, R) + z.SINKS) : z.KEYS, 32), blocks = ceil(z.T * R, rows) * heads;
  best = { time: Infinity };
  for (let SPLITS = 1; SPLITS <= Math.max(1, Math.min(64, keys / 4)); SPLITS++) {
    const t = time(0.75 * (keys / SPLITS + 4), 3 * blocks * SPLITS) + (SPLITS > 1 ? 5 + SPLITS * z.B * z.T * z.H * z.DH * 8 / 5e6 : 0);
    if (t < best.time) best = { SPLITS, time: t };
  }
  return { CHUNK, SPLITS: best.SPLITS };
}

/** The launch that joins the splits of rows. */
function joinKernel(m, z, out, ws, more, heads) {
  const rows = heads * more.TILES * 16, lanes = z.DH <= 64 ? 16 : z.DH <= 128 ? 32 : 64;
  // Of many splits a workgroup a row (32 rows of 128 splits 14.3 us by a wavefront each, 5 so).
  const parts = more.SPLITS >= 16 && rows < 2 ** 20 ? 256 / lanes : 1;
  return m('winjoin', grid(parts > 1 ? rows : ceil(rows, 256 / lanes)), 256, parts > 1 ? 'float lds[1024]' : null,
    `window_join<${S}, ${lanes}, ${parts}>(${out('o')}, ${out('lse')}, ${ws}, ${parts > 1 ? 'lds, blockIdx.x' : `nullptr, blockIdx.x * ${256 / lanes}u + threadIdx.x / ${lanes}u`})`, more);
}

function forwardKernels(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null);
  if (z.T * (z.H / z.HK) > FEW_ROWS) return wideForward(s, parts, joined);
  const R = z.H / z.HK, heads = z.B * z.HK;
  // The keys that the rows see at most, in tiles of 16, dealt to as many workgroups as fill the chip four times, eight tiles each or more.
  // (32 tokens of 8 heads over 1028 keys: 16.8 us by nine tiles, 21.6 by five.)
  const most = ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW + ceil(16, R) + 32 + z.SINKS) : z.KEYS, 16);
  const SPLITS = Math.max(1, Math.min(256, Math.floor(most / 8), ceil(4 * CUS, heads)));
  const types = {};
  let at = 0;
  const more = { TILES: 1, SPLITS };
  const place = (name, bytes) => { more[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  place('OUT', SPLITS > 1 ? 4 * SPLITS * heads * 16 * z.DH : 0);
  place('STATS', SPLITS > 1 ? 8 * SPLITS * heads * 16 : 0);
  const m = maker(s, e, types);
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', ws = `reinterpret_cast<char*>(${e.ws})`;
  const kernels = [m('win', grid(heads * SPLITS), 256, `float lds[tcmi::window_lds<${z.DH}>()]`,
    `window_rows<${S}>(A.in[0], A.in[1], A.in[2], ${L}, ${out('o')}, ${out('lse')}, ${ws}, lds, blockIdx.x)`, more)];
  if (SPLITS > 1) kernels.push(joinKernel(m, z, out, ws, more, heads));
  return { kernels, workspace: at };
}

function backwardKernels(s, parts, joined) {
  const { z } = s, e = entry(joined ? parts : null);
  const R = z.H / z.HK, heads = z.B * z.HK;
  const out = (p) => (parts.includes(p) ? e.out(p) : 'nullptr');
  const L = s.lengths ? 'A.in[3]' : 'nullptr', first = s.lengths ? 4 : 3;
  const args = `{A.in[0], A.in[1], A.in[2], ${L}, A.in[${first}], A.in[${first + 1}], A.in[${first + 2}], ${e.ws}}`;
  const dq = parts.includes('dq'), dk = parts.includes('dk'), dv = parts.includes('dv');
  const types = { HB: 'int', WAVES: 'int' }, more = {};
  // dy·o of every row, where the gradients of keys do not form it.
  const masses = z.DH > 128 && (dk || dv);
  let at = masses ? align(4 * z.B * z.T * z.H, 256) : 0;
  const place = (name, bytes) => { more[name] = at; types[name] = 'size_t'; at = align(at + bytes, 256); };
  const m = maker(s, e, types), ws = `reinterpret_cast<char*>(${e.ws})`;
  const kernels = [];
  const add = (n) => ceil(z.DH % 4 ? n : n / 4, 256), KP = align(z.KEYS, 64), RP = align(z.T * R, 64), packed = packs(z), lanes = lanesOf(z.DH);
  const hold = z.DH <= 64;
  if (packed) {
    Object.assign(more, { WAVES: 4, HB: 1, SPLITS: 1 });
    place('KSCALE', 4 * heads * KP);
    place('VSCALE', 4 * heads * KP);
    place('KDOTS', formBytes(z, KP, 2));
    place('VDOTS', formBytes(z, KP, 2));
    place('KSUMS', dq ? formBytes(z, KP, 3) : 0);
    place('ROWSTATS', 16 * heads * RP);
    for (const [name, planes] of [['QDOTS', 2], ['DDOTS', 2], ['QSUMS', 3], ['DSUMS', 3]]) place(name, dk || dv ? formBytes(z, RP, planes) : 0);
    const keys = ceil(heads * KP, 256 / lanes), place256 = (first) => `(blockIdx.x - ${first}u) * ${256 / lanes}u + threadIdx.x / ${lanes}u`;
    kernels.push(m('winpack', grid(keys + ceil(heads * RP, 256 / lanes)), 256, null,
      `window_pack_both<${S}, ${dq}, ${dk || dv}, ${keys}u>(${args}, ${ws}, blockIdx.x, ${place256(0)}, ${place256(keys)})`, Object.assign({ VSUMS: 0 }, more)));
  }
  if (masses) {
    kernels.push(m('winmass', grid(ceil(z.B * z.T * z.H, 64)), 256, null, `window_wide_mass<${S}>(A.in[0], A.in[${first}], A.in[${first + 2}], ${e.ws}, blockIdx.x * 64u + threadIdx.x / 64u * 16u)`));
  }
  // The gradients of queries and of keys run side by side, and what joins their parts.
  const jobs = [], joins = [], waves = packed && z.DH > 64 ? 8 : 4;
  if (packed) more.WAVES = waves;
  const keyBlocks = blocksOf(hold && packed, z.KEYS, heads, ceil(Math.min(z.T, z.WINDOW || z.T) * R, 32)), rowBlocks = blocksOf(hold && packed, z.T * R, heads, ceil(z.WINDOW ? Math.min(z.KEYS, z.WINDOW) : z.KEYS, 64));
  const keyRows = 16 * waves * keyBlocks, rows = 16 * waves * rowBlocks;
  // (Of heads above 64 a workgroup a CU, by its registers, and where operands are split once by LDS too.)
  const { CHUNK, SPLITS } = deal(z, heads, (hold ? 2 : 1) * CUS, keyRows, rows);
  const place4 = (name, floats) => place(name, 4 * floats);
  if (dk || dv) {
    // Eight wavefronts where a packed tile takes most of LDS.
    const HB = keyBlocks, tiles = ceil(z.KEYS, keyRows), all = ceil(z.T * R, 32), most = z.WINDOW ? Math.min(all, ceil((z.WINDOW + keyRows) * R, 32) + 1) : all;
    const sinks = z.WINDOW ? Math.min(tiles, ceil(Math.min(z.SINKS, z.KEYS), keyRows)) : 0;
    const CHUNKS = ceil(most, CHUNK), CHUNKS_MOST = sinks ? Math.max(CHUNKS, ceil(all, CHUNK)) : CHUNKS, FEW = Math.min(z.KEYS, sinks * keyRows);
    Object.assign(more, { CHUNK, CHUNKS, CHUNKS_MOST, FEW, ROWS_EACH: keyRows });
    const floats = CHUNKS_MOST > 1 ? (CHUNKS * z.KEYS + (CHUNKS_MOST - CHUNKS) * FEW) * z.B * z.HK * z.DH : 0;
    place4('DKPARTS', dk ? floats : 0);
    place4('DVPARTS', dv ? floats : 0);
    // The sinks' chunks, then the other tiles', the keys that most queries see first. (Workgroups go to the XCDs in turn: an odd number of chunks a
    // tile, one more than there are where that is even, gives each of them first and last ones alike. 512 tokens of 8 heads 93.6 us, 89.4 so.)
    const few = sinks * CHUNKS_MOST, ODD = CHUNKS | 1;
    const where = (block) => {
      const id = `(${block} / ${heads}u)`, at = `(${id} - ${few}u)`;
      return `${block} % ${heads}u, ${id} < ${few}u ? ${id} / ${CHUNKS_MOST}u : ${sinks}u + ${at} / ${ODD}u, ${id} < ${few}u ? ${id} % ${CHUNKS_MOST}u : ${at} % ${ODD}u`;
    };
    // Both at once, or of the largest heads, which its registers do not hold both of, one after the other.
    for (const [k, v] of dk && dv && z.DH > 128 ? [[false, true], [true, false]] : [[dk, dv]]) {
      jobs.push({ HB, blocks: (few + (tiles - sinks) * ODD) * heads, lds: (sizes) => (packed ? `tcmi::WindowPackedRows<${sizes}>::LDS` : `tcmi::WindowBack<${sizes}>::LDS`),
        call: (sizes, block) => `${packed ? 'window_packed_dkv' : 'window_wide_dkv'}<${sizes}, ${k}, ${v}>(${args}, ${out('dk')}, ${out('dv')}, ${ws}, lds, ${where(block)})` });
    }
    for (const [is, p, by] of [[dk, 'dk', `static_cast<float>(${S}::scale())`], [dv, 'dv', '1.f']]) {
      if (is && CHUNKS_MOST > 1) joins.push({ blocks: add(z.B * z.KEYS * z.HK * z.DH), call: (sizes, block) => `window_wide_join<${sizes}>(${out(p)}, reinterpret_cast<const float*>(${ws} + ${sizes}::${p.toUpperCase()}PARTS), ${L}, ${by}, ${block} * 256u + threadIdx.x)` });
    }
  }
  if (dq) {
    const HB = rowBlocks, tiles = ceil(z.T * R, rows), lines = z.B * z.T * z.H;
    more.SPLITS = SPLITS;
    place4('DQPARTS', SPLITS > 1 ? SPLITS * lines * z.DH : 0);
    const sums = (sizes) => `reinterpret_cast<float*>(${ws} + ${sizes}::DQPARTS)`;
    const where = (block) => `${block} % ${heads}u, ${tiles - 1}u - ${block} / ${heads * SPLITS}u, ${block} / ${heads}u % ${SPLITS}u`;
    jobs.push({ HB, blocks: tiles * heads * SPLITS, lds: (sizes) => (packed ? `tcmi::WindowPacked<${sizes}>::DQ` : `tcmi::WindowBack<${sizes}>::LDS`),
      call: (sizes, block) => (packed ? `window_packed_dq<${sizes}>(${args}, ${out('dq')}, ${sums(sizes)}, ${ws}, lds, ${where(block)})`
        : `window_wide_dq<${sizes}>(${args}, ${out('dq')}, ${sums(sizes)}, lds, ${where(block)})`) });
    if (SPLITS > 1) joins.push({ blocks: add(lines * z.DH), call: (sizes, block) => `window_wide_add<${sizes}>(${out('dq')}, ${sums(sizes)}, ${block} * 256u + threadIdx.x)` });
  }
  for (const j of jobs.concat(joins)) j.more = Object.assign({}, more, packed ? { HB: j.HB || 1 } : {});
  kernels.push(m.jobs('winback', 64 * waves, jobs));
  if (joins.length) kernels.push(m.jobs('winadd', 256, joins));
  return { kernels, workspace: at };
}

/** The flops of one product over the pairs of a query and a key that it sees, were every sequence full. */
function seen(z) {
  const first = z.LAST ? z.KEYS - z.T : 0, p0 = Math.max(0, first), p1 = Math.min(z.KEYS, first + z.T) - 1;
  // Of the positions below p: the keys up to each, less those before the window, and the sinks among those.
  const to = (p) => {
    const n = Math.max(0, p - (z.WINDOW || p)), few = Math.min(n, z.SINKS);
    return p * (p + 1) / 2 - n * (n + 1) / 2 + few * (few + 1) / 2 + (n - few) * z.SINKS;
  };
  return p0 <= p1 ? 2 * z.B * z.H * z.DH * (to(p1 + 1) - to(p0)) : 0;
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
