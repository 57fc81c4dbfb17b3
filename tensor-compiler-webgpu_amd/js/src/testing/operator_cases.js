'use strict';
// Graphs of the operators that are one node each (ir/operators.js), from plain
// descriptions: those of their GPU tests (CASES; FORMS, whose tests name them) and of their measurement (MEASURED).
//   { family: 'rotary', x, positions, gain?, gradient?, options }   a second x where `twin`
//       gives its shape; `twice`: rotated, and the result again
//   { family: 'loss', N, d, V, bias?, gradient?, wrt?, after? }     wrt: 'h', 'W', 'b' (default all); `after`: the
//       losses' cotangent depends on the losses, so their gradients cannot run beside them
//   { family: 'orthogonalize', x, count, options, twice }
//   { family: 'embedding', tokens, V, d, scale?, gradient?, one? }          one: the token of nine rows of ten
//   { family: 'residual', x, options: { norm, residual, eps }, vectors: ['gain', 'bias', ...], gate: 'full'?, keep: 'h' | 'n'?,
//       gradient?, wrt? }                                                     keep, wrt: default all
//   { family: 'window', q, k, lengths?, options, gradient?, wrt? }          wrt: 'q', 'k', 'v' (default all)

const { Graph } = require('../ir/graph');
const { grad } = require('../autodiff');

function operatorGraph(c) {
  const g = new Graph();
  let outs = [], names = [], wrt = [], grads = [];
  if (c.family === 'rotary') {
    const at = g.input('at', c.positions);
    [c.x].concat(c.twin ? [c.twin] : []).forEach((shape, k) => {
      const x = g.input(`x${k}`, shape);
      const gain = c.gain ? g.input(`g${k}`, [shape[shape.length - 1]]) : null;
      const y = g.rotary(x, at, Object.assign({ gain }, c.options || {}));
      outs.push(c.twice ? g.rotary(y, at, Object.assign({ gain }, c.options || {})) : y);
      names.push(`y${k}`);
      wrt.push(x);
      grads.push(`dx${k}`);
      if (c.gain) { wrt.push(gain); grads.push(`dg${k}`); }
    });
  } else if (c.family === 'loss') {
    const h = g.input('h', [c.N, c.d]), W = g.input('W', [c.d, c.V]), t = g.input('t', [c.N]);
    const b = c.bias ? g.input('b', [c.V]) : null;
    const loss = g.linearCrossEntropy(h, W, t, b);
    outs = [c.after ? g.mul(loss, loss) : loss];
    names = ['loss'];
    const all = { h, W, b };
    for (const k of c.wrt || (c.bias ? ['h', 'W', 'b'] : ['h', 'W'])) { wrt.push(all[k]); grads.push(`d${k}`); }
  } else if (c.family === 'orthogonalize') {
    for (let k = 0; k < (c.count || 1); k++) {
      const y = g.orthogonalize(g.input(`x${k}`, c.x), c.options);
      outs.push(c.twice ? g.orthogonalize(y, c.options) : y);
      names.push(`y${k}`);
    }
  } else if (c.family === 'embedding') {
    const t = g.input('tokens', c.tokens), table = g.input('table', [c.V, c.d]);
    outs = [g.embedding(t, table, { scale: c.scale })];
    names = ['e'];
    wrt.push(table);
    grads.push('dtable');
  } else if (c.family === 'residual') {
    const x = g.input('x', c.x), y = g.input('y', c.x), all = { x, y };
    for (const k of c.vectors || []) all[k] = g.input(k, k === 'gate' && c.gate === 'full' ? c.x : c.x.slice(-1));
    const r = g.residualNorm(x, y, Object.assign({}, all, c.options));
    names = c.keep ? [c.keep] : Object.keys(r);
    outs = names.map((k) => r[k]);
    for (const k of c.wrt || Object.keys(all)) { wrt.push(all[k]); grads.push(`d${k}`); }
  } else if (c.family === 'window') {
    const all = { q: g.input('q', c.q), k: g.input('k', c.k), v: g.input('v', c.k) };
    outs = [g.windowAttention(all.q, all.k, all.v, Object.assign({ lengths: c.lengths ? g.input('lengths', [c.q[0]]) : null }, c.options))];
    names = ['o'];
    for (const k of c.wrt || ['q', 'k', 'v']) { wrt.push(all[k]); grads.push(`d${k}`); }
  } else throw new Error(`no operator '${c.family}'`);
  if (!c.gradient) return { graph: g, keep: outs, names };
  const G = grad(g, outs, wrt);
  return { graph: G.graph, keep: outs.concat(G.grads), names: names.concat(grads) };
}

const rotary = (name, x, positions, more) => Object.assign({ name, family: 'rotary', x, positions }, more);
const loss = (name, N, d, V, more) => Object.assign({ name, family: 'loss', N, d, V }, more);
const orth = (name, x, more) => Object.assign({ name, family: 'orthogonalize', x }, more);

const embedding = (name, tokens, V, d, more) => Object.assign({ name, family: 'embedding', tokens, V, d }, more);
const residual = (name, x, vectors, options, more) => Object.assign({ name, family: 'residual', x, vectors, options }, more);
const window = (name, q, k, options, more) => Object.assign({ name, family: 'window', q, k, options }, more);

// Cases of the operators for long contexts and large vocabularies.
const CONTEXT = [
  // One row and one token; few; tables of one digit, of two and of three; tokens of several tiles and chunks.
  embedding('one', [1], 1, 1, { gradient: true }),
  embedding('token', [3], 50, 64, { scale: 8, gradient: true }),
  embedding('scalar', [], 7, 12, { gradient: true }),
  embedding('step', [4, 33], 96, 64, { scale: 0.5, gradient: true }),
  embedding('odd', [131], 517, 37, { gradient: true }),
  embedding('same', [700], 1, 20, { scale: -2, gradient: true }),
  embedding('two', [3001], 2, 260, { gradient: true }),
  embedding('wide', [65], 513, 1030, { gradient: true }),
  embedding('narrow', [2000], 300, 3, { gradient: true }),
  embedding('many', [2500], 70001, 4, { gradient: true }),
  embedding('most', [300], 300000, 8, { gradient: true }),
  embedding('counted', [17003], 300, 8, { gradient: true }),
  embedding('counted-twice', [20480], 1000, 2, { gradient: true }),
  // Of a table of few rows, the most of them, and one more; sorted tokens that are all one.
  embedding('few-most', [3001], 128, 70, { scale: 2, gradient: true }),
  embedding('few-more', [3001], 129, 70, { scale: 2, gradient: true }),
  embedding('few-long', [40000], 5, 7, { gradient: true }),
  embedding('same-sorted', [1500], 130, 20, { scale: -2, gradient: true, one: 77 }),
  embedding('two-sorted', [3001], 200, 260, { gradient: true, one: 3 }),
  embedding('values', [9, 5], 11, 24, { scale: 0 }),
  // Norms of both kinds, with what may stand beside them; rows from one float to the longest; only some results.
  residual('plain', [5, 64], ['gain'], {}, { gradient: true }),
  residual('sum', [7, 24], [], { residual: 0.5 }, { gradient: true }),
  residual('layer', [4, 33, 96], ['gain', 'bias'], {}, { gradient: true }),
  residual('sandwich', [3, 7, 64], ['gain', 'postGain'], { residual: 0.7 }, { gradient: true }),
  residual('all', [37, 260], ['gain', 'bias', 'postGain', 'postBias', 'gate'], { residual: 1.5, eps: 1e-3 }, { gradient: true }),
  residual('full-gate', [19, 130], ['gain', 'bias', 'postGain', 'postBias', 'gate'], { residual: -1 }, { gradient: true, gate: 'full' }),
  residual('gated', [33, 40], ['gain', 'gate'], {}, { gradient: true }),
  residual('gate-alone', [33, 41], ['gate'], { residual: 0 }, { gradient: true }),
  residual('post-alone', [21, 37], ['postGain', 'postBias'], {}, { gradient: true }),
  residual('layer-gain', [9, 48], ['gain', 'postGain'], { norm: 'layer' }, { gradient: true }),
  residual('one', [1], ['gain', 'postGain', 'gate'], {}, { gradient: true }),
  residual('float', [5, 1], ['gain', 'bias'], {}, { gradient: true }),
  residual('odd', [13, 515], ['gain', 'postGain', 'gate'], {}, { gradient: true }),
  residual('wide', [70, 1028], ['gain', 'postGain'], {}, { gradient: true }),
  residual('wider', [6, 4099], ['gain', 'bias', 'postGain', 'postBias', 'gate'], {}, { gradient: true }),
  residual('longest', [3, 16384], ['gain', 'bias', 'postGain', 'postBias', 'gate'], {}, { gradient: true }),
  residual('rows', [9001, 20], ['gain', 'postGain', 'gate'], {}, { gradient: true }),
  residual('only-n', [40, 64], ['gain', 'postGain'], {}, { gradient: true, keep: 'n' }),
  residual('only-h', [40, 64], ['gain', 'postGain'], {}, { gradient: true, keep: 'h' }),
  residual('only-dy', [40, 64], ['gain', 'postGain', 'gate'], {}, { gradient: true, wrt: ['y'] }),
  residual('only-vectors', [40, 64], ['gain', 'postGain', 'gate'], {}, { gradient: true, wrt: ['gate', 'gain'] }),
  residual('values', [11, 100], ['gain', 'bias', 'postGain', 'gate'], { norm: 'layer' }, {}),
  // One token and many, over its own keys or a cache; windows and sinks of one key, of a tile's, of all; heads alone and shared;
  // sequences of their own lengths, some of no key.
  window('one', [1, 1, 1, 1], [1, 1, 1, 1], {}, { gradient: true }),
  window('token', [3, 1, 8, 64], [3, 50, 2, 64], { window: 20, sinks: 4 }, { lengths: true, gradient: true }),
  window('token-all', [5, 1, 4, 32], [5, 700, 4, 32], {}, { lengths: true }),
  window('token-far', [2, 1, 6, 80], [2, 5003, 2, 80], { window: 4000, sinks: 3 }, { lengths: true }),
  window('tokens', [3, 5, 6, 24], [3, 90, 2, 24], { window: 7 }, { lengths: true, gradient: true }),
  window('tokens-beyond', [6, 9, 3, 16], [6, 11, 1, 16], { window: 3, sinks: 1 }, { lengths: true, gradient: true }),
  window('step', [2, 64, 4, 64], [2, 64, 4, 64], {}, { gradient: true }),
  window('first', [6, 33, 4, 16], [6, 33, 2, 16], { queries: 'first', window: 9, sinks: 2 }, { lengths: true, gradient: true }),
  window('self', [2, 40, 2, 32], [2, 40, 1, 32], { window: 1 }, { gradient: true }),
  window('self-sink', [2, 40, 2, 32], [2, 40, 1, 32], { window: 1, sinks: 1, scale: 0.3 }, { gradient: true }),
  window('sinks-all', [1, 50, 2, 48], [1, 50, 2, 48], { window: 2, sinks: 50 }, { gradient: true }),
  window('sinks-tile', [1, 90, 2, 16], [1, 90, 2, 16], { window: 17, sinks: 17 }, { gradient: true }),
  window('odd', [2, 37, 3, 15], [2, 37, 3, 15], { window: 11, sinks: 2 }, { gradient: true }),
  window('odd-heads', [1, 21, 15, 9], [1, 21, 3, 9], { window: 30 }, { gradient: true }),
  window('long', [1, 530, 2, 64], [1, 530, 1, 64], { window: 100, sinks: 5 }, { gradient: true }),
  window('longer', [1, 700, 3, 128], [1, 700, 1, 128], {}, { gradient: true }),
  window('wide', [1, 150, 2, 256], [1, 150, 1, 256], { window: 70 }, { gradient: true }),
  window('late', [2, 70, 4, 96], [2, 300, 2, 96], { window: 120, sinks: 4 }, { gradient: true }),
  window('more-queries', [2, 20, 2, 32], [2, 7, 2, 32], { queries: 'first' }, { gradient: true }),
  // By operands split once (several workgroups read each key).
  window('packed', [2, 300, 8, 64], [2, 300, 1, 64], { window: 70, sinks: 5 }, { lengths: true, gradient: true }),
  window('packed-odd', [1, 517, 6, 15], [1, 517, 2, 15], { window: 200, sinks: 20 }, { gradient: true }),
  window('packed-late', [4, 200, 8, 80], [4, 700, 2, 80], { window: 150, sinks: 3 }, { lengths: true, gradient: true }),
  window('packed-first', [3, 333, 6, 96], [3, 333, 2, 96], { queries: 'first', window: 190 }, { lengths: true, gradient: true }),
  window('packed-heads', [1, 601, 2, 128], [1, 601, 2, 128], { scale: -0.05 }, { gradient: true }),
  window('packed-small', [1, 1100, 1, 24], [1, 1100, 1, 24], {}, { gradient: true }),
  window('packed-sinks', [1, 520, 4, 32], [1, 520, 2, 32], { window: 258, sinks: 300 }, { gradient: true }),
  window('packed-k', [1, 140, 4, 64], [1, 140, 1, 64], {}, { gradient: true, wrt: ['k'] }),
  window('packed-v', [1, 140, 4, 64], [1, 140, 1, 64], {}, { gradient: true, wrt: ['v'] }),
  window('packed-q', [1, 140, 4, 64], [1, 140, 1, 64], {}, { gradient: true, wrt: ['q'] }),
  // Gradients of few rows and large heads.
  window('token-large', [2, 1, 3, 200], [2, 40, 1, 200], { window: 9, sinks: 2 }, { lengths: true, gradient: true }),
  window('few-large', [3, 7, 2, 130], [3, 7, 2, 130], {}, { gradient: true }),
  window('few-long', [1, 2, 4, 128], [1, 1500, 2, 128], {}, { gradient: true }),
  window('only-q', [2, 64, 4, 32], [2, 64, 2, 32], { window: 20 }, { gradient: true, wrt: ['q'] }),
  window('only-k', [2, 64, 4, 32], [2, 64, 2, 32], { window: 20 }, { gradient: true, wrt: ['k'] }),
  window('only-v', [2, 64, 4, 32], [2, 64, 2, 32], { window: 20 }, { gradient: true, wrt: ['v'] }),
];

const CASES = [
  // One token and many; heads before and after the tokens; one position a token and one a sequence's token.
  rotary('token', [3, 1, 5, 64], [3, 1], { gain: true, gradient: true }),
  rotary('step', [4, 33, 4, 64], [33], { gain: true, gradient: true, twin: [4, 33, 2, 64] }),
  rotary('twins', [3, 40, 2, 64], [40], { gain: true, gradient: true, twin: [3, 40, 2, 64] }),
  rotary('twice', [3, 40, 2, 64], [40], { gain: true, gradient: true, twice: true }),
  rotary('heads-first', [2, 3, 17, 32], [2, 17], { gain: true, gradient: true, options: { axis: 2 } }),
  rotary('one-head', [29, 48], [29], { gain: true, gradient: true }),
  // Three axes, and frequencies that start over on each; adjacent pairs; a part of the head unrotated.
  rotary('video', [1, 45, 3, 96], [1, 45, 3], { gain: true, gradient: true, options: { sections: [12, 18, 18] } }),
  rotary('plane', [2, 16, 2, 40], [2, 16, 2], { gain: false, gradient: true, options: { sections: [8, 8], restart: true, pairs: 'adjacent' } }),
  rotary('adjacent', [2, 9, 4, 128], [2, 9], { gain: true, gradient: true, options: { pairs: 'adjacent', sections: [32] } }),
  rotary('partial', [2, 9, 4, 64], [9], { gain: true, gradient: true, options: { sections: [8] } }),
  // No multiple of four anywhere, an odd head, no rotation at all, the longest head.
  rotary('odd', [3, 7, 3, 15], [3, 7], { gain: true, gradient: true, options: { sections: [5] } }),
  rotary('odd-adjacent', [7, 1, 7], [7], { gain: true, gradient: true, options: { pairs: 'adjacent', axis: 0 } }),
  rotary('norm-only', [5, 2, 24], [5], { gain: true, gradient: true, options: { sections: [0], axis: 0 } }),
  rotary('long-head', [3, 1, 4096], [3], { gain: true, gradient: true, options: { axis: 0 } }),
  rotary('wide', [2, 700, 9, 32], [2, 700], { gain: true, gradient: true }),
  // Rows from one to several pieces of tiles, classes from one to more than a tile, ragged and not; some gradients only.
  loss('one', 1, 1, 1, { gradient: true }),
  loss('few', 5, 16, 7, { bias: true, gradient: true }),
  loss('square', 16, 8, 16, { gradient: true }),
  loss('tile', 128, 64, 128, { bias: true, gradient: true }),
  loss('step', 300, 96, 96, { bias: true, gradient: true }),
  loss('ragged', 131, 37, 517, { bias: true, gradient: true }),
  loss('deep', 40, 515, 260, { gradient: true }),
  loss('wide', 70, 20, 5003, { bias: true, gradient: true }),
  loss('rows', 3001, 20, 30, { bias: true, gradient: true }),
  loss('values', 200, 24, 300, { bias: true }),
  loss('only-h', 50, 24, 300, { bias: true, gradient: true, wrt: ['h'] }),
  loss('only-W', 50, 24, 300, { bias: true, gradient: true, wrt: ['W'] }),
  loss('only-b', 50, 24, 300, { bias: true, gradient: true, wrt: ['b'] }),
  loss('pieces', 700, 24, 150, { bias: true, gradient: true, tuning: { loss: { piece: 1 } } }),
  loss('piece-values', 400, 24, 150, { bias: true, tuning: { loss: { piece: 1 } } }),
  loss('squared', 50, 24, 300, { bias: true, gradient: true, after: true }),
  // Rows that are few, up to the most of them, by tiles of 64 and of 256 classes; one row more, and the same again.
  loss('row', 1, 515, 1000, { bias: true, gradient: true }),
  loss('few-odd', 33, 37, 517, { bias: true, gradient: true }),
  loss('few-most', 64, 64, 132, { gradient: true }),
  loss('few-classes', 17, 9, 129, { bias: true, gradient: true }),
  loss('few-wide', 9, 20, 33001, { bias: true, gradient: true }),
  loss('few-values', 49, 70, 132, {}),
  loss('one-more', 65, 1, 130, { gradient: true }),
  loss('more', 77, 17, 131, { bias: true, gradient: true }),
  loss('more-deep', 100, 515, 260, { gradient: true }),
  loss('more-h', 150, 24, 300, { bias: true, gradient: true, wrt: ['h'] }),
  loss('more-W', 150, 24, 300, { bias: true, gradient: true, wrt: ['W'] }),
  loss('more-b', 150, 24, 300, { bias: true, gradient: true, wrt: ['b'] }),
  loss('more-squared', 150, 24, 300, { bias: true, gradient: true, after: true }),
  // Classes that are few, in whole rows: one, an odd count, the most of them, one more; 16 and 32 rows a workgroup; deep and shallow.
  loss('narrow-one', 6, 5, 1, { bias: true, gradient: true }),
  loss('narrow-odd', 131, 37, 33, { bias: true, gradient: true }),
  loss('narrow-most', 200, 512, 128, { gradient: true }),
  loss('narrow-more', 200, 513, 128, { gradient: true }),
  loss('narrow-rows', 4100, 70, 95, { bias: true, gradient: true }),
  loss('narrow-deep', 70, 1030, 96, { bias: true, gradient: true }),
  loss('narrow-h', 150, 24, 100, { bias: true, gradient: true, wrt: ['h'] }),
  loss('narrow-b', 150, 24, 100, { bias: true, gradient: true, wrt: ['b'] }),
  loss('narrow-values', 150, 24, 6, { bias: true }),
  loss('narrow-squared', 150, 24, 100, { bias: true, gradient: true, after: true }),
  loss('pairs-few', 77, 520, 117, { bias: true, gradient: true }),
  loss('pairs-rows', 3001, 20, 130, { bias: true, gradient: true }),
  // Matrices from one element to several tiles, wide and tall, alone, stacked and side by side.
  orth('one', [1, 1]),
  orth('row', [1, 70]),
  orth('column', [70, 1]),
  orth('small', [8, 8]),
  orth('square', [128, 128]),
  orth('wide', [40, 300]),
  orth('tall', [300, 130]),
  orth('odd', [65, 67]),
  orth('stack', [3, 2, 33, 20]),
  orth('twins', [96, 64], { count: 3 }),
  orth('steps', [50, 70], { options: { steps: 2, coefficients: [1.5, -0.5, 0], eps: 0 } }),
  // Sides of 64 and one more, of each count of tiles, wide and tall, even rows of four and not; alone, stacked and side by side.
  orth('thin-most', [64, 200]),
  orth('thin-tall', [999, 64]),
  orth('thin-odd', [31, 517]),
  orth('thin-columns', [517, 31]),
  orth('thin-47', [4099, 47]),
  orth('thin-16', [2050, 16]),
  orth('thin-row', [2, 9001]),
  orth('thin-stack', [2, 3, 130, 12]),
  orth('thin-twins', [48, 100], { count: 3 }),
  orth('thin-steps', [70, 60], { options: { steps: 9, coefficients: [2, -1.5, 0.5], eps: 1e-3 } }),
  orth('more-than-thin', [65, 500]),
  orth('twins-large', [96, 70], { count: 3 }),
  orth('stack-large', [3, 70, 90], { options: { steps: 2, coefficients: [1.5, -0.5, 0], eps: 0 } }),
  orth('none', [20, 30], { options: { steps: 0 } }),
];

const FORMS = [
  // Coefficients near 0 and at it, of a matrix that the products of pairs take: their scales' exponents are the largest.
  orth('linear', [96, 100], { options: { steps: 1, coefficients: [1, 0, 0] } }),
  orth('nearly-linear', [100, 70], { options: { steps: 2, coefficients: [0.5, -1e-12, 0] } }),
  // Losses by products of pairs whose rows' magnitudes are far apart: whole, and in pieces with K split.
  loss('far-rows', 128, 64, 512, { bias: true, gradient: true }),
  loss('far-rows-pieces', 330, 40, 700, { bias: true, gradient: true, tuning: { loss: { piece: 1 } } }),
  // The loss by large tiles: of the logits alone, of the gradients with K split and whole, in pieces.
  loss('tall-logits', 517, 131, 9001, { bias: true, gradient: true }),
  loss('tall-logits-pieces', 517, 131, 9001, { bias: true, gradient: true, tuning: { loss: { piece: 2 ** 24 } } }),
  loss('tall-values', 517, 131, 9001, { bias: true }),
  loss('large-split', 1301, 201, 16001, { bias: true, gradient: true }),
  loss('large-whole', 2499, 1999, 2401, { bias: true, gradient: true }),
  loss('large-pieces', 513, 1001, 7001, { gradient: true, tuning: { loss: { piece: 2 ** 24 } } }),
  loss('tall-after', 517, 131, 9001, { bias: true, gradient: true, after: true }),
  // Matrices by 64 x 64 tiles whose upper half is computed, split along K, wide and tall.
  orth('half', [771, 1301]),
  orth('half-tall', [1301, 771]),
  // By 128 x 128 tiles, X by each of the larger: stacks wide and tall, and one whose leftover tiles are split.
  orth('square-tall-tiles', [128, 200, 250]),
  orth('square-tall-tiles-tall', [128, 250, 200]),
  orth('square-wide-tiles', [256, 100, 250]),
  orth('square-wide-tiles-tall', [128, 300, 250]),
  orth('square-tiles', [171, 100, 300]),
  orth('square-tiles-tall', [171, 300, 100]),
  orth('square-split', [60, 500, 520], { options: { steps: 2 } }),
  // Equal stacks side by side, and matrices whose workgroups are dealt to the XCDs (eight of them, or a multiple).
  orth('stack-twins', [8, 100, 90], { count: 3 }),
  orth('stack-twins-odd', [3, 90, 100], { count: 2 }),
  orth('eight', [90, 101], { count: 8 }),
  orth('twice', [96, 100], { twice: true, count: 2, options: { steps: 2 } }),
  // Attention of few rows, of many, of many that share their split operands; heads of whole tiles and not. With gradients, and without.
  ...[false, true].reduce((all, gradient) => all.concat([
    ['few', [2, 5, 6, 24], [2, 30, 2, 24], { window: 11, sinks: 2 }], ['more', [2, 9, 4, 24], [2, 30, 2, 24], { window: 11, sinks: 2 }], ['few-whole', [1, 13, 2, 64], [1, 13, 2, 64], {}],
    ['wide', [2, 80, 2, 64], [2, 80, 2, 64], { window: 37, sinks: 3 }], ['wide-large', [1, 70, 2, 160], [1, 70, 2, 160], {}],
    ['packed', [1, 300, 4, 64], [1, 300, 2, 64], { window: 260, sinks: 5 }], ['packed-odd', [1, 280, 4, 40], [1, 280, 2, 40], {}],
  ].map(([name, q, k, options]) => window(`window-${name}${gradient ? '' : '-forward'}`, q, k, options, { gradient }))), []),
  embedding('embedding-order', [900], 40, 36, { scale: 3, gradient: true }),
  window('window-few-splits', [2, 1, 4, 64], [2, 2000, 2, 64], { sinks: 2, window: 1900 }, { gradient: true }),
  window('window-few-large', [2, 4, 6, 160], [2, 21, 2, 160], { window: 11, sinks: 2 }, { gradient: true }),
  residual('residual-small-rms', [37, 64], ['gain'], { eps: 0 }, { gradient: true }),
  residual('residual-small-layer', [37, 64], ['gain'], { eps: 0, norm: 'layer' }, { gradient: true }),
  // Two blocks of rows, and in the gradients of keys, a wavefront (window.js blocksOf): sizes that end inside their tiles, heads of whole tiles and not.
  window('window-blocks', [32, 151, 16, 20], [32, 151, 4, 20], { window: 130, sinks: 3 }, { lengths: true, gradient: true }),
  window('window-blocks-odd', [32, 69, 32, 37], [32, 139, 4, 37], {}, { lengths: true, gradient: true }),
  window('window-blocks-first', [32, 150, 16, 64], [32, 150, 4, 64], { queries: 'first', window: 125, sinks: 70 }, { lengths: true, gradient: true }),
  window('window-blocks-large', [32, 141, 16, 112], [32, 141, 4, 112], { window: 130, sinks: 5 }, { lengths: true, gradient: true }),
  window('window-blocks-largest', [16, 139, 32, 128], [16, 201, 4, 128], {}, { lengths: true }),
  // Of each form, with a scale that leaves scores in powers of two exact where the operands are few bits.
  ...[
    ['few', [2, 5, 6, 24], [2, 30, 2, 24], { window: 11, sinks: 2 }], ['wide', [2, 80, 2, 64], [2, 80, 2, 64], { window: 37, sinks: 3 }], ['wide-large', [1, 70, 2, 160], [1, 70, 2, 160], {}],
    ['packed', [1, 300, 4, 64], [1, 300, 2, 64], { window: 260, sinks: 5 }], ['packed-odd', [1, 280, 4, 40], [1, 280, 2, 40], {}], ['packed-large', [1, 300, 4, 128], [1, 300, 2, 128], {}],
    ['packed-blocks', [32, 150, 16, 24], [32, 150, 4, 24], { window: 130, sinks: 3 }],
  ].map(([name, q, k, options]) => window(`window-exact-${name}`, q, k, Object.assign({ scale: Math.LN2 / 4 }, options), { gradient: true })),
];

const r = (B, T, H, dh, axes, gradient, twin) => rotary(null, [B, T, H, dh], axes === 1 ? [B, T] : [B, T, axes],
  { gain: true, gradient, twin: [B, T, twin, dh], options: { axis: 1, base: 10000, eps: 1e-5,
    sections: axes === 1 ? [dh / 2] : [dh / 2 - 2 * Math.floor(3 * dh / 16), Math.floor(3 * dh / 16), Math.floor(3 * dh / 16)] } });
const MEASURED = [
  r(32, 1, 8, 64, 1, false, 2), r(64, 128, 4, 64, 1, true, 4), r(1, 8191, 16, 128, 3, true, 4), r(2, 32768, 32, 128, 1, false, 8),
  loss(null, 128, 64, 96, { bias: true }), loss(null, 8192, 256, 96, { bias: true, gradient: true }), loss(null, 4096, 512, 32768, {}),
  loss(null, 1001, 515, 50021, { bias: true, gradient: true }), loss(null, 8192, 1024, 65536, { gradient: true }),
  orth(null, [256, 256], { count: 16 }), orth(null, [1300, 777]), orth(null, [4096, 4096], { count: 2 }),
];

// The sizes of perf/more_operators.py.
const e = (N, V, d, gradient) => embedding(null, [N], V, d, { scale: Math.sqrt(d), gradient });
const n = (N, d, vectors, options, gradient) => residual(null, [N, d], vectors, Object.assign({ eps: 1e-5 }, options), { gradient });
const w = (B, T, S, H, Hk, dh, options, more) => window(null, [B, T, H, dh], [B, S, Hk, dh], Object.assign({ sinks: 0, queries: T === S ? 'first' : 'last' }, options), more);
const MEASURED_CONTEXT = [
  e(32, 32768, 1024, false), e(8192, 96, 256, true), e(32768, 65536, 1024, true),
  n(32, 1024, ['gain', 'postGain'], { residual: 0.75, norm: 'rms' }, false), n(8192, 256, ['gain', 'bias'], { norm: 'layer' }, true),
  n(8189, 4095, ['gain', 'postGain', 'gate'], { residual: 0.75, norm: 'rms' }, true),
  w(32, 1, 4096, 8, 2, 64, { window: 1024, sinks: 4 }, { lengths: true }), w(4, 1, 131072, 8, 2, 64, {}, { lengths: true }),
  w(64, 128, 128, 4, 4, 64, {}, { gradient: true }), w(3, 1001, 1001, 6, 3, 80, { window: 257, sinks: 3 }, { lengths: true, gradient: true }),
  w(2, 16384, 16384, 16, 4, 128, { window: 1024, sinks: 4 }, {}), w(1, 8192, 8192, 8, 2, 64, {}, { gradient: true }),
];

module.exports = { operatorGraph, CASES, FORMS, MEASURED, CONTEXT, MEASURED_CONTEXT };
