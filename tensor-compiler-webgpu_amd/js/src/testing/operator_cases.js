'use strict';
// Graphs of the operators that are one node each (ir/operators.js), from plain
// descriptions: those of their GPU tests (CASES; FORMS, whose tests name them) and of their measurement (MEASURED).
//   { family: 'rotary', x, positions, gain?, gradient?, options }   a second x where `twin`
//       gives its shape; `twice`: rotated, and the result again
//   { family: 'loss', N, d, V, bias?, gradient?, wrt?, after? }     wrt: 'h', 'W', 'b' (default all); `after`: the
//       losses' cotangent depends on the losses, so their gradients cannot run beside them
//   { family: 'orthogonalize', x, count, options, twice }

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
  } else throw new Error(`no operator '${c.family}'`);
  if (!c.gradient) return { graph: g, keep: outs, names };
  const G = grad(g, outs, wrt);
  return { graph: G.graph, keep: outs.concat(G.grads), names: names.concat(grads) };
}

const rotary = (name, x, positions, more) => Object.assign({ name, family: 'rotary', x, positions }, more);
const loss = (name, N, d, V, more) => Object.assign({ name, family: 'loss', N, d, V }, more);
const orth = (name, x, more) => Object.assign({ name, family: 'orthogonalize', x }, more);

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

module.exports = { operatorGraph, CASES, FORMS, MEASURED };
