'use strict';
// Operators of a transformer's training step that are one node each, beside the
// reference's op set (src/ir/shapes.js:51 in abho7/tensor-compiler-webgpu, whose graphs
// never hold them): their attributes and shape rules, for the builder (graph.js) and
// inferShape (shapes.js). Every value is float32, class indices and positions included.
//
// rotary            [x, positions] or [x, positions, gain] -> x's shape. Rows of the last
//   axis (dh elements: one head of one token) are normalised by their root mean square
//   and the gain, where there is one, and rotated: pair j of dims (a, b) by
//   angle(j) = position on axis axes[j] · frequencies[j] to (a cos - b sin, b cos + a sin).
//   `axis` is the tokens' axis. R = frequencies.length pairs are rotated: dims (j, j + R)
//   for pairs 'halves', (2j, 2j + 1) for 'adjacent'; dims from 2R on are not.
// rotaryGrad        [x, positions, (gain,) dy], attrs.part 'dx' | 'dgain'.
// linearCrossEntropy  [h, W, targets] or [h, W, targets, bias] -> [N]. Row r's loss is
//   logsumexp(z) - z[targets[r]], z = h[r]·W + bias; 0 for a row left out, whose target is
//   not a whole number in 0..V-1 (padding: -1).
// linearCrossEntropyGrad  [h, W, targets, (bias,) dloss], attrs.part 'dh' | 'dW' | 'dbias'.
// orthogonalize     [x] -> x's shape: each matrix of the last two axes divided by its
//   Frobenius norm plus eps, then `steps` times X <- a·X + (b·A + c·A·A)·X, A = X·Xᵀ (on the
//   side of fewer rows). An optimizer's operator: it has no gradient.

const isNumber = (v) => typeof v === 'number' && Number.isFinite(v);

/**
 * The rotation's frequencies and axes from its options: `sections`, the rotated pairs of
 * each position axis in turn (default: all dh/2 on one), `base` (10000): pair j turns by
 * base^(-j/R) a position, R the pairs in all; with `restart`, each section counts its own
 * pairs from 0 over its own length. `frequencies` and `axes` given in full take their place.
 */
function rotaryPairs(dh, options) {
  const o = options || {};
  if (o.frequencies) {
    const frequencies = Array.from(o.frequencies, Number);
    return { frequencies, axes: o.axes ? Array.from(o.axes, Number) : frequencies.map(() => 0) };
  }
  const sections = o.sections === undefined ? [Math.floor(dh / 2)] : Array.from(o.sections, Number);
  const base = o.base === undefined ? 10000 : o.base;
  if (!sections.every((s) => Number.isInteger(s) && s >= 0)) throw new Error(`rotary: sections are counts of pairs, not ${JSON.stringify(o.sections)}`);
  if (!(isNumber(base) && base > 0)) throw new Error(`rotary: base ${base}`);
  const R = sections.reduce((a, b) => a + b, 0);
  const frequencies = [], axes = [];
  sections.forEach((s, axis) => {
    for (let k = 0; k < s; k++) {
      frequencies.push(o.restart ? base ** (-k / s) : base ** (-frequencies.length / R));
      axes.push(axis);
    }
  });
  return { frequencies, axes, count: sections.length };
}

const product = (s) => s.reduce((a, b) => a * b, 1);
const same = (a, b) => a.length === b.length && a.every((d, i) => d === b[i]);

/** Operator rules for shapes.js: op -> { arity: [least, most], rule(shapes, attrs, op) }, throwing `ShapeError`. */
function operatorRules(ShapeError, fmt) {
  const need = (ok, message) => { if (!ok) throw new ShapeError(message); };

  function rotaryShape([x, pos, gain], attrs, op) {
    need(x.length >= 2, `${op} of ${fmt(x)}: tokens and a head take two axes or more`);
    const r = x.length, dh = x[r - 1], a = attrs.axis;
    need(Number.isInteger(a) && a >= 0 && a < r - 1, `${op} of ${fmt(x)}: no token axis ${a}`);
    need(Number.isInteger(attrs.positionAxes) && attrs.positionAxes >= 1 && attrs.positionAxes <= 256, `${op}: ${attrs.positionAxes} position axes (1 to 256)`);
    const { frequencies: f, axes } = attrs;
    need(Array.isArray(f) && f.every(isNumber) && 2 * f.length <= dh, `${op}: at most ${Math.floor(dh / 2)} finite frequencies for heads of ${dh}`);
    need(Array.isArray(axes) && axes.length === f.length && axes.every((i) => Number.isInteger(i) && i >= 0 && i < attrs.positionAxes),
      `${op}: each pair takes one of ${attrs.positionAxes} position axes`);
    need(attrs.pairs === 'halves' || attrs.pairs === 'adjacent', `${op}: pairs are 'halves' or 'adjacent', not '${attrs.pairs}'`);
    const tail = attrs.positionAxes > 1 ? [attrs.positionAxes] : [];
    need(same(pos, [x[a]].concat(tail)) || (a > 0 && same(pos, [x[0], x[a]].concat(tail))),
      `${op}: positions of ${fmt(pos)} for ${fmt(x)}: expected ${fmt([x[a]].concat(tail))}${a > 0 ? ` or ${fmt([x[0], x[a]].concat(tail))}` : ''}`);
    if (gain) {
      need(same(gain, [dh]), `${op}: a gain of ${fmt(gain)} for heads of ${dh}`);
      need(isNumber(attrs.eps) && attrs.eps >= 0, `${op}: eps ${attrs.eps}`);
    }
    return x.slice();
  }

  function lossShape([h, W, t, bias], attrs, op) {
    need(h.length === 2 && W.length === 2 && h[1] === W[0], `${op} of ${fmt(h)} by ${fmt(W)}: [rows, d] by [d, classes]`);
    need(same(t, [h[0]]), `${op}: targets of ${fmt(t)} for ${h[0]} rows`);
    if (bias) need(same(bias, [W[1]]), `${op}: a bias of ${fmt(bias)} for ${W[1]} classes`);
    need(W[1] <= 2 ** 24, `${op}: ${W[1]} classes (a float32 names 2^24)`);
    return [h[0]];
  }

  return {
    rotary: { arity: [2, 3], rule: rotaryShape },
    rotaryGrad: {
      arity: [3, 4],
      rule(s, attrs, op) {
        const x = rotaryShape(s.slice(0, -1), attrs, op), dy = s[s.length - 1];
        need(same(dy, x), `${op}: a gradient of ${fmt(dy)} for ${fmt(x)}`);
        need(attrs.part === 'dx' || (attrs.part === 'dgain' && s.length === 4), `${op}: no part '${attrs.part}'`);
        return attrs.part === 'dx' ? x : s[2].slice();
      },
    },
    linearCrossEntropy: { arity: [3, 4], rule: lossShape },
    linearCrossEntropyGrad: {
      arity: [4, 5],
      rule(s, attrs, op) {
        const rows = lossShape(s.slice(0, -1), attrs, op), dy = s[s.length - 1];
        need(same(dy, rows), `${op}: a gradient of ${fmt(dy)} for ${rows[0]} losses`);
        const part = { dh: s[0], dW: s[1], dbias: s.length === 5 ? s[3] : undefined }[attrs.part];
        need(part, `${op}: no part '${attrs.part}'`);
        return part.slice();
      },
    },
    orthogonalize: {
      arity: [1, 1],
      rule([x], attrs, op) {
        need(x.length >= 2, `${op} of ${fmt(x)}: a matrix takes two axes or more`);
        need(Number.isInteger(attrs.steps) && attrs.steps >= 0 && attrs.steps <= 64, `${op}: steps ${attrs.steps}`);
        need(Array.isArray(attrs.coefficients) && attrs.coefficients.length === 3 && attrs.coefficients.every(isNumber),
          `${op}: three finite coefficients, not ${JSON.stringify(attrs.coefficients)}`);
        need(isNumber(attrs.eps) && attrs.eps >= 0, `${op}: eps ${attrs.eps}`);
        need(Number.isFinite(singularBound(attrs)), `${op}: the coefficients ${JSON.stringify(attrs.coefficients)} let singular values grow past 16 in ${attrs.steps} steps`);
        return x.slice();
      },
    },
  };
}

/**
 * The largest singular value that `steps` of the polynomial p(s) = a·s + b·s^3 + c·s^5 can
 * reach from [0, 1]: each step's largest |p| over the last one's interval (p at its ends
 * and where p' = a + 3b·s^2 + 5c·s^4 is 0). Infinity past 16, the range that the kernels'
 * halves are scaled for.
 */
function singularBound(attrs) {
  const [a, b, c] = attrs.coefficients;
  const p = (s) => Math.abs(s * (a + s * s * (b + s * s * c)));
  let top = 1, most = 1;
  for (let k = 0; k < attrs.steps; k++) {
    const at = [top];
    const root = (s2) => { if (s2 > 0 && s2 < top * top) at.push(Math.sqrt(s2)); };
    // The roots of 5c·t² + 3b·t + a in t = s², q the sum of two terms of one sign: a root stays where c is next to 0.
    const d = 9 * b * b - 20 * a * c;
    if (d >= 0) {
      const q = -0.5 * (3 * b + (b < 0 ? -1 : 1) * Math.sqrt(d));
      root(q / (5 * c));
      root(a / q);
    }
    top = Math.max(...at.map(p));
    most = Math.max(most, top);
    if (!(most <= 16)) return Infinity;
  }
  return most;
}

module.exports = { rotaryPairs, operatorRules, singularBound, product };
