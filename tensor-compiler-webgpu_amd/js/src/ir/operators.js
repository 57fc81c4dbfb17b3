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
// embedding         [tokens, table] -> tokens' shape and the table's columns: scale · table[token],
//   zeros where the token is not a whole number in 0..rows-1 (padding: -1).
// embeddingGrad     [tokens, dy], attrs.rows the table's rows -> [rows, d]: each row scale times the
//   sum of its tokens' rows of dy.
// residualNorm      [x, y, (gain, (bias,)) (postGain, (postBias,)) (gate)], attrs.part 'h' | 'n'. Rows of the last
//   axis: h = residual·x + gate·N(y), n = N(h). N(v) = (v - mean) / sqrt(mean of (v - mean)² + eps)·gain + bias for norm
//   'layer', v / sqrt(mean of v² + eps)·gain for 'rms'; of y it is there with a postGain (else N(y) = y), of h with a gain.
//   A gate of [d] or of x's shape. Which operands there are: attrs.pre, bias, post, postBias, gate.
// residualNormGrad  [x, y, (gain,) (postGain, (postBias,)) (gate,) (dh,) (dn)], attrs.has names the last two; attrs.part
//   'dx' | 'dy' | 'dgain' | 'dbias' | 'dpostGain' | 'dpostBias' | 'dgate'.
// windowAttention   [q, k, v] or [q, k, v, lengths]: q [B, T, H, dh], k and v [B, S, Hk, dh] (query heads h·H/Hk ... share key
//   head h), lengths [B]; attrs.part 'o' (q's shape) or 'lse' [B, T, H], the logarithm of the sums that o was divided by. Sequence
//   b has its first L = lengths[b] keys (rounded down, within 0..S, NaN as 0; default S). Query t stands at position t
//   (attrs.queries 'first') or L - T + t ('last') and sees the keys j <= position that are within attrs.window (position - window < j; 0:
//   all) or among the first attrs.sinks. A query whose position is not in 0..L-1 sees nothing: zeros, and -Infinity in lse.
// windowAttentionGrad  [q, k, v, (lengths,) o, lse, dy], attrs.part 'dq' | 'dk' | 'dv'.

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

  function embeddingShape([t, table], attrs, op) {
    need(table.length === 2, `${op}: a table of ${fmt(table)}: [rows, d]`);
    need(table[0] <= 2 ** 24, `${op}: ${table[0]} rows (a float32 names 2^24)`);
    need(isNumber(attrs.scale), `${op}: scale ${attrs.scale}`);
    return t.concat([table[1]]);
  }

  /** The operands of a residualNorm after x and y, by name; `grad`: those that its gradient reads. */
  function residualOperands(s, attrs, op, grad) {
    const names = [attrs.pre && 'gain', attrs.bias && !grad && 'bias', attrs.post && 'postGain', attrs.postBias && 'postBias', attrs.gate && 'gate'].filter(Boolean);
    const more = grad ? attrs.has : [];
    const [x, y] = s, d = x[x.length - 1];
    need(x.length >= 1 && same(x, y), `${op} of ${fmt(x)} and ${fmt(y)}: a stream and a branch of one shape`);
    need(s.length === 2 + names.length + more.length, `${op}: ${s.length} operands for ${['x', 'y'].concat(names, more).join(', ')}`);
    need(attrs.norm === 'rms' || attrs.norm === 'layer', `${op}: norms are 'rms' or 'layer', not '${attrs.norm}'`);
    need(attrs.norm === 'layer' || !(attrs.bias || attrs.postBias), `${op}: a norm by the root mean square has no bias`);
    need((attrs.pre || !attrs.bias) && (attrs.post || !attrs.postBias), `${op}: a bias without its gain`);
    need(isNumber(attrs.eps) && attrs.eps >= 0, `${op}: eps ${attrs.eps}`);
    need(isNumber(attrs.residual), `${op}: a residual scale of ${attrs.residual}`);
    const at = {};
    names.forEach((n, k) => {
      at[n] = s[2 + k];
      need(same(at[n], [d]) || (n === 'gate' && same(at[n], x)), `${op}: a ${n} of ${fmt(at[n])} for rows of ${d}`);
    });
    more.forEach((n, k) => {
      const g = s[2 + names.length + k];
      need((n === 'dh' || (n === 'dn' && attrs.pre)) && same(g, x), `${op}: a gradient ${n} of ${fmt(g)} for ${fmt(x)}`);
    });
    return at;
  }

  function windowShape([q, k, v, lengths], attrs, op) {
    need(q.length === 4 && k.length === 4, `${op} of ${fmt(q)} by ${fmt(k)}: [batch, tokens, heads, head size]`);
    need(same(k, v), `${op}: keys of ${fmt(k)} and values of ${fmt(v)}`);
    need(q[0] === k[0] && q[3] === k[3] && q[2] % k[2] === 0, `${op} of ${fmt(q)} by ${fmt(k)}: equal batches and head sizes, and a whole number of query heads to a key head`);
    if (lengths) {
      need(same(lengths, [q[0]]), `${op}: lengths of ${fmt(lengths)} for ${q[0]} sequences`);
      need(k[1] <= 2 ** 24, `${op}: lengths up to ${k[1]} keys (a float32 names 2^24)`);
    }
    const whole = (n) => Number.isInteger(n) && n >= 0 && n < 2 ** 31;
    need(whole(attrs.window), `${op}: a window of ${attrs.window}`);
    need(whole(attrs.sinks), `${op}: ${attrs.sinks} sinks`);
    need(isNumber(attrs.scale), `${op}: scale ${attrs.scale}`);
    need(attrs.queries === 'first' || attrs.queries === 'last', `${op}: queries are the 'first' or the 'last', not '${attrs.queries}'`);
    return { o: q.slice(), lse: q.slice(0, 3) };
  }

  return {
    embedding: { arity: [2, 2], rule: embeddingShape },
    embeddingGrad: {
      arity: [2, 2],
      rule([t, dy], attrs, op) {
        const d = dy[dy.length - 1];
        need(Number.isInteger(attrs.rows) && attrs.rows >= 1, `${op}: ${attrs.rows} rows`);
        need(same(dy, embeddingShape([t, [attrs.rows, d]], attrs, op)), `${op}: a gradient of ${fmt(dy)} for tokens of ${fmt(t)}`);
        return [attrs.rows, d];
      },
    },
    residualNorm: {
      arity: [2, 7],
      rule(s, attrs, op) {
        residualOperands(s, attrs, op, false);
        need(attrs.part === 'h' || (attrs.part === 'n' && attrs.pre), `${op}: no part '${attrs.part}'`);
        return s[0].slice();
      },
    },
    residualNormGrad: {
      arity: [3, 8],
      rule(s, attrs, op) {
        need(Array.isArray(attrs.has) && attrs.has.length >= 1 && attrs.has.length <= 2 && new Set(attrs.has).size === attrs.has.length, `${op}: gradients ${JSON.stringify(attrs.has)}`);
        const at = residualOperands(s, attrs, op, true), dn = attrs.has.includes('dn');
        const part = { dx: s[0], dy: s[1], dgain: dn ? at.gain : undefined, dbias: dn && attrs.bias ? at.gain : undefined, dpostGain: at.postGain, dpostBias: at.postBias, dgate: at.gate }[attrs.part];
        need(part, `${op}: no part '${attrs.part}'`);
        return part.slice();
      },
    },
    windowAttention: {
      arity: [3, 4],
      rule(s, attrs, op) {
        const part = windowShape(s, attrs, op)[attrs.part];
        need(part, `${op}: no part '${attrs.part}'`);
        return part;
      },
    },
    windowAttentionGrad: {
      arity: [6, 7],
      rule(s, attrs, op) {
        const to = windowShape(s.slice(0, -3), attrs, op), [o, lse, dy] = s.slice(-3);
        need(same(o, to.o) && same(lse, to.lse) && same(dy, to.o), `${op}: ${fmt(o)}, ${fmt(lse)} and a gradient of ${fmt(dy)} for queries of ${fmt(s[0])}`);
        const part = { dq: s[0], dk: s[1], dv: s[2] }[attrs.part];
        need(part, `${op}: no part '${attrs.part}'`);
        return part.slice();
      },
    },
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
