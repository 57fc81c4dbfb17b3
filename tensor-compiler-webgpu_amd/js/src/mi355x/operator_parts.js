'use strict';
// What the launches of the operators that are one node each (operators.js) are built from: a
// kernel's record, how its text reaches its launch's argument block, and the mark of parts that run as one launch.

const { kernelText } = require('./codegen');

const ceil = (a, b) => Math.ceil(a / b);
const align = (n, to) => ceil(n, to) * to;

/** A double as a C++ literal that reads back as itself. */
function double(v) {
  const t = String(v);
  return /[.e]/.test(t) ? t : `${t}.0`;
}

/** One kernel record. */
function kernel(kind, text, grid, threads, more) {
  const k = kernelText(kind, text);
  return Object.assign({ name: k.name, source: k.source, grid, block: [threads, 1, 1], lds: 0 }, more || {});
}

/**
 * How a kernel's text reaches its launch: alone, `A` (TcmiArgs) with the part's output in
 * A.out; as one of `parts` in a joint launch, member k of its argument block for the k-th part, the
 * operands and the workspace in member 0's. With several `groups` of them (a joint launch of equal nodes), workgroups'
 * z index is the group, its members one after another, its workspace `floats` long.
 */
function entry(parts, groups, floats) {
  if (!parts) return { sig: 'const TcmiArgs A', open: '', out: () => 'A.out', ws: 'A.ws' };
  const n = parts.length;
  if (groups > 1) {
    return { sig: `const TcmiBatch<${n * groups}> B`, open: `  const TcmiPtrs* const M = B.m + ${n}u * blockIdx.z;\n  const TcmiPtrs& A = M[0];\n`,
      out: (part) => `M[${parts.indexOf(part)}].out`, ws: `A.ws + blockIdx.z * (size_t)${floats}u` };
  }
  return { sig: `const TcmiBatch<${n}> B`, open: '  const TcmiPtrs& A = B.m[0];\n', out: (part) => `B.m[${parts.indexOf(part)}].out`, ws: 'A.ws' };
}

/** Members of a kernel's struct of sizes: whole numbers of the types that `types` names (default uint32_t), truth values. */
function constants(z, types) {
  return Object.keys(z).map((k) => (typeof z[k] === 'boolean' ? `  static constexpr bool ${k} = ${z[k]};`
    : (types || {})[k] === 'int' ? `  static constexpr int ${k} = ${z[k]};`
      : `  static constexpr ${(types || {})[k] || 'uint32_t'} ${k} = ${z[k]}u;`)).join('\n');
}

/**
 * Marks kernel `k` as the first of part `part` of a launch whose parts `build(parts, groups)` forms
 * together, in `order`. They read the same first `operands` operands (default: all). `groups`: whether it forms those
 * parts of several nodes of one key.
 */
function joint(k, part, order, key, build, operands, groups) {
  Object.defineProperty(k, 'part', { value: part });
  Object.defineProperty(k, 'joint', { value: { name: JSON.stringify(key), order, build, operands, groups: !!groups } });
}

module.exports = { ceil, align, double, constants, kernel, entry, joint };
