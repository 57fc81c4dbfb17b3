'use strict';
// Runs MI355X launch lists: the drop-in for the reference's WebGPU runner.
//
// HipRunner.run(graph, lowered, inputs, { canary }) has the contract of
// GpuRunner.run (src/gpu/runtime.js:60-128 in abho7/tensor-compiler-webgpu):
// one buffer per node, inputs and constants uploaded, every launch in order on
// one stream, every node read back, and with `canary` each buffer padded past
// its end with 0xdeadbeef that must survive. It returns { values, canaryIntact }
// (a Float32Array per node) and throws on any HIP error; a fatal error makes
// the runner `lost` for good (runtime.js:23,61).
//
// runLocal(graph, lowered, values) is the node-local executor
// (src/gpu/harness-m3b.js:86-140): each launch reads float32-rounded reference
// operands and writes its own output, so no launch sees another's error.
//
// prepare(graph, lowered) makes a Program: buffers, packed argument blocks and
// function handles made once, then run() issues every launch with one native
// call (or replays a captured HIP graph) — what the trainer and bench use.
// With { arena: { keep } } its node buffers are placed by live range in one
// allocation (arena.js): only inputs, constants and `keep` stay readable. With
// { streams: n } (2..4) independent launches are issued on n streams
// (schedule.js), one native call per run as before.

const crypto = require('crypto');
const fs = require('fs');
const path = require('path');
const { size } = require('../ir/shapes');
const { addon, CACHE } = require('./addon');
const { kernelSources } = require('./lower');
const { MAX_IN, MAX_P } = require('./codegen');
const { planArena } = require('./arena');
const { scheduleLaunches } = require('./schedule');

const CANARY_BITS = 0xdeadbeef;
const CANARY_PAD = 256;           // words past the end of every buffer
const ARG_BYTES = MAX_IN * 8 + 8 + 8 + MAX_P * 4;
const PTR_BYTES = MAX_IN * 8 + 8 + 8;     // one member of a batched launch's block

const PRELUDE = '#include "tcmi_device.h"\n';

/** One translation unit holding `sources` (name -> text), in name order so the text is canonical. */
function translationUnit(sources) {
  const names = Array.from(sources.keys()).sort();
  return PRELUDE + names.map((n) => sources.get(n)).join('\n');
}

// The kernel index: for every kernel compiled before (here or at build time),
// the translation unit it was compiled in, so a later process loads that unit's
// cached code object instead of compiling the kernel again in a new unit.
// <cache>/index/<key>.tu holds a unit's text, <key>.names its kernels' names.
const INDEX = path.join(CACHE, 'index');
let indexMap = null;   // kernel name -> unit key, read once per process

function unitKey(text) { return crypto.createHash('sha256').update(text).digest('hex').slice(0, 32); }

function writeAtomic(file, text) {
  const tmp = `${file}.${process.pid}.tmp`;
  fs.writeFileSync(tmp, text);
  fs.renameSync(tmp, file);
}

function loadIndex() {
  if (indexMap) return indexMap;
  indexMap = new Map();
  let files = [];
  try { files = fs.readdirSync(INDEX); } catch (e) { return indexMap; }
  for (const f of files) {
    if (!f.endsWith('.names')) continue;
    const key = f.slice(0, -'.names'.length);
    for (const name of fs.readFileSync(path.join(INDEX, f), 'utf8').split('\n')) if (name) indexMap.set(name, key);
  }
  return indexMap;
}

/** Record that the kernels `names` are in unit `text`; an index that cannot be written only costs compile time. */
function indexUnit(names, text) {
  const key = unitKey(text);
  const map = loadIndex();
  for (const n of names) map.set(n, key);
  try {
    fs.mkdirSync(INDEX, { recursive: true });
    const tu = path.join(INDEX, `${key}.tu`);
    if (!fs.existsSync(tu)) writeAtomic(tu, text);
    writeAtomic(path.join(INDEX, `${key}.names`), names.join('\n') + '\n');
  } catch (e) {
    // read-only cache: nothing to record
  }
}

/** The text of indexed unit `key`, or null. */
function unitText(key) {
  try {
    return fs.readFileSync(path.join(INDEX, `${key}.tu`), 'utf8');
  } catch (e) {
    return null;
  }
}

/**
 * Compile (into the on-disk cache only; no GPU needed) every kernel of `lists`
 * as one module; with `select(name)`, only the kernels it accepts.
 */
function precompile(lists, arch, select) {
  const all = new Map();
  for (const l of lists) for (const [name, src] of kernelSources(l)) if (!select || select(name)) all.set(name, src);
  if (!all.size) return 0;
  const text = translationUnit(all);
  addon().precompile(text, '', arch || 'gfx950');
  indexUnit(Array.from(all.keys()), text);
  return all.size;
}

/** Pack one kernel's argument block (TcmiArgs in tcmi_device.h). */
function packArgs(view, offset, inPtrs, outPtr, wsPtr, params) {
  const put64 = (at, v) => {
    view.setUint32(at, v % 4294967296, true);
    view.setUint32(at + 4, Math.floor(v / 4294967296), true);
  };
  if (inPtrs.length > MAX_IN) throw new Error(`launch has ${inPtrs.length} operands (max ${MAX_IN})`);
  if (params.length > MAX_P) throw new Error(`launch has ${params.length} parameters (max ${MAX_P})`);
  for (let k = 0; k < MAX_IN; k++) put64(offset + 8 * k, k < inPtrs.length ? inPtrs[k] : 0);
  put64(offset + MAX_IN * 8, outPtr);
  put64(offset + MAX_IN * 8 + 8, wsPtr);
  for (let k = 0; k < MAX_P; k++) view.setUint32(offset + MAX_IN * 8 + 16 + 4 * k, k < params.length ? params[k] : 0, true);
}

/** Pack one member of a batched launch's argument block (TcmiPtrs in tcmi_device.h). */
function packPtrs(view, offset, inPtrs, outPtr, wsPtr) {
  const put64 = (at, v) => {
    view.setUint32(at, v % 4294967296, true);
    view.setUint32(at + 4, Math.floor(v / 4294967296), true);
  };
  if (inPtrs.length > MAX_IN) throw new Error(`launch has ${inPtrs.length} operands (max ${MAX_IN})`);
  for (let k = 0; k < MAX_IN; k++) put64(offset + 8 * k, k < inPtrs.length ? inPtrs[k] : 0);
  put64(offset + MAX_IN * 8, outPtr);
  put64(offset + MAX_IN * 8 + 8, wsPtr);
}

/**
 * The perf lowering's buffer sharing: alias (node -> node whose buffer it uses) and
 * folded (no buffer: folded into its consumers, or dead).
 */
function sharing(lowered) {
  const alias = new Map(lowered.aliases || []);
  for (const [k, v] of alias) if (alias.has(v)) throw new Error(`alias chain ${k} -> ${v} is not resolved`);
  return { alias, folded: new Set((lowered.folded || []).concat(lowered.dead || [])) };
}

/**
 * Refuse a launch list with a kernel that reads and writes one element past its
 * buffers (the off-by-one sabotage) unless every buffer carries a canary pad.
 */
function requirePad(lowered, padded) {
  if (padded) return;
  for (const l of lowered.launches) for (const k of l.kernels) {
    if (k.needsPad) throw new Error(`launch of node ${l.node} (${k.name}) runs past its buffers: run it with canaries`);
  }
}

function constData(node) {
  const n = size(node.shape);
  const v = node.attrs.value;
  if (typeof v === 'number') return new Float32Array(Math.max(1, n)).fill(v);
  return Float32Array.from(v);
}

class HipRunner {
  static create() {
    const a = addon();
    a.init();
    return new HipRunner(a);
  }

  constructor(a) {
    this.a = a;
    this.loaded = new Map();    // kernel name (a hash of its source) -> function handle
    this.units = new Map();     // indexed unit key -> its loaded module (null: unreadable)
  }

  get lost() { return this.a.lost(); }

  info() { return Object.assign({ version: this.a.version(), compileOptions: this.a.compileOptions() }, this.a.info()); }

  /**
   * Function handles for every kernel of `lowered` (one launch list, or an
   * array of them): the kernels not loaded yet are compiled together as one
   * module (one hiprtc call, cached on disk by its text). `apart`: every launch by itself.
   */
  functions(lowered, apart) {
    const lists = Array.isArray(lowered) ? lowered : [lowered];
    const missing = new Map();
    for (const l of lists) for (const [name, src] of kernelSources(l, apart)) if (!this.loaded.has(name)) missing.set(name, src);
    // Kernels compiled before in some unit: load that unit's module once per
    // process (a code-object cache hit) and take their functions from it.
    const index = loadIndex();
    for (const name of Array.from(missing.keys())) {
      const key = index.get(name);
      if (!key) continue;
      if (!this.units.has(key)) {
        const text = unitText(key);
        this.units.set(key, text === null ? null : this.a.compile(text, ''));
      }
      const module = this.units.get(key);
      if (module === null) continue;
      this.loaded.set(name, this.a.function(module, name));
      missing.delete(name);
    }
    if (missing.size) {
      const text = translationUnit(missing);
      const module = this.a.compile(text, '');
      for (const name of missing.keys()) this.loaded.set(name, this.a.function(module, name));
      indexUnit(Array.from(missing.keys()), text);
    }
    return this.loaded;
  }

  alloc(bytes) { return this.a.malloc(Math.max(16, Math.ceil(bytes / 16) * 16)); }

  /**
   * Launch every kernel of `lowered` with node buffers `bufs` (node id -> device address),
   * each batch of the perf lowering as one launch of its batched kernel.
   */
  launchAll(lowered, fns, bufs, outOf, ws) {
    const argBuf = new ArrayBuffer(ARG_BYTES);
    const view = new DataView(argBuf);
    const bytes = new Uint8Array(argBuf);
    const batchAt = new Map((lowered.batches || []).map((b) => [b.start, b]));
    const L = lowered.launches;
    for (let i = 0; i < L.length;) {
      const b = batchAt.get(i);
      if (b) {
        const block = new ArrayBuffer(b.count * PTR_BYTES);
        const bv = new DataView(block);
        for (let m = 0; m < b.count; m++) {
          const l = L[i + m];
          packPtrs(bv, m * PTR_BYTES, l.inputs.map((id) => bufs[id]), outOf ? outOf(l) : bufs[l.node], ws + m * b.wsStride);
        }
        for (const k of b.kernels) this.a.launch(fns.get(k.name), k.grid, k.block, k.lds, new Uint8Array(block));
        i += b.count;
        continue;
      }
      const l = L[i++];
      const out = outOf ? outOf(l) : bufs[l.node];
      packArgs(view, 0, l.inputs.map((id) => bufs[id]), out, ws, l.params);
      for (const k of l.kernels) this.a.launch(fns.get(k.name), k.grid, k.block, k.lds, bytes);
    }
  }

  async run(graph, lowered, inputs, options) {
    const canary = !!(options && options.canary);
    if (this.a.lost()) throw new Error('device lost');
    requirePad(lowered, canary);
    const a = this.a;
    const fns = this.functions(lowered);
    const n = graph.nodes.map((node) => size(node.shape));
    const cap = n.map((k) => (canary ? k + CANARY_PAD : k));
    const { alias, folded } = sharing(lowered);
    const bufs = [];
    const owned = [];
    let ws = 0;
    try {
      for (let i = 0; i < graph.nodes.length; i++) {
        if (alias.has(i)) bufs.push(bufs[alias.get(i)]);
        else if (folded.has(i)) bufs.push(0);
        else { const h = this.alloc(cap[i] * 4); bufs.push(h); owned.push(h); }
      }
      ws = this.alloc(lowered.workspace || 16);
      for (const node of graph.nodes) {
        const h = bufs[node.id];
        if (!h || alias.has(node.id)) continue;
        if (canary) a.fill32(h, 0, CANARY_BITS, cap[node.id]);
        if (node.op === 'input') {
          const v = inputs[node.attrs.name];
          if (v === undefined) throw new Error(`no value for input '${node.attrs.name}'`);
          if (v.length !== n[node.id]) throw new Error(`input '${node.attrs.name}' has ${v.length} values, needs ${n[node.id]}`);
          a.h2d(h, 0, v instanceof Float32Array ? v : Float32Array.from(v));
        } else if (node.op === 'const') {
          a.h2d(h, 0, constData(node).subarray(0, n[node.id]));
        }
      }
      this.launchAll(lowered, fns, bufs, null, ws);
      a.sync();
      const values = [], canaryIntact = [];
      for (const node of graph.nodes) {
        if (!bufs[node.id]) { values.push(null); canaryIntact.push(true); continue; }
        const out = new Float32Array(n[node.id]);
        a.d2h(bufs[node.id], 0, out);
        values.push(out);
        if (canary) canaryIntact.push(a.countNot32(bufs[node.id], n[node.id] * 4, CANARY_BITS, CANARY_PAD) === 0);
      }
      return { values, canaryIntact };
    } finally {
      for (const h of owned) a.free(h);
      if (ws) a.free(ws);
    }
  }

  /** Node-local run: every launch on float32 reference operands `values` (per node). */
  async runLocal(graph, lowered, values, options) {
    const canary = !!(options && options.canary);
    const a = this.a;
    requirePad(lowered, canary);
    const fns = this.functions(lowered);
    const n = graph.nodes.map((node) => size(node.shape));
    const ref = [], outs = new Map();
    let ws = 0;
    try {
      for (const node of graph.nodes) {
        const h = this.alloc((n[node.id] + (canary ? CANARY_PAD : 0)) * 4);
        ref.push(h);
        a.h2d(h, 0, Float32Array.from(values[node.id]));
      }
      for (const l of lowered.launches) {
        const cap = n[l.node] + (canary ? CANARY_PAD : 0);
        const h = this.alloc(cap * 4);
        outs.set(l.node, h);
        if (canary) a.fill32(h, 0, CANARY_BITS, cap);
      }
      ws = this.alloc(lowered.workspace || 16);
      this.launchAll(lowered, fns, ref, (l) => outs.get(l.node), ws);
      a.sync();
      const result = new Array(graph.nodes.length);
      const canaryIntact = new Array(graph.nodes.length);
      for (const [id, h] of outs) {
        const out = new Float32Array(n[id]);
        a.d2h(h, 0, out);
        result[id] = out;
        if (canary) canaryIntact[id] = a.countNot32(h, n[id] * 4, CANARY_BITS, CANARY_PAD) === 0;
      }
      if (canary) result.canaryIntact = canaryIntact;
      return result;
    } finally {
      for (const h of ref) a.free(h);
      for (const h of outs.values()) a.free(h);
      if (ws) a.free(ws);
    }
  }

  /**
   * A prepared program: one buffer per node, constants uploaded, every launch's
   * argument block packed once. `only(l)` keeps a subset of launches.
   */
  prepare(graph, lowered, options) {
    return new Program(this, graph, lowered, options || {});
  }
}

class Program {
  /**
   * options.only: launch filter; options.buffers: node buffers to use (device addresses,
   * owned by the caller); options.arena: { keep } to place the buffers by live range in
   * one allocation, or an arena plan of the same launch list that `buffers` follows;
   * options.streams: issue independent launches on up to 4 streams.
   */
  constructor(runner, graph, lowered, { only, buffers, arena, streams } = {}) {
    requirePad(lowered, false);
    const a = runner.a;
    this.a = a;
    this.graph = graph;
    this.lowered = lowered;
    const fns = runner.functions(lowered, !!only || streams > 1);
    this.n = graph.nodes.map((node) => size(node.shape));
    const { alias, folded } = sharing(lowered);
    this.owned = [];
    this.arena = null;
    if (buffers) {
      this.bufs = buffers.slice();
      if (arena && arena.offsets) this.arena = arena;
    } else if (arena) {
      if (only) throw new Error('an arena is planned over the whole launch list: no launch filter');
      const plan = planArena(graph, lowered, { keep: arena.keep });
      const base = runner.alloc(plan.size);
      this.owned.push(base);
      this.arena = plan;
      this.bufs = [];
      for (const node of graph.nodes) {
        if (alias.has(node.id)) this.bufs.push(this.bufs[alias.get(node.id)]);
        else if (folded.has(node.id)) this.bufs.push(0);
        else this.bufs.push(base + plan.offsets.get(node.id));
      }
    } else {
      this.bufs = [];
      for (const node of graph.nodes) {
        if (alias.has(node.id)) this.bufs.push(this.bufs[alias.get(node.id)]);
        else if (folded.has(node.id)) this.bufs.push(0);
        else { const h = runner.alloc(this.n[node.id] * 4); this.bufs.push(h); this.owned.push(h); }
      }
    }
    this.ws = runner.alloc(lowered.workspace || 16);
    for (const node of graph.nodes) {
      if (node.op === 'const' && !buffers) a.h2d(this.bufs[node.id], 0, constData(node).subarray(0, this.n[node.id]));
    }
    const launches = lowered.launches.filter((l) => !only || only(l));
    // Dispatch units: a batch's members go as one launch of its batched kernel
    // (whole launch lists on one stream; a filtered or multi-stream program
    // launches every member by itself, in the same order).
    const batchAt = new Map(!only && !(streams > 1) ? (lowered.batches || []).map((b) => [b.start, b]) : []);
    const units = [];
    for (let i = 0; i < launches.length;) {
      const b = batchAt.get(i);
      const members = launches.slice(i, i + (b ? b.count : 1));
      units.push({ kernels: b ? b.kernels : members[0].kernels, members, wsStride: b ? b.wsStride : 0 });
      i += members.length;
    }
    let count = 0, argBytes = 0;
    for (const u of units) for (const k of u.kernels) { count++; argBytes += u.members.length > 1 ? u.members.length * PTR_BYTES : ARG_BYTES; }
    this.count = count;
    this.fns = new Float64Array(count);
    this.dims = new Uint32Array(count * 7);
    this.args = new Uint8Array(argBytes);
    this.offsets = new Uint32Array(count + 1);
    const view = new DataView(this.args.buffer);
    let i = 0, at = 0;
    for (const u of units) {
      for (const k of u.kernels) {
        this.offsets[i] = at;
        if (u.members.length > 1) {
          u.members.forEach((l, m) => {
            packPtrs(view, at, l.inputs.map((id) => this.bufs[id]), this.bufs[l.node], this.ws + m * u.wsStride);
            at += PTR_BYTES;
          });
        } else {
          const l = u.members[0];
          packArgs(view, at, l.inputs.map((id) => this.bufs[id]), this.bufs[l.node], this.ws, l.params);
          at += ARG_BYTES;
        }
        this.fns[i] = fns.get(k.name);
        this.dims.set([k.grid[0], k.grid[1], k.grid[2], k.block[0], k.block[1], k.block[2], k.lds], i * 7);
        i++;
      }
    }
    this.offsets[count] = at;
    this.launches = launches;
    this.dispatches = count;
    this.graphHandle = 0;
    this.dag = null;
    if (streams && streams > 1) {
      // Buffers an arena reuses would add write-after-read hazards the schedule does not track.
      if (this.arena) throw new Error('streams > 1 is not supported with an arena');
      this.dag = scheduleLaunches(launches, streams, (id) => (alias.has(id) ? alias.get(id) : id));
      a.dagReserve(this.dag.events);
    }
  }

  /** Throw unless node `id` keeps its own bytes across the launches (always, without an arena). */
  persistent(id, what) {
    if (this.arena && !this.arena.pinned.has(this.arena.owner(id))) {
      throw new Error(`node ${id} cannot be ${what}: its arena bytes are reused by later launches (add it to keep)`);
    }
  }

  write(id, data) {
    this.persistent(id, 'written');
    this.a.h2d(this.bufs[id], 0, data instanceof Float32Array ? data : Float32Array.from(data));
  }

  read(id) {
    if (!this.bufs[id]) throw new Error(`node ${id} is not materialised (folded into its consumers, or nothing kept reads it)`);
    this.persistent(id, 'read');
    const out = new Float32Array(this.n[id]);
    this.a.d2h(this.bufs[id], 0, out);
    return out;
  }

  /** Enqueue every launch once (asynchronous). */
  run() {
    const d = this.dag;
    if (d) this.a.launchDag(this.fns, this.dims, this.args, this.offsets, d.streams, d.streamOf, d.recordEvent, d.waitBegin, d.waits);
    else this.a.launchMany(this.fns, this.dims, this.args, this.offsets);
  }

  /** Enqueue every launch `k` times over, in one native call (timing back-to-back runs). */
  runTimes(k) {
    if (this.dag) {
      for (let r = 0; r < k; r++) this.run();
      return;
    }
    if (!this.repeated || this.repeated.k !== k) {
      const n = this.count, bytes = this.args.length;
      const fns = new Float64Array(n * k), dims = new Uint32Array(n * k * 7);
      const args = new Uint8Array(bytes * k), offsets = new Uint32Array(n * k + 1);
      for (let r = 0; r < k; r++) {
        fns.set(this.fns, r * n);
        dims.set(this.dims, r * n * 7);
        args.set(this.args, r * bytes);
        for (let i = 0; i < n; i++) offsets[r * n + i] = r * bytes + this.offsets[i];
      }
      offsets[n * k] = k * bytes;
      this.repeated = { k, fns, dims, args, offsets };
    }
    const r = this.repeated;
    this.a.launchMany(r.fns, r.dims, r.args, r.offsets);
  }

  /** Capture one run() as a HIP graph; later replay() calls enqueue it whole. */
  capture() {
    if (this.graphHandle) return;
    if (this.dag) {
      // Switched off: capturing config 5's step over three streams ended the process with
      // a segmentation fault inside the runtime (config 1's step captured and replayed
      // correctly); until its cause is known, multi-stream programs run eagerly only.
      throw new Error('a program issued over several streams is not captured into a HIP graph');
    }
    this.a.captureBegin();
    try { this.run(); } finally { this.graphHandle = this.a.captureEnd(); }
  }

  replay() {
    if (!this.graphHandle) this.capture();
    this.a.graphLaunch(this.graphHandle);
  }

  sync() { this.a.sync(); }

  destroy() {
    if (this.graphHandle) this.a.graphDestroy(this.graphHandle);
    for (const h of this.owned) this.a.free(h);
    this.a.free(this.ws);
  }
}

/**
 * Independent programs issued together over `streams` streams (1..4), every
 * program's launches in order on its stream, in one native call that forks the
 * side streams off the library stream first and joins them back at the end
 * (tcmi_launch_dag), so one program's kernel ramp and tail overlap another
 * program's kernels. Programs go to streams longest first, each to the stream
 * with the fewest algorithmic bytes so far, so the streams end together. The
 * programs must share no buffer that one of them writes (checked by address: each
 * must own its buffers, as prepare() makes them) and must each be issued on one
 * stream.
 */
class Concurrent {
  constructor(runner, programs, streams) {
    if (!(streams >= 1 && streams <= 4)) throw new Error(`streams must be 1..4, got ${streams}`);
    this.a = runner.a;
    const written = new Map();   // device address -> program index
    programs.forEach((p, i) => {
      if (p.dag) throw new Error('a program issued over several streams cannot join a concurrent group');
      for (const l of p.launches) {
        const w = p.bufs[l.node];
        if (written.has(w) && written.get(w) !== i) throw new Error(`programs ${written.get(w)} and ${i} both write buffer ${w}`);
        written.set(w, i);
      }
      if (written.has(p.ws) && written.get(p.ws) !== i) throw new Error(`programs ${written.get(p.ws)} and ${i} share a workspace`);
      written.set(p.ws, i);
    });
    programs.forEach((p, i) => {
      for (const l of p.launches) {
        for (const id of l.inputs) {
          const w = written.get(p.bufs[id]);
          if (w !== undefined && w !== i) throw new Error(`program ${i} reads buffer ${p.bufs[id]} that program ${w} writes`);
        }
      }
    });
    const count = programs.reduce((c, p) => c + p.count, 0);
    const bytes = programs.reduce((c, p) => c + p.args.length, 0);
    this.fns = new Float64Array(count);
    this.dims = new Uint32Array(count * 7);
    this.args = new Uint8Array(bytes);
    this.offsets = new Uint32Array(count + 1);
    this.streamOf = new Uint8Array(count);
    const work = programs.map((p) => p.launches.reduce((q, l) => q + l.bytes, 0));
    const load = new Array(streams).fill(0), streamOfProgram = new Array(programs.length);
    programs.map((_, i) => i).sort((x, y) => work[y] - work[x] || x - y).forEach((i) => {
      let best = 0;
      for (let t = 1; t < streams; t++) if (load[t] < load[best]) best = t;
      streamOfProgram[i] = best;
      load[best] += work[i];
    });
    this.load = load;
    let k = 0, at = 0;
    programs.forEach((p, i) => {
      this.fns.set(p.fns, k);
      this.dims.set(p.dims, k * 7);
      this.args.set(p.args, at);
      for (let j = 0; j < p.count; j++) this.offsets[k + j] = at + p.offsets[j];
      this.streamOf.fill(streamOfProgram[i], k, k + p.count);
      k += p.count;
      at += p.args.length;
    });
    this.offsets[count] = at;
    this.streams = streams;
    this.recordEvent = new Int32Array(count).fill(-1);
    this.waitBegin = new Uint32Array(count + 1);
    this.waits = new Uint32Array(0);
  }

  /** Enqueue every program once (asynchronous). */
  run() {
    this.a.launchDag(this.fns, this.dims, this.args, this.offsets, this.streams, this.streamOf, this.recordEvent, this.waitBegin, this.waits);
  }
}

module.exports = { HipRunner, Program, Concurrent, packArgs, packPtrs, translationUnit, precompile, CANARY_BITS, CANARY_PAD, ARG_BYTES, PTR_BYTES, PRELUDE };
