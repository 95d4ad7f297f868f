// The 8-bit key/value cache, attention over it, and the norm and rotation of new query and key rows
// (include/supra_kv.h). The reference keeps a context's projected K and V in float32 for a whole run
// (app/models/dit.js:137-144) and attends to them at every step (dit.js:180-185); a cache holds them in a quarter of
// the memory, and lets sequences grow.
//
//   new KvCache(gpu, { pages, Hkv, D })       pages of 32 tokens; .release()
//   sequences(gpu, { lens, rows, blocks })     the sequences of a call: tokens in the cache, rows of the call (those
//       tokens' last ones, or queries of a cross-attention), pages of each; .release(). rows defaults to lens.
//   write(gpu, cache, seqs, { k, v, kOff, vOff, ldk, ldv })   quantises rows into the cache
//   read(gpu, cache, seqs, { k, v, ... })      -> { k, v }, Tensors [T, Hkv*D] where not given
//   attention(gpu, cache, seqs, { q, H, causal, scale, qOff, ldq, out, oOff, ldo }) -> Tensor [T, H*D]
//   frequencies(gpu, rotaryDim, theta)         float64 angles per position, theta^(-2i/rotaryDim); .release()
//   qkNormRope(gpu, { T, H, Hkv, D, q, k, qOff, kOff, ldq, ldk, qOut, kOut, qoOff, koOff, ldqo, ldko, qWeight, kWeight,
//       eps, norm, rotaryDim, pairs, ropeScale, freq, positions }) -> { q, k }; outputs where not given: in place
// Rows are float32 Tensors (offsets and strides in floats, as elsewhere in this shim).
"use strict";

var BLOCK = 32;  // SA_KV_BLOCK

function invalid(msg) {
  var e = new Error(msg);
  e.code = "SA_ERR_INVALID";
  return e;
}

// Tensor -> its device buffer; a raw device buffer passes through; null/undefined -> null.
function raw(t, name) {
  if (t === undefined || t === null) return null;
  if (typeof t === "object" && "buf" in t && "shape" in t) {
    if (!t.buf) throw invalid(name + " is a released or invalid Tensor");
    return t.buf;
  }
  return t;
}

function KvCache(gpu, opts) {
  var bytes = gpu.native.kvCacheBytes(opts.pages, opts.Hkv, opts.D);  // checks the sizes
  this.gpu = gpu;
  this.pages = opts.pages;
  this.Hkv = opts.Hkv;
  this.D = opts.D;
  this.k = gpu.empty([bytes], "u8");
  this.v = gpu.empty([bytes], "u8");
  this.kScale = gpu.empty([opts.pages * opts.Hkv], "u8");
  this.vScale = gpu.empty([opts.pages * opts.Hkv], "u8");
}

KvCache.prototype.release = function () {
  [this.k, this.v, this.kScale, this.vScale].forEach(function (t) { t.release(); });
};

// blocks[b]: the pages of sequence b, in order (those of its lens[b] tokens at least).
function sequences(gpu, opts) {
  var lens = Int32Array.from(opts.lens), B = lens.length;
  var rows = Int32Array.from(opts.rows || opts.lens);
  if (rows.length !== B || opts.blocks.length !== B) throw invalid("lens, rows and blocks must have one entry for each sequence");
  var start = new Int32Array(B + 1), maxRows = 0, maxLen = 0, maxBlocks = 0;
  for (var b = 0; b < B; b++) {
    if (lens[b] < 0 || rows[b] < 0) throw invalid("lens and rows must be >= 0");
    if (opts.blocks[b].length * BLOCK < lens[b]) throw invalid("sequence " + b + " has " + lens[b] + " tokens and " + opts.blocks[b].length + " pages");
    start[b + 1] = start[b] + rows[b];
    maxRows = Math.max(maxRows, rows[b]);
    maxLen = Math.max(maxLen, lens[b]);
    maxBlocks = Math.max(maxBlocks, opts.blocks[b].length);
  }
  var table = new Int32Array(Math.max(1, B * maxBlocks)).fill(-1);
  for (b = 0; b < B; b++) table.set(opts.blocks[b], b * maxBlocks);
  var seqLen = gpu.fromArray(lens.length ? lens : new Int32Array(1));
  var blockTable = gpu.fromArray(table), rowStart = gpu.fromArray(start);
  return {
    B: B, T: start[B], maxRows: maxRows, maxBlocks: maxBlocks, maxLen: maxLen, seqLen: seqLen, blockTable: blockTable, rowStart: rowStart,
    release: function () { seqLen.release(); blockTable.release(); rowStart.release(); },
  };
}

function common(cache, seqs) {
  return {
    pages: cache.pages, Hkv: cache.Hkv, D: cache.D, kCache: raw(cache.k, "cache"), vCache: raw(cache.v, "cache"),
    kScale: raw(cache.kScale, "cache"), vScale: raw(cache.vScale, "cache"), B: seqs.B, T: seqs.T, maxRows: seqs.maxRows,
    maxBlocks: seqs.maxBlocks, rowStart: raw(seqs.rowStart, "sequences"), seqLen: raw(seqs.seqLen, "sequences"),
    blockTable: raw(seqs.blockTable, "sequences"),
  };
}

function rowsOf(cache, seqs, o) {
  var a = common(cache, seqs);
  a.k = raw(o.k, "k");
  a.v = raw(o.v, "v");
  a.kOff = o.kOff || 0;
  a.vOff = o.vOff || 0;
  a.ldk = o.ldk || 0;
  a.ldv = o.ldv || 0;
  return a;
}

function write(gpu, cache, seqs, opts) {
  var args = rowsOf(cache, seqs, opts);
  gpu.op({ name: "kv.write", flops: 0 }, function () {
    gpu.native.kvWrite(args);
  });
}

function read(gpu, cache, seqs, opts) {
  var o = Object.assign({}, opts), width = cache.Hkv * cache.D;
  if (!o.k) o.k = gpu.empty([seqs.T, width]);
  if (!o.v) o.v = gpu.empty([seqs.T, width]);
  var args = rowsOf(cache, seqs, o);
  gpu.op({ name: "kv.read", flops: 0 }, function () {
    gpu.native.kvRead(args);
  });
  return { k: o.k, v: o.v };
}

function attention(gpu, cache, seqs, opts) {
  var H = opts.H || cache.Hkv;
  var out = opts.out || gpu.empty([seqs.T, H * cache.D]);
  var args = Object.assign(common(cache, seqs), {
    H: H, causal: opts.causal ? 1 : 0, scale: opts.scale === undefined || opts.scale === null ? 1 / Math.sqrt(cache.D) : opts.scale,
    maxLen: seqs.maxLen, q: raw(opts.q, "q"), qOff: opts.qOff || 0, ldq: opts.ldq || 0, out: raw(out, "out"), oOff: opts.oOff || 0, ldo: opts.ldo || 0,
  });
  var bytes = gpu.native.kvAttentionWorkspaceBytes(args), ws = null;
  if (bytes > 0) {
    ws = gpu.empty([bytes], "u8");
    args.workspace = ws.buf;
    args.workspaceBytes = bytes;
  }
  try {
    // at the longest sequence, of which the others are a part: 4 * rows * keys * D * H, as ops.attention counts
    gpu.op({ name: "kv.attention", flops: 4 * seqs.T * seqs.maxLen * cache.D * H }, function () {
      gpu.native.kvAttention(args);
    });
  } finally {
    if (ws) ws.release();  // stream-ordered pool reuse
  }
  return out;
}

function frequencies(gpu, rotaryDim, theta) {
  var f = new Float64Array(rotaryDim / 2);
  for (var i = 0; i < f.length; i++) f[i] = Math.pow(theta === undefined ? 10000 : theta, (-2 * i) / rotaryDim);
  return gpu.fromArray(new Uint8Array(f.buffer));
}

var PAIRS = { half: 0, near: 1 };
var NORM = { none: 0, rms: 1 };

function qkNormRope(gpu, o) {
  var pairs = PAIRS[o.pairs === undefined ? "half" : o.pairs], norm = NORM[o.norm === undefined ? "rms" : o.norm];
  if (pairs === undefined) throw invalid("unknown pairs " + o.pairs);
  if (norm === undefined) throw invalid("unknown norm " + o.norm);
  var qOut = o.qOut || o.q, kOut = o.kOut || o.k;
  var args = {
    T: o.T, H: o.q ? o.H : 0, Hkv: o.k ? o.Hkv : 0, D: o.D, rotaryDim: o.rotaryDim === undefined ? (o.freq ? o.D : 0) : o.rotaryDim, pairs: pairs, norm: norm,
    eps: o.eps === undefined ? 1e-6 : o.eps, ropeScale: o.ropeScale === undefined ? 1 : o.ropeScale,
    q: raw(o.q, "q"), k: raw(o.k, "k"), qOff: o.qOff || 0, kOff: o.kOff || 0, ldq: o.ldq || 0, ldk: o.ldk || 0,
    qOut: raw(qOut, "qOut"), kOut: raw(kOut, "kOut"),
    qoOff: o.qOut ? o.qoOff || 0 : o.qOff || 0, koOff: o.kOut ? o.koOff || 0 : o.kOff || 0,
    ldqo: o.qOut ? o.ldqo || 0 : o.ldq || 0, ldko: o.kOut ? o.ldko || 0 : o.ldk || 0,
    qWeight: raw(o.qWeight, "qWeight"), kWeight: raw(o.kWeight, "kWeight"), invFreq: raw(o.freq, "freq"), positions: raw(o.positions, "positions"),
  };
  gpu.op({ name: "qkNormRope", flops: 0 }, function () {
    gpu.native.qkNormRope(args);
  });
  return { q: qOut, k: kOut };
}

module.exports = {
  BLOCK: BLOCK, KvCache: KvCache, sequences: sequences, write: write, read: read, attention: attention, frequencies: frequencies,
  qkNormRope: qkNormRope,
};
