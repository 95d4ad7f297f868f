// CPU checks of the 8-bit cache in the JS binding (no GPU): exports, how the shim's calls map onto the addon's, and
// what is refused before the device is touched.
// Usage: node tests/node/kv_cpu.js
"use strict";

var assert = require("assert");
var path = require("path");

var root = path.join(__dirname, "..", "..", "supra2-img-web_amd", "js");
var sa = require(path.join(root, "index.js"));
var device = require(path.join(root, "device.js"));
var native = device.loadNative();

var checks = 0;
function check(name, fn) {
  fn();
  checks++;
  process.stdout.write("ok " + name + "\n");
}
function invalid(re) {
  return function (e) { return e.code === "SA_ERR_INVALID" && (!re || re.test(e.message)); };
}

check("addon exports", function () {
  ["qkNormRope", "kvCacheBytes", "kvWrite", "kvRead", "kvAttention", "kvAttentionWorkspaceBytes"].forEach(function (f) {
    assert.strictEqual(typeof native[f], "function", f);
  });
  assert.strictEqual(native.SA_KV_BLOCK, sa.kv.BLOCK);
  assert.strictEqual(native.SA_ROPE_NEAR, 1);
  assert.strictEqual(native.SA_NORM_RMS, 1);
  assert.strictEqual(native.kvCacheBytes(7, 3, 128), 7 * 3 * 32 * 128);
});

check("calls that are refused", function () {
  assert.throws(function () { native.kvCacheBytes(0, 1, 64); }, invalid());
  assert.throws(function () { native.kvCacheBytes(1, 1, 80); }, function (e) { return e.code === "SA_ERR_UNSUPPORTED"; });
  assert.throws(function () { native.kvCacheBytes(1.5, 1, 64); }, invalid(/pages must be an integer/));
  assert.throws(function () { native.kvCacheBytes(Math.pow(2, 40), 1, 64); }, invalid(/int32/));
  assert.throws(function () { native.kvWrite({}); }, invalid());
  assert.throws(function () { native.kvRead({ pages: 1, Hkv: 1, D: 64, kCache: {} }); }, invalid(/kCache must be a device buffer/));
  assert.throws(function () { native.kvAttention({ pages: 1, Hkv: 1, D: 64, B: 1, T: 1, maxRows: 1, maxBlocks: 1, H: 1 }); }, invalid(/non-NULL/));
  assert.throws(function () { native.kvAttentionWorkspaceBytes({ pages: 1, Hkv: 1, D: 64, causal: 0.5 }); }, invalid());
  assert.throws(function () { native.qkNormRope({ T: 1, H: 1, D: 64, q: 5 }); }, invalid(/q must be a device buffer/));
});

// A device made of objects: records the calls.
function fake() {
  var calls = [];
  var n = {
    calls: calls, deviceCount: function () { return 1; },
    malloc: function (bytes) { return { bytes: bytes }; }, free: function () {},
    upload: function (buf, arr) { buf.data = Array.from(arr); },
    copy: function (dst, doff, src, soff, bytes) { calls.push(["copy", doff, soff, bytes]); },
    kvCacheBytes: native.kvCacheBytes,
    kvAttentionWorkspaceBytes: function () { return n.workspace || 0; },
  };
  ["kvWrite", "kvRead", "kvAttention", "qkNormRope"].forEach(function (f) {
    n[f] = function (a) { calls.push([f, a]); };
  });
  return n;
}

check("sequences and cache arrays", function () {
  var n = fake(), gpu = new device.GPU(n);
  var cache = new sa.kv.KvCache(gpu, { pages: 6, Hkv: 2, D: 64 });
  assert.ok(cache.k.buf.bytes >= 6 * 2 * 32 * 64 && cache.vScale.buf.bytes >= 12);
  var s = sa.kv.sequences(gpu, { lens: [40, 0, 33], rows: [3, 0, 33], blocks: [[5, 1], [], [0, 2, 3]] });
  assert.deepStrictEqual([s.B, s.T, s.maxRows, s.maxBlocks, s.maxLen], [3, 36, 33, 3, 40]);
  assert.deepStrictEqual(s.rowStart.buf.data, [0, 3, 3, 36]);
  assert.deepStrictEqual(s.blockTable.buf.data, [5, 1, -1, -1, -1, -1, 0, 2, 3]);
  assert.deepStrictEqual(s.seqLen.buf.data, [40, 0, 33]);
  assert.throws(function () { sa.kv.sequences(gpu, { lens: [33], blocks: [[1]] }); }, invalid(/33 tokens and 1 pages/));
  assert.throws(function () { sa.kv.sequences(gpu, { lens: [1, 2], blocks: [[1]] }); }, invalid(/one entry/));
  assert.throws(function () { sa.kv.sequences(gpu, { lens: [-1], blocks: [[1]] }); }, invalid(/>= 0/));
});

check("write, read and attention", function () {
  var n = fake(), gpu = new device.GPU(n);
  var cache = new sa.kv.KvCache(gpu, { pages: 2, Hkv: 2, D: 64 });
  var s = sa.kv.sequences(gpu, { lens: [40], rows: [4], blocks: [[1, 0]] });
  var qkv = gpu.empty([4, 512]);
  sa.kv.write(gpu, cache, s, { k: qkv, v: qkv, kOff: 256, vOff: 384, ldk: 512, ldv: 512 });
  var w = n.calls.pop();
  assert.strictEqual(w[0], "kvWrite");
  assert.deepStrictEqual([w[1].kOff, w[1].vOff, w[1].ldk, w[1].T, w[1].B, w[1].maxBlocks], [256, 384, 512, 4, 1, 2]);
  assert.strictEqual(w[1].kCache, cache.k.buf);
  var back = sa.kv.read(gpu, cache, s, {});
  assert.deepStrictEqual(back.k.shape, [4, 128]);
  assert.strictEqual(n.calls.pop()[1].v, back.v.buf);
  var out = sa.kv.attention(gpu, cache, s, { q: qkv, H: 4, causal: true, ldq: 512 });
  var a = n.calls.pop()[1];
  assert.deepStrictEqual(out.shape, [4, 256]);
  assert.deepStrictEqual([a.H, a.causal, a.scale, a.maxLen, a.ldq, a.workspaceBytes], [4, 1, 0.125, 40, 512, undefined]);
  n.workspace = 4096;
  sa.kv.attention(gpu, cache, s, { q: qkv, H: 4, ldq: 512, scale: 0.5 });
  a = n.calls.pop()[1];
  assert.deepStrictEqual([a.causal, a.scale, a.workspaceBytes], [0, 0.5, 4096]);
  assert.ok(a.workspace.bytes >= 4096);
  qkv.release();
  assert.throws(function () { sa.kv.attention(gpu, cache, s, { q: qkv, H: 4 }); }, invalid(/released/));
});

check("norm and rotation", function () {
  var n = fake(), gpu = new device.GPU(n);
  var qkv = gpu.empty([3, 512]), freq = sa.kv.frequencies(gpu, 64, 100);
  assert.deepStrictEqual(Array.from(new Float64Array(Uint8Array.from(freq.buf.data).buffer)).slice(0, 2), [1, Math.pow(100, -2 / 64)]);
  var r = sa.kv.qkNormRope(gpu, { T: 3, H: 4, Hkv: 2, D: 64, q: qkv, k: qkv, kOff: 256, ldq: 512, ldk: 512, freq: freq, positions: gpu.empty([3], "i32") });
  var a = n.calls.pop()[1];
  assert.strictEqual(r.q, qkv);
  assert.deepStrictEqual([a.koOff, a.ldko, a.qoOff, a.rotaryDim, a.pairs, a.norm, a.eps], [256, 512, 0, 64, 0, 1, 1e-6]);
  sa.kv.qkNormRope(gpu, { T: 3, H: 4, D: 64, q: qkv, qOut: gpu.empty([3, 256]), ldq: 512, norm: "none", pairs: "near" });
  a = n.calls.pop()[1];
  assert.deepStrictEqual([a.Hkv, a.k, a.ldqo, a.rotaryDim, a.pairs, a.norm], [0, null, 0, 0, 1, 0]);
  assert.throws(function () { sa.kv.qkNormRope(gpu, { T: 1, H: 1, D: 64, q: qkv, pairs: "other" }); }, invalid(/unknown pairs/));
});

check("DiT contexts in a cache", function () {
  var n = fake(), gpu = new device.GPU(n);
  var kvs = [77, 0, 1].map(function (L) { return gpu.empty([Math.max(1, L), 1152]); });
  var ctx = sa.dit.cacheContexts(gpu, kvs, [77, 0, 1]);
  assert.strictEqual(ctx.cache.pages, 4);
  var w = n.calls.filter(function (c) { return c[0] === "kvWrite"; })[0][1];
  assert.deepStrictEqual([w.T, w.vOff, w.ldk, w.Hkv, w.D, w.maxBlocks], [78, 576, 1152, 9, 64, 3]);
  assert.deepStrictEqual(n.calls.filter(function (c) { return c[0] === "copy"; }), [["copy", 0, 0, 77 * 4608], ["copy", 77 * 4608, 0, 4608]]);
  assert.deepStrictEqual(ctx.seqs.blockTable.buf.data, [0, 1, 2, -1, -1, -1, 3, -1, -1]);
  var out = sa.dit.crossAttention(gpu, gpu.empty([768, 576]), ctx);
  var a = n.calls.pop();
  assert.strictEqual(a[0], "kvAttention");
  assert.deepStrictEqual([a[1].causal, a[1].H, a[1].T, a[1].maxRows, a[1].scale], [0, 9, 768, 256, 0.125]);
  assert.deepStrictEqual(out.shape, [768, 576]);
  ctx.release();
  assert.throws(function () { sa.dit.cacheContexts(gpu, kvs, [1]); }, RangeError);
  kvs[0].release();
  assert.throws(function () { sa.dit.cacheContexts(gpu, kvs, [77, 0, 1]); }, invalid(/released/));
});

process.stdout.write("all " + checks + " checks passed\n");
