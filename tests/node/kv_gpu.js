// GPU run of the 8-bit cache through the JS shim; outputs go back to Python for the oracle comparison.
// Usage: node tests/node/kv_gpu.js <dir>   (reads <dir>/manifest.json and <dir>/*.bin)
"use strict";

var fs = require("fs");
var path = require("path");

var sa = require(path.join(__dirname, "..", "..", "supra2-img-web_amd", "js", "index.js"));

var dir = process.argv[2];
var m = JSON.parse(fs.readFileSync(path.join(dir, "manifest.json"), "utf8"));

function load(name) {
  var b = fs.readFileSync(path.join(dir, name));
  return new Float32Array(b.buffer.slice(b.byteOffset, b.byteOffset + b.byteLength));
}

function save(gpu, name, t) {
  return gpu.read(t).then(function (a) {
    fs.writeFileSync(path.join(dir, name), Buffer.from(a.buffer, a.byteOffset, a.byteLength));
  });
}

sa.GPU.create({ profile: true }).then(function (gpu) {
  // two prompts: norms and rotation in place on the packed rows, cache write, causal attention, read back
  var p = m.prompts, W = (p.H + 2 * p.Hkv) * p.D;
  var qkv = gpu.fromArray(load("qkv.bin"), [p.T, W]);
  var freq = sa.kv.frequencies(gpu, p.D, 10000);
  var pos = gpu.fromArray(Int32Array.from(p.positions));
  sa.kv.qkNormRope(gpu, { T: p.T, H: p.H, Hkv: p.Hkv, D: p.D, q: qkv, k: qkv, kOff: p.H * p.D, ldq: W, ldk: W, freq: freq, positions: pos,
    qWeight: gpu.fromArray(load("wq.bin")), kWeight: gpu.fromArray(load("wk.bin")) });
  var cache = new sa.kv.KvCache(gpu, { pages: p.pages, Hkv: p.Hkv, D: p.D });
  var seqs = sa.kv.sequences(gpu, { lens: p.lens, blocks: p.blocks });
  sa.kv.write(gpu, cache, seqs, { k: qkv, v: qkv, kOff: p.H * p.D, vOff: (p.H + p.Hkv) * p.D, ldk: W, ldv: W });
  var o = sa.kv.attention(gpu, cache, seqs, { q: qkv, H: p.H, causal: true, ldq: W });
  var back = sa.kv.read(gpu, cache, seqs, {});
  // the DiT's cross-attention over cached contexts, and the refusals of released and too small buffers
  var d = m.dit;
  var kvs = d.lens.map(function (L, b) { return gpu.fromArray(load("kv" + b + ".bin"), [L, 1152]); });
  var ctx = sa.dit.cacheContexts(gpu, kvs, d.lens);
  var x = sa.dit.crossAttention(gpu, gpu.fromArray(load("q.bin"), [d.lens.length * 256, 576]), ctx);
  var small = gpu.empty([4]), refused = [];
  [function () { sa.kv.write(gpu, cache, seqs, { k: small, v: qkv, ldv: W }); }, function () { sa.kv.attention(gpu, cache, seqs, { q: qkv, H: p.H, ldq: W, out: small }); },
    function () { sa.kv.attention(gpu, cache, seqs, { q: qkv, H: p.H, ldq: W, out: qkv }); }, function () { sa.kv.read(gpu, cache, seqs, { k: back.k, v: back.k }); }].forEach(function (f) {
    try { f(); refused.push("none"); } catch (e) { refused.push(e.code); }
  });
  return save(gpu, "rotated.bin", qkv).then(function () { return save(gpu, "o.bin", o); })
    .then(function () { return save(gpu, "k.bin", back.k); }).then(function () { return save(gpu, "v.bin", back.v); })
    .then(function () { return save(gpu, "x.bin", x); }).then(function () { return gpu.profiler.report(); })
    .then(function (rows) {
      fs.writeFileSync(path.join(dir, "result.json"), JSON.stringify({ refused: refused, names: rows.map(function (r) { return r.name; }) }));
    });
}).catch(function (e) {
  process.stderr.write(String(e && e.stack ? e.stack : e) + "\n");
  process.exit(1);
});
