// Runs one case of the operators for batches of prompts (4-bit weights, embedding rows, attention behind a shared
// prefix) through the JS op layer for the parity tests: reads a JSON spec whose inputs are raw little-endian
// files, writes the outputs the same way.  node run_batch.mjs case.json
//
// Cases:
//   ops       quantizeQ4, linear (both precisions, bf16 and residual results, a LoRA), embedRows, attentionPrefix
//   encode    Qwen3.encodeBatch of a synthetic text encoder, with and without a kept prefix, and encode of each
//             prompt; on bf16 weights or after quantizeQ4, with the embedding rows from the host or the device
//   adapter   the LLM adapter's prompt weights
//   pipeline  LatentPipeline.encodeBatch beside encode

import fs from "fs";
import { GPU } from "../../anima-studio_amd/js/gpu.mjs";
import * as ops from "../../anima-studio_amd/js/ops.mjs";
import { SyntheticWeights } from "../../anima-studio_amd/js/weights.mjs";
import { ropeTable } from "../../anima-studio_amd/js/common.mjs";
import { AnimaDiT, adapt, syntheticAdapter } from "../../anima-studio_amd/js/dit.mjs";
import { attachLoras, linearRegistry } from "../../anima-studio_amd/js/lora.mjs";
import { LatentPipeline } from "../../anima-studio_amd/js/pipeline.mjs";
import { Qwen3 } from "../../anima-studio_amd/js/qwen3.mjs";

const ARR = { f32: Float32Array, u8: Uint8Array, u16: Uint16Array };

function load(path, dtype) {
  const b = fs.readFileSync(path);
  return new ARR[dtype || "f32"](b.buffer.slice(b.byteOffset, b.byteOffset + b.length));
}

function save(path, arr) {
  fs.writeFileSync(path, Buffer.from(arr.buffer, arr.byteOffset, arr.byteLength));
}

const message = async (f) => {
  try {
    await f();
  } catch (e) {
    return e.message;
  }
  return "";
};

async function opsCase(gpu, c) {
  const put = async (n, t) => save(`${c.out}.${n}`, await gpu.read(t));
  const { M, N, K } = c;
  for (const mid of [false, true]) {
    const tag = mid ? "mid" : "sym";
    const W = ops.quantizeQ4(gpu, { kind: "bf16", N, K, name: "w", buf: gpu.upload(load(c.w, "u16")) }, { group: c.group, mid });
    await put(`${tag}.q`, W.buf);
    await put(`${tag}.s`, W.groupScale);
    if (mid) await put(`${tag}.z`, W.groupMid);
    const x = gpu.fromArray(load(c.x), [M, K]);
    await put(`${tag}.fp32`, ops.linear(gpu, x, W));
    await put(`${tag}.bf16`, ops.linear(gpu, x, W, { precision: "bf16", outBf16: true }));
    const r = gpu.fromArray(load(c.r), [M, N]);
    ops.linear(gpu, x, W, { out: r, resid: true });
    await put(`${tag}.resid`, r);
    W.lora = [{ A: gpu.upload(load(c.A)), B: gpu.upload(load(c.B)), r: 8, scale: 0.5, off: 0, n: N }];
    await put(`${tag}.lora`, ops.linear(gpu, x, W));
    await put(`${tag}.rows`, ops.embedRows(gpu, W, c.ids, { weights: c.weights, scale: 2 }));
  }
  const kept = ops.quantizeQ4(gpu, { kind: "bf16", N: 4, K: 48, buf: null });
  const { H, lens, P } = c, group = c.attnGroup, D = 128, KH = H / group, T = lens.reduce((a, b) => a + b, 0);
  const q = gpu.fromArray(load(c.q), [T, H * D]), kv = gpu.fromArray(load(c.kv), [P + T, 2 * KH * D]);
  const cs = ropeTable(gpu, P + Math.max(...lens), D, 1e6), ld = 2 * KH * D;
  for (const precision of ["fp32", "bf16"]) {
    const d = { H, D, group, cs, precision, ldq: H * D, ldk: ld, ldv: ld, vOff: KH * D };
    const prefix = ops.attentionPrefixPrepare(gpu, Object.assign({ k: kv, v: kv, len: P }, d));
    const own = kv.view(P * ld, [T, ld]);
    await put(`attn.${precision}`, ops.attentionPrefix(gpu, Object.assign({ q, k: own, v: own, lens, prefix }, d)));
  }
  console.log(JSON.stringify({ kind: kept.kind }));
}

async function encode(gpu, c) {
  const te = Qwen3.synthetic(gpu, new SyntheticWeights(gpu, 23), { layers: c.layers, vocab: c.vocab });
  const first = await gpu.read(await te.encode(c.prompts[0]));
  await te.embedOnDevice();
  const second = await gpu.read(await te.encode(c.prompts[0]));
  const log = { device: first.reduce((n, v, i) => n + (v !== second[i]), 0), converted: 0 };
  if (c.q4) {
    log.converted = te.quantizeQ4(c.q4);
    log.again = te.quantizeQ4(c.q4) + te.quantizeF8();
    await te.embedOnDevice({ q4: c.q4 });
  }
  const put = async (name, ts) => {
    for (let i = 0; i < ts.length; i++) {
      save(`${c.out}.${name}.${i}`, await gpu.read(ts[i]));
      ts[i].release();
    }
  };
  for (const prec of ["fp32", "bf16"]) {
    te.precision = prec;
    await put(`${prec}.batch`, await te.encodeBatch(c.prompts));
    await put(`${prec}.one`, [await te.encode(c.prompts[0])]);
    const prefix = await te.keepPrefix(c.prompts[0].slice(0, c.keep));
    await put(`${prec}.kept`, await te.encodeBatch(c.prompts, { prefix }));
    await put(`${prec}.kept2`, await te.encodeBatch(c.prompts.slice().reverse(), { prefix }));
    await put(`${prec}.only`, await te.encodeBatch([c.prompts[0].slice(0, c.keep)], { prefix }));
    te.precision = prec === "fp32" ? "bf16" : "fp32";
    log[`${prec}.precision`] = await message(() => te.encodeBatch(c.prompts, { prefix }));
    te.precision = prec;
    log[`${prec}.other`] = await message(() => te.encodeBatch([[c.vocab - 1]], { prefix }));
    attachLoras({ te: linearRegistry(te) }, []);
    log[`${prec}.lora`] = await message(() => te.encodeBatch(c.prompts, { prefix }));
    prefix.release();
    log[`${prec}.released`] = await message(() => te.encodeBatch(c.prompts, { prefix }));
  }
  log.outside = await message(() => te.encodeBatch([[0, c.vocab]]));
  const values = async (name, W) => {
    save(`${c.out}.w.${name}`, await gpu.read(W.buf ? (W.buf.release ? W.buf : W) : W));
    if (W.groupScale) save(`${c.out}.w.${name}.s`, await gpu.read(W.groupScale));
    if (W.groupMid) save(`${c.out}.w.${name}.z`, await gpu.read(W.groupMid));
  };
  for (let i = 0; i < te.layers.length; i++)
    for (const k of ["ln1", "ln2", "qn", "kn", "qkv", "o", "gate", "up", "down"]) await values(`${i}.${k}`, te.layers[i][k]);
  await values("norm", te.norm);
  await values("embed", te.deviceTable);
  te.release();
  console.log(JSON.stringify(log));
}

async function adapter(gpu, c) {
  const A = syntheticAdapter(gpu, new SyntheticWeights(gpu, 29), { blocks: 1, vocab: 64 });
  const hidden = gpu.fromArray(load(c.hidden), [c.Ls, 1024]);
  for (const name of Object.keys(c.weights)) save(`${c.out}.${name}`, await gpu.read(await adapt(gpu, A, hidden, c.ids, c.weights[name])));
}

async function pipeline(gpu, c) {
  const src = new SyntheticWeights(gpu, 31, { mode: "bf16", blocks: 1 });
  const dit = AnimaDiT.synthetic(gpu, src), te = Qwen3.synthetic(gpu, src, { layers: 1, vocab: 97 });
  const p = new LatentPipeline(gpu, dit, { te, adapter: syntheticAdapter(gpu, src, { blocks: 1, vocab: 64 }) });
  te.precision = "fp32";
  const same = await p.encode(c.prompts[0]);
  const conds = await p.encodeBatch(c.prompts);
  const again = await p.encodeBatch([c.prompts[1], c.prompts[0], c.prompts[1]]);
  console.log(JSON.stringify({ n: conds.length, hit: conds[0] === same, again: again.map((t) => conds.indexOf(t)), stats: p.stats,
    cached: p.ctxCache.size, none: (await p.encodeBatch([])).length, left: p.ctxCache.size }));
  p.clearContexts();
}

const c = JSON.parse(fs.readFileSync(process.argv[2], "utf8"));
GPU.create({})
  .then(async (gpu) => {
    await { ops: opsCase, encode, adapter, pipeline }[c.case](gpu, c);
    gpu.destroy();
  })
  .catch((e) => {
    console.error(e);
    process.exit(1);
  });
