// Runs one case of the e4m3 operators through the JS op layer (ops.mjs -> N-API -> libanima.so) for
// the parity tests: reads a JSON spec whose inputs are raw little-endian files, writes the outputs
// the same way.  node run_f8.mjs case.json
//
// Cases:
//   block   residualNorm -> linear -> quantRowsF8 -> linear (bf16) -> residualNorm -> linearGlu ->
//           linear, on bf16 weights converted by quantizeF8 or on an e4m3 safetensors file
//   groups  residualNorm of rows in groups with gates and modulations of their own, and of each group by itself
//   qwen3   Qwen3.encode of a synthetic text encoder after quantizeF8 (both precisions; recorded,
//           replayed and eager) and its weights; an encoding with a LoRA of zeros attached
//   ditsteps  a synthetic DiT's residual stream after each block, and after the e4m3 blocks op by op
//   dit     a synthetic DiT's velocities: bf16 weights, after quantizeF8, and with LoRAs of zeros; graph replays

import fs from "fs";
import { GPU } from "../../anima-studio_amd/js/gpu.mjs";
import * as ops from "../../anima-studio_amd/js/ops.mjs";
import { SafeTensors, SyntheticWeights, concatLinears } from "../../anima-studio_amd/js/weights.mjs";
import { ropeTable } from "../../anima-studio_amd/js/common.mjs";
import { AnimaDiT, ForwardGraph } from "../../anima-studio_amd/js/dit.mjs";
import { Qwen3 } from "../../anima-studio_amd/js/qwen3.mjs";

const ARR = { f32: Float32Array, u8: Uint8Array, u16: Uint16Array };

function load(path, dtype) {
  const b = fs.readFileSync(path);
  return new ARR[dtype || "f32"](b.buffer.slice(b.byteOffset, b.byteOffset + b.length));
}

function save(path, arr) {
  fs.writeFileSync(path, Buffer.from(arr.buffer, arr.byteOffset, arr.byteLength));
}

// a LoRA entry of zeros on W: its linears then take the fp32 input
function zeroLora(gpu, W) {
  const A = gpu.upload(new Float32Array(8 * W.K)), B = gpu.upload(new Float32Array(W.N * 8));
  W.lora = [{ A, B, r: 8, scale: 1, off: 0, n: W.N }];
}

async function block(gpu, c) {
  const st = c.file ? SafeTensors.open(c.file) : null;
  const weight = (name, N, K) => {
    if (st) return st.linear(gpu, name + ".");
    return ops.quantizeF8(gpu, { kind: "bf16", N, K, name, buf: gpu.upload(load(c.w[name], "u16")) });
  };
  const { M, C, F } = c;
  const Wa = weight("a", C, C), Wb = weight("b", C, C), Wg = weight("gate", F, C), Wu = weight("up", F, C), Wd = weight("down", C, F);
  const two = concatLinears(gpu, [Object.assign({}, weight("gate", F, C)), weight("up", F, C)]);
  const x = gpu.fromArray(load(c.x), [M, C]);
  const mod = gpu.upload(load(c.mod));
  const h = ops.residualNorm(gpu, x, C, { norm: "layer", mod, shiftOff: 0, scaleOff: C, f8: true });
  const y = ops.linear(gpu, null, Wa, { xq: h, act: "gelu" });
  const yq = ops.quantRowsF8(gpu, y, C);
  const z = ops.linear(gpu, null, Wb, { xq: yq, precision: "bf16", outBf16: true });
  const h2 = ops.residualNorm(gpu, x, C, { y: z, gate: mod, gOff: 2 * C, weight: gpu.upload(load(c.norm)), h: true, f8: true });
  const g = ops.linearGlu(gpu, null, Wg, Wu, { xq: h2, f8: true });
  const gf = ops.linearGlu(gpu, h2.h, Wg, Wu, {});
  const both = two ? ops.linear(gpu, null, two, { xq: h2 }) : null;
  const x1 = await gpu.read(x);
  ops.linear(gpu, null, Wd, { xq: g, out: x, resid: true, gate: mod, gOff: 2 * C });
  const out = { x: await gpu.read(x), x1, y: await gpu.read(y), z: await gpu.read(z), h2: await gpu.read(h2.h), gf: await gpu.read(gf) };
  for (const [n, r] of [["h", h], ["yq", yq], ["h2", h2], ["g", g]]) {
    out[n + ".q"] = await gpu.read(r.q);
    out[n + ".s"] = await gpu.read(r.s);
  }
  for (const [n, W] of [["a", Wa], ["b", Wb], ["gate", Wg], ["up", Wu], ["down", Wd]]) {
    out[`w.${n}.q`] = await gpu.read(W.buf);
    out[`w.${n}.s`] = await gpu.read(W.scale);
  }
  if (both) out.both = await gpu.read(both);
  for (const k of Object.keys(out)) save(`${c.out}.${k}`, out[k]);
}

async function groups(gpu, c) {
  const { M, C, per, ld } = c;
  const gate = gpu.upload(load(c.gate)), mod = gpu.upload(load(c.mod)), y = gpu.fromArray(load(c.y), [M, C]);
  const run = async (tag, x, opts) => {
    const r = ops.residualNorm(gpu, x, C, Object.assign({ gate, mod, norm: "layer", h: true, f8: true }, opts));
    for (const [n, t] of [["x", x], ["h", r.h], ["q", r.q], ["s", r.s]]) save(`${c.out}.${tag}.${n}`, await gpu.read(t));
  };
  await run("all", gpu.fromArray(load(c.x), [M, C]), { y, groupRows: per, gateLd: ld, modLd: 2 * ld, gOff: 4, shiftOff: 0, scaleOff: ld });
  const x = gpu.fromArray(load(c.x), [M, C]);
  for (let g = 0, m = 0; m < M; g++, m += per) {
    const n = Math.min(per, M - m);
    await run(g, x.view(m * C, [n, C]), { y: y.view(m * C, [n, C]), gOff: g * ld + 4, shiftOff: 2 * g * ld, scaleOff: 2 * g * ld + ld });
  }
}

// the encoder's layers in fp32 precision, op by op on fp32 rows
function encoderSteps(gpu, te, rows, L) {
  const { hidden: D, heads: H, kvHeads: KH, headDim: HD } = te.cfg;
  const x = gpu.fromArray(rows, [L, D]), cs = ropeTable(gpu, L, HD, te.cfg.theta), ld = (H + 2 * KH) * HD;
  for (const l of te.layers) {
    const h = ops.residualNorm(gpu, x, D, { weight: l.ln1 }).h;
    const qkv = ops.linear(gpu, h, l.qkv, {});
    const a = ops.attention(gpu, { q: qkv, k: qkv, v: qkv, Lq: L, Lk: L, H, D: HD, ldq: ld, ldk: ld, ldv: ld, qOff: 0,
      kOff: H * HD, vOff: (H + KH) * HD, group: H / KH, causal: true, qNorm: l.qn, kNorm: l.kn, cs, precision: "fp32" });
    ops.linear(gpu, a, l.o, { out: x, resid: true });
    const h2 = ops.residualNorm(gpu, x, D, { weight: l.ln2 }).h;
    ops.linear(gpu, ops.linearGlu(gpu, h2, l.gate, l.up, {}), l.down, { out: x, resid: true });
  }
  return ops.residualNorm(gpu, x, D, { weight: te.norm }).h;
}

async function qwen3(gpu, c) {
  const te = Qwen3.synthetic(gpu, new SyntheticWeights(gpu, 17), { layers: c.layers, vocab: c.vocab });
  (await te.encode(c.ids)).release(); // a graph over the bf16 weights, dropped by quantizeF8
  console.log(JSON.stringify({ converted: te.quantizeF8(), again: te.quantizeF8() }));
  for (const prec of ["fp32", "bf16"]) {
    te.precision = prec;
    for (const tag of ["", ".replay", ".replay2"]) save(`${c.out}.${prec}${tag}`, await gpu.read(await te.encode(c.ids)));
    te.graphs = false;
    save(`${c.out}.${prec}.eager`, await gpu.read(await te.encode(c.ids)));
    te.graphs = true;
  }
  for (let i = 0; i < te.layers.length; i++) {
    const l = te.layers[i];
    for (const k of ["ln1", "ln2", "qn", "kn"]) save(`${c.out}.w.${i}.${k}`, await gpu.read(l[k]));
    for (const k of ["qkv", "o", "gate", "up", "down"]) {
      save(`${c.out}.w.${i}.${k}`, await gpu.read(l[k].buf));
      save(`${c.out}.w.${i}.${k}.s`, await gpu.read(l[k].scale));
    }
  }
  save(`${c.out}.w.norm`, await gpu.read(te.norm));
  save(`${c.out}.w.embed`, await gpu.read(te.table));
  te.precision = "fp32";
  save(`${c.out}.steps`, await gpu.read(encoderSteps(gpu, te, await te.embedRows(c.ids), c.ids.length)));
  zeroLora(gpu, te.layers[0].o);
  save(`${c.out}.lora`, await gpu.read(await te.encode(c.ids)));
  te.release();
}

async function dit(gpu, c) {
  const model = AnimaDiT.synthetic(gpu, new SyntheticWeights(gpu, c.seed, { mode: "bf16", blocks: c.blocks }));
  const lat = c.latents.map((p) => load(p));
  const forward = async (tag) => {
    const tc = model.timeCond(c.sigma);
    const cond = model.prepareContext(c.ctx.map((p) => gpu.fromArray(load(p), [c.Lk, 1024])));
    const v = await model.forward(lat, c.h, c.w, cond, tc);
    v.forEach((vb, b) => save(`${c.out}.${tag}.${b}`, vb));
    tc.release();
    cond.release();
  };
  model.precision = "fp32";
  await forward("bf16w");
  console.log(JSON.stringify({ converted: model.quantizeF8() }));
  await forward("f8");
  model.precision = "bf16";
  await forward("f8bf16");
  // recorded into a graph and replayed with other latents, an eager forward before each
  const cond = model.prepareContext(c.ctx.map((p) => gpu.fromArray(load(p), [c.Lk, 1024])));
  const n = lat.length * lat[0].length;
  const x = gpu.empty([lat.length, 16, c.h, c.w]), tc = model.timeCond(c.sigma);
  gpu.write(x, lat[0], 0);
  gpu.write(x, lat[1], lat[0].length * 4);
  const fg = await ForwardGraph.capture(model, x, c.h, c.w, cond, tc);
  const differ = [];
  for (let i = 0; i < 3; i++) {
    gpu.write(x, lat[i % 2].map((v) => v * (i + 1)), 0);
    const e = await gpu.read(await model.forwardDevice(x, c.h, c.w, cond, tc));
    const g = await gpu.read(fg.run(tc));
    differ.push(e.reduce((k, v, j) => k + (v !== g[j]), 0));
  }
  console.log(JSON.stringify({ differ, n }));
  fg.release();
  model.precision = "fp32";
  for (const b of model.blocks)
    for (const W of [b.self.qkv, b.self.o, b.cross.q, b.cross.o, b.l1, b.l2]) if (W) zeroLora(gpu, W);
  await forward("f8lora");
}

// A DiT block on e4m3 weights op by op: fp32 rows between the ops (bf16 rows widened on the host), which each product
// quantizes itself.  x: [B * L, 2048], updated in place.
async function blockSteps(gpu, model, i, x, cond, tc, B, L, cs) {
  const D = 2048, H = 16, HD = 128, M = B * L, precision = model.precision;
  const b = model.blocks[i], m = tc.blocks[i];
  const wide = async (t) => {
    if (t.dtype !== "bf16") return t;
    const u = await gpu.read(t), f = new Float32Array(u.length), bits = new Uint32Array(f.buffer);
    u.forEach((v, j) => { bits[j] = v * 65536; });
    return gpu.fromArray(f, t.shape);
  };
  const norm = (mod) => ops.residualNorm(gpu, x, D, { norm: "layer", mod, shiftOff: 0, scaleOff: D }).h;
  const into = (y, W, mod) => ops.linear(gpu, y, W, { M, out: x, resid: true, gate: mod, gOff: 2 * D, precision });
  const qkv = ops.linear(gpu, norm(m.self), b.self.qkv, { precision });
  const a = ops.attention(gpu, { q: qkv, k: qkv, v: qkv, B, Lq: L, Lk: L, H, D: HD, ldq: 3 * D, ldk: 3 * D, ldv: 3 * D, qOff: 0,
    kOff: D, vOff: 2 * D, qNorm: b.self.qn, kNorm: b.self.kn, cs, precision, oBf16: precision === "bf16" });
  into(await wide(a), b.self.o, m.self);
  const q = ops.linear(gpu, norm(m.cross), b.cross.q, { precision });
  const k = ops.linear(gpu, cond.ctx, b.cross.k, {}), v = ops.linear(gpu, cond.ctx, b.cross.v, {});
  ops.rmsnorm(gpu, k, b.cross.kn, HD, 1e-6, k);
  const c = ops.attention(gpu, { q, k, v, B, Lq: L, Lk: cond.Lk, H, D: HD, ldq: D, ldk: D, ldv: D, qNorm: b.cross.qn, precision,
    oBf16: precision === "bf16" });
  into(await wide(c), b.cross.o, m.cross);
  const h = ops.linear(gpu, norm(m.mlp), b.l1, { act: "gelu", precision, outBf16: precision === "bf16" });
  into(await wide(h), b.l2, m.mlp);
}

async function ditsteps(gpu, c) {
  const src = new SyntheticWeights(gpu, c.seed, { blocks: c.kinds.length });
  src.quantKind = (i) => c.kinds[i];
  const model = AnimaDiT.synthetic(gpu, src);
  console.log(JSON.stringify({ converted: model.quantizeF8() }));
  const B = c.latents.length, L = (c.h / 2) * (c.w / 2), tc = model.timeCond(c.sigma);
  for (const precision of ["fp32", "bf16"]) {
    model.precision = precision;
    const cond = model.prepareContext(c.ctx.map((p) => gpu.fromArray(load(p), [c.Lk, 1024])));
    const xs = [];
    await model.forward(c.latents.map((p) => load(p)), c.h, c.w, cond, tc, async (i, x) => xs.push(await gpu.read(x)));
    for (let i = 1; i < xs.length; i++) {
      if (c.kinds[i] !== "bf16") continue;
      const x = gpu.fromArray(xs[i - 1], [B * L, 2048]);
      await blockSteps(gpu, model, i, x, cond, tc, B, L, model.ropeTable(c.h / 2, c.w / 2));
      save(`${c.out}.${precision}.${i}`, xs[i]);
      save(`${c.out}.${precision}.${i}.steps`, await gpu.read(x));
    }
    cond.release();
  }
}

const c = JSON.parse(fs.readFileSync(process.argv[2], "utf8"));
GPU.create({})
  .then(async (gpu) => {
    await { block, groups, qwen3, dit, ditsteps }[c.case](gpu, c);
    gpu.destroy();
  })
  .catch((e) => {
    console.error(e);
    process.exit(1);
  });
