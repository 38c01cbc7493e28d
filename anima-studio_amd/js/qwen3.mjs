// The Qwen3-0.6B text encoder of Anima (app/models/qwen3.js:1-79) on this build's ops: 28 layers
// of RMSNorm -> q/k/v linears -> per-head q/k RMSNorm -> 1D RoPE -> causal GQA attention (16 query
// heads over 8 kv heads, on the flash kernels) -> o linear (residual) -> RMSNorm -> gate/up
// linears -> SiLU(gate) * up -> down linear (residual); the final RMSNorm's output is the hidden
// state the DiT's context is built from.  Node-12 syntax only.

import * as ops from "./ops.mjs";
import { ropeTable } from "./common.mjs";
import { concatLinears } from "./weights.mjs";
import { native } from "./gpu.mjs";
import { loraGeneration } from "./lora.mjs";

const LINEARS = ["qkv", "q", "k", "v", "o", "gate", "up", "down"];

function releaseGraph(gpu, g) {
  native.graphDestroy(gpu.ctx, g.graph);
  for (const t of [g.out, g.x, g.cs]) t.release();
}

// a weight object or a tensor
function releaseWeight(t) {
  if (!t) return;
  if (t.buf && t.buf.release) t.buf.release();
  else if (t.release) t.release();
  for (const f of ["scale", "srel", "codebook", "bias", "groupScale", "groupMid"]) if (t[f] && t[f].release) t[f].release();
}

// q, k and v of a layer stacked into one [(H + 2 KH) HD, D] linear (one GEMM per layer instead
// of three; the q/k RMSNorm and RoPE then run inside the attention's loads).  Formats that
// cannot be stacked (W4 parts with different codebooks) keep the three linears.
function stackQKV(gpu, l) {
  const qkv = concatLinears(gpu, [l.q, l.k, l.v]);
  if (!qkv) return;
  l.qkv = qkv;
  delete l.q;
  delete l.k;
  delete l.v;
}

const hasLora = (l) => LINEARS.some((k) => l[k] && l[k].lora && l[k].lora.length > 0);
// whether a layer runs on e4m3 rows from norm to norm (layersF8)
const isF8 = (l) => !!l.qkv && ["qkv", "o", "gate", "up", "down"].every((k) => l[k].kind === "f8") &&
  l.gate.K === l.up.K && l.gate.N === l.up.N && !hasLora(l);

// The number of ids that all prompts begin with, or 0 where sharing them saves fewer than SHARE_ROWS rows: the
// prefix costs two more calls a layer.  The 28 layers of 8 prompts with 77 shared ids and 40 of their own
// (539 rows saved) take 4.4 ms shared and 5.0 apart, of 2 with 77 and 77 (77 rows) 4.1 and 3.6.
const SHARE_ROWS = 256;
function commonPrefix(prompts) {
  let n = 0;
  while (n < prompts[0].length && prompts.every((p) => p[n] === prompts[0][n])) n++;
  return (prompts.length - 1) * n < SHARE_ROWS ? 0 : n;
}

export const QWEN3 = { layers: 28, hidden: 1024, heads: 16, kvHeads: 8, headDim: 128, mlp: 3072, theta: 1e6, vocab: 151936 };

export class Qwen3 {
  // Weights from a safetensors file in the reference's names (qwen3.js:8-31).
  static async load(gpu, st, onProgress) {
    const m = new Qwen3(gpu, QWEN3);
    m.layers = [];
    for (let i = 0; i < QWEN3.layers; i++) {
      const p = `model.layers.${i}.`;
      m.layers.push({
        ln1: st.vector(gpu, p + "input_layernorm.weight"),
        ln2: st.vector(gpu, p + "post_attention_layernorm.weight"),
        qn: st.vector(gpu, p + "self_attn.q_norm.weight"),
        kn: st.vector(gpu, p + "self_attn.k_norm.weight"),
        q: st.linear(gpu, p + "self_attn.q_proj."),
        k: st.linear(gpu, p + "self_attn.k_proj."),
        v: st.linear(gpu, p + "self_attn.v_proj."),
        o: st.linear(gpu, p + "self_attn.o_proj."),
        gate: st.linear(gpu, p + "mlp.gate_proj."),
        up: st.linear(gpu, p + "mlp.up_proj."),
        down: st.linear(gpu, p + "mlp.down_proj."),
      });
      stackQKV(gpu, m.layers[i]);
      if (onProgress) onProgress((i + 1) / QWEN3.layers);
    }
    m.norm = st.vector(gpu, "model.norm.weight");
    m.embedRows = (ids) => st.rows("model.embed_tokens.weight", ids);
    m.loadTable = () => st.table(gpu, "model.embed_tokens.weight");
    return m;
  }

  // Seeded random-init weights of the same architecture (bf16 linears, norm weights near 1, an
  // embedding table of `vocab` rows held on the host); opts: { layers, vocab }.
  static synthetic(gpu, src, opts) {
    const o = opts || {};
    const cfg = Object.assign({}, QWEN3, { layers: o.layers || QWEN3.layers, vocab: o.vocab || 4096 });
    const m = new Qwen3(gpu, cfg);
    const { hidden: D, heads: H, kvHeads: KH, headDim: HD, mlp: F } = cfg;
    m.layers = [];
    for (let i = 0; i < cfg.layers; i++) {
      // the checkpoint's module names (qwen3.js:8-31), so that LoRA files address these linears
      const p = `model.layers.${i}.`;
      m.layers.push({
        ln1: src.vector(gpu, p + "input_layernorm.weight", D), ln2: src.vector(gpu, p + "post_attention_layernorm.weight", D),
        qn: src.vector(gpu, p + "self_attn.q_norm.weight", HD), kn: src.vector(gpu, p + "self_attn.k_norm.weight", HD),
        q: src.bf16Linear(gpu, p + "self_attn.q_proj", H * HD, D, 1.0), k: src.bf16Linear(gpu, p + "self_attn.k_proj", KH * HD, D, 1.0),
        v: src.bf16Linear(gpu, p + "self_attn.v_proj", KH * HD, D, 1.0), o: src.bf16Linear(gpu, p + "self_attn.o_proj", D, H * HD, 0.5),
        gate: src.bf16Linear(gpu, p + "mlp.gate_proj", F, D, 1.0), up: src.bf16Linear(gpu, p + "mlp.up_proj", F, D, 1.0),
        down: src.bf16Linear(gpu, p + "mlp.down_proj", D, F, 0.5),
      });
      stackQKV(gpu, m.layers[i]);
    }
    m.norm = src.vector(gpu, "model.norm.weight", D);
    const table = gpu.empty([cfg.vocab * D]);
    src.fill(table, "f32", "model.embed_tokens.weight", -1, 1);
    m.table = table;
    m.embedRows = async (ids) => {
      const all = await gpu.read(table);
      const out = new Float32Array(ids.length * D);
      ids.forEach((id, i) => out.set(all.subarray(id * D, (id + 1) * D), i * D));
      return out;
    };
    m.loadTable = async () => {
      const buf = gpu.empty([cfg.vocab, D]);
      gpu.copy(buf, table, cfg.vocab * D * 4);
      return { kind: "f32", N: cfg.vocab, K: D, buf };
    };
    return m;
  }

  constructor(gpu, cfg) {
    this.gpu = gpu;
    this.cfg = cfg;
    // precision of the attention ("fp32": 32-bit products), and of the products of e4m3 layers and of 4-bit weights
    this.precision = "bf16";
    this.graphs = true; // replay the layers from a recorded HIP graph (per token count and precision)
    this.graphCache = new Map();
    this.deviceTable = null; // the embedding table, after embedOnDevice
    this.conversions = 0; // of the weights; a kept prefix belongs to one
  }

  // Loads the embedding table to the device, where every encoding then takes its rows from (ops.embedRows)
  // instead of reading them on the host.  opts.q4: { group, mid } converts it to 4 bits (ops.quantizeQ4); else
  // the rows are the same values.
  async embedOnDevice(opts) {
    const table = await this.loadTable();
    if (opts && opts.q4) ops.quantizeQ4(this.gpu, table, opts.q4);
    releaseWeight(this.deviceTable);
    this.deviceTable = table;
    this.conversions++;
  }

  // ids' rows of the embedding table, read: a function that writes them to a tensor [ids.length, D]
  async rowsOf(ids) {
    const t = this.deviceTable;
    if (!t) {
      const rows = await this.embedRows(ids);
      return (x) => this.gpu.write(x, rows);
    }
    for (const id of ids) if (!(Number.isInteger(id) && id >= 0 && id < t.N)) throw new Error(`token id ${id} outside the embedding table [${t.N},${t.K}]`);
    return (x) => ops.embedRows(this.gpu, this.deviceTable, ids, { out: x }); // (the table of that moment: t may have been replaced)
  }

  // ids -> Tensor [L, 1024] (qwen3.js:38-78).  With this.graphs (the default) the 28 layers run as a
  // HIP graph recorded once per (token count, attention precision): the host only uploads the
  // embedding rows and replays it (the same kernels and arguments as the eager pass, so the same
  // result), which removes the per-kernel launch cost of ~280 short kernels.
  async encode(ids) {
    const gpu = this.gpu;
    const { hidden: D, headDim: HD } = this.cfg;
    const Lt = ids.length;
    const fill = await this.rowsOf(ids);
    // LoRA side paths (attachLoras) run eagerly: a graph recorded before an attach would not hold them
    const lora = this.layers.some(hasLora);
    if (!this.graphs || lora) {
      const x = gpu.empty([Lt, D]);
      fill(x);
      const cs = ropeTable(gpu, Lt, HD, this.cfg.theta);
      const out = this.layersDevice(x, cs, Lt);
      cs.release();
      x.release();
      return out;
    }
    const key = `${Lt}:${this.precision}`;
    let g = this.graphCache.get(key);
    if (!g) {
      g = this.recordGraph(fill, Lt);
      if (this.graphCache.size >= 4) {
        const [k0, g0] = this.graphCache.entries().next().value;
        this.graphCache.delete(k0);
        releaseGraph(gpu, g0);
      }
    } else {
      this.graphCache.delete(key);  // most recently used last
    }
    this.graphCache.set(key, g);
    fill(g.x);
    native.graphLaunch(gpu.ctx, g.graph);
    const out = gpu.empty([Lt, D]);
    gpu.copy(out, g.out, Lt * D * 4);
    return out;
  }

  // The fixed residual-stream buffer, RoPE table and output of one token count, and the graph of
  // the layers over them (recorded after one eager pass, so the pool already holds its buffers).
  recordGraph(fill, Lt) {
    const gpu = this.gpu;
    const { hidden: D, headDim: HD } = this.cfg;
    const x = gpu.empty([Lt, D]);
    fill(x);
    const cs = ropeTable(gpu, Lt, HD, this.cfg.theta);
    this.layersDevice(x, cs, Lt).release();
    native.graphBegin(gpu.ctx);
    let out = null, graph = 0;
    try {
      out = this.layersDevice(x, cs, Lt);
    } finally {
      if (out) graph = native.graphEnd(gpu.ctx);
      else {
        try {
          native.graphDestroy(gpu.ctx, native.graphEnd(gpu.ctx));
        } catch (e) {
          // the capture was already invalid: graphEnd discarded it
        }
        x.release();
        cs.release();
      }
    }
    return { x, cs, out, graph };
  }

  // Converts the layers' bf16 linears to e4m3 with one scale per 128 x 128 block (ops.quantizeF8): half
  // the bytes, and the layers then run on e4m3 rows (layersF8).  An option for a caller who accepts
  // 8-bit weights and activations; the checkpoint's form is the default.
  // Returns the number of linears converted.
  quantizeF8() {
    return this.convert((W) => ops.quantizeF8(this.gpu, W).kind === "f8");
  }

  // Converts the layers' bf16 linears to 4 bits with one scale per opts.group values (ops.quantizeQ4; opts.mid: and
  // a middle value): close to a quarter of the bytes.  An option as quantizeF8.  The activations are fp32 rows, which the
  // products at this.precision "bf16" (the default) round to 11 bits where they run on the matrix cores, and at "fp32" keep.
  // Returns the number of linears converted.
  quantizeQ4(opts) {
    return this.convert((W) => ops.quantizeQ4(this.gpu, W, opts).kind === "q4");
  }

  convert(one) {
    let n = 0;
    for (const l of this.layers)
      for (const k of LINEARS) if (l[k] && (l[k].kind === "bf16" || l[k].kind === "f32") && one(l[k])) n++;
    for (const g of this.graphCache.values()) releaseGraph(this.gpu, g);
    this.graphCache.clear();
    if (n) this.conversions++;
    return n;
  }

  // What a kept prefix has to have in common with an encoding that reads it
  stateKey() {
    return `${this.precision}:${this.conversions}:${loraGeneration()}`;
  }

  checkPrefix(kept) {
    if (!kept) return;
    if (kept.owner !== this) throw new Error("encodeBatch: opts.prefix is of another encoder");
    if (!kept.hidden.buf) throw new Error("encodeBatch: opts.prefix has been released");
    if (kept.key !== this.stateKey()) throw new Error("encodeBatch: opts.prefix is of another precision, other weights or other LoRAs");
  }

  // The tokens that a series of prompts begins with (a template), encoded once for encodeBatch's opts.prefix:
  // each layer's keys and values as ops.attentionPrefixPrepare lays them out, and the tokens' hidden states (under
  // the causal mask neither depends on what follows).  Belongs to the caller (release()); it is of no use to
  // another encoder, or after a change of the precision, the weights or the LoRAs, and encodeBatch then refuses it.
  async keepPrefix(ids) {
    if (!ids.length) throw new Error("keepPrefix: no tokens");
    const kv = [], key = this.stateKey();
    const hidden = await this.runBatch(ids, { P: ids.length, lens: [], keep: kv });
    return { owner: this, ids: Array.from(ids), kv, hidden, key, release() { for (const t of kv.concat([hidden])) t.release(); } };
  }

  // Several prompts (arrays of ids) at once -> one Tensor [length, D] each, as encode gives it.  The tokens that
  // they all begin with, where they are enough (or opts.prefix of keepPrefix, which all have to begin with), pass
  // the layers once, and the rest of all prompts in one pass behind them: every weight is read once for the batch.
  async encodeBatch(prompts, opts) {
    const gpu = this.gpu, D = this.cfg.hidden;
    const kept = (opts && opts.prefix) || null;
    prompts.forEach((p, i) => {
      if (!p.length) throw new Error(`encodeBatch: prompt ${i} has no tokens`);
      if (kept && !kept.ids.every((id, j) => id === p[j])) throw new Error(`encodeBatch: prompt ${i} does not begin with opts.prefix`);
    });
    this.checkPrefix(kept);
    if (!prompts.length) return [];
    const P = kept ? kept.ids.length : commonPrefix(prompts), lens = prompts.map((p) => p.length - P);
    const ids = kept ? [] : Array.from(prompts[0]).slice(0, P);
    for (const p of prompts) for (let i = P; i < p.length; i++) ids.push(p[i]);
    const all = ids.length ? await this.runBatch(ids, { P: kept ? 0 : P, lens, kept }) : null;
    const head = kept ? kept.hidden : all;
    let row = kept ? 0 : P;
    const out = prompts.map((p, i) => {
      const t = gpu.empty([p.length, D]);
      if (P) gpu.copy(t, head, P * D * 4);
      if (lens[i]) gpu.copy(t.at(P * D), all.at(row * D), lens[i] * D * 4);
      row += lens[i];
      return t;
    });
    if (all) all.release();
    return out;
  }

  // The layers over batch.P rows of a prefix (at positions 0 ...) and behind them batch.lens rows of each sequence
  // (behind those, or behind batch.kept): the normed hidden states of all rows.
  async runBatch(ids, batch) {
    const gpu = this.gpu, { hidden: D, headDim: HD } = this.cfg;
    const fill = await this.rowsOf(ids);
    this.checkPrefix(batch.kept); // (again: the rows may have been waited for)
    const x = gpu.empty([ids.length, D]);
    fill(x);
    const P = batch.kept ? batch.kept.ids.length : batch.P;
    const cs = ropeTable(gpu, P + batch.lens.reduce((a, n) => Math.max(a, n), 0), HD, this.cfg.theta);
    const out = this.layersDevice(x, cs, ids.length, batch);
    cs.release();
    x.release();
    return out;
  }

  // Layer i's attention of a batch on its normed rows h: the prefix's rows among themselves, then all
  // sequences behind the prefix's prepared keys and values.
  batchAttention(l, i, h, hr, cs, batch) {
    const gpu = this.gpu, precision = this.precision;
    const { heads: H, kvHeads: KH, headDim: HD } = this.cfg, { P, lens } = batch;
    const rows = h.shape[0], T = rows - P, ld = (H + 2 * KH) * HD;
    const qkv = l.qkv ? this.project(h, l.qkv, { xr: hr }) : null;
    const [q, k, v] = qkv ? [qkv, qkv, qkv] : [l.q, l.k, l.v].map((W) => this.project(h, W, { xr: hr }));
    const d = { H, D: HD, group: H / KH, qNorm: l.qn, kNorm: l.kn, cs, precision, causal: true, ldq: qkv ? ld : H * HD,
      ldk: qkv ? ld : KH * HD, ldv: qkv ? ld : KH * HD, kOff: qkv ? H * HD : 0, vOff: qkv ? (H + KH) * HD : 0 };
    const a = gpu.empty([rows, H * HD]);
    let prefix = batch.kept ? batch.kept.kv[i] : null;
    if (P) {
      ops.attention(gpu, Object.assign({ q, k, v, Lq: P, Lk: P, out: a }, d));
      if (T || batch.keep) prefix = ops.attentionPrefixPrepare(gpu, Object.assign({ k, v, len: P }, d));
    }
    if (T) {
      const own = (t, ldt) => t.view(P * ldt, [T, ldt]);
      ops.attentionPrefix(gpu, Object.assign({ q: own(q, d.ldq), k: own(k, d.ldk), v: own(v, d.ldv), lens, prefix, out: own(a, H * HD) }, d));
    }
    if (batch.keep) batch.keep.push(prefix);
    else if (P && prefix) prefix.release();
    for (const t of qkv ? [qkv] : [q, k, v]) t.release();
    return a;
  }

  // ops.linear, on 4-bit weights at the encoder's precision
  project(x, W, opts) {
    return ops.linear(this.gpu, x, W, W.kind === "q4" ? Object.assign({ precision: this.precision }, opts) : opts);
  }

  // The layers on e4m3 weights: every product reads e4m3 rows that the kernel before it wrote.  A
  // layer is seven launches: seam (residual addition + norm), qkv, attention, its rows to e4m3, o,
  // seam, gate / up / SiLU, down; the last seam is the final norm.
  layersF8(x, cs, Lt) {
    const gpu = this.gpu;
    const { hidden: D, heads: H, kvHeads: KH, headDim: HD } = this.cfg;
    const ld = (H + 2 * KH) * HD, precision = this.precision, bf16 = precision === "bf16";
    let y = null;
    const seam = (weight, f8) => {
      const r = ops.residualNorm(gpu, x, D, { y, weight, f8 });
      if (y) y.release();
      y = null;
      return r;
    };
    for (const l of this.layers) {
      const h = seam(l.ln1, true);
      const qkv = ops.linear(gpu, null, l.qkv, { xq: h, precision });
      h.release();
      const a = ops.attention(gpu, { q: qkv, k: qkv, v: qkv, Lq: Lt, Lk: Lt, H, D: HD, ldq: ld, ldk: ld, ldv: ld, qOff: 0,
        kOff: H * HD, vOff: (H + KH) * HD, group: H / KH, causal: true, qNorm: l.qn, kNorm: l.kn, cs, precision,
        oBf16: bf16 });
      qkv.release();
      const aq = ops.quantRowsF8(gpu, a, H * HD);
      a.release();
      y = ops.linear(gpu, null, l.o, { xq: aq, precision, outBf16: bf16 });
      aq.release();
      const h2 = seam(l.ln2, true);
      const gu = ops.linearGlu(gpu, null, l.gate, l.up, { xq: h2, precision, f8: true });
      h2.release();
      y = ops.linear(gpu, null, l.down, { xq: gu, precision, outBf16: bf16 });
      gu.release();
    }
    return seam(this.norm, false).h;
  }

  // The decoder layers and the final RMSNorm on the residual stream x [Lt, D] (updated in place);
  // returns the normed hidden states (a new tensor).  batch: the rows of runBatch instead of one sequence.
  layersDevice(x, cs, Lt, batch) {
    const gpu = this.gpu;
    const { hidden: D, heads: H, kvHeads: KH, headDim: HD } = this.cfg;
    if (!batch && this.layers.length && this.layers.every(isF8)) return this.layersF8(x, cs, Lt);
    for (let i = 0; i < this.layers.length; i++) {
      const l = this.layers[i];
      const h = ops.rmsnorm(gpu, x, l.ln1, D);
      const hr = ops.needsRotation(l.qkv || l.q) ? ops.rotate(gpu, h) : null;
      let a;
      if (batch) {
        a = this.batchAttention(l, i, h, hr, cs, batch);
      } else if (l.qkv) {
        // one GEMM for q, k and v; their per-head RMSNorm and RoPE run in the attention's loads
        const qkv = this.project(h, l.qkv, { xr: hr });
        const ld = (H + 2 * KH) * HD;
        a = ops.attention(gpu, { q: qkv, k: qkv, v: qkv, Lq: Lt, Lk: Lt, H, D: HD, ldq: ld, ldk: ld, ldv: ld, qOff: 0,
          kOff: H * HD, vOff: (H + KH) * HD, group: H / KH, causal: true, qNorm: l.qn, kNorm: l.kn, cs,
          precision: this.precision });
        qkv.release();
      } else {
        const q = this.project(h, l.q, { xr: hr });
        const k = this.project(h, l.k, { xr: hr });
        const v = this.project(h, l.v, { xr: hr });
        const qn = ops.rmsnorm(gpu, q, l.qn, HD);
        const kn = ops.rmsnorm(gpu, k, l.kn, HD);
        q.release();
        k.release();
        ops.rope(gpu, qn, cs, Lt, H, HD);
        ops.rope(gpu, kn, cs, Lt, KH, HD);
        a = ops.attention(gpu, { q: qn, k: kn, v, Lq: Lt, Lk: Lt, H, D: HD, ldq: H * HD, ldk: KH * HD, ldv: KH * HD,
          group: H / KH, causal: true, precision: this.precision });
        qn.release();
        kn.release();
        v.release();
      }
      if (hr) hr.release();
      h.release();
      this.project(a, l.o, { out: x, resid: true });
      a.release();
      const h2 = ops.rmsnorm(gpu, x, l.ln2, D);
      const h2r = ops.needsRotation(l.gate) ? ops.rotate(gpu, h2) : null;
      const g = this.project(h2, l.gate, { xr: h2r });
      const u = this.project(h2, l.up, { xr: h2r });
      if (h2r) h2r.release();
      h2.release();
      const gu = ops.elementwise(gpu, "silu_mul", g, u);
      g.release();
      u.release();
      this.project(gu, l.down, { out: x, resid: true });
      gu.release();
    }
    return ops.rmsnorm(gpu, x, this.norm, D);
  }

  release() {
    for (const g of this.graphCache.values()) releaseGraph(this.gpu, g);
    this.graphCache.clear();
    for (const l of this.layers || []) for (const key of Object.keys(l)) releaseWeight(l[key]);
    releaseWeight(this.norm);
    releaseWeight(this.table);
    releaseWeight(this.deviceTable);
    this.deviceTable = null;
    this.layers = [];
  }
}
