// Batches of prompts on a text encoder of every kind of weight: writes Qwen3.encodeBatch's and Qwen3.encode's hidden states of
// each prompt, in both precisions.  node run_kinds.mjs case.json, with { kind, layers, vocab, prompts, keep, out }:
//   bf16, f8 (quantizeF8), i8, w4       one kind in every linear
//   unstacked                           w4 whose q, k and v have different codebooks: three products
//   mixed                               e4m3 in the first layer, 4-bit scales in the rest

import fs from "fs";
import { GPU } from "../../anima-studio_amd/js/gpu.mjs";
import * as ops from "../../anima-studio_amd/js/ops.mjs";
import { SyntheticWeights } from "../../anima-studio_amd/js/weights.mjs";
import { Qwen3 } from "../../anima-studio_amd/js/qwen3.mjs";

const c = JSON.parse(fs.readFileSync(process.argv[2], "utf8"));

function source(gpu) {
  const src = new SyntheticWeights(gpu, 23, { mode: c.kind === "i8" ? "int8" : "w4a8", blocks: 3 });
  if (c.kind === "i8" || c.kind === "w4" || c.kind === "unstacked") {
    src.bf16Linear = (g, name, N, K) => {
      const W = src.blockLinear(g, name, N, K, 1);
      if (c.kind === "unstacked") {
        const f = name.endsWith("k_proj") ? 0.75 : name.endsWith("v_proj") ? 1.25 : 1;
        W.codebookData = W.codebookData.map((v) => v * f);
        W.codebook = g.upload(W.codebookData);
      }
      return W;
    };
  }
  return src;
}

GPU.create({})
  .then(async (gpu) => {
    const te = Qwen3.synthetic(gpu, source(gpu), { layers: c.layers, vocab: c.vocab });
    if (c.kind === "f8") te.quantizeF8();
    if (c.kind === "mixed") {
      te.layers.forEach((l, i) => {
        for (const k of Object.keys(l)) if (l[k].kind === "bf16") i === 0 ? ops.quantizeF8(gpu, l[k]) : ops.quantizeQ4(gpu, l[k]);
      });
    }
    const kinds = te.layers.map((l) => Object.keys(l).filter((k) => l[k].kind).map((k) => `${k}:${l[k].kind}`).sort().join(" "));
    for (const prec of ["fp32", "bf16"]) {
      te.precision = prec;
      const prefix = await te.keepPrefix(c.prompts[0].slice(0, c.keep));
      const sets = { batch: await te.encodeBatch(c.prompts), kept: await te.encodeBatch(c.prompts, { prefix }) };
      sets.one = [];
      for (const p of c.prompts) sets.one.push(await te.encode(p));
      prefix.release();
      for (const name of Object.keys(sets))
        for (let i = 0; i < c.prompts.length; i++) {
          fs.writeFileSync(`${c.out}.${prec}.${name}.${i}`, Buffer.from((await gpu.read(sets[name][i])).buffer));
          sets[name][i].release();
        }
    }
    te.release();
    console.log(JSON.stringify(kinds));
    gpu.destroy();
  })
  .catch((e) => {
    console.error(e);
    process.exit(1);
  });
