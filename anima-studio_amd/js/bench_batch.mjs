// Batches of prompts on a synthetic text encoder of 28 layers, on bf16 weights and on 4-bit ones (groups of 64): the prompts
// one by one (encode, which replays a graph), together (encodeBatch, the shared tokens once), together behind a kept
// prefix, and together without a shared token.  Milliseconds a batch, host included; one line of JSON a batch.
//
//   node bench_batch.mjs [--precision bf16|fp32] [--steps 10]

import { GPU } from "./gpu.mjs";
import { SyntheticWeights } from "./weights.mjs";
import { Qwen3 } from "./qwen3.mjs";

function arg(name, def) {
  const i = process.argv.indexOf("--" + name);
  return i < 0 ? def : process.argv[i + 1];
}

// [shared tokens, prompts, tokens of their own]
const BATCHES = [[77, 2, 40], [77, 8, 40], [77, 32, 40], [400, 32, 60]];
const VOCAB = 4096;

async function main() {
  const gpu = await GPU.create({});
  const te = Qwen3.synthetic(gpu, new SyntheticWeights(gpu, 23), { vocab: VOCAB });
  const steps = Number(arg("steps", 10));
  te.precision = arg("precision", "bf16");
  await te.embedOnDevice();
  const ids = (n, seed) => Array.from({ length: n }, (_, i) => (i * 7919 + seed * 104729) % (VOCAB - 96));
  const time = async (f) => {
    for (let i = 0; i < 3; i++) await f();
    await gpu.sync();
    const t0 = process.hrtime.bigint();
    for (let i = 0; i < steps; i++) await f();
    await gpu.sync();
    return Number(process.hrtime.bigint() - t0) / 1e6 / steps;
  };
  const all = async (prompts, opts) => {
    for (const t of await te.encodeBatch(prompts, opts)) t.release();
  };
  for (const weights of ["bf16", "q4"]) {
    if (weights === "q4") te.quantizeQ4();
    for (const [shared, n, own] of BATCHES) {
      const head = ids(shared, 1), prompts = Array.from({ length: n }, (_, i) => head.concat([VOCAB - 96 + i], ids(own - 1, i + 2)));
      const apart = prompts.map((p, i) => [VOCAB - 96 + i].concat(p.slice(1)));
      const prefix = await te.keepPrefix(head);
      const ms = {
        one_by_one: await time(async () => {
          for (const p of prompts) (await te.encode(p)).release();
        }),
        together: await time(() => all(prompts)),
        kept: await time(() => all(prompts, { prefix })),
        not_shared: await time(() => all(apart)),
      };
      prefix.release();
      for (const k of Object.keys(ms)) ms[k] = Number(ms[k].toFixed(2));
      console.log(JSON.stringify({ weights, precision: te.precision, prompts: n, shared, own, ms }));
    }
  }
  te.release();
  gpu.destroy();
}

main().catch((e) => {
  console.error(e);
  process.exit(1);
});
