"""What a batch of prompts keeps between its calls and its turns of the event loop, on the CPU: the native calls are recorded
instead of made."""

import pytest

from test_batch_js import NODE, RECORD, node

pytestmark = pytest.mark.skipif(NODE is None, reason="node is not installed")

# two-layer encoders of width 256, and a promise that is settled from outside
ENCODER = (RECORD + "const W = (N, K) => ({ kind: 'bf16', N, K, buf: ++last });"
           "const encoder = (Qwen3, layers) => { const te = new Qwen3(gpu, { hidden: 256, heads: 2, kvHeads: 1, headDim: 128, mlp: 256, theta: 1e6 });"
           " te.layers = Array.from({ length: layers }, () => ({ qkv: W(512, 256), o: W(256, 256), gate: W(256, 256), up: W(256, 256), down: W(256, 256),"
           "  ln1: tensor([256]), ln2: tensor([256]), qn: tensor([128]), kn: tensor([128]) }));"
           " te.norm = tensor([256]); te.embedRows = async (ids) => new Float32Array(ids.length * 256); return te; };"
           "const err = async (f) => { try { await f(); return ''; } catch (e) { return e.message; } };")


def test_prefix_of_another_encoder():
    """A kept prefix belongs to the encoder that made it: another one has other weights, and may have other layers."""
    got = node(ENCODER + "import('./qwen3.mjs').then(async ({ Qwen3 }) => {"
               "const a = encoder(Qwen3, 2), b = encoder(Qwen3, 2), c = encoder(Qwen3, 3), prefix = await a.keepPrefix([1, 2]);"
               "const go = (te) => err(() => te.encodeBatch([[1, 2, 3]], { prefix }));"
               "console.log(JSON.stringify([await go(a), await go(b), await go(c)])); })")
    assert got[0] == "" and all("another encoder" in e for e in got[1:]), got


# a pipeline whose text encoder and adapter wait until they are told to go on; conditionings count their releases
PIPELINE = (RECORD + "import('./pipeline.mjs').then(async ({ LatentPipeline }) => { const lora = await import('./lora.mjs');"
            "const conds = [], hidden = [], waits = []; let ready = [];"
            "const dit = { prepareContext: ([c]) => { c.release(); const t = { n: conds.length, freed: 0, release() { this.freed++; } }; conds.push(t); return t; } };"
            "const h = () => { const t = tensor([3, 1024]); hidden.push(t); return t; };"
            "const gate = () => new Promise((ok, no) => waits.push({ ok, no }));"
            "const te = { encode: async () => { await gate(); return h(); }, encodeBatch: async (p) => { await gate(); return p.map(h); } };"
            "const A = { blocks: [], outProj: { kind: 'bf16', N: 1024, K: 1024, buf: 1 }, norm: tensor([1024]), embedRows: async (ids) => { await gate(); return new Float32Array(ids.length * 1024); } };"
            "gpu.read = async (t) => new Float32Array(t.size);"
            "const p = new LatentPipeline(gpu, dit, { te, adapter: A });"
            "const prompt = (key) => ({ key, qwenIds: [1, 2], t5Ids: [3], t5Weights: null });"
            "const tick = () => new Promise((r) => setTimeout(r, 1));"
            "const go = async (n) => { for (let i = 0; i < n; i++) { await tick(); const w = waits.shift(); if (w) w.ok(); } await tick(); };"
            "const done = async (q) => { let r; q.then((v) => { r = { v }; }, (e) => { r = { e: e.message }; }); for (let i = 0; i < 40 && !r; i++) await go(1); return r; };"
            "const out = {};")


def test_overlapping_calls():
    """encodeBatch beside calls that want other prompts: what it returns is whole, in order, and not released."""
    got = node(PIPELINE +
               "const a = (await done(p.encode(prompt('a')))).v;"
               "const batch = p.encodeBatch([prompt('b'), prompt('a'), prompt('c'), prompt('b')]);"
               "await go(2);"  # b is there, c under way
               "const d = p.encode(prompt('d'));"
               "const r = (await done(batch)).v, dd = (await done(d)).v;"
               "out.whole = r.map((t) => t && t.freed); out.order = [r[1] === a, r[0] === r[3], new Set(r.concat([dd])).size];"
               "out.hidden = hidden.every((t) => t.released === 1); out.held = p.ctxHeld.size;"
               # the next call drops what it does not want, once
               "const e = (await done(p.encode(prompt('d')))).v; out.next = [e === dd, conds.map((t) => t.freed), p.ctxCache.size];"
               # the same prompt twice at once: one conditioning in the end
               "const two = [p.encodeBatch([prompt('e')]), p.encodeBatch([prompt('e')]), p.encode(prompt('e'))];"
               "const n = conds.length, x = []; for (const q of two) x.push(...[].concat((await done(q)).v));"
               "out.same = [new Set(x).size, conds.length - n, p.ctxCache.get('e') === x[0], x[0].freed];"
               # the cache cleared under a call that returns an entry of it
               "const hit = p.encodeBatch([prompt('e'), prompt('f')]); await tick(); p.clearContexts(); out.cleared = (await done(hit)).v.map((t) => t.freed);"
               "console.log(JSON.stringify(out)); });")
    assert got["whole"] == [0, 0, 0, 0] and got["order"] == [True, True, 4] and got["hidden"] and got["held"] == 0
    assert got["next"] == [True, [1, 1, 1, 0], 1]
    assert got["same"] == [1, 1, True, 0] and got["cleared"] == [0, 0]


def test_failures_release():
    """An adapter that fails, and LoRAs attached on the way: an error, every hidden state released once, nothing held, nothing stale."""
    got = node(PIPELINE +
               "const fail = p.encodeBatch([prompt('a'), prompt('b'), prompt('c')]); fail.catch(() => {}); await go(2); await tick();"
               "waits.shift().no(new Error('lost')); out.fail = (await done(fail)).e; out.hidden = hidden.map((t) => t.released);"
               "out.held = p.ctxHeld.size; out.keys = Array.from(p.ctxCache.keys());"
               "const b = p.encodeBatch([prompt('a'), prompt('x'), prompt('y')]); b.catch(() => {}); await go(2); lora.attachLoras({}, []);"
               "out.lora = (await done(b)).e; const z = (await done(p.encode(prompt('z')))).v;"
               "out.left = [Array.from(p.ctxCache.keys()), z.freed, p.ctxHeld.size, hidden.every((t) => t.released === 1)];"
               "console.log(JSON.stringify(out)); });")
    assert got["fail"] == "lost" and got["hidden"] == [1, 1, 1] and got["held"] == 0 and got["keys"] == ["a"]
    assert "LoRAs were attached" in got["lora"] and got["left"] == [["z"], 0, 0, True]


def test_ids_that_are_no_row():
    """Ids from the host that no 32-bit index holds: rows of zeros, as any outside the table; the encoder refuses them."""
    got = node(ENCODER + "import('./ops.mjs').then(async (ops) => { const { Qwen3 } = await import('./qwen3.mjs');"
               "const sent = []; const from = gpu.fromArray; gpu.fromArray = (a, s) => { sent.push(Array.from(a)); return from(a, s); };"
               "ops.embedRows(gpu, { kind: 'f32', N: 10, K: 128, buf: 1 }, [0, 9, 10, -1, 4294967296, 4294967299, NaN, undefined, 1.5, -0.5, Infinity]);"
               "const te = encoder(Qwen3, 1); te.deviceTable = { kind: 'f32', N: 10, K: 256, buf: 1 };"
               "console.log(JSON.stringify([sent[0], await err(() => te.encodeBatch([[1, 1.5]])), await err(() => te.encodeBatch([[NaN]]))])); })")
    assert got[0] == [0, 9] + [-1] * 9
    assert "token id 1.5 outside" in got[1] and "token id NaN outside" in got[2]


def test_table_replaced_under_an_encoding():
    """embedOnDevice that ends between an encoding's check of its ids and its launches: the rows come from the new table."""
    got = node(ENCODER + "import('./qwen3.mjs').then(async ({ Qwen3 }) => { const te = encoder(Qwen3, 1);"
               "const table = () => ({ kind: 'f32', N: 10, K: 256, buf: tensor([10, 256]) }); te.loadTable = async () => table();"
               "await te.embedOnDevice(); const old = te.deviceTable; calls.splice(0);"
               "const r = te.embedOnDevice(), e = te.encodeBatch([[1, 2]]); await r; const t = await e; await te.encodeBatch([[3]]);"
               "const used = calls.filter((c) => c[0] === 'embedRows').map((c) => c[2].buf);"
               "console.log(JSON.stringify([t.length, old.buf.released, used.map((b) => b === te.deviceTable.buf.buf)])); })")
    assert got == [1, 1, [True, True]]
