"""Batches of prompts through the JavaScript host: 4-bit weights, embedding rows and attention behind a shared prefix by
themselves (ops.mjs), and together as the text encoder runs them (qwen3.mjs encodeBatch, pipeline.mjs).

Tolerances of an encoding against 64 bits on the same weights: 1e-5 in the 2-norm in fp32 precision, as the encoder's own
test (two layers are 14 products and two attentions, each off by about 2^-22 of its result), and 1e-2 in bf16, where the
attentions are off by 0.003 to 0.005 and the products of 4-bit weights by 2^-12 of x."""

import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from helpers import PKG_DIR, ROOT, report

JS = os.path.join(PKG_DIR, "js")
NODE = shutil.which("node")
RUN = os.path.join(ROOT, "tests", "js", "run_batch.mjs")

pytestmark = pytest.mark.skipif(NODE is None, reason="node is not installed")


def node(code):
    r = subprocess.run([NODE, "--input-type=module", "-e", code], cwd=JS, capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout)


def run_case(tmp_path, spec):
    path = tmp_path / "case.json"
    path.write_text(json.dumps(spec))
    print(f"[case] js batch {spec['case']}", flush=True)
    r = subprocess.run([NODE, RUN, str(path)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-3000:]
    return json.loads(r.stdout) if r.stdout else None


def write(tmp_path, name, arr):
    p = tmp_path / name
    np.ascontiguousarray(arr).tofile(p)
    return str(p)


def widen(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def values64(q, s, z, N, K, g):
    """The values of a 4-bit weight."""
    q = q.reshape(N, K // 2)
    c = np.stack([q & 15, q >> 4], -1).reshape(N, K // g, g).astype(np.float64) - 8
    w = c * widen(s).reshape(N, -1, 1).astype(np.float64)
    if z is not None:
        w = w + widen(z).reshape(N, -1, 1)
    return w.reshape(N, K)


# ------------------------------------------------------------------ on the CPU


def test_exports():
    ks, names = node("import { native } from './gpu.mjs'; import * as ops from './ops.mjs'; "
                     "console.log(JSON.stringify([Object.keys(native), Object.keys(ops)]))")
    for k in ("weightQuantQ4", "embedRows", "attentionPrefix"):
        assert k in ks, k
    for k in ("quantizeQ4", "embedRows", "attentionPrefix", "attentionPrefixPrepare"):
        assert k in names, k


# the native calls recorded instead of made: [name, arguments], buffers numbered from 1
RECORD = ("import Module from 'module'; const calls = [];"
          "Module._extensions['.node'] = (m) => { m.exports = new Proxy({}, { get: (t, k) => (...a) => { calls.push([k, ...a]); return 64; } }); };"
          "let last = 0; const tensor = (s, d) => ({ buf: ++last, shape: s, dtype: d || 'f32', bytes: 0, released: 0,"
          " get size() { return this.shape.reduce((a, b) => a * b, 1); }, at() { return this.buf; },"
          " view(i, s) { return Object.assign(tensor(s, this.dtype), { buf: this.buf + i / 1e9 }); }, release() { this.released++; } });"
          "const gpu = { ctx: 1, empty: tensor, copy() {}, write() {}, fromArray: (a, s) => Object.assign(tensor(s), { data: Array.from(a),"
          " dtype: a instanceof Int32Array ? 'i32' : 'f32' }) };"
          "const msg = (f) => { try { f(); return ''; } catch (e) { return e.message; } };")


def test_refusals():
    got = node(RECORD + "import('./ops.mjs').then((ops) => {"
               "const q4 = { kind: 'q4', N: 32, K: 128, name: 'w', group: 64 }, f = (s) => tensor(s || [4, 128]);"
               "const table = { kind: 'f32', N: 10, K: 128, buf: 1 };"
               "const at = (o) => ops.attentionPrefix(gpu, Object.assign({ q: f([5, 256]), k: f([5, 128]), v: f([5, 128]), lens: [2, 3],"
               "  H: 2, D: 128, group: 2, ldq: 256, ldk: 128, ldv: 128 }, o));"
               "const prefix = ops.attentionPrefixPrepare(gpu, { k: f([7, 128]), v: f([7, 128]), len: 7, H: 2, D: 128, group: 2, ldk: 128, ldv: 128 });"
               "console.log(JSON.stringify({"
               " group: msg(() => ops.quantizeQ4(gpu, { kind: 'bf16', N: 2, K: 128, name: 'w' }, { group: 48 })),"
               " rows: msg(() => ops.linear(gpu, f(), q4, { xq: { q: tensor([4, 128], 'i8'), s: f([4]) } })),"
               " x: msg(() => ops.linear(gpu, tensor([4, 128], 'bf16'), q4)),"
               " out: msg(() => ops.linear(gpu, f(), q4, { outBf16: true, out: f([4, 32]) })),"
               " precision: msg(() => ops.linear(gpu, f(), q4, { precision: 'fp16' })),"
               " glu: msg(() => ops.linearGlu(gpu, f(), q4, q4, {})),"
               " kind: msg(() => ops.embedRows(gpu, { kind: 'i8', N: 4, K: 128 }, [1])),"
               " weights: msg(() => ops.embedRows(gpu, table, [1, 2], { weights: [1] })),"
               " short: msg(() => ops.embedRows(gpu, table, [1, 2], { out: f([1, 128]) })),"
               " ids: msg(() => ops.embedRows(gpu, table, f([2]))),"
               " q: msg(() => at({ q: f([4, 256]) })), k: msg(() => at({ k: tensor([5, 128], 'bf16') })),"
               " v: msg(() => at({ vOff: 4 })), o: msg(() => at({ out: f([5, 128]) })), obf: msg(() => at({ out: f([5, 256]), oBf16: true })),"
               " other: msg(() => at({ prefix, precision: 'bf16' })), heads: msg(() => at({ prefix, group: 1 })),"
               " fine: [msg(() => at({ prefix })), msg(() => at({})), msg(() => ops.embedRows(gpu, table, [1, -1], { weights: [1, 2], scale: 2 })),"
               "  msg(() => ops.linear(gpu, f(), q4, { precision: 'bf16', outBf16: true }))] })); })")
    assert got.pop("fine") == [""] * 4
    want = {"group": "groups of 48", "rows": "quantized rows for a q4 weight", "x": "a bf16 tensor, expected f32",
            "out": "a f32 tensor, expected bf16", "precision": "unknown precision fp16", "glu": "expected f8", "kind": "a i8 table",
            "weights": "1 weights for 2 rows", "short": "do not fit", "ids": "a f32 tensor, expected i32", "q": "q of 1024 values",
            "k": "a bf16 tensor", "v": "v of 640 values", "o": "out of 640 values", "obf": "a f32 tensor, expected bf16",
            "other": "another precision", "heads": "other heads"}
    for k, w in want.items():
        assert w in got[k], (k, got[k])


def test_arguments():
    """What reaches the library."""
    got = node(RECORD + "import('./ops.mjs').then((ops) => {"
               "const W = ops.quantizeQ4(gpu, { kind: 'bf16', N: 8, K: 256, buf: tensor([8, 256], 'bf16') }, { group: 32, mid: true });"
               "const same = ops.quantizeQ4(gpu, { kind: 'bf16', N: 8, K: 80, buf: 5 });"
               "ops.linear(gpu, tensor([3, 256]), W, { precision: 'bf16' });"
               "const p = ops.attentionPrefixPrepare(gpu, { k: tensor([9, 256]), v: tensor([9, 256]), len: 9, H: 4, D: 128, group: 2, ldk: 256,"
               "  ldv: 256, precision: 'bf16' });"
               "ops.attentionPrefix(gpu, { q: tensor([4, 512]), k: tensor([4, 256]), v: tensor([4, 256]), lens: [1, 0, 3], prefix: p, H: 4, D: 128,"
               "  group: 2, ldq: 512, ldk: 256, ldv: 256, precision: 'bf16', causal: false, oBf16: true });"
               "const last = (n) => calls.filter((c) => c[0] === n).pop();"
               "const lin = last('linear'), at = last('attentionPrefix')[2], prep = calls.filter((c) => c[0] === 'attentionPrefix')[0][2];"
               "console.log(JSON.stringify({ kinds: [W.kind, same.kind], quant: last('weightQuantQ4').slice(3, 7), shapes: [W.buf.shape, W.groupScale.shape],"
               " w: [lin[2].kindId, lin[2].group, lin[2].groupScale > 0, lin[2].groupMid > 0], d: [lin[3].M, lin[3].precision],"
               " kv: last('attentionKvBytes').slice(1), prep: [Array.from(prep.lens), prep.prepareInto > 0, prep.prepareBytes, prep.P],"
               " at: [Array.from(at.lens), at.P, at.causal, at.oBf16, at.precision, at.ldo, at.prefixKv === prep.prepareInto] })); })")
    assert got == {"kinds": ["q4", "bf16"], "quant": [1, 8, 256, 32], "shapes": [[1024], [8, 8]], "w": [6, 32, True, True], "d": [3, 0],
                   "kv": [1, 2, 9, 0], "prep": [[9], True, 64, 0], "at": [[1, 0, 3], 9, 0, 1, 0, 512, True]}


def test_batch_calls():
    """encodeBatch: the rows, lengths and positions of a batch's calls; prompts that are refused; whole-prompt prefixes."""
    got = node(RECORD + "import('./qwen3.mjs').then(async ({ Qwen3 }) => {"
               "const te = new Qwen3(gpu, { hidden: 256, heads: 2, kvHeads: 1, headDim: 128, mlp: 256, theta: 1e6 });"
               "const W = (N, K) => ({ kind: 'bf16', N, K, buf: ++last });"
               "te.layers = [{ qkv: W(512, 256), o: W(256, 256), gate: W(256, 256), up: W(256, 256), down: W(256, 256), ln1: tensor([256]), ln2: tensor([256]),"
               " qn: tensor([128]), kn: tensor([128]) }, { q: W(256, 256), k: W(128, 256), v: W(128, 256), o: W(256, 256), gate: W(256, 256), up: W(256, 256),"
               " down: W(256, 256), ln1: tensor([256]), ln2: tensor([256]), qn: tensor([128]), kn: tensor([128]) }];"
               "te.norm = tensor([256]); te.embedRows = async (ids) => new Float32Array(ids.length * 256);"
               "const trace = () => calls.splice(0).filter((c) => /^attention(Prefix)?$/.test(c[0])).map((c) => [c[0], c[2].Lq || Array.from(c[2].lens),"
               "  c[2].P || 0, c[2].prepareInto ? 1 : 0, c[2].ldq || 0, c[2].sinOff]);"
               "const out = {}, err = async (f) => { try { await f(); return ''; } catch (e) { return e.message; } };"
               "const long = new Array(128).fill(5);"
               "const shapes = (await te.encodeBatch([long.concat([3, 4]), long.concat([7]), long])).map((t) => t.shape); out.shapes = shapes; out.shared = trace();"
               "await te.encodeBatch([[1, 2], [3]]); out.none = trace();"
               "await te.encodeBatch([[1, 2], [1, 2]]); out.few = trace();"
               "await te.encodeBatch([long.concat(long), long.concat(long)]); out.same = trace();"
               "const prefix = await te.keepPrefix([1, 2]); out.keep = trace();"
               "await te.encodeBatch([[1, 2, 3], [1, 2, 4, 5]], { prefix }); out.kept = trace();"
               "await te.encodeBatch([[1, 2]], { prefix }); out.whole = trace();"
               "out.empty = (await te.encodeBatch([])).length; out.e = [await err(() => te.encodeBatch([[1], []])),"
               " await err(() => te.encodeBatch([[1, 3]], { prefix })), await err(() => te.keepPrefix([]))];"
               "te.conversions++; out.e.push(await err(() => te.encodeBatch([[1, 2]], { prefix })));"
               "te.deviceTable = { kind: 'f32', N: 8, K: 256, buf: 1 }; out.e.push(await err(() => te.encodeBatch([[1, 8]])));"
               "console.log(JSON.stringify(out)); })")
    assert got["shapes"] == [[130, 256], [129, 256], [128, 256]] and got["empty"] == 0

    def calls(n, P, lens, cs, keep=False):
        r = []
        for ld in (512, 256):
            if n:
                r.append(["attention", n, 0, 0, ld, cs * 64])
                if lens or keep:
                    r.append(["attentionPrefix", [n], 0, 1, 0, cs * 64])
            if lens:
                r.append(["attentionPrefix", lens, P, 0, ld, cs * 64])
        return r

    assert got["shared"] == calls(128, 128, [2, 1, 0], 130)
    assert got["none"] == calls(0, 0, [2, 1], 2)
    assert got["few"] == calls(0, 0, [2, 2], 2)
    assert got["same"] == calls(256, 256, [], 256)
    assert got["keep"] == calls(2, 2, [], 2, True)
    assert got["kept"] == calls(0, 2, [1, 2], 4)
    assert got["whole"] == []
    for e, w in zip(got["e"], ("prompt 1 has no tokens", "does not begin with opts.prefix", "no tokens", "other weights", "token id 8 outside")):
        assert w in e, got["e"]


def test_table(tmp_path):
    """SafeTensors.table: the values that rows() reads one by one, whatever the file's type; more rows than one piece holds."""
    from test_f8_js import safetensors

    rng = np.random.default_rng(2)
    v = rng.normal(0, 1, (5000, 8)).astype(np.float32)
    v[0] = [0.0, -0.0, np.inf, -np.inf, np.nan, 1e-42, 3e38, -1.5]
    q, sc = rng.integers(-128, 128, (4097, 8)).astype(np.int8), rng.normal(0, 1, 4097).astype(np.float32)
    half = v.astype(np.float16)
    path = safetensors(tmp_path / "t.safetensors", {
        "a.weight": ("BF16", v.shape, bf16(v).tobytes()), "b.weight": ("F32", v.shape, v.tobytes()), "c.weight": ("F16", half.shape, half.tobytes()),
        "d.weight": ("I8", q.shape, q.tobytes()), "d.weight_scale": ("F32", sc.shape, sc.tobytes()), "d.comfy_quant": ("U8", (2,), b"{}")})
    got = node("import { SafeTensors } from './weights.mjs'; import fs from 'fs';"
               "const gpu = { empty: (s, d) => ({ bytes: Buffer.alloc(s[0] * s[1] * (d === 'bf16' ? 2 : 4)), dtype: d, release() {} }),"
               " write(t, a, off) { Buffer.from(a.buffer, a.byteOffset, a.byteLength).copy(t.bytes, off || 0); } };"
               f"const st = SafeTensors.open({json.dumps(path)});"
               "(async () => { const r = {}; for (const n of ['a', 'b', 'c', 'd']) { const t = await st.table(gpu, n + '.weight');"
               f" fs.writeFileSync({json.dumps(str(tmp_path))} + '/' + n, t.buf.bytes); r[n] = [t.kind, t.N, t.K, t.buf.dtype]; }}"
               " console.log(JSON.stringify(r)); })();")
    assert got == {"a": ["bf16", 5000, 8, "bf16"], "b": ["f32", 5000, 8, "f32"], "c": ["f32", 5000, 8, "f32"], "d": ["f32", 4097, 8, "f32"]}
    np.testing.assert_array_equal(np.fromfile(tmp_path / "a", np.uint16).reshape(v.shape), bf16(v))
    np.testing.assert_array_equal(np.fromfile(tmp_path / "b", np.uint32), v.view(np.uint32).reshape(-1))
    np.testing.assert_array_equal(np.fromfile(tmp_path / "c", np.float32).reshape(v.shape), half.astype(np.float32))
    np.testing.assert_array_equal(np.fromfile(tmp_path / "d", np.float32).reshape(q.shape), (q.astype(np.float64) * sc[:, None]).astype(np.float32))


# ------------------------------------------------------------------ on the device


@pytest.mark.gpu
def test_js_ops(tmp_path):
    """The operators one by one, bit for bit where the definition is exact."""
    import test_q4_gpu as ref

    rng = np.random.default_rng(3)
    M, N, K, g = 21, 96, 192, 32
    out = str(tmp_path / "o")
    w, x, r = widen(bf16(rng.normal(0, 0.05, (N, K)))), rng.normal(size=(M, K)).astype(np.float32), rng.normal(size=(M, N)).astype(np.float32)
    A, B = rng.normal(0, 0.1, (8, K)).astype(np.float32), rng.normal(0, 0.1, (N, 8)).astype(np.float32)
    ids, wt = [3, 95, -1, 0, 96], [1.0, 0.5, 2.0, 1.25, 1.0]
    lens, P, H, Hkv = [2, 70, 0, 1], 75, 4, 2
    q, kv = rng.normal(size=(sum(lens), H * 128)).astype(np.float32), rng.normal(size=(P + sum(lens), 2 * Hkv * 128)).astype(np.float32)
    spec = {"case": "ops", "M": M, "N": N, "K": K, "group": g, "ids": ids, "weights": wt, "lens": lens, "P": P, "H": H, "attnGroup": H // Hkv, "out": out}
    for n, a in (("w", bf16(w)), ("x", x), ("r", r), ("A", A), ("B", B), ("q", q), ("kv", kv)):
        spec[n] = write(tmp_path, n, a)
    assert run_case(tmp_path, spec) == {"kind": "bf16"}

    def get(name, dtype=np.float32):
        return np.fromfile(f"{out}.{name}", dtype)

    x64 = x.astype(np.float64)
    for mid in (False, True):
        t = "mid" if mid else "sym"
        c, s, z = ref.quant_ref(w, g, mid)
        np.testing.assert_array_equal(get(f"{t}.q", np.uint8), ref.pack(c).reshape(-1))
        np.testing.assert_array_equal(get(f"{t}.s", np.uint16), s.reshape(-1))
        if mid:
            np.testing.assert_array_equal(widen(get("mid.z", np.uint16)), widen(z).reshape(-1))
        v = values64(ref.pack(c), s, z if mid else None, N, K, g)
        y = x64 @ v.T
        assert report(f"{t} fp32", get(f"{t}.fp32").reshape(M, N), y)[0] <= 1e-6
        assert report(f"{t} bf16", widen(get(f"{t}.bf16", np.uint16)).reshape(M, N), y)[0] <= 2.0 ** -8
        assert report(f"{t} resid", get(f"{t}.resid").reshape(M, N), y + r)[0] <= 1e-6
        assert report(f"{t} lora", get(f"{t}.lora").reshape(M, N), y + 0.5 * (x64 @ A.T.astype(np.float64)) @ B.T)[0] <= 1e-5
        rows = get(f"{t}.rows").reshape(len(ids), K)
        for i, (d, f) in enumerate(zip(ids, wt)):
            want = (2 * f * v[d]) if 0 <= d < N else np.zeros(K)
            # (a value with a middle is rounded once, and its weighted form once)
            assert np.all(np.abs(rows[i] - want) <= 2.0 ** -23 * np.abs(want)), (t, d)
    k, v = kv[:, : Hkv * 128].reshape(-1, Hkv, 128), kv[:, Hkv * 128:].reshape(-1, Hkv, 128)
    from oracle import qwen3_ref as qr
    cos, sin = qr.rope_table(P + max(lens), 128, 1e6)
    want, at = [], 0
    for n in lens:
        pos = np.arange(P, P + n)
        kk = np.concatenate([k[:P], k[P + at: P + at + n]]).astype(np.float64)
        vv = np.concatenate([v[:P], v[P + at: P + at + n]]).astype(np.float64)
        qq = np.zeros((P + n, H, 128))
        qq[P:] = qr.rope(q[at: at + n].reshape(n, H, 128).astype(np.float64), cos[pos], sin[pos])
        kk = qr.rope(kk, cos[: P + n], sin[: P + n])
        want.append(qr.causal_gqa(qq, kk, vv, H // Hkv)[P:].reshape(n, H * 128))
        at += n
    want = np.concatenate(want)
    assert report("attention fp32", get("attn.fp32").reshape(want.shape), want)[0] <= 1e-5
    assert report("attention bf16", get("attn.bf16").reshape(want.shape), want)[0] <= 1e-2


@pytest.mark.gpu
@pytest.mark.parametrize("q4", [None, {"group": 64}, {"group": 32, "mid": True}], ids=["bf16", "q4", "q4mid"])
def test_js_encode_batch(tmp_path, q4):
    """The operators together: a two-layer encoder's batches against 64 bits on the same weights, each prompt by itself,
    with and without a kept prefix.  Rows from the device's table are those of the host's, bit for bit; a kept prefix
    of another state is refused."""
    from oracle import qwen3_ref

    V, L = 97, 2
    rng = np.random.default_rng(11)
    head = [int(v) for v in rng.integers(0, V - 1, size=90)]
    prompts = [head + [int(v) for v in rng.integers(0, V - 1, size=n)] for n in (9, 0, 130, 1)]
    out = str(tmp_path / "e")
    log = run_case(tmp_path, {"case": "encode", "layers": L, "vocab": V, "prompts": prompts, "keep": 66, "q4": q4, "out": out})
    assert log["device"] == 0 and log["converted"] == (10 if q4 else 0) and log.get("again", 0) == 0
    for p in ("fp32", "bf16"):
        assert "another precision" in log[p + ".precision"] and "does not begin" in log[p + ".other"]
        assert "other LoRAs" in log[p + ".lora"] and "released" in log[p + ".released"]
    assert "token id 97 outside" in log["outside"]

    def get(name, dtype=np.float32):
        return np.fromfile(f"{out}.{name}", dtype)

    D, H, KH, Dh, g = 1024, 16, 8, 128, (q4 or {}).get("group")

    def weight(n, N, K, plain):
        if q4 is None:
            return plain(n).astype(np.float64).reshape(N, K)
        return values64(get(f"w.{n}", np.uint8), get(f"w.{n}.s", np.uint16), get(f"w.{n}.z", np.uint16) if q4.get("mid") else None, N, K, g)

    W = {"norm": get("w.norm").astype(np.float64), "embed": weight("embed", V, D, lambda n: get(f"w.{n}"))}
    for i in range(L):
        for n in ("ln1", "ln2", "qn", "kn"):
            W[f"{i}.{n}"] = get(f"w.{i}.{n}").astype(np.float64)
        F = get(f"w.{i}.gate", np.uint8).size // (D * 2) if q4 is None else get(f"w.{i}.gate", np.uint8).size * 2 // D
        for n, N, K in (("qkv", (H + 2 * KH) * Dh, D), ("o", D, H * Dh), ("gate", F, D), ("up", F, D), ("down", D, F)):
            W[f"{i}.{n}"] = weight(f"{i}.{n}", N, K, lambda n: widen(get(f"w.{n}", np.uint16)))
        W[f"{i}.q"], W[f"{i}.k"], W[f"{i}.v"] = np.split(W[f"{i}.qkv"], [H * Dh, (H + KH) * Dh])
    want = [qwen3_ref.encode(W, p, L) for p in prompts]
    only = want[0][:66]
    for prec, bar in (("fp32", 1e-5), ("bf16", 1e-2)):
        sets = {"batch": want, "one": want[:1], "kept": want, "kept2": want[::-1], "only": [only]}
        for name, refs in sets.items():
            for i, r in enumerate(refs):
                got = get(f"{prec}.{name}.{i}").reshape(r.shape)
                assert report(f"{prec} {name} {i}", got, r)[0] <= bar
        # the rows of the prefix are computed once
        first = get(f"{prec}.batch.0").reshape(-1, D)[:90]
        for i in range(1, 4):
            assert np.array_equal(first, get(f"{prec}.batch.{i}").reshape(-1, D)[:90])


@pytest.mark.gpu
def test_js_adapter_weights(tmp_path):
    """Prompt weights of up to 24 bits on the device, others on the host: one rounding of each product in both, zeros behind."""
    rng = np.random.default_rng(13)
    n, out = 19, str(tmp_path / "a")
    ids = [int(v) for v in rng.integers(0, 64, size=n)]
    w = {"none": None, "short": [float(np.float32(v)) for v in rng.uniform(0.5, 1.5, size=n)], "long": [float(v) for v in rng.uniform(0.5, 1.5, size=n)]}
    run_case(tmp_path, {"case": "adapter", "Ls": 23, "ids": ids, "weights": w, "out": out,
                        "hidden": write(tmp_path, "h", rng.normal(size=(23, 1024)).astype(np.float32))})
    got = {k: np.fromfile(f"{out}.{k}", np.float32).reshape(512, 1024) for k in w}
    assert all(not g[n:].any() for g in got.values()) and np.abs(got["none"][:n]).min(1).all()
    for k in ("short", "long"):
        np.testing.assert_array_equal(got[k][:n], (got["none"][:n].astype(np.float64) * np.array(w[k])[:, None]).astype(np.float32))


@pytest.mark.gpu
def test_js_pipeline(tmp_path):
    """A prompt that is cached is not encoded again, the same prompt twice is encoded once, and others leave the cache."""
    rng = np.random.default_rng(17)

    def prompt(key, ids):
        return {"key": key, "qwenIds": ids, "t5Ids": [int(v) for v in rng.integers(0, 64, size=7)], "t5Weights": None}

    prompts = [prompt("a", [1, 2, 3, 4, 5]), prompt("b", [1, 2, 3, 9]), prompt("c", [7])]
    got = run_case(tmp_path, {"case": "pipeline", "prompts": prompts})
    assert got["n"] == 3 and got["hit"] and got["again"] == [1, 0, 1] and got["cached"] == 2 and got["none"] == 0 and got["left"] == 0
    assert got["stats"]["encodeMisses"] == 3 and got["stats"]["encodeHits"] == 4
