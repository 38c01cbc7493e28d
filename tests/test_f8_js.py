"""The e4m3 operators through the JavaScript host (ops.mjs, weights.mjs, qwen3.mjs, dit.mjs).

Encodings and velocities are compared with others whose e4m3 rows come from slightly different values.  A relative
difference d moves a value across a rounding boundary with probability d / step and then changes it by step, between
2^-4 and 2^-3 of itself: a row tensor then differs by up to sqrt(2^-3 d) in the 2-norm, and this is the d of the
next one.  From an fp32 rounding, d = 1e-6, that is 3.5e-4, then 6.6e-3, then 2.9e-2: after a few products the two
have roundings as independent as any two (no bar proportional to 1e-6 holds; 7.4e-3 was seen after eight).  Each of
k row tensors then differs by sqrt(2) times a rounding, at most 2^-4 of a value and uniform in that range:
ROUNDING sqrt(2 k) in all, which is the bar.  The encoder's wiring is also pinned bit for bit, by the same ops
called one by one on fp32 rows (which the operators quantize to the same bytes).
"""

import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import oracle as orc
from helpers import PKG_DIR, ROOT, report

JS = os.path.join(PKG_DIR, "js")
NODE = shutil.which("node")
RUN_F8 = os.path.join(ROOT, "tests", "js", "run_f8.mjs")

pytestmark = pytest.mark.skipif(NODE is None, reason="node is not installed")


ROUNDING = 2.0 ** -4 / 3 ** 0.5


def node(code):
    r = subprocess.run([NODE, "--input-type=module", "-e", code], cwd=JS, capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    return json.loads(r.stdout)


def run_case(tmp_path, spec):
    path = tmp_path / "case.json"
    path.write_text(json.dumps(spec))
    print(f"[case] js f8 {spec['case']}", flush=True)
    r = subprocess.run([NODE, RUN_F8, str(path)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-3000:]
    return r.stdout


def write(tmp_path, name, arr):
    p = tmp_path / name
    np.ascontiguousarray(arr).tofile(p)
    return str(p)


def safetensors(path, tensors):
    """{name: (dtype, shape, bytes)} as a safetensors file."""
    header, off = {}, 0
    for n, (dt, shape, b) in tensors.items():
        header[n] = {"dtype": dt, "shape": list(shape), "data_offsets": [off, off + len(b)]}
        off += len(b)
    h = json.dumps(header).encode()
    with open(path, "wb") as f:
        f.write(len(h).to_bytes(8, "little") + h + b"".join(b for _, _, b in tensors.values()))
    return str(path)


# ------------------------------------------------------------------ on the CPU


def test_exports():
    ks, names = node("import { native } from './gpu.mjs'; import * as ops from './ops.mjs'; "
                     "console.log(JSON.stringify([Object.keys(native), Object.keys(ops)]))")
    for k in ("quantRowsF8", "weightQuantF8", "linearGlu", "residualNorm"):
        assert k in ks, k
    for k in ("quantRowsF8", "quantizeF8", "linearGlu", "residualNorm"):
        assert k in names, k


# a GPU object without a device: what is refused before any native call
FAKE = ("const gpu = { ctx: null, empty: (s, d) => ({ buf: 0, shape: s, dtype: d || 'f32', size: s.reduce((a, b) => a * b, 1), "
        "release() {} }), upload: (a) => ({ buf: 0, data: Array.from(a), release() {} }), copy() {} };"
        "const msg = (f) => { try { f(); return ''; } catch (e) { return e.message; } };")
MSG = "const msg = (f) => { try { f(); return ''; } catch (e) { return e.message; } };"


def test_refusals():
    got = node("import * as ops from './ops.mjs';" + FAKE +
               "const f8 = { kind: 'f8', N: 32, K: 128, buf: 0, scale: 0, name: 'w' }, i8 = Object.assign({}, f8, { kind: 'i8' });"
               "const rows = (d) => ({ q: gpu.empty([4, 128], d), s: gpu.empty([4]) });"
               "const lora = Object.assign({}, f8, { lora: [{}] });"
               "console.log(JSON.stringify({"
               "int8_rows: msg(() => ops.linear(gpu, null, f8, { xq: rows('i8') })),"
               "e4m3_rows: msg(() => ops.linear(gpu, null, i8, { xq: rows('u8') })),"
               "width: msg(() => ops.linear(gpu, null, f8, { xq: { q: gpu.empty([4, 256], 'u8'), s: gpu.empty([2, 4]) } })),"
               "scales: msg(() => ops.linearGlu(gpu, null, f8, f8, { xq: { q: gpu.empty([4, 128], 'u8'), s: gpu.empty([1, 3]) } })),"
               "bf16_out: msg(() => ops.linear(gpu, gpu.empty([4, 128]), i8, { outBf16: true })),"
               "lora_rows: msg(() => ops.linear(gpu, null, lora, { xq: rows('u8') })),"
               "lora_bf16: msg(() => ops.linear(gpu, gpu.empty([4, 128]), lora, { outBf16: true })),"
               "precision: msg(() => ops.linear(gpu, gpu.empty([4, 128]), f8, { precision: 'fp16' })),"
               "glu_kind: msg(() => ops.linearGlu(gpu, null, f8, i8, { xq: rows('u8') })),"
               "glu_rows: msg(() => ops.linearGlu(gpu, null, f8, f8, { xq: rows('i8') })),"
               "glu_lora: msg(() => ops.linearGlu(gpu, null, f8, lora, { xq: rows('u8') })),"
               "norm: msg(() => ops.residualNorm(gpu, gpu.empty([4, 128]), 128, { norm: 'batch' })),"
               "y: msg(() => ops.residualNorm(gpu, gpu.empty([4, 128]), 128, { y: gpu.empty([3, 128]) })),"
               "}))")
    assert "int8 rows for a f8 weight" in got["int8_rows"]
    assert "e4m3 rows for a i8 weight" in got["e4m3_rows"]
    assert "rows [4,256] with 8 scales for K = 128" in got["width"] and "rows [4,128] with 3 scales" in got["scales"]
    assert "bf16 results are for f8" in got["bf16_out"]
    assert "needs its input" in got["lora_rows"]
    assert "no bf16 result with a LoRA" in got["lora_bf16"]
    assert "unknown precision fp16" in got["precision"]
    assert "expected f8" in got["glu_kind"] and "int8 rows" in got["glu_rows"] and "has a LoRA" in got["glu_lora"]
    assert "unknown norm batch" in got["norm"] and "y of 384" in got["y"]


def test_m_of_e4m3_rows():
    """opts.M beside e4m3 rows: their scales lie [blocks][rows], so a prefix or more rows than there are is refused
    (the kernels take M as the scales' stride); int8 rows, with one scale each, can be cut."""
    got = node("import * as ops from './ops.mjs';" + FAKE +
               "const f8 = { kind: 'f8', N: 32, K: 384, buf: 0, scale: 0, name: 'w' };"
               "const f8rows = () => ({ q: gpu.empty([8, 384], 'u8'), s: gpu.empty([3, 8]) });"
               "const i8rows = () => ({ q: gpu.empty([8, 384], 'i8'), s: gpu.empty([8]) });"
               "const tries = {};"
               "for (const M of [4, 7, 8, 9, 16, undefined]) {"
               "  tries['linear ' + M] = msg(() => ops.linear(gpu, null, f8, { M, xq: f8rows() }));"
               "  tries['glu ' + M] = msg(() => ops.linearGlu(gpu, null, f8, f8, { M, xq: f8rows() }));"
               "}"
               "tries.int8 = msg(() => ops.linear(gpu, null, Object.assign({}, f8, { kind: 'i8' }), { M: 4, xq: i8rows() }));"
               "console.log(JSON.stringify(tries))")
    for op in ("linear", "glu"):
        for M in (4, 7, 9, 16):
            assert f"M = {M} for 8 e4m3 rows" in got[f"{op} {M}"], (op, M)
        # what passes reaches the library, which has no context here
        assert got[f"{op} 8"] == got[f"{op} undefined"] == got["int8"]
    assert "rows" not in got["int8"]


# the native calls recorded instead of made: [name, arguments], buffers numbered from 1
RECORD = ("import Module from 'module'; const calls = [];"
          "Module._extensions['.node'] = (m) => { m.exports = new Proxy({}, { get: (t, k) => (...a) => { calls.push([k, ...a]); return 64; } }); };"
          "let last = 0; const tensor = (s, d) => ({ buf: ++last, shape: s, dtype: d || 'f32', bytes: 0,"
          " get size() { return this.shape.reduce((a, b) => a * b, 1); }, at() { return this.buf; }, release() {} });"
          "const gpu = { ctx: 1, empty: tensor, copy() {} };")


def test_residual_norm_groups():
    """groupRows, gateLd and modLd reach the library; vectors too short for the groups, and a result without e4m3 rows
    in a linear's place, are refused."""
    got = node(RECORD + MSG + "import('./ops.mjs').then((ops) => {"
               "const x = tensor([6, 128]), norm = (o) => ops.residualNorm(gpu, x, 128, o);"
               "norm({ gate: tensor([3, 128]), gOff: 0, mod: tensor([3, 256]), scaleOff: 128, groupRows: 2, modLd: 256 });"
               "norm({ gate: tensor([1152]), gOff: 512, gateLd: 256, groupRows: 2 });"
               "norm({ gate: tensor([128]) });"
               "const none = norm({});"
               "const d = calls.filter((c) => c[0] === 'residualNorm').map((c) => [c[2].groupRows, c[2].gateLd, c[2].modLd]);"
               "console.log(JSON.stringify({ d,"
               " gate: msg(() => norm({ gate: tensor([2, 128]), groupRows: 2 })),"
               " off: msg(() => norm({ gate: tensor([3, 128]), gOff: 4, groupRows: 2 })),"
               " mod: msg(() => norm({ mod: tensor([3, 256]), scaleOff: 128, groupRows: 2, modLd: 260 })),"
               " one: msg(() => norm({ gate: tensor([100]) })),"
               " rows: msg(() => ops.linear(gpu, null, { kind: 'f8', N: 32, K: 128, name: 'w' }, { xq: none })),"
               " glu: msg(() => ops.linearGlu(gpu, null, { kind: 'f8', N: 32, K: 128 }, { kind: 'f8', N: 32, K: 128 }, { xq: none })) })); })")
    assert got["d"] == [[2, 0, 256], [2, 256, 0], [0, 0, 0], [0, 0, 0]]
    assert "gate of 256 values, 384 for 3 groups" in got["gate"] and "gate of 384 values, 388" in got["off"]
    assert "mod of 768 values, 776" in got["mod"] and "gate of 100 values, 128" in got["one"]
    assert "without rows q and scales s" in got["rows"] and "without rows q and scales s" in got["glu"]


def test_types_of_tensors():
    """bf16 tensors where the kernels read or write fp32 rows, twice the bytes, and the other way round."""
    got = node(RECORD + MSG + "import('./ops.mjs').then((ops) => {"
               "const W = { kind: 'f8', N: 32, K: 128, name: 'w' }, f = () => tensor([4, 128]), b = () => tensor([4, 128], 'bf16');"
               "console.log(JSON.stringify({"
               " x: msg(() => ops.linear(gpu, b(), W, {})), glu: msg(() => ops.linearGlu(gpu, b(), W, W, {})),"
               " norm: msg(() => ops.residualNorm(gpu, b(), 128, {})),"
               " out: msg(() => ops.linear(gpu, f(), W, { out: tensor([4, 32], 'bf16') })),"
               " bf16_out: msg(() => ops.linear(gpu, f(), W, { out: tensor([4, 32]), outBf16: true })),"
               " glu_out: msg(() => ops.linearGlu(gpu, f(), W, W, { out: tensor([4, 32], 'bf16') })),"
               " fine: [msg(() => ops.linear(gpu, f(), W, { out: tensor([4, 32]) })),"
               "  msg(() => ops.linear(gpu, f(), W, { out: tensor([4, 32], 'bf16'), outBf16: true })),"
               "  msg(() => ops.linearGlu(gpu, f(), W, W, { out: tensor([4, 32]) })),"
               "  msg(() => ops.residualNorm(gpu, f(), 128, { y: b() }))] })); })")
    assert got.pop("fine") == [""] * 4
    for name, m in got.items():
        assert "a bf16 tensor, expected f32" in m if name != "bf16_out" else "a f32 tensor, expected bf16" in m, (name, m)


def test_context_of_mixed_kinds():
    """Cross-attention k / v of several kinds in one model: each linear gets the rows that its weight reads."""
    kinds = [("i8", "i8"), ("f8", "f8"), ("bf16", "bf16"), ("w4", "f8"), ("f8", "i8")]
    got = node(RECORD + "import('./dit.mjs').then(({ AnimaDiT }) => {"
               "const W = (kind) => ({ kind, N: 2048, K: 1024, buf: ++last, scale: ++last, name: kind });"
               f"const m = new AnimaDiT(gpu); m.blocks = {json.dumps(kinds)}.map(([k, v]) => ({{ cross: {{ k: W(k), v: W(v), kn: tensor([128]) }} }}));"
               "m.prepareContext([tensor([40, 1024]), tensor([40, 1024])]);"
               "console.log(JSON.stringify(calls.filter((c) => c[0] === 'linear').map((c) => [c[2].kindId, !!c[3].xq, !!c[3].x, c[3].M])));"
               "})")
    ids = {"bf16": 0, "i8": 1, "w4": 2, "f8": 5}
    assert got == [[ids[k], k in ("i8", "w4"), k not in ("i8", "w4"), 80] for pair in kinds for k in pair]


def test_checkpoint_and_stacking(tmp_path):
    """SafeTensors.linear on block-scaled e4m3, and concatLinears of whole blocks only."""
    rng = np.random.default_rng(3)

    def tensors(name, n, k, nb, kb):
        return {f"{name}.weight": ("F8_E4M3", (n, k), rng.integers(0, 120, n * k, dtype=np.uint8).tobytes()),
                f"{name}.weight_scale_inv": ("F32", (nb, kb), np.arange(nb * kb, dtype=np.float32).tobytes())}

    t = {**tensors("a", 200, 144, 2, 2), **tensors("bad", 200, 144, 2, 1), **tensors("c", 128, 144, 1, 2),
         "plain.weight": ("F8_E4M3", (16, 16), bytes(256))}
    path = safetensors(tmp_path / "w.safetensors", t)
    got = node("import { SafeTensors, concatLinears } from './weights.mjs';" + FAKE +
               f"const st = SafeTensors.open({json.dumps(path)});"
               "const a = st.linear(gpu, 'a.'), c = st.linear(gpu, 'c.');"
               "const stack = (ws) => { const w = concatLinears(gpu, ws.map((v) => Object.assign({}, v)));"
               "  return w && [w.kind, w.N, w.K, w.buf.size, w.buf.dtype, w.scale.size]; };"
               "console.log(JSON.stringify({ a: [a.kind, a.N, a.K, a.buf.data, a.scale.data, a.name],"
               " bad: msg(() => st.linear(gpu, 'bad.')), plain: msg(() => st.linear(gpu, 'plain.')),"
               " ca: stack([c, a]), ac: stack([a, c]) }))")
    assert got["a"][:3] == ["f8", 200, 144] and got["a"][5] == "a"
    assert bytes(got["a"][3]) == t["a.weight"][2] and got["a"][4] == [0, 1, 2, 3]
    assert "expected [2, 2]" in got["bad"] and "F8_E4M3" in got["plain"]
    assert got["ca"] == ["f8", 328, 144, 328 * 144, "u8", 6]
    assert got["ac"] is None


# ------------------------------------------------------------------ on the GPU


@pytest.mark.gpu
@pytest.mark.parametrize("file", [False, True])
def test_js_block(tmp_path, file):
    import test_f8_gpu as ref

    M, C, F = 37, 208, 384
    rng = np.random.default_rng(8)
    shapes = {"a": (C, C), "b": (C, C), "gate": (F, C), "up": (F, C), "down": (C, F)}
    out = str(tmp_path / "o")
    spec = {"case": "block", "M": M, "C": C, "F": F, "out": out}
    x = rng.normal(size=(M, C)).astype(np.float32)
    mod = (0.3 * rng.normal(size=3 * C)).astype(np.float32)
    norm = rng.uniform(0.5, 1.5, C).astype(np.float32)
    spec.update(x=write(tmp_path, "x", x), mod=write(tmp_path, "mod", mod), norm=write(tmp_path, "norm", norm))
    W, blob = {}, {}
    for i, (n, (N, K)) in enumerate(shapes.items()):
        if file:
            W[n] = ref.f8_weight(40 + i, N, K)
            blob[f"{n}.weight"] = ("F8_E4M3", (N, K), W[n][0].tobytes())
            blob[f"{n}.weight_scale_inv"] = ("F32", W[n][1].shape, W[n][1].tobytes())
        else:
            bits, val = ref.bf16((rng.normal(size=(N, K)) / np.sqrt(K)).astype(np.float32))
            spec.setdefault("w", {})[n] = write(tmp_path, "w" + n, bits)
            W[n] = val
    if file:
        spec["file"] = safetensors(tmp_path / "w.safetensors", blob)
    run_case(tmp_path, spec)

    def get(name, dtype=np.float32):
        return np.fromfile(f"{out}.{name}", dtype)

    for n, (N, K) in shapes.items():
        q, s = get(f"w.{n}.q", np.uint8).reshape(N, K), get(f"w.{n}.s").reshape(-(-N // 128), -(-K // 128))
        if file:
            assert np.array_equal(q, W[n][0]) and np.array_equal(s, W[n][1])
        else:  # (the conversion itself is pinned with the C entry point)
            assert np.abs(ref.weight64(q, s) - W[n]).max() <= 2.0 ** -4 * np.abs(W[n]).max()
        W[n] = ref.weight64(q, s)

    def rows(n, K):
        return ref.rows64(get(n + ".q", np.uint8).reshape(M, K), get(n + ".s").reshape(-(-K // 128), M))

    def check(name, got, want, bound, steps=2):
        d = np.abs(got - want)
        assert (d <= bound + steps * ref.U * np.abs(want) + 1e-30).all(), f"{name}: {(d / (bound + 1e-30)).max()}"

    h = rows("h", C)
    x64 = x.astype(np.float64)
    n64 = (x64 - x64.mean(1, keepdims=True)) / np.sqrt(x64.var(1, keepdims=True) + 1e-6) * (1 + mod[C:2 * C].astype(np.float64)) + mod[:C]
    # an e4m3 value is off by 2^-4 of itself, 2^-10 scale at the least
    assert (np.abs(h - n64) <= 2.0 ** -4 * np.abs(n64) * 1.001 + 2.0 ** -9 * np.abs(n64).max(1, keepdims=True) / 448 + 1e-5).all()
    y, dy = ref.product64(h, W["a"], False)
    check("y", get("y").reshape(M, C), ref.act64(y, "gelu"), ref.act_error(y, "gelu", dy))
    q, s = ref.quant_ref(get("y").reshape(M, C))
    assert np.array_equal(get("yq.q", np.uint8).reshape(M, C), q) and np.array_equal(get("yq.s").reshape(-1, M), s)
    z, dz = ref.product64(rows("yq", C), W["b"], True)
    zg = (get("z", np.uint16).astype(np.uint32) << 16).view(np.float32).reshape(M, C).astype(np.float64)
    check("z", zg, z, dz + 2.0 ** -8 * (np.abs(z) + dz))
    x1 = x + mod[2 * C:].astype(np.float64) * zg
    check("x1", get("x1").reshape(M, C), x1, 3 * ref.U * (np.abs(x) + np.abs(x1 - x)))
    g1 = get("x1").reshape(M, C).astype(np.float64)
    h2 = g1 / np.sqrt((g1 * g1).mean(1, keepdims=True) + 1e-6) * norm
    check("h2", get("h2").reshape(M, C), h2, 40 * ref.U * np.abs(h2))
    q, s = ref.quant_ref(get("h2").reshape(M, C))
    assert np.array_equal(get("h2.q", np.uint8).reshape(M, C), q) and np.array_equal(get("h2.s").reshape(-1, M), s)
    gt, dg = ref.product64(rows("h2", C), W["gate"], False)
    up, du = ref.product64(rows("h2", C), W["up"], False)
    a, da = ref.act64(gt, "silu"), ref.act_error(gt, "silu", dg)
    f, df = a * up, da * (np.abs(up) + du) + np.abs(a) * du
    check("glu", get("gf").reshape(M, F), f, df)
    if os.path.exists(out + ".both"):
        both = get("both").reshape(M, 2 * F)
        check("gate | up", both, np.concatenate([gt, up], 1), np.concatenate([dg, du], 1))
    assert os.path.exists(out + ".both")
    d, dd = ref.product64(rows("g", F), W["down"], False)
    gate = mod[2 * C:].astype(np.float64)
    check("x", get("x").reshape(M, C), g1 + gate * d, np.abs(gate) * dd + 3 * ref.U * (np.abs(g1) + np.abs(gate * d)))


@pytest.mark.gpu
@pytest.mark.parametrize("M,per", [(20, 10), (21, 8)])
def test_js_groups(tmp_path, M, per):
    """Rows in groups (the last one short) with gates and modulations of their own: the same bits as each group alone."""
    C, ld, out = 272, 288, str(tmp_path / "g")
    rng = np.random.default_rng(M)
    n = -(-M // per)
    spec = {"case": "groups", "M": M, "C": C, "per": per, "ld": ld, "out": out}
    for k, size in (("x", M * C), ("y", M * C), ("gate", n * ld), ("mod", 2 * n * ld)):
        spec[k] = write(tmp_path, k, rng.normal(size=size).astype(np.float32))
    run_case(tmp_path, spec)

    def get(tag, name, dtype=np.float32):
        return np.fromfile(f"{out}.{tag}.{name}", dtype)

    for name, dtype, rows in (("x", np.float32, True), ("h", np.float32, True), ("q", np.uint8, True), ("s", np.float32, False)):
        whole = get("all", name, dtype)
        parts = [get(g, name, dtype).reshape(min(per, M - g * per), C) if rows else
                 get(g, name, dtype).reshape(-1, min(per, M - g * per)) for g in range(n)]
        assert np.array_equal(whole.reshape(M, C) if rows else whole.reshape(-1, M), np.concatenate(parts, 0 if rows else 1)), name


def encode_ref(W, ids, layers):
    """The encoder in 64 bits with the e4m3 rows that every product reads (qwen3.mjs layersF8)."""
    import test_f8_gpu as ref
    from oracle import qwen3_ref as r

    def rows(x):
        return ref.rows64(*ref.quant_ref(x))

    D, H, KH, Dh = r.CFG["hidden"], r.CFG["heads"], r.CFG["kv_heads"], r.CFG["head_dim"]
    L = len(ids)
    x = W["embed"][np.asarray(ids)]
    cos, sin = r.rope_table(L, Dh, r.CFG["theta"])
    for i in range(layers):
        def g(n):
            return W[f"{i}.{n}"]

        qkv = rows(r.rmsnorm(x, g("ln1"))) @ g("qkv").T
        q, k, v = (t.reshape(L, -1, Dh) for t in np.split(qkv, [H * Dh, (H + KH) * Dh], 1))
        q, k = r.rope(r.rmsnorm(q, g("qn")), cos, sin), r.rope(r.rmsnorm(k, g("kn")), cos, sin)
        a = r.causal_gqa(q, k, v, H // KH).reshape(L, H * Dh)
        x = x + rows(a) @ g("o").T
        h = rows(r.rmsnorm(x, g("ln2")))
        gt, up = h @ g("gate").T, h @ g("up").T
        x = x + rows(gt / (1.0 + np.exp(-gt)) * up) @ g("down").T
    return r.rmsnorm(x, W["norm"])


@pytest.mark.gpu
def test_js_qwen3_f8(tmp_path):
    """A 2-layer encoder on e4m3 weights (8 row tensors) against 64 bits with the same roundings to e4m3; the fp32
    encoding bit for bit against the ops one by one; recorded, replayed and eager encodings equal; and the path
    of a LoRA (of zeros) on one linear, which quantizes fp32 inputs inside every call."""
    import test_f8_gpu as ref

    out = str(tmp_path / "te")
    ids = [int(v) for v in np.random.default_rng(5).integers(0, 97, size=37)]
    log = run_case(tmp_path, {"case": "qwen3", "layers": 2, "vocab": 97, "ids": ids, "out": out})
    assert json.loads(log.splitlines()[0]) == {"converted": 10, "again": 0}

    def get(name, dtype=np.float32):
        return np.fromfile(f"{out}.{name}", dtype)

    D = 1024
    W = {"norm": get("w.norm").astype(np.float64), "embed": get("w.embed").reshape(97, D).astype(np.float64)}
    for i in range(2):
        for n in ("ln1", "ln2", "qn", "kn"):
            W[f"{i}.{n}"] = get(f"w.{i}.{n}").astype(np.float64)
        for n, K in (("qkv", D), ("o", 2048), ("gate", D), ("up", D), ("down", None)):
            q = get(f"w.{i}.{n}", np.uint8)
            q = q.reshape(-1, K) if K else q.reshape(D, -1)
            W[f"{i}.{n}"] = ref.weight64(q, get(f"w.{i}.{n}.s").reshape(-1, -(-q.shape[1] // 128)))
    want = encode_ref(W, ids, 2)
    bar = ROUNDING * 16 ** 0.5
    assert np.array_equal(get("fp32"), get("steps"))
    for prec in ("fp32", "bf16"):
        got = get(prec)
        assert np.isfinite(got).all()
        assert report(f"qwen3 f8 {prec} vs 64 bits", got.reshape(-1, D), want)[0] <= bar
        for tag in (".replay", ".replay2", ".eager"):
            assert np.array_equal(got, get(prec + tag)), prec + tag
    assert report("qwen3 f8 with a LoRA of zeros", get("lora"), get("fp32"))[0] <= bar


@pytest.mark.gpu
def test_js_dit_f8(tmp_path):
    """A 2-block DiT (12 row tensors): on e4m3 weights, its norms writing e4m3 rows, against the same weights
    reading fp32 rows (LoRAs of zeros); with bf16 attention and products; and against the bf16 weights, where the
    12 products' weights are off as well."""
    out = str(tmp_path / "v")
    h, w, Lk = 16, 24, 40
    lat = [orc.randn(60 + b, 16 * h * w) for b in range(2)]
    ctx = [orc.randn(70 + b, Lk * 1024) for b in range(2)]
    spec = {"case": "dit", "seed": 9, "blocks": 2, "sigma": 0.7, "h": h, "w": w, "Lk": Lk, "out": out,
            "latents": [write(tmp_path, f"l{b}", v) for b, v in enumerate(lat)],
            "ctx": [write(tmp_path, f"c{b}", v) for b, v in enumerate(ctx)]}
    log = run_case(tmp_path, spec)
    # qkv (stacked), o, cross q / k / v / o, the two of the feed-forward
    assert json.loads(log.splitlines()[0]) == {"converted": 16}
    assert json.loads(log.splitlines()[1])["differ"] == [0, 0, 0]  # replays against eager forwards
    bar = ROUNDING * 24 ** 0.5
    for b in range(2):
        v = {t: np.fromfile(f"{out}.{t}.{b}", np.float32) for t in ("bf16w", "f8", "f8bf16", "f8lora")}
        assert all(np.isfinite(t).all() for t in v.values())
        assert report("dit f8 rows from norms vs from fp32 rows", v["f8"], v["f8lora"])[0] <= bar
        assert report("dit f8 bf16 vs fp32", v["f8bf16"], v["f8"])[0] <= bar
        assert 1e-3 < report("dit f8 vs bf16 weights", v["f8"], v["bf16w"])[0] <= bar


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", [["bf16", "bf16", "bf16"], ["i8", "bf16"], ["w4", "bf16", "i8", "bf16"]])
def test_js_dit_f8_steps(tmp_path, kinds):
    """The DiT's e4m3 blocks (of bf16 ones converted) between others, in both precisions: the residual stream bit for bit
    as the block's ops one by one give it, on fp32 rows that every product quantizes itself."""
    out = str(tmp_path / "s")
    h, w, Lk = 16, 24, 40
    spec = {"case": "ditsteps", "seed": 11, "kinds": kinds, "sigma": 0.6, "h": h, "w": w, "Lk": Lk, "out": out,
            "latents": [write(tmp_path, f"l{b}", orc.randn(80 + b, 16 * h * w)) for b in range(2)],
            "ctx": [write(tmp_path, f"c{b}", orc.randn(90 + b, Lk * 1024)) for b in range(2)]}
    log = run_case(tmp_path, spec)
    assert json.loads(log.splitlines()[0]) == {"converted": 8 * kinds.count("bf16")}
    n = 0
    for prec in ("fp32", "bf16"):
        for i in range(1, len(kinds)):
            if kinds[i] == "bf16":
                got, want = (np.fromfile(f"{out}.{prec}.{i}{t}", np.float32) for t in ("", ".steps"))
                assert np.isfinite(got).all() and np.array_equal(got, want), (prec, i, np.abs(got - want).max())
                n += 1
    assert n == 2 * kinds[1:].count("bf16")
