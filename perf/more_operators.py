"""Cases of the text encoder's operators for a batch of prompts: rows of an embedding table, products with 4-bit weights,
and attention of many sequences behind one shared prefix.

A case is a plain dict; `op` names the operator:

  embed      `t` rows of a table of `n` rows, `k` wide ("f32", "bf16" or "q4" values), each times its prompt weight
             (`weights`) and a common `scale`; indexes outside the table (padding) give rows of zeros
  linear     a product with a 4-bit weight of groups of `g` along k, with (`mid`) or without a middle value a group: `m`
             rows, `k` -> `n`; `epi`: "store", "resid" (out += r) or "gated" (out += gate * r); `out`: "f32" rows from
             products as exact as 32 bits are, or "bf16" rows (stored), from products as exact as that needs
  attention  `b` sequences of `lmin` to `lmax` rows, packed one behind the other, each behind the same `p` keys; `h`
             heads over `hkv` key heads of 128; causal, or every row of a sequence sees all of its rows; `out`: "bf16" rows,
             from products of bf16 values, or "f32" rows, from 32-bit products

Values of a 4-bit weight: s (c - 8) + z with codes c of 0 to 15 (even k in the low half of a byte), and s, z in bf16, one
for each group.  Attention: rows of q and k are RMS-normed for each head (eps 1e-6) and rotated at their position, `p` plus
the row's place in its sequence; the prefix's keys come normed and rotated.
"""

import importlib
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
HD = 128
THETA = 1e6


def listed():
    return [
        # the first token of a prompt from the text encoder's table: latency
        {"name": "embed_1x1024_bf16", "op": "embed", "t": 1, "n": 151936, "k": 1024, "table": "bf16", "g": 0, "mid": False,
         "weights": False, "scale": 1.0},
        # a batch of padded prompts with prompt weights, from a table kept in 4 bits
        {"name": "embed_8191x2048_q4", "op": "embed", "t": 8191, "n": 65536, "k": 2048, "table": "q4", "g": 64, "mid": True,
         "weights": True, "scale": 0.5},
        # one token through the text encoder's stacked q/k/v projection: latency
        {"name": "linear_1x4096x1024", "op": "linear", "m": 1, "n": 4096, "k": 1024, "g": 64, "mid": False, "epi": "store",
         "act": "none", "out": "f32"},
        # one row through an image model's widest product, groups of 32 with a middle: the weights' bytes
        {"name": "linear_1x8192x2048_g32", "op": "linear", "m": 1, "n": 8192, "k": 2048, "g": 32, "mid": True,
         "epi": "store", "act": "gelu", "out": "f32"},
        # a short prompt through the output projection, added to the residual stream
        {"name": "linear_43x1024x2048_resid", "op": "linear", "m": 43, "n": 1024, "k": 2048, "g": 64, "mid": True,
         "epi": "resid", "act": "none", "out": "f32"},
        # sizes that divide nothing but the group
        {"name": "linear_515x1316x1440_g32", "op": "linear", "m": 515, "n": 1316, "k": 1440, "g": 32, "mid": False,
         "epi": "gated", "act": "silu", "out": "f32"},
        # a batch of prompts through the stacked q/k/v projection, 32-bit products
        {"name": "linear_2048x4096x1024", "op": "linear", "m": 2048, "n": 4096, "k": 1024, "g": 128, "mid": True,
         "epi": "store", "act": "none", "out": "f32"},
        # two images of 1024 x 1024 through a DiT's first MLP product, bf16 rows: the largest
        {"name": "linear_8192x8192x2048_bf16", "op": "linear", "m": 8192, "n": 8192, "k": 2048, "g": 64, "mid": False,
         "epi": "store", "act": "gelu", "out": "bf16"},
        # positive and negative prompt, one token each behind a run of quality tags: latency
        {"name": "attn_2x1_p77", "op": "attention", "b": 2, "lmin": 1, "lmax": 1, "p": 77, "h": 16, "hkv": 8, "causal": True,
         "out": "bf16"},
        # ragged prompts behind a system text, 32-bit products, three heads to a key head
        {"name": "attn_9x3-211_p1000_f32", "op": "attention", "b": 9, "lmin": 3, "lmax": 211, "p": 1000, "h": 15, "hkv": 5,
         "causal": True, "out": "f32"},
        # single tokens of many sequences behind a long text: the prefix's bytes
        {"name": "attn_64x1_p8192", "op": "attention", "b": 64, "lmin": 1, "lmax": 1, "p": 8192, "h": 32, "hkv": 8,
         "causal": True, "out": "bf16"},
        # a list of prompts behind a long text: the largest
        {"name": "attn_64x64-192_p4096", "op": "attention", "b": 64, "lmin": 64, "lmax": 192, "p": 4096, "h": 16, "hkv": 8,
         "causal": True, "out": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["embed", "linear", "linear", "linear", "attention", "attention", "attention"])
    if op == "embed":
        table = rng.choice(["f32", "bf16", "q4"])
        g = rng.choice([32, 64, 128]) if table == "q4" else 0
        return {"op": op, "t": _log_int(rng, 1, 8192), "n": _log_int(rng, 2, 151936), "k": _log_int(rng, g or 32, 2048, g or 4),
                "table": table, "g": g, "mid": table == "q4" and rng.choice([True, False]),
                "weights": rng.choice([True, False]), "scale": rng.choice([1.0, 0.5, 32.0])}
    if op == "linear":
        g = rng.choice([32, 64, 128])
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192), _log_int(rng, g, 8192, g)
        n = max(64, min(n, (1 << 37) // (m * k)))
        epi = rng.choice(["store", "store", "resid", "gated"])
        return {"op": op, "m": m, "n": n, "k": k, "g": g, "mid": rng.choice([True, False]), "epi": epi,
                "act": rng.choice(["none", "none", "gelu", "silu"]),
                "out": rng.choice(["f32", "bf16"]) if epi == "store" else "f32"}
    h, hkv = rng.choice([(16, 8), (16, 16), (8, 1), (15, 5), (32, 8), (3, 3)])
    out = rng.choice(["bf16", "bf16", "f32"])
    case = {"op": op, "b": _log_int(rng, 1, 64), "lmin": 0, "lmax": _log_int(rng, 1, 600), "p": rng.choice([0, 1, 1, 1]) and
            _log_int(rng, 1, 8192), "h": h, "hkv": hkv, "causal": rng.choice([True, True, False]), "out": out}
    case["lmin"] = rng.choice([1, 1, 0, case["lmax"]])
    most = work(listed()[-1])["flops"] // (1 if out == "bf16" else 4)
    while work(case)["flops"] > most:
        case["b"] = (case["b"] + 1) // 2
        case["p"] = case["p"] * 3 // 4
    return case


def _lens(case):
    """The sequences' rows: from lmin to lmax, some at either end, one at least of them with a row."""
    rng = random.Random("%d %d %d" % (case["b"], case["lmin"], case["lmax"]))
    lens = [rng.choice([rng.randint(case["lmin"], case["lmax"])] * 6 + [case["lmin"], case["lmax"]]) for _ in range(case["b"])]
    if not any(lens):
        lens[-1] = case["lmax"]
    return lens


# ---------------------------------------------------------------- inputs


class _State:
    pass


class _Inputs:
    """Seeded device tensors, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=self.g, device="cuda") * std + mean

    def rows(self, m, k):
        """Activations: normal, with channels of larger scale as trained models have them."""
        return self.normal((m, k)) * torch.exp(self.normal((k,), 0.7))

    def q4(self, n, k, g, mid, std):
        """A 4-bit weight of standard deviation `std`: codes of a rounded normal distribution."""
        c = (self.normal((n, k), 2.5).round_().clamp_(-8, 7) + 8).to(torch.uint8)
        w = {"n": n, "k": k, "g": g, "codes": c[:, 0::2] | (c[:, 1::2] << 4),
             "s": (torch.exp(self.normal((n, k // g), 0.2)) * (std / 2.5)).to(torch.bfloat16), "z": None}
        if mid:
            w["z"] = self.normal((n, k // g), 0.2 * std).to(torch.bfloat16)
        return w


def _angles(rows):
    """Rotation angles [rows][64] in 64 bits (frequencies in 32, as a model's table has them)."""
    f = (1.0 / THETA ** (torch.arange(0, HD, 2, dtype=torch.float64, device="cuda") / HD)).float().double()
    return torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * f


def _inputs(case, seed):
    g, t, op = _Inputs(seed), {}, case["op"]
    if op == "embed":
        n, k = case["n"], case["k"]
        if case["table"] == "q4":
            t["w"] = g.q4(n, k, case["g"], case["mid"], 0.05)
        else:
            w = g.normal((n, k), 0.05)
            t["table"] = w.to(torch.bfloat16) if case["table"] == "bf16" else w
        ids = torch.randint(0, n, (case["t"],), generator=g.g, device="cuda", dtype=torch.int32)
        pad = torch.rand((case["t"],), generator=g.g, device="cuda") < 0.1
        t["ids"] = torch.where(pad & (torch.arange(case["t"], device="cuda") > 0), -1, ids).to(torch.int32)
        if case["weights"]:
            t["weights"] = 1.0 + 0.1 * torch.randint(-5, 6, (case["t"],), generator=g.g, device="cuda").float()
        return t
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        t["x"] = g.rows(m, k)
        t["w"] = g.q4(n, k, case["g"], case["mid"], 1.0 / math.sqrt(k))
        t["bias"] = g.normal((n,), 0.1)
        if case["epi"] == "gated":
            t["gate"] = g.normal((n,), 0.5)
        if case["epi"] != "store":
            t["out"] = g.normal((m, n))
        return t
    lens, p, h, hkv = _lens(case), case["p"], case["h"], case["hkv"]
    rows = sum(lens)
    t["qkv"] = g.rows(rows, (h + 2 * hkv) * HD)
    t["qn"], t["kn"] = g.normal((HD,), 0.1, 1.4), g.normal((HD,), 0.1, 1.4)
    a = _angles(p + max(lens))
    t["cos"], t["sin"] = torch.cos(a).float(), torch.sin(a).float()
    if p:
        k = g.normal((p, hkv, HD))
        k = k / torch.sqrt((k * k).mean(2, keepdim=True) + EPS) * t["kn"]
        c, s = t["cos"][:p, None], t["sin"][:p, None]
        t["pk"] = torch.cat([k[:, :, :64] * c - k[:, :, 64:] * s, k[:, :, 64:] * c + k[:, :, :64] * s], 2).contiguous()
        t["pv"] = g.normal((p, hkv, HD))
    return t


def prepare(case, seed):
    s = _State()
    s.case, s.t = case, _inputs(case, seed)
    t, op = s.t, case["op"]
    dtype = torch.bfloat16 if case.get("out") == "bf16" else torch.float32
    if op == "embed":
        s.out = torch.empty((case["t"], case["k"]), device="cuda")
    elif op == "linear":
        s.out = t["out"] if case["epi"] != "store" else torch.empty((case["m"], case["n"]), device="cuda", dtype=dtype)
    else:
        s.lens = _lens(case)
        s.out = torch.empty((sum(s.lens), case["h"] * HD), device="cuda", dtype=dtype)
        s.table = torch.cat([t["cos"], t["sin"]])
        # places of the packed rows in a padded batch, and back
        s.seq = torch.tensor([b for b, n in enumerate(s.lens) for _ in range(n)], device="cuda")
        s.pos = torch.tensor([i for n in s.lens for i in range(n)], device="cuda")
    s.weight = s.prefix = s.hlens = None
    torch.cuda.synchronize()
    if own:
        _keep(s)
    return s


# ---------------------------------------------------------------- plain form (32 bits)


def _values32(w, rows=None):
    """The values that (some rows of) a 4-bit weight stand for."""
    codes, sc, z = w["codes"], w["s"], w["z"]
    if rows is not None:
        codes, sc, z = codes[rows], sc[rows], None if z is None else z[rows]
    c = torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1, w["g"]).float() - 8.0
    v = c * sc.float()[:, :, None]
    if z is not None:
        v = v + z.float()[:, :, None]
    return v.view(codes.shape[0], -1)


def _act(v, act):
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v / (1.0 + torch.exp(-v)) if act == "silu" else v


def _norm_rope(x, w, c, s):
    """x [rows][heads][128]: RMS norm for each head, then the rotation of dims (d, d + 64)."""
    x = x / torch.sqrt((x * x).mean(2, keepdim=True) + EPS) * w
    c, s = c[:, None], s[:, None]
    return torch.cat([x[:, :, :64] * c - x[:, :, 64:] * s, x[:, :, 64:] * c + x[:, :, :64] * s], 2)


def _plain_attention(s):
    case, t = s.case, s.t
    h, hkv, p, b, n = case["h"], case["hkv"], case["p"], case["b"], max(s.lens)
    grp = h // hkv
    c, sn = t["cos"][p + s.pos], t["sin"][p + s.pos]
    rows = t["qkv"].shape[0]
    q = _norm_rope(t["qkv"][:, : h * HD].reshape(rows, h, HD), t["qn"], c, sn) * (1.0 / math.sqrt(HD))
    k = _norm_rope(t["qkv"][:, h * HD: (h + hkv) * HD].reshape(rows, hkv, HD), t["kn"], c, sn)
    v = t["qkv"][:, (h + hkv) * HD:].reshape(rows, hkv, HD)
    # a padded batch for the sequences' own keys: [b, hkv, n (x grp), 128]
    qb, kb, vb = (torch.zeros((b, n, x.shape[1], HD), device="cuda") for x in (q, k, v))
    for dst, src in ((qb, q), (kb, k), (vb, v)):
        dst[s.seq, s.pos] = src
    qb = qb.view(b, n, hkv, grp, HD).permute(0, 2, 1, 3, 4).reshape(b * hkv, n * grp, HD)
    kb, vb = (x.permute(0, 2, 1, 3).reshape(b * hkv, n, HD) for x in (kb, vb))
    sc = torch.bmm(qb, kb.transpose(1, 2).contiguous()).view(b, hkv, n, grp, n)
    i = torch.arange(n, device="cuda")
    lens = torch.tensor(s.lens, device="cuda")
    seen = (i[None, None, :] < lens[:, None, None]) & ((i[None, :] <= i[:, None])[None] if case["causal"] else torch.ones((), dtype=torch.bool, device="cuda"))
    sc = torch.where(seen[:, None, :, None, :], sc, float("-inf"))
    sc = sc.permute(0, 2, 1, 3, 4)[s.seq, s.pos].reshape(rows, h, n)
    top = sc.amax(2)
    if p:
        # the shared keys, once for all rows: [hkv, rows x grp, p]
        qp = q.view(rows, hkv, grp, HD).permute(1, 0, 2, 3).reshape(hkv, rows * grp, HD)
        sp = torch.bmm(qp, t["pk"].permute(1, 2, 0).contiguous()).view(hkv, rows, grp, p)
        top = torch.maximum(top, sp.amax(3).permute(1, 0, 2).reshape(rows, h))
        ep = torch.exp(sp - top.view(rows, hkv, grp).permute(1, 0, 2)[:, :, :, None])
        del sp
    e = torch.exp(sc - top[:, :, None])
    total = e.sum(2)
    eb = torch.zeros((b, n, h, n), device="cuda")
    eb[s.seq, s.pos] = e
    eb = eb.view(b, n, hkv, grp, n).permute(0, 2, 1, 3, 4).reshape(b * hkv, n * grp, n)
    o = torch.bmm(eb, vb).view(b, hkv, n, grp, HD).permute(0, 2, 1, 3, 4)[s.seq, s.pos].reshape(rows, h, HD)
    if p:
        total = total + ep.sum(3).permute(1, 0, 2).reshape(rows, h)
        op = torch.bmm(ep.view(hkv, rows * grp, p), t["pv"].permute(1, 0, 2).contiguous())
        o = o + op.view(hkv, rows, grp, HD).permute(1, 0, 2, 3).reshape(rows, h, HD)
    return (o / total[:, :, None]).reshape(rows, h * HD).to(s.out.dtype)


def _plain(s):
    case, t, op = s.case, s.t, s.case["op"]
    if op == "embed":
        ids = t["ids"].long().clamp(min=0)
        v = _values32(t["w"], ids) if "w" in t else t["table"][ids].float()
        f = case["scale"] * t["weights"] if "weights" in t else torch.full((case["t"],), case["scale"], device="cuda")
        return torch.where((t["ids"] >= 0)[:, None], v * f[:, None], 0.0)
    if op == "linear":
        r = _act(t["x"] @ _values32(t["w"]).t() + t["bias"], case["act"])
        if case["epi"] == "store":
            return r.to(s.out.dtype)
        return s.out.add_(r * t["gate"] if case["epi"] == "gated" else r)
    return _plain_attention(s)


# ---------------------------------------------------------------- the framework's operators

_module = _context = None


def _ctx():
    """The program's one context."""
    global _module, _context
    if _context is None:
        _module = importlib.import_module("anima-studio_amd")
        _context = _module.Context(0)
    return _context


def _ptr(t):
    return None if t is None else t.data_ptr()


def _keep(s):
    """What a program keeps from call to call: the weight object, the prefix's keys and values in the attention's form."""
    ctx, case, t = _ctx(), s.case, s.t
    if case["op"] != "attention":
        w, kinds = t.get("w"), {"f32": _module.W_F32, "bf16": _module.W_BF16}
        if w is None:
            s.weight = _module.weight(kinds[case["table"]], case["n"], case["k"], _ptr(t["table"]))
        else:
            s.weight = _module.weight(_module.W_Q4, w["n"], w["k"], _ptr(w["codes"]), group=w["g"], group_scale=_ptr(w["s"]),
                                      group_mid=_ptr(w["z"]), bias=_ptr(t.get("bias")))
        return
    s.hlens = np.asarray(s.lens, np.int32)
    s.precision = _module.PREC_BF16 if case["out"] == "bf16" else _module.PREC_FP32
    if case["p"]:
        p, hkv = case["p"], case["hkv"]
        s.prefix = torch.empty(ctx.attention_kv_bytes(1, hkv, p, s.precision), dtype=torch.uint8, device="cuda")
        ctx.attention_prefix(k=_ptr(t["pk"]), v=_ptr(t["pv"]), lens=[p], H=hkv, ldk=hkv * HD, ldv=hkv * HD, precision=s.precision,
                             prepare_into=_ptr(s.prefix))
        ctx.sync()


def _own(s):
    ctx, case, t, op = _ctx(), s.case, s.t, s.case["op"]
    if op == "embed":
        ctx.embed_rows(s.weight, _ptr(t["ids"]), case["t"], _ptr(s.out), weights=_ptr(t.get("weights")), scale=case["scale"])
        return s.out
    if op == "linear":
        epi = {"store": _module.EPI_STORE, "resid": _module.EPI_RESID, "gated": _module.EPI_GATED}[case["epi"]]
        bf16 = case["out"] == "bf16"
        ctx.linear(s.weight, case["m"], _ptr(s.out), x=_ptr(t["x"]), act=case["act"], epilogue=epi, gate=_ptr(t.get("gate")),
                   precision=_module.PREC_BF16 if bf16 else _module.PREC_FP32, out_bf16=bf16)
        return s.out
    h, hkv, ld = case["h"], case["hkv"], (case["h"] + 2 * case["hkv"]) * HD
    ctx.attention_prefix(q=_ptr(t["qkv"]), k=_ptr(t["qkv"]), v=_ptr(t["qkv"]), o=_ptr(s.out), lens=s.hlens, H=h, D=HD,
                         group=h // hkv, ldq=ld, ldk=ld, ldv=ld, k_off=h * HD, v_off=(h + hkv) * HD, P=case["p"],
                         prefix_kv=_ptr(s.prefix), causal=int(case["causal"]), q_norm=_ptr(t["qn"]), k_norm=_ptr(t["kn"]),
                         rope_cs=_ptr(s.table), rope_sin_off=t["cos"].numel(), eps=EPS, precision=s.precision,
                         o_bf16=case["out"] == "bf16")
    return s.out


def run(state):
    if own:
        return _own(state)
    return _plain(state)


def work(case):
    op = case["op"]
    if op == "embed":
        t, k = case["t"], case["k"]
        row = {"f32": 4 * k, "bf16": 2 * k}.get(case["table"]) or k // 2 + (k // case["g"]) * (4 if case["mid"] else 2)
        return {"bytes": t * (row + 4 * k + 4 + (4 if case["weights"] else 0)), "flops": t * k}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        out = m * n * (2 if case["out"] == "bf16" else 4 if case["epi"] == "store" else 8)
        return {"bytes": 4 * m * k + n * k // 2 + n * (k // case["g"]) * (4 if case["mid"] else 2) + out + 4 * n,
                "flops": 2 * m * n * k}
    lens, h, hkv, p = _lens(case), case["h"], case["hkv"], case["p"]
    e = 2 if case["out"] == "bf16" else 4
    pairs = sum(n * p + (n * (n + 1) // 2 if case["causal"] else n * n) for n in lens)
    return {"bytes": 2 * p * hkv * HD * e + sum(lens) * (4 * (h + 2 * hkv) + e * h) * HD, "flops": 4 * pairs * h * HD}


# ---------------------------------------------------------------- 64 bits


def _exact_values(w, rows=None):
    codes = w["codes"] if rows is None else w["codes"][rows]
    v = torch.empty((codes.shape[0], w["k"]), dtype=torch.float64, device="cuda")
    v[:, 0::2] = (codes % 16).double() - 8
    v[:, 1::2] = torch.div(codes, 16, rounding_mode="floor").double() - 8
    for j in range(w["k"] // w["g"]):
        part = v[:, j * w["g"]: (j + 1) * w["g"]]
        part *= (w["s"] if rows is None else w["s"][rows])[:, j: j + 1].double()
        if w["z"] is not None:
            part += (w["z"] if rows is None else w["z"][rows])[:, j: j + 1].double()
    return v


def _exact_heads(x, w, angles):
    """[rows][heads][128] -> the same normed and rotated, as complex numbers turned by their angle."""
    x = x.double()
    x = x * torch.rsqrt(torch.sum(x * x, 2, keepdim=True) / HD + EPS) * w.double()
    z = torch.complex(x[..., :64].contiguous(), x[..., 64:].contiguous()) * angles[:, None]
    return torch.cat([z.real, z.imag], 2)


def exact(case, seed):
    t, op = _inputs(case, seed), case["op"]
    if op == "embed":
        live = torch.nonzero(t["ids"] >= 0)[:, 0]
        rows = t["ids"][live].long()
        out = torch.zeros((case["t"], case["k"]), dtype=torch.float64, device="cuda")
        v = _exact_values(t["w"], rows) if "w" in t else t["table"][rows].double()
        out[live] = v * case["scale"] * (t["weights"][live, None].double() if "weights" in t else 1.0)
        return out
    if op == "linear":
        r = torch.mm(t["x"].double(), _exact_values(t["w"]).t()) + t["bias"].double()
        if case["act"] == "gelu":
            r = r * torch.special.ndtr(r)
        elif case["act"] == "silu":
            r = r * torch.sigmoid(r)
        if case["epi"] == "gated":
            r = r * t["gate"].double()
        return r if case["epi"] == "store" else t["out"].double() + r
    h, hkv, p = case["h"], case["hkv"], case["p"]
    # the rotation as the table has it (its 32-bit cosines and sines are inputs)
    turn = torch.complex(t["cos"].double(), t["sin"].double())
    outs, at = [], 0
    for n in _lens(case):
        x = t["qkv"][at: at + n]
        at += n
        q = _exact_heads(x[:, : h * HD].reshape(n, h, HD), t["qn"], turn[p: p + n])
        k = _exact_heads(x[:, h * HD: (h + hkv) * HD].reshape(n, hkv, HD), t["kn"], turn[p: p + n])
        v = x[:, (h + hkv) * HD:].reshape(n, hkv, HD).double()
        if p:
            k, v = torch.cat([t["pk"].double(), k]), torch.cat([t["pv"].double(), v])
        k, v = (y.repeat_interleave(h // hkv, 1).transpose(0, 1) for y in (k, v))
        score = torch.bmm(q.transpose(0, 1).contiguous(), k.transpose(1, 2).contiguous()) / math.sqrt(HD)
        if case["causal"]:
            score = score.masked_fill(torch.ones((n, p + n), device="cuda").triu(p + 1).bool(), float("-inf"))
        outs.append(torch.bmm(torch.softmax(score, 2), v.contiguous()).transpose(0, 1).reshape(n, h * HD))
    return torch.cat(outs)
