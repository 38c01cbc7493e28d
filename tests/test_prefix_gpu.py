"""Attention of many sequences behind one shared prefix on the device, against a 64-bit form of each sequence by itself.

Tolerances.  fp32: a score is off by the roundings of the norms, the rotations and the products: at most 40 2^-24 |q| |k| scale;
a weight by twice that of itself, the sums by 2^-24 (32 + keys / 16); so an output element is off by at most
(80 |q| |k| scale + 32 + keys / 16) 2^-24 of the largest value of v that the row sees.
bf16: q and k are rounded to 11 bits, the weights and v to 8, each value off by 2^-11 and 2^-8 of itself at the most, by 2^-12.3 and
2^-9.3 in the root mean square.  A score is off by sqrt(2) 2^-12.3 sqrt(sum (q_d k_d)^2) scale, which is 0.0006 where q and k have
normed rows of 1.4; an output row, a mean of many independent values, by sqrt(0.0006^2 + 2 2^-18.6) = 0.0023 of the root of sum
(p v)^2.  The tests ask for five times that, 0.012, of every row of 128 values.  A bf16 result adds 2^-8 of itself."""

import numpy as np
import pytest

from helpers import amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    with amd().Context(0) as c:
        yield c


def widen(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def norm(x, w, eps=1e-6):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w if w is not None else x


def rope(x, cs, pos):
    if cs is None:
        return x
    c, s = cs[0][pos][:, None], cs[1][pos][:, None]
    return np.concatenate([x[..., :64] * c - x[..., 64:] * s, x[..., 64:] * c + x[..., :64] * s], -1)


class Case:
    """A batch behind a prefix: inputs on the host and the device, the prepared prefix, one call, and its 64-bit form."""

    def __init__(self, ctx, lens, P, H, Hkv, precision, *, causal=1, normed=True, roped=True, scale=0.0, o_bf16=False, seed=0, pad=0,
                 std=1.0, table=None):
        m = amd()
        rng = np.random.default_rng(seed + sum(lens) + P)
        self.ctx, self.lens, self.P, self.H, self.Hkv, self.precision = ctx, list(lens), P, H, Hkv, precision
        self.causal, self.scale, self.o_bf16 = causal, scale, o_bf16
        self.T, self.ld = sum(lens), (H + 2 * Hkv) * 128 + pad
        self.qkv = (rng.normal(0, std, (self.T, self.ld))).astype(np.float32)
        self.qn, self.kn = (rng.normal(1.4, 0.1, (2, 128)).astype(np.float32) if normed else (None, None))
        rows = table or P + max(lens)
        ang = np.arange(rows)[:, None] * (1e6 ** (-np.arange(0, 128, 2) / 128.0)).astype(np.float32).astype(np.float64)
        self.cs = (np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)) if roped else None
        self.pk, self.pv = rng.normal(0, std, (2, P, Hkv, 128)).astype(np.float32)
        self.d = {}
        if P:
            up = [ctx.upload(self.pk), ctx.upload(self.pv)]
            self.prefix = ctx.empty((ctx.attention_kv_bytes(1, Hkv, P, precision),), np.uint8)
            ctx.attention_prefix(k=up[0], v=up[1], lens=[P], H=H, group=H // Hkv, ldk=Hkv * 128, ldv=Hkv * 128, precision=precision,
                                 prepare_into=self.prefix, k_norm=self.put("kn", self.kn),
                                 rope_cs=self.put("cs", np.concatenate([t.reshape(-1) for t in self.cs]) if roped else None),
                                 rope_sin_off=self.cs[0].size if roped else 0)
        else:
            self.prefix = None

    def put(self, name, a):
        if a is None:
            return None
        if name not in self.d:
            self.d[name] = self.ctx.upload(a)
        return self.d[name]

    def call(self, qkv=None, out=None, o_off=0, ldo=None):
        m, H, Hkv = amd(), self.H, self.Hkv
        qkv = qkv or self.put("qkv", self.qkv)
        o = out or self.ctx.empty((max(self.T, 1), ldo or H * 128), np.uint16 if self.o_bf16 else np.float32)
        self.ctx.attention_prefix(q=qkv, k=qkv, v=qkv, o=o, lens=self.lens, H=H, group=H // Hkv, ldq=self.ld, ldk=self.ld, ldv=self.ld,
                                  k_off=H * 128, v_off=(H + Hkv) * 128, P=self.P, prefix_kv=self.prefix, scale=self.scale,
                                  causal=self.causal, precision=self.precision, q_norm=self.put("qn", self.qn),
                                  k_norm=self.put("kn", self.kn),
                                  rope_cs=self.put("cs", np.concatenate([t.reshape(-1) for t in self.cs]) if self.cs else None),
                                  rope_sin_off=self.cs[0].size if self.cs else 0, o_bf16=self.o_bf16, o_off=o_off, ldo=ldo)
        return o

    def get(self, **kw):
        r = self.call(**kw).numpy()
        return widen(r) if self.o_bf16 else r

    def ref(self):
        """-> out [T][H][128] and the tolerance of each element."""
        H, Hkv, P = self.H, self.Hkv, self.P
        cs = tuple(t.astype(np.float64) for t in self.cs) if self.cs else None
        kn = self.kn.astype(np.float64) if self.kn is not None else None
        qn = self.qn.astype(np.float64) if self.qn is not None else None
        pk = rope(norm(self.pk.astype(np.float64), kn), cs, np.arange(P)) if P else np.zeros((0, Hkv, 128))
        pv = self.pv.astype(np.float64)
        scale = self.scale or 1 / np.sqrt(128.0)
        outs, tols, at = [], [], 0
        for n in filter(None, self.lens):
            x = self.qkv[at: at + n].astype(np.float64)
            at += n
            pos = P + np.arange(n)
            q = rope(norm(x[:, : H * 128].reshape(n, H, 128), qn), cs, pos)
            k = rope(norm(x[:, H * 128: (H + Hkv) * 128].reshape(n, Hkv, 128), kn), cs, pos)
            v = x[:, (H + Hkv) * 128: (H + 2 * Hkv) * 128].reshape(n, Hkv, 128)
            k, v = np.concatenate([pk, k]), np.concatenate([pv, v])
            k, v = np.repeat(k, H // Hkv, 1), np.repeat(v, H // Hkv, 1)
            s = np.einsum("ihd,jhd->hij", q, k) * scale
            if self.causal:
                s = np.where(np.arange(P + n)[None, None, :] <= P + np.arange(n)[None, :, None], s, -np.inf)
            p = np.exp(s - s.max(2, keepdims=True))
            p /= p.sum(2, keepdims=True)
            o = np.einsum("hij,jhd->ihd", p, v)
            if self.precision == amd().PREC_FP32:
                size = np.sqrt((q * q).sum(2))[:, :, None] * np.sqrt((k * k).sum(2)).max(0)[None, :, None] * abs(scale)
                tol = (80 * size + 32 + (P + n) / 16) * 2.0 ** -24 * np.abs(v).max((0, 2))[None, :, None] + 0 * o
            else:
                spread = np.sqrt(np.einsum("hij,jhd->ihd", p * p, v * v).sum(2, keepdims=True))  # of a whole row
                tol = 0.012 * spread + 0 * o
            outs.append(o)
            tols.append(tol)
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, got=None):
        got = self.get() if got is None else got
        ref, tol = self.ref()
        got = got.reshape(ref.shape)
        if self.precision == amd().PREC_FP32:
            err = np.abs(got - ref)
        else:  # whole rows
            err = np.sqrt(((got - ref) ** 2).sum(2, keepdims=True))
            if self.o_bf16:
                tol = tol + 2.0 ** -8 * np.sqrt((ref * ref).sum(2, keepdims=True))
        assert np.isfinite(got).all()
        assert np.all(err <= tol), (err / tol).max()


LENS = {"one": [1], "ones": [1] * 40, "many": [1] * 300, "pair": [1, 1], "ragged": [3, 0, 64, 1, 65, 17, 0, 130, 2], "empty_ends": [0, 5, 0],
        "long": [777], "long_behind_short": [1, 2, 500, 1], "blocks": [64, 64, 128], "tens": [11] * 30}


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("P", [0, 1, 63, 64, 65, 300, 1024])
@pytest.mark.parametrize("lens", list(LENS))
def test_lengths(ctx, lens, P, precision):
    Case(ctx, LENS[lens], P, 4, 2, precision).check()


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (16, 8), (5, 5), (6, 2), (8, 1), (15, 3), (32, 8), (33, 1)])
@pytest.mark.parametrize("lens,P", [([9, 1, 40], 100), ([2], 700), ([70, 50, 100], 0)])
def test_heads(ctx, lens, P, H, Hkv, precision):
    Case(ctx, lens, P, H, Hkv, precision).check()


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("normed,roped,scale,causal", [(False, False, 0.0, 1), (True, False, 0.2, 1), (False, True, 0.0, 0),
                                                       (True, True, 0.0, 0), (True, True, -0.1, 1)])
@pytest.mark.parametrize("lens,P", [([9, 1, 140], 100), ([30, 30], 0), ([130], 200)])
def test_forms(ctx, lens, P, normed, roped, scale, causal, precision):
    Case(ctx, lens, P, 4, 2, precision, causal=causal, normed=normed, roped=roped, scale=scale, pad=12).check()


@pytest.mark.parametrize("lens,P", [([9, 1, 140], 100), ([1] * 20, 640), ([300], 1)])
def test_bf16_rows(ctx, lens, P):
    """O as bf16 is the fp32 O rounded to nearest even, bit for bit."""
    a, b = Case(ctx, lens, P, 4, 2, 0), Case(ctx, lens, P, 4, 2, 0, o_bf16=True)
    b.check()
    u = a.get().view(np.uint32)
    np.testing.assert_array_equal(((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16), b.call().numpy())


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P", [([1], 8192), ([3, 1], 5000), ([1] * 130, 2500), ([200] * 3, 4100), ([2000, 100], 64), ([600] * 8, 600)])
def test_long(ctx, lens, P, precision):
    Case(ctx, lens, P, 2, 1, precision).check()


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P", [([64] * 32, 70), ([65, 1, 30] * 24 + [77], 130)])
def test_many_tiles(ctx, lens, P, precision):
    """Tiles of 256 rows enough for every compute unit (32 heads, a kv head each): several sequences to a tile, not split."""
    Case(ctx, lens, P, 32, 32, precision).check()


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P,H,Hkv", [([3, 1], 640, 2, 1), ([64] * 32, 640, 32, 32), ([200], 0, 2, 2), ([300, 90], 200, 2, 1)])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_rise(ctx, lens, P, H, Hkv, precision, falling):
    """Scores of 2^90 times the weight every 64 keys (or a 2^90th): a row is the mean of the values at its last (first) such
    keys, whose scores are the same.  q and k are powers of two times signs, so that only the common factor scale rounds."""
    c = Case(ctx, lens, P, H, Hkv, precision, normed=False, roped=False)
    sign = np.where(np.random.default_rng(1).random(128) < 0.5, -1.0, 1.0).astype(np.float32)
    level = lambda j: (-1.0 if falling else 1.0) * (j // 64).astype(np.float32)[:, None, None] * 0.5
    c.pk = (level(np.arange(P)) * sign * np.ones((1, Hkv, 1))).astype(np.float32)
    if P:
        up = [ctx.upload(c.pk), ctx.upload(c.pv)]
        ctx.attention_prefix(k=up[0], v=up[1], lens=[P], H=H, group=H // Hkv, ldk=Hkv * 128, ldv=Hkv * 128, precision=precision,
                             prepare_into=c.prefix)
    at = 0
    c.qkv[:, : H * 128] = np.tile(sign, H)
    for n in lens:
        c.qkv[at: at + n, H * 128: (H + Hkv) * 128] = (level(P + np.arange(n)) * sign * np.ones((1, Hkv, 1))).reshape(n, -1)
        at += n
    c.scale = float(90 / 64 * np.log(2.0))  # a level is 128 * 0.5 * scale
    got = c.get().reshape(c.T, H, 128)
    ref, _ = c.ref()
    v = max(np.abs(c.pv).max() if P else 0, np.abs(c.qkv[:, (H + Hkv) * 128:]).max())
    # equal weights at one level, rounded alike and divided by the sum of what they were rounded to: a value of v is off by half a
    # bf16 step (8 significant bits: 2^-8 of a value just above a power of two), a sum of up to 64 by 64 2^-24
    assert np.abs(got - ref).max() <= (2.0 ** -8 if precision == 0 else 0.0) * v + 128 * 2.0 ** -24 * v


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
def test_longest_prefix(ctx, precision):
    """2^22 keys: 2 GiB of k in fp32, prepared planes of 1 and 2 GiB.  Values of 1 plus noise, so that a result is 1 but for the
    mean of the noise: the sums of 4 million weights, in chains of at most 65536 keys a part and 64 parts, are off by 2^-24 a step of
    16 keys (fp32: of half of one) in the worst case, a bf16 value by 2^-8 of itself, and the errors of q, k and the weights meet the noise
    alone."""
    m = amd()
    P, T = 1 << 22, 3
    k, v = ctx.empty((P, 128)), ctx.empty((P, 128))
    ctx.fill_random(k, P * 128, "f32", 1, -1.0, 1.0)
    ctx.fill_random(v, P * 128, "f32", 2, 0.75, 1.25)
    prefix = ctx.empty((ctx.attention_kv_bytes(1, 1, P, precision),), np.uint8)
    ctx.attention_prefix(k=k, v=v, lens=[P], H=2, group=2, ldk=128, ldv=128, precision=precision, prepare_into=prefix)
    hk, hv = k.numpy(), v.numpy()
    k.release()
    v.release()
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (T, 4 * 128)).astype(np.float32)
    x[:, :256] *= np.float32(0.5)
    # the last block of the prefix counts: row 0 of head 0 looks for its last key
    x[0, :128] = 40.0 * hk[-1]
    dx, out = ctx.upload(x), ctx.empty((T, 256))
    ctx.attention_prefix(q=dx, k=dx, v=dx, o=out, lens=[2, 1], H=2, group=2, ldq=512, ldk=512, ldv=512, k_off=256, v_off=384, P=P,
                         prefix_kv=prefix, precision=precision)
    got = out.numpy().reshape(T, 2, 128)
    prefix.release()
    ctx.trim()
    s = np.concatenate([(x[:, h * 128: h * 128 + 128].astype(np.float64) @ hk[i: i + (1 << 19)].T.astype(np.float64))
                        for h in range(2) for i in range(0, P, 1 << 19)], 1).reshape(T, 2, P) / np.sqrt(128.0)
    for t in range(T):
        own = [0] if t == 0 else [0, 1] if t == 1 else [2]
        ko, vo = x[own, 256:384].astype(np.float64), x[own, 384:].astype(np.float64)
        for h in range(2):
            so = ko @ x[t, h * 128: h * 128 + 128].astype(np.float64) / np.sqrt(128.0)
            top = max(s[t, h].max(), so.max())
            p, po = np.exp(s[t, h] - top), np.exp(so - top)
            l = p.sum() + po.sum()
            ref = (sum(p[i: i + (1 << 19)] @ hv[i: i + (1 << 19)].astype(np.float64) for i in range(0, P, 1 << 19)) + po @ vo) / l
            # 65536 keys in steps of 16 (fp32: 32), then 64 parts
            tol = 1.25 * 2.0 ** -24 * (65536 / (16 if precision == m.PREC_BF16 else 32) + 64) + (2.0 ** -8 if precision == m.PREC_BF16 else 1e-5)
            assert np.abs(got[t, h] - ref).max() <= tol * max(1.0, np.abs(ref).max()), (t, h, np.abs(got[t, h] - ref).max())


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
def test_two_contexts(ctx, precision):
    """Calls of two contexts at once, each on its stream with scratch of its own."""
    with amd().Context(0) as other:
        a, b = Case(ctx, [40, 1, 17], 200, 4, 2, precision), Case(other, [40, 1, 17], 200, 4, 2, precision)
        ra, rb = a.get(), b.get()
        outs = [(a.call(), b.call()) for _ in range(4)]
        for x, y in outs:
            np.testing.assert_array_equal(x.numpy(), ra)
            np.testing.assert_array_equal(y.numpy(), rb)
        np.testing.assert_array_equal(ra, rb)


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P", [([5, 70, 1], 100), ([5, 70, 1], 0), ([1] * 70, 64), ([300, 200], 130)])
@pytest.mark.parametrize("std", [30.0, 1e-3])
def test_large_and_small_scores(ctx, lens, P, precision, std):
    """Without norms: scores of thousands (one key takes all), and of nothing (every key the same).  The largest weights
    of the bf16 form may differ from the 64-bit ones where two scores are within their roundings, so there the rows are
    compared with the fp32 form's bound on scores rounded to bf16 inputs: finite, and within the values seen."""
    c = Case(ctx, lens, P, 4, 2, precision, normed=False, roped=False, std=std)
    got = c.get()
    assert np.isfinite(got).all()
    if precision == 1 or std < 1:
        c.check(got)
    else:
        top = max(np.abs(c.qkv).max(), np.abs(c.pv).max() if P else 0)
        assert np.abs(got).max() <= top * (1 + 2.0 ** -6)


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("lens,P", [([5, 70, 1, 8], 100), ([33, 1, 64, 40], 0), ([1] * 70, 64), ([300, 200, 100, 5], 130)])
@pytest.mark.parametrize("what", ["k", "v", "q"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
def test_sequences_do_not_reach_each_other(ctx, lens, P, precision, causal, what, bad):
    """NaN, infinities and the largest numbers in one sequence's rows: every other sequence's results keep their bits; under a
    causal mask, so do the rows before it."""
    c = Case(ctx, lens, P, 4, 2, precision, causal=causal, normed=False)
    good = c.get()
    b = len(lens) // 2
    at = sum(lens[:b])
    row = at + lens[b] // 2
    off = {"q": 0, "k": 4 * 128, "v": 6 * 128}[what]
    x = c.qkv.copy()
    x[row, off + 7] = bad
    got = c.get(qkv=ctx.upload(x))
    same = np.ones(c.T, bool)
    if what == "q":
        same[row] = False
    else:
        same[(row if causal else at): at + lens[b]] = False
    np.testing.assert_array_equal(got[same], good[same])
    if not np.isfinite(bad):
        hit = got[row].reshape(4, 128)
        heads = [0] if what == "q" else [0, 1]
        assert all((~np.isfinite(hit[h])).any() for h in heads)
        rest = [h for h in range(4) if h not in heads]
        np.testing.assert_array_equal(hit[rest], good[row].reshape(4, 128)[rest])


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
def test_rows_behind_the_last_sequence_stay(ctx, precision):
    """Rows and columns beyond the result are left as they were."""
    c = Case(ctx, [5, 0, 70], 77, 4, 2, precision, pad=4)
    buf = np.full((90, 4 * 128 + 20), 3.0, np.float32)
    out = ctx.upload(buf)
    got = c.call(out=out, o_off=8, ldo=buf.shape[1]).numpy()
    c.check(np.ascontiguousarray(got[:75, 8: 8 + 512]))
    buf[:75, 8: 520] = got[:75, 8: 520]
    np.testing.assert_array_equal(got, buf)


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
def test_no_rows(ctx, precision):
    c = Case(ctx, [3], 10, 4, 2, precision)
    c.lens = [0, 0]
    out = ctx.upload(np.full((3, 512), 5.0, np.float32))
    c.call(out=out)
    assert (out.numpy() == 5.0).all()


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("lens,P", [([40, 1, 17], 200), ([1], 3000), ([600], 64)])
def test_replayed_from_a_graph(ctx, lens, P, precision):
    """Two captured calls with scratch of their own, replayed in turn with eager calls and other inputs between them."""
    a, b = Case(ctx, lens, P, 4, 2, precision), Case(ctx, [7, 90], P, 2, 2, precision, seed=5)
    outs, graphs = [], []
    for c in (a, b):
        o = c.call()
        ctx.sync()
        ctx.graph_begin()
        c.call(out=o)
        graphs.append(ctx.graph_end())
        outs.append(o)
    try:
        for i in range(3):
            for c, o, g in zip((a, b), outs, graphs):
                x = c.qkv * np.float32(1 + i) + np.float32(0.1 * i)
                c.put("qkv", c.qkv).write(x)
                ref = c.call().numpy()
                ctx.graph_launch(g)
                np.testing.assert_array_equal(o.numpy(), ref)
    finally:
        for g in graphs:
            ctx.graph_destroy(g)


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
def test_against_the_attention_of_each_sequence(ctx, precision):
    """The framework's own causal attention of the whole prompt, prefix and rows in one sequence: the same rows within both
    sides' tolerance.  Its bf16 form rounds q and k to 8 bits: a score is off by eight times 0.0006, so a row by
    sqrt(0.005^2 + 2 2^-18.6) = 0.006 in the root mean square, 0.03 at five times that, beside this side's 0.012."""
    m = amd()
    c = Case(ctx, [37, 5, 90], 150, 4, 2, precision)
    got = c.get().reshape(c.T, 4, 128)
    ref, tol = c.ref()
    at, ld = 0, 8 * 128
    for n in c.lens:
        x = np.concatenate([np.concatenate([np.zeros((150, 512), np.float32), c.pk.reshape(150, 256), c.pv.reshape(150, 256)], 1),
                            c.qkv[at: at + n]])
        L = 150 + n
        dx, o = ctx.upload(x), ctx.empty((L, 512))
        cs = np.concatenate([t[:L].reshape(-1) for t in c.cs]) if c.cs[0].shape[0] == L else np.concatenate(
            [np.ascontiguousarray(t[:L]).reshape(-1) for t in c.cs])
        ctx.attention(q=dx, k=dx, v=dx, o=o, B=1, Lq=L, Lk=L, H=4, D=128, ldq=ld, ldk=ld, ldv=ld, k_off=512, v_off=768, group=2, causal=1,
                      precision=precision, q_norm=c.put("qn", c.qn), k_norm=c.put("kn", c.kn), rope_cs=ctx.upload(cs), rope_sin_off=L * 64)
        d = got[at: at + n] - o.numpy()[150:].reshape(n, 4, 128)
        err = np.abs(d) if precision == m.PREC_FP32 else np.sqrt((d * d).sum(2, keepdims=True))
        assert np.all(err <= (2 if precision == m.PREC_FP32 else 3.5) * tol[at: at + n])
        at += n
