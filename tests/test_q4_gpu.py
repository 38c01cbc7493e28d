"""4-bit weights with group scales and embedding rows on the device, against 64-bit forms.

Tolerances.  S = sum_k |x_k w_k|.  A product is off by the rounding of x (kept to 2^-23 of itself, or to 2^-12 where
ANIMA_PREC_BF16 lets the call round it to 11 bits), of w (one rounding, 2^-24) and of the sums: the longest chain of 32-bit
additions has at most K / 16 steps and a few dozen more where parts are joined, each off by 2^-24 of at most S.
So 2^-24 (32 + K / 16) S, and 2^-12 S more.  The slope of an activation is at most 1.13, the GELU polynomial is off by 2^-22 of its
argument and the rest of the epilogue by a few 2^-24 of its terms.  A bf16 result is off by 2^-8 of itself more."""

import numpy as np
import pytest

from helpers import amd, ran

pytestmark = pytest.mark.gpu

BIT_EPS = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    with amd().Context(0) as c:
        yield c


def bf16(x):
    """float32 -> bf16 bits, to nearest even (finite values)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    return ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def widen(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def values(codes, s, z, g):
    """64-bit values of a 4-bit weight (codes [N][K], s and z as floats or None)."""
    v = (codes.astype(np.float64) - 8) * np.repeat(s.astype(np.float64), g, 1)
    return v if z is None else v + np.repeat(z.astype(np.float64), g, 1)


class Q4:
    """A random 4-bit weight on the device and its values."""

    def __init__(self, ctx, rng, N, K, g, mid, bias=None, spread=0.3):
        codes = rng.integers(0, 16, (N, K)).astype(np.uint8)
        s = widen(bf16(np.exp(rng.normal(0, spread, (N, K // g))) / (5 * np.sqrt(K))))
        z = widen(bf16(rng.normal(0, 1, (N, K // g)) / np.sqrt(K))) if mid else None
        self.values = values(codes, s, z, g)
        self.bufs = [ctx.upload(pack(codes)), ctx.upload(bf16(s)), ctx.upload(bf16(z)) if mid else None]
        self.bias = bias
        self.dbias = ctx.upload(bias) if bias is not None else None
        self.w = amd().weight(amd().W_Q4, N, K, self.bufs[0], group=g, group_scale=self.bufs[1], group_mid=self.bufs[2],
                              bias=self.dbias)


def erf(x):
    import torch

    return torch.erf(torch.from_numpy(x)).numpy()


def act64(r, act):
    if act == "gelu":
        return 0.5 * r * (1 + erf(r * np.sqrt(0.5)))
    return r / (1 + np.exp(-r)) if act == "silu" else r


def bound(x, w, K, precision, out_bf16, ref, r0):
    m = amd()
    S = np.abs(x) @ np.abs(w).T
    t = BIT_EPS * (32 + K / 16) * S + (2.0 ** -12 * S if precision == m.PREC_BF16 else 0.0)
    t = 1.13 * t + 2.0 ** -21 * np.abs(r0) + 8 * BIT_EPS * np.abs(ref)
    return t + 2.0 ** -8 * np.abs(ref) if out_bf16 else t


# (the largest cases: a few workgroups of the largest tiles in every direction; k loops of one step to many)
SHAPES = [(1, 1, 32, 32), (1, 5, 64, 64), (1, 1000, 1024, 64), (1, 4096, 256, 128), (2, 17, 96, 32), (3, 130, 2048, 128),
          (4, 129, 1440, 32), (5, 64, 128, 64), (7, 333, 4096, 64), (8, 100, 1184, 32), (9, 65, 320, 64), (15, 1024, 512, 128),
          (16, 48, 32, 32), (17, 70, 64, 64), (31, 257, 1056, 32), (33, 127, 384, 128), (43, 1024, 2048, 64), (64, 96, 8192, 128),
          (65, 514, 96, 32), (100, 300, 640, 64), (127, 129, 1088, 64), (128, 128, 256, 32), (129, 260, 160, 32), (200, 1000, 512, 128),
          (257, 513, 288, 32), (300, 64, 4160, 64), (515, 516, 1440, 32), (1024, 384, 128, 128),
          # (products that the matrix kernels take: the smaller ones above are the vector kernel's)
          (14, 2668, 4032, 32), (31, 2101, 1056, 32), (64, 1025, 1184, 32), (48, 1500, 2176, 128), (20, 2050, 2112, 64), (129, 2260, 160, 32),
          (257, 1513, 288, 32), (66, 1031, 2048, 128), (130, 700, 1056, 32)]


@pytest.mark.parametrize("precision", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("mid", [False, True], ids=["sym", "mid"])
@pytest.mark.parametrize("M,N,K,g", SHAPES)
def test_products(ctx, M, N, K, g, mid, precision):
    rng = np.random.default_rng(M * 1000 + N + K)
    W = Q4(ctx, rng, N, K, g, mid)
    x = (rng.normal(0, 1, (M, K)) * np.exp(rng.normal(0, 0.7, K))).astype(np.float32)
    dx, out = ctx.upload(x), ctx.empty((M, N))
    ctx.linear(W.w, M, out, x=dx, precision=precision)
    ref = x.astype(np.float64) @ W.values.T
    err = np.abs(out.numpy() - ref)
    tol = bound(x.astype(np.float64), W.values, K, precision, False, ref, ref)
    assert np.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("precision,M,N,K,g,mid,name", [
    (1, 1025, 4092, 288, 32, True, "gemm.q4.128"), (1, 515, 3700, 1312, 32, True, "gemm.q4.128"), (0, 2050, 3900, 320, 64, True, "gemm.q4.64"),
    (0, 1030, 3600, 1152, 128, False, "gemm.q4.64"), (1, 2049, 4092, 1056, 32, True, "gemm.q4.256"), (0, 4100, 3901, 544, 32, True, "gemm.q4.256"),
    (0, 2050, 3901, 576, 64, False, "gemm.q4.128"), (1, 640, 1701, 4160, 64, True, "gemm.q4.128"), (0, 640, 1701, 4160, 64, True, "gemm.q4.64"), (1, 70, 260, 256, 64, True, "gemv.q4"), (1, 70, 2600, 256, 64, True, "gemm.q4.64"), (0, 300, 64, 4160, 64, True, "gemm.q4.64"),
    (1, 20, 40, 16416, 32, True, "gemm.q4.64"), (1, 20, 40, 8224, 32, False, "gemv.q4"), (0, 64, 300, 1024, 64, True, "gemm.q4.few"), (1, 20, 2700, 8224, 32, False, "gemm.q4.few"),
    (0, 64, 1300, 1024, 64, True, "gemm.q4.few"), (0, 5000, 65, 64, 32, True, "gemm.q4.64"), (0, 100, 101, 512, 32, True, "gemv.q4"), (1, 300000, 3, 32, 32, False, "gemm.q4.64"), (1, 40, 100, 8192, 128, True, "gemm.q4.64"),
    (1, 4, 300, 1024, 64, True, "gemv.q4")])
def test_variants(ctx, precision, M, N, K, g, mid, name):
    """Each kernel by its profiler name, at ragged sizes, with an activation and bf16 rows."""
    rng = np.random.default_rng(M + K)
    W = Q4(ctx, rng, N, K, g, mid)
    x = rng.normal(0, 1, (M, K)).astype(np.float32)
    dx, out = ctx.upload(x), ctx.empty((M, N), np.uint16)
    assert ran(ctx, lambda: ctx.linear(W.w, M, out, x=dx, act="gelu", precision=precision, out_bf16=True)) == {name}
    r0 = x.astype(np.float64) @ W.values.T
    ref = act64(r0, "gelu")
    err = np.abs(widen(out.numpy()) - ref)
    tol = bound(x.astype(np.float64), W.values, K, precision, True, ref, r0)
    assert np.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("M", [1, 3, 20, 150])
@pytest.mark.parametrize("epi,act,add,alpha,out_bf16", [
    (0, "none", False, 0.0, True), (0, "gelu", False, 0.0, True), (0, "silu", True, 0.5, False), (0, "gelu", True, 0.0, False),
    (1, "none", False, 0.0, False), (1, "silu", True, -2.0, False), (2, "none", False, 0.0, False), (2, "gelu", True, 0.25, False)])
@pytest.mark.parametrize("N,ragged,K", [(132, False, 224), (67, True, 224), (256, True, 224), (2668, False, 1056), (2667, True, 1056)])
def test_epilogues(ctx, M, epi, act, add, alpha, out_bf16, N, ragged, K):
    """Every epilogue, with rows of out, add and x further apart than they are wide, and gate and buffers at odd offsets."""
    m = amd()
    g = 32
    rng = np.random.default_rng(M + N)
    W = Q4(ctx, rng, N, K, g, True, bias=rng.normal(0, 1, N).astype(np.float32))
    ldx, ldc, lda, goff = (K + 8, N + 3, N + 1, 5) if ragged else (K, N, N, 0)
    x = rng.normal(0, 1, (M, ldx)).astype(np.float32)
    before = rng.normal(0, 1, (M, ldc)).astype(np.float32)
    delta = rng.normal(0, 1, (M, lda)).astype(np.float32)
    gate = rng.normal(0, 1, N + 5).astype(np.float32)
    dx, dd, dg = ctx.upload(x), ctx.upload(delta), ctx.upload(gate)
    out = ctx.upload(bf16(before)) if out_bf16 else ctx.upload(before)
    ctx.linear(W.w, M, out, x=dx, ldx=ldx, ldc=ldc, act=act, epilogue=epi, gate=dg if epi == 2 else None, gate_off=goff, alpha=alpha,
               add=dd if add else None, ld_add=lda if add else 0, precision=m.PREC_FP32, out_bf16=out_bf16)
    xs = x[:, :K].astype(np.float64)
    r0 = (alpha or 1.0) * (xs @ W.values.T) + W.bias + (delta[:, :N] if add else 0.0)
    r = act64(r0, act)
    b = before[:, :N].astype(np.float64)
    ref = r if epi == 0 else b + r if epi == 1 else b + gate[goff: goff + N] * r
    got = widen(out.numpy()) if out_bf16 else out.numpy()
    tol = max(abs(alpha), 1.0) * bound(xs, W.values, K, m.PREC_FP32, out_bf16, ref, r0)
    tol += 4 * BIT_EPS * (np.abs(W.bias) + (np.abs(delta[:, :N]) if add else 0.0))
    if epi == 2:
        tol = tol * np.maximum(1.0, np.abs(gate[goff: goff + N])) + 4 * BIT_EPS * np.abs(b)
    if epi == 1:
        tol = tol + 4 * BIT_EPS * np.abs(b)
    err = np.abs(got[:, :N] - ref)
    assert np.all(err <= tol), (err / tol).max()
    if ldc > N:  # what lies between the rows stays
        np.testing.assert_array_equal(got[:, N:], widen(bf16(before))[:, N:] if out_bf16 else before[:, N:])


@pytest.mark.parametrize("M,N,K", [(1, 200, 512), (12, 200, 512), (80, 200, 512), (300, 520, 512), (12, 2700, 2048), (80, 900, 2048)])
@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("rows", ["tiny", "huge", "one", "zero", "mixed"])
def test_ranges_of_rows(ctx, M, N, K, g, rows):
    """Rows of any magnitude beside each other, scales of any magnitude beside each other: each result to the accuracy of
    its own row and column."""
    rng = np.random.default_rng(M + g)
    W = Q4(ctx, rng, N, K, g, True)
    f = {"tiny": 2.0 ** -100, "huge": 2.0 ** 100, "one": 1.0, "zero": 0.0}.get(rows)
    f = np.full((M, 1), f) if f is not None else 2.0 ** rng.integers(-60, 60, (M, 1))
    x = (rng.normal(0, 1, (M, K)) * f).astype(np.float32)
    scale = 2.0 ** rng.integers(-20, 20, (N, 1))  # columns of other magnitudes
    s, z = widen(W.bufs[1].numpy()) * scale.astype(np.float32), widen(W.bufs[2].numpy()) * scale.astype(np.float32)
    W.bufs[1].write(bf16(s))
    W.bufs[2].write(bf16(z))
    w = W.values * scale
    dx, out = ctx.upload(x), ctx.empty((M, N))
    ctx.linear(W.w, M, out, x=dx, precision=amd().PREC_FP32)
    ref = x.astype(np.float64) @ w.T
    err = np.abs(out.numpy() - ref)
    tol = bound(x.astype(np.float64), w, K, 1, False, ref, ref) + 2.0 ** -149
    assert np.all(err <= tol), (err / np.maximum(tol, 1e-300)).max()


@pytest.mark.parametrize("M,N,K", [(1, 70, 256), (12, 70, 256), (80, 200, 256), (300, 300, 256), (24, 2100, 1024), (80, 900, 1024)])
def test_outliers_and_small_scales(ctx, M, N, K):
    """One activation 10^4 times the rest, and groups whose scales are 2^20 apart within a column: the parts beside the large
    ones count with 2^-24 of the row's largest magnitude times the column's."""
    rng = np.random.default_rng(5)
    W = Q4(ctx, rng, N, K, 32, False)
    s = widen(W.bufs[1].numpy()) * (2.0 ** -rng.integers(0, 21, (N, K // 32))).astype(np.float32)
    W.bufs[1].write(bf16(s))
    codes = np.stack([W.bufs[0].numpy() & 15, W.bufs[0].numpy() >> 4], 2).reshape(N, K)
    w = values(codes, s, None, 32)
    x = rng.normal(0, 1, (M, K)).astype(np.float32)
    x[np.arange(M), rng.integers(0, K, M)] *= 1e4
    dx, out = ctx.upload(x), ctx.empty((M, N))
    ctx.linear(W.w, M, out, x=dx, precision=amd().PREC_FP32)
    ref = x.astype(np.float64) @ w.T
    tol = bound(x.astype(np.float64), w, K, 1, False, ref, ref)
    tol += K * 2.0 ** -24 * 2.0 ** -12 * np.abs(x).max(1)[:, None] * np.abs(w).max(1)[None, :]
    err = np.abs(out.numpy() - ref)
    assert np.all(err <= tol), (err / tol).max()


@pytest.mark.parametrize("M,N,K", [(1, 150, 192), (6, 150, 192), (40, 150, 192), (200, 150, 192), (24, 2100, 1024), (200, 900, 1024)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_rows_that_are_not_finite(ctx, M, N, K, bad):
    """A row of x with a NaN or an infinity gives NaN or infinities; no other row changes."""
    rng = np.random.default_rng(9)
    W = Q4(ctx, rng, N, K, 64, True)
    x = rng.normal(0, 1, (M, K)).astype(np.float32)
    out, dx = ctx.empty((M, N)), ctx.upload(x)
    ctx.linear(W.w, M, out, x=dx, precision=1)
    good = out.numpy()
    y = x.copy()
    y[M // 2, 70] = bad
    dx.write(y)
    ctx.linear(W.w, M, out, x=dx, precision=1)
    got = out.numpy()
    assert not np.isfinite(got[M // 2]).any()
    keep = np.arange(M) != M // 2
    np.testing.assert_array_equal(got[keep], good[keep])


@pytest.mark.parametrize("M,N,K", [(1, 260, 512), (5, 260, 512), (50, 260, 512), (300, 260, 512), (50, 2100, 1024), (17, 4100, 2048)])
def test_rows_do_not_depend_on_their_neighbours(ctx, M, N, K):
    """The same row twice in a batch gives the same bits, and a batch gives the same bits twice."""
    rng = np.random.default_rng(4)
    W = Q4(ctx, rng, N, K, 64, True)
    x = rng.normal(0, 1, (M, K)).astype(np.float32)
    x[-1] = x[0]
    out, dx = ctx.empty((M, N)), ctx.upload(x)
    ctx.linear(W.w, M, out, x=dx, precision=1)
    a = out.numpy()
    np.testing.assert_array_equal(a[0], a[-1])
    ctx.linear(W.w, M, out, x=dx, precision=1)
    np.testing.assert_array_equal(a, out.numpy())


def test_no_rows(ctx):
    W = Q4(ctx, np.random.default_rng(0), 8, 32, 32, False)
    out = ctx.upload(np.full(8, 7.0, np.float32))
    ctx.linear(W.w, 0, out, x=out)
    assert (out.numpy() == 7.0).all()


@pytest.mark.parametrize("M,N,K", [(1, 384, 1024), (24, 384, 1024), (160, 384, 1024), (300, 384, 1024), (24, 2100, 1024), (200, 300, 4096)])
def test_replayed_from_a_graph(ctx, M, N, K):
    """A captured product, replayed several times with other work and other inputs between the replays."""
    rng = np.random.default_rng(2)
    W = Q4(ctx, rng, N, K, 64, True)
    xs = [rng.normal(0, 1, (M, K)).astype(np.float32) for _ in range(3)]
    dx, out, other = ctx.upload(xs[0]), ctx.empty((M, N)), ctx.empty((M, N))
    ctx.linear(W.w, M, out, x=dx)
    ctx.sync()
    ctx.graph_begin()
    ctx.linear(W.w, M, out, x=dx)
    g = ctx.graph_end()
    try:
        for x in xs:
            dx.write(x)
            ctx.linear(W.w, M, other, x=dx)
            ref = other.numpy()
            ctx.graph_launch(g)
            np.testing.assert_array_equal(out.numpy(), ref)
    finally:
        ctx.graph_destroy(g)


# ---------------------------------------------------------------- conversion


def quant_ref(w, g, mid):
    """The conversion's definition, in fp32."""
    N, K = w.shape
    v = w.reshape(N, K // g, g)
    lo, hi = v.min(2), v.max(2)
    f = np.float32
    if mid:
        s = widen(bf16((hi - lo) / f(15)))
        z = widen(bf16((s.astype(np.float64) * 8 + lo).astype(np.float32)))  # (exact in 64 bits: rounded once)
    else:
        s, z = widen(bf16(np.maximum(-lo, hi) / f(7))), np.zeros_like(lo)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.rint((v - z[:, :, None]) / s[:, :, None])
    c = np.where(s[:, :, None] == 0, 0, np.clip(c, -8, 7))
    return (c + 8).astype(np.uint8).reshape(N, K), bf16(s), bf16(z)


@pytest.mark.parametrize("mid", [False, True], ids=["sym", "mid"])
@pytest.mark.parametrize("is_bf16", [True, False], ids=["bf16", "f32"])
@pytest.mark.parametrize("N,K,g", [(1, 32, 32), (3, 64, 64), (70, 1152, 128), (33, 2048, 64), (5, 96, 32)])
def test_conversion(ctx, N, K, g, is_bf16, mid):
    rng = np.random.default_rng(N + K)
    w = (rng.normal(0.01, 0.05, (N, K)) * np.exp(rng.normal(0, 1, (N, 1)))).astype(np.float32)
    w[0, :g] = 0.0
    w[-1, -g:] = 0.625
    if N > 2:
        w[1] *= np.float32(2.0 ** -60)
        w[2] = np.abs(w[2])
    if is_bf16:
        w = widen(bf16(w))
    dw = ctx.upload(bf16(w)) if is_bf16 else ctx.upload(w)
    q, s, z = ctx.empty((N, K // 2), np.uint8), ctx.empty((N, K // g), np.uint16), ctx.empty((N, K // g), np.uint16)
    ctx.weight_quant_q4(dw, N, K, g, q, s, z if mid else None, bf16=is_bf16)
    c, rs, rz = quant_ref(w, g, mid)
    np.testing.assert_array_equal(s.numpy(), rs)
    if mid:
        np.testing.assert_array_equal(widen(z.numpy()), widen(rz))
    np.testing.assert_array_equal(q.numpy(), pack(c))
    # a weight is off by half a step and what the clamp and the roundings of s and z (2^-8 each) take
    step = np.repeat(widen(rs), g, 1).astype(np.float64)
    got = values(c, widen(rs), widen(rz) if mid else None, g)
    zz = np.repeat(np.abs(widen(rz)), g, 1)
    assert np.all(np.abs(got - w) <= 0.5 * step + 2.0 ** -8 * (8 * step + zz) + 2.0 ** -8 * np.abs(w) * (step == 0) + 1e-45)


def test_conversion_of_what_is_not_finite(ctx):
    """A NaN or an infinity stays in its group."""
    w = np.random.default_rng(1).normal(0, 1, (4, 128)).astype(np.float32)
    ref, rs, _ = quant_ref(w, 32, False)
    w[1, 40], w[2, 5] = np.nan, np.inf
    q, s = ctx.empty((4, 64), np.uint8), ctx.empty((4, 4), np.uint16)
    ctx.weight_quant_q4(ctx.upload(w), 4, 128, 32, q, s, bf16=False)
    got, gs = q.numpy().reshape(4, 4, 16), s.numpy()
    keep = np.ones((4, 4), bool)
    keep[1, 1] = keep[2, 0] = False
    np.testing.assert_array_equal(gs[keep], rs[keep])
    np.testing.assert_array_equal(got[keep], pack(ref).reshape(4, 4, 16)[keep])
    assert np.isnan(widen(gs)[1, 1]) and not np.isfinite(widen(gs)[2, 0])


# ---------------------------------------------------------------- embedding rows


@pytest.mark.parametrize("kind", ["f32", "bf16", "q4", "q4mid"])
@pytest.mark.parametrize("T,N,K,ldo", [(1, 1, 32, 0), (1, 3000, 1024, 0), (5, 7, 96, 100), (300, 1000, 160, 160), (4099, 50, 2048, 0),
                                       (70, 64, 2080, 2084)])
@pytest.mark.parametrize("weights,scale", [(False, 0.0), (True, 0.0), (True, 32.0), (False, 0.5)])
def test_embed_rows(ctx, kind, T, N, K, ldo, weights, scale):
    """Bit for bit: a row's value times the rounded product of scale and weight, rounded once; padding rows are zeros, and
    what lies between the rows stays."""
    m = amd()
    rng = np.random.default_rng(T + K)
    if kind.startswith("q4"):
        W = Q4(ctx, rng, N, K, 32, kind == "q4mid")
        table, v = W.w, W.values.astype(np.float32)
    else:
        v = rng.normal(0, 1, (N, K)).astype(np.float32)
        if kind == "bf16":
            v = widen(bf16(v))
        W = ctx.upload(bf16(v) if kind == "bf16" else v)
        table = m.weight(m.W_BF16 if kind == "bf16" else m.W_F32, N, K, W)
    ids = rng.integers(0, N, T).astype(np.int32)
    ids[rng.random(T) < 0.2] = -1
    if T > 3:
        ids[:4] = [N, -(1 << 31), (1 << 31) - 1, N - 1]
    f = rng.choice([0.0, 1.0, 1.1, -0.7], T).astype(np.float32)
    ld = ldo or K
    out = ctx.upload(np.full((T, ld), 9.0, np.float32))
    ctx.embed_rows(table, ctx.upload(ids), T, out, weights=ctx.upload(f) if weights else None, scale=scale, ldo=ldo)
    fac = (np.float32(scale or 1.0) * (f if weights else np.ones(T, np.float32))).astype(np.float32)
    inside = (ids >= 0) & (ids < N)
    ref = np.where(inside[:, None], v[np.where(inside, ids, 0)] * fac[:, None], np.float32(0))
    got = out.numpy()
    np.testing.assert_array_equal(got[:, :K], ref)
    assert (got[:, K:] == 9.0).all()


def test_embed_replayed_from_a_graph(ctx):
    """The indexes are read as they are when the replay runs."""
    m = amd()
    v = np.random.default_rng(0).normal(0, 1, (10, 64)).astype(np.float32)
    dv, ids, out = ctx.upload(v), ctx.upload(np.zeros(5, np.int32)), ctx.empty((5, 64))
    table = m.weight(m.W_F32, 10, 64, dv)
    ctx.graph_begin()
    ctx.embed_rows(table, ids, 5, out)
    g = ctx.graph_end()
    try:
        for i in ([1, 2, 3, -1, 0], [9, 9, 9, 9, 9], [4, 10, 5, 6, 7]):
            ids.write(np.asarray(i, np.int32))
            ctx.graph_launch(g)
            ref = np.stack([v[j] if 0 <= j < 10 else 0 * v[0] for j in i])
            np.testing.assert_array_equal(out.numpy(), ref)
    finally:
        ctx.graph_destroy(g)


def test_large_table(ctx):
    """Rows whose elements lie past 2^31, and past 2^32 bytes."""
    m = amd()
    N, K = 1 << 20, 2080  # 4.4 GB in bf16
    dw = ctx.empty((N * K,), np.uint16)
    ctx.fill_random(dw, N * K, "bf16", 7, -1.0, 1.0)
    ids = np.asarray([N - 1, N // 2 + 1, 0, N - 2], np.int32)
    out = ctx.empty((4, K))
    ctx.embed_rows(m.weight(m.W_BF16, N, K, dw), ctx.upload(ids), 4, out)
    got = out.numpy()
    row = np.empty(K, np.uint16)
    for t, i in enumerate(ids):
        m.lib().anima_d2h(ctx.h, row.ctypes.data, dw.ptr + int(i) * K * 2, row.nbytes)
        np.testing.assert_array_equal(got[t], widen(row))
    dw.release()
    ctx.trim()


def test_names(ctx):
    """The profiler names of the operators."""
    W = Q4(ctx, np.random.default_rng(0), 64, 64, 32, False)
    x, out, ids = ctx.upload(np.ones((1, 64), np.float32)), ctx.empty((1, 64)), ctx.upload(np.zeros(1, np.int32))
    assert ran(ctx, lambda: ctx.linear(W.w, 1, out, x=x)) == {"gemv.q4"}
    assert ran(ctx, lambda: ctx.embed_rows(W.w, ids, 1, out)) == {"embed_rows"}
