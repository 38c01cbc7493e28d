"""The e4m3 operators through the C ABI against 64-bit references.

Quantization is defined step by step in 32 bits, so its bytes and scales are compared for equality.  Products
are compared with 64-bit sums of the same e4m3 values.  With A = sum of the magnitudes of an output's terms, an
fp32 sum of 128 products per block and ceil(K / 128) blocks, in any order and in up to 16 partial sums, is off by
at most (128 + blocks + 16) 2^-24 A when every addition rounds to nearest, twice that when the matrix core
truncates; the epilogue's bias, factor and addition add one rounding (2^-24) each.  With precision "bf16" the 8-bit
matrix instructions drop, of each of eight products but the largest, what lies 2^-13 below the largest: at most
7 * 2^-13 of the largest, so 7 * 2^-13 A more; and as the dropped parts have either sign, in the 2-norm 1e-4 (seven
parts uniform up to 2^-13 of a largest product of about twice the mean square: 2^-13 * 2 * sqrt(7 / 12 / 8) = 6.6e-5).
Norms are compared with
64-bit norms: sums of squares are off by at most 2^-24 (log2 of the row's threads + terms per thread <= 41) of
themselves, and every other step rounds once.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

import oracle as orc
from helpers import amd, ran

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = np.float32(2.0 ** -100)


@pytest.fixture(scope="module")
def ctx():
    c = amd().Context(0)
    yield c
    c.close()


def randn(seed, n):
    """The oracle's normal values; it fills 16 and more."""
    return orc.randn(seed, max(n, 16))[:n]


def case(msg):
    print(f"[case] {msg}", flush=True)


# ------------------------------------------------------------------ references


def to_e4m3(x):
    """fp32 -> e4m3 bytes, round to nearest even."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def from_e4m3(q):
    return torch.from_numpy(np.ascontiguousarray(q)).view(torch.float8_e4m3fn).to(torch.float64).numpy()


def bf16(x):
    """fp32 -> (bf16 bits, their values)."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16)
    return t.view(torch.uint16).numpy(), t.float().numpy()


def quant_ref(x):
    """The definition: fp32 rows -> (bytes, scales [blocks][rows])."""
    x = np.asarray(x, np.float32)
    M, K = x.shape
    KB = -(-K // 128)
    q, s = np.zeros((M, K), np.uint8), np.zeros((KB, M), np.float32)
    with np.errstate(all="ignore"):
        for b in range(KB):
            v = x[:, 128 * b:128 * b + 128]
            a = np.maximum(np.abs(v).max(1), TINY)  # (a NaN stays)
            s[b] = a / np.float32(448)
            q[:, 128 * b:128 * b + 128] = to_e4m3(v * (np.float32(448) * (np.float32(1) / a))[:, None])
    return q, s


def rows64(q, s):
    return from_e4m3(q) * np.repeat(s.T.astype(np.float64), 128, 1)[:, :q.shape[1]]


def weight64(w, scale):
    N, K = w.shape
    return from_e4m3(w) * np.repeat(np.repeat(scale.astype(np.float64), 128, 0)[:N], 128, 1)[:, :K]


def random_e4m3(seed, n, k):
    return to_e4m3(np.clip(110 * randn(seed, n * k).reshape(n, k), -448, 448))


def f8_weight(seed, N, K, gain=1.0):
    rng = np.random.default_rng(seed)
    scale = (rng.uniform(0.5, 1.5, (-(-N // 128), -(-K // 128))) * gain / (110 * math.sqrt(K))).astype(np.float32)
    return random_e4m3(seed, N, K), scale


def act64(x, act):
    if act == "gelu":
        return 0.5 * x * (1 + torch.erf(torch.from_numpy(x / math.sqrt(2))).numpy())
    return x / (1 + np.exp(-x)) if act == "silu" else x


def act_error(x, act, dx):
    """Bound of an activation's error for an input off by dx: slopes below 1.13, and the functions' own errors:
    gelu's error function within 1.6e-7, silu's exponential and quotient within 4 roundings."""
    if act == "none":
        return dx
    own = 1.6e-7 * np.abs(x) if act == "gelu" else 4 * U * np.abs(act64(x, act))
    return 1.13 * dx + own + 2 * U * np.abs(act64(x, act))


def product64(x64, w64, fast=True):
    """(sums, bound of the kernel's error); fast: precision "bf16"."""
    K = x64.shape[1]
    c = 2 * (128 + -(-K // 128) + 16) * U + (7 * 2.0 ** -13 if fast else 0.0)
    return x64 @ w64.T, c * (np.abs(x64) @ np.abs(w64).T)


def near(got, ref):
    """The 2-norm bar of the 8-bit matrix instructions' sums."""
    return np.linalg.norm(got - ref) <= 1e-4 * np.linalg.norm(ref)


class Guarded:
    """A device buffer of `shape` with 1 KiB of a pattern behind it that must survive."""

    def __init__(self, ctx, shape, dtype, init=None):
        self.shape, self.dtype, self.ctx = shape, np.dtype(dtype), ctx
        self.n = int(np.prod(shape)) * self.dtype.itemsize
        host = np.full(self.n + 1024, 0xA5, np.uint8)
        if init is not None:
            host[:self.n] = np.ascontiguousarray(init).view(np.uint8).reshape(-1)
        self.buf = ctx.upload(host)
        self.ptr = self.buf.ptr

    def numpy(self):
        host = self.buf.numpy()
        assert np.all(host[self.n:] == 0xA5), "written past the end"
        return host[:self.n].view(self.dtype).reshape(self.shape).copy()


# ------------------------------------------------------------------ rows and weights to e4m3


def special_rows(seed, M, K):
    """Rows over many magnitudes; some zero, tiny, huge, or with one outlier."""
    x = randn(seed, M * K).reshape(M, K).astype(np.float32)
    x *= np.float32(2.0) ** np.random.default_rng(seed).integers(-20, 20, (M, 1)).astype(np.float32)
    x[0] = 0
    if M > 4:
        x[1] *= np.float32(1e-36)
        x[2] *= np.float32(1e30)
        x[3, K // 2] = 1e6
        x[4, :] = np.float32(1e-42)  # below 2^-100: zero at the smallest scale
    return x


@pytest.mark.parametrize("M,K,ldx", [(1, 16, 0), (1, 128, 0), (7, 144, 0), (43, 2048, 4096), (129, 1008, 1020), (300, 8192, 0),
                                     (2, 16400, 0), (4099, 64, 64)])
@pytest.mark.parametrize("wide", [False, True])
def test_quant_rows(ctx, M, K, ldx, wide):
    case(f"quant_rows_f8 M={M} K={K} ldx={ldx} bf16={wide}")
    ld = ldx or K
    if wide and ld % 8:
        ld += 4
    x = special_rows(M + K, M, ld)
    bits, vals = bf16(x) if wide else (x, x)
    q, s = Guarded(ctx, (M, K), np.uint8), Guarded(ctx, (-(-K // 128), M), np.float32)
    ctx.quant_rows_f8(ctx.upload(bits), M, K, q.ptr, s.ptr, ldx=ld if ld != K else ldx, bf16=wide)
    rq, rs = quant_ref(vals[:, :K])
    gq, gs = q.numpy(), s.numpy()
    assert np.array_equal(gs, rs)
    assert np.array_equal(gq, rq)
    # what the rows stand for: half a step of 3 mantissa bits, or of the smallest step
    bound = np.maximum(2.0 ** -4 * np.abs(vals[:, :K]), 2.0 ** -10 * np.repeat(rs.T, 128, 1)[:, :K]).astype(np.float64)
    assert np.all(np.abs(rows64(gq, gs) - vals[:, :K]) <= bound * (1 + 4 * U) + 2.0 ** -149)


def test_quant_rows_not_finite(ctx):
    case("quant_rows_f8 with NaN and infinities")
    x = special_rows(9, 6, 384)
    x[0, 5], x[1, 130], x[2, 300], x[3, 383] = np.nan, np.inf, -np.inf, -np.nan
    q, s = Guarded(ctx, (6, 384), np.uint8), Guarded(ctx, (3, 6), np.float32)
    ctx.quant_rows_f8(ctx.upload(x), 6, 384, q.ptr, s.ptr)
    rq, rs = quant_ref(x)
    gq, gs = q.numpy(), s.numpy()
    assert np.array_equal(gs, rs, equal_nan=True)
    g, r = from_e4m3(gq), from_e4m3(rq)
    assert np.array_equal(g, r, equal_nan=True)
    assert np.all(np.isnan(g[0, :128])) and np.isfinite(g[0, 128:]).all()
    assert np.isinf(gs[1, 1]) and np.isnan(g[1, 130]) and np.all(g[1, 131:256] == 0)


@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (130, 144), (500, 1008), (1024, 2048)])
@pytest.mark.parametrize("wide", [False, True])
def test_weight_quant(ctx, N, K, wide):
    case(f"weight_quant_f8 N={N} K={K} bf16={wide}")
    w = special_rows(N + 3, N, K)
    bits, vals = bf16(w) if wide else (w, w)
    q, s = Guarded(ctx, (N, K), np.uint8), Guarded(ctx, (-(-N // 128), -(-K // 128)), np.float32)
    ctx.weight_quant_f8(ctx.upload(bits), N, K, q.ptr, s.ptr, bf16=wide)
    gq, gs = q.numpy(), s.numpy()
    for i in range(gs.shape[0]):
        for j in range(gs.shape[1]):
            v = vals[128 * i:128 * i + 128, 128 * j:128 * j + 128]
            a = max(np.abs(v).max(), TINY)
            assert gs[i, j] == a / np.float32(448)
            assert np.array_equal(gq[128 * i:128 * i + 128, 128 * j:128 * j + 128], to_e4m3(v * (np.float32(448) * (np.float32(1) / a))))


# ------------------------------------------------------------------ products


def inputs(ctx, seed, M, K, kind, ld=0):
    """(keyword arguments of the call, the 64-bit values of the rows it multiplies)."""
    if kind == "f32":
        x = (randn(seed, M * (ld or K)) * 2).astype(np.float32).reshape(M, ld or K)
        return dict(x=ctx.upload(x), ldx=ld), rows64(*quant_ref(x[:, :K]))
    q = random_e4m3(seed, M, ld or K)
    s = np.random.default_rng(seed).uniform(0.5, 1.5, (-(-K // 128), M)).astype(np.float32) / 100
    return dict(xq=ctx.upload(q), xs=ctx.upload(s), ldx=ld), rows64(q[:, :K], s)


LINEAR = [(1, 64, 16), (1, 4096, 1024), (2, 33, 48), (5, 130, 144), (16, 128, 128), (17, 257, 272), (43, 1024, 2048), (63, 1000, 3088),
          (64, 512, 128), (65, 640, 1152), (130, 260, 2064), (200, 4100, 512), (300, 384, 4096), (517, 1316, 1424), (1025, 516, 256),
          (2300, 2052, 144)]


@pytest.mark.parametrize("M,N,K", LINEAR)
@pytest.mark.parametrize("kind", ["f8", "f32"])
@pytest.mark.parametrize("epi,act,fast", [("store", "none", True), ("store", "none", False), ("resid", "gelu", False),
                                          ("gated", "silu", True)])
def test_linear(ctx, M, N, K, kind, epi, act, fast):
    case(f"linear f8 M={M} N={N} K={K} x={kind} {epi} {act} fast={fast}")
    m = amd()
    w, scale = f8_weight(N + K, N, K)
    args, x64 = inputs(ctx, M + K, M, K, kind)
    bias = randn(5, N).astype(np.float32)
    gate = randn(6, N + 8).astype(np.float32)
    out0 = randn(7, M * N).reshape(M, N).astype(np.float32)
    W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale), bias=ctx.upload(bias))
    out = Guarded(ctx, (M, N), np.float32, out0)
    ctx.linear(W, M, out.ptr, act=act, alpha=0.75, epilogue=dict(store=m.EPI_STORE, resid=m.EPI_RESID, gated=m.EPI_GATED)[epi],
               gate=ctx.upload(gate), gate_off=8, precision=m.PREC_BF16 if fast else m.PREC_FP32, **args)
    y, dy = product64(x64, weight64(w, scale), fast)
    v = 0.75 * y + bias
    dv = 0.75 * dy + 3 * U * (np.abs(0.75 * y) + np.abs(bias))
    r, dr = act64(v, act), act_error(v, act, dv)
    if epi == "gated":
        r, dr = r * gate[8:], (dr + U * np.abs(r)) * np.abs(gate[8:])
    ref = r if epi == "store" else out0 + r
    got = out.numpy().astype(np.float64)
    assert np.all(np.abs(got - ref) <= dr + 2 * U * (np.abs(r) + np.abs(ref)))
    if epi == "store":
        assert near(got, ref)
        # bf16 rows, into wider rows: half a step of 8 significant bits more
        ldc = N + (4 if N % 4 == 0 else 3)
        out = Guarded(ctx, (M, ldc), np.uint16, np.full((M, ldc), 0x3F80, np.uint16))
        ctx.linear(W, M, out.ptr, act=act, alpha=0.75, ldc=ldc, out_bf16=True, precision=m.PREC_BF16 if fast else m.PREC_FP32, **args)
        bits = out.numpy()
        gb = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).double().numpy()[:, :N]
        assert np.all(np.abs(gb - ref) <= (dr + 2 * U * np.abs(ref)) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(ref))
        assert np.all(bits[:, N:] == 0x3F80)


@pytest.mark.parametrize("M,N,K", [(3, 70, 160), (50, 96, 1040), (190, 300, 528), (700, 1030, 400)])
@pytest.mark.parametrize("kind", ["f8", "f32"])
def test_linear_strides_and_alignment(ctx, M, N, K, kind):
    """Rows of x inside wider rows, out inside wider rows that start off 16 bytes, an added term; columns beside
    the output keep their values."""
    case(f"linear f8 strides M={M} N={N} K={K} x={kind}")
    m = amd()
    w, scale = f8_weight(N, N, K)
    args, x64 = inputs(ctx, M, M, K, kind, ld=K + 32)
    ldc, ld_add = N + 5, N + 3
    out0 = randn(8, M * ldc + 1).astype(np.float32)
    add = randn(9, M * ld_add).reshape(M, ld_add).astype(np.float32)
    W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale))
    out = Guarded(ctx, (M * ldc + 1,), np.float32, out0)
    ctx.linear(W, M, out.ptr + 4, ldc=ldc, add=ctx.upload(add), ld_add=ld_add, **args)
    y, dy = product64(x64, weight64(w, scale))
    flat = out.numpy()
    got = flat[1:].reshape(M, ldc)
    ref = y + add[:, :N]
    assert np.all(np.abs(got[:, :N] - ref) <= dy + 2 * U * (np.abs(y) + np.abs(ref)))
    assert flat[0] == out0[0] and np.array_equal(got[:, N:], out0[1:].reshape(M, ldc)[:, N:])


@pytest.mark.parametrize("M,N,K", [(6, 96, 400), (40, 300, 1168), (150, 130, 272), (600, 512, 384)])
def test_linear_not_finite(ctx, M, N, K):
    """A row with a NaN gives NaN in that row alone; bytes past a row's K columns are never multiplied."""
    case(f"linear f8 NaN rows M={M} N={N} K={K}")
    m = amd()
    w, scale = f8_weight(N, N, K)
    W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale))
    x = randn(3, M * (K + 16)).reshape(M, K + 16).astype(np.float32)
    x[:, K:] = np.nan  # past the row
    x[M // 2, K - 1] = np.nan
    x[1, 0] = np.inf
    bad = np.zeros(M, bool)
    bad[[1, M // 2]] = True
    out = Guarded(ctx, (M, N), np.float32)
    ctx.linear(W, M, out.ptr, x=ctx.upload(x), ldx=K + 16)
    got = out.numpy()
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    q = random_e4m3(4, M, K + 16)
    q[:, K:] = 0x7F  # NaN past the row
    q[M // 2, 0] = 0xFF
    bad = np.zeros(M, bool)
    bad[M // 2] = True
    s = np.full((-(-K // 128), M), 0.01, np.float32)
    out = Guarded(ctx, (M, N), np.float32)
    ctx.linear(W, M, out.ptr, xq=ctx.upload(q), xs=ctx.upload(s), ldx=K + 16)
    got = out.numpy()
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


def test_linear_far_offsets(ctx):
    """A weight of more than 2^31 bytes and an output of more than 2^31 values."""
    m = amd()
    L = m.lib()
    N, K, M = 270000, 8192, 2
    case(f"linear f8 far weight N={N} K={K}")
    w = ctx.empty((N, K), np.uint8)
    ctx.fill_random(w, N * K, "u8", 11, 0, 0x6F)
    scale = ctx.empty((-(-N // 128), K // 128))
    ctx.fill_random(scale, scale.shape[0] * scale.shape[1], "f32", 12, 1e-4, 2e-4)
    args, x64 = inputs(ctx, 13, M, K, "f8")
    out = ctx.empty((M, N))
    ctx.linear(m.weight(m.W_F8, N, K, w, scale=scale), M, out, **args)
    got, sc = out.numpy(), scale.numpy()
    for n in (0, 127, 128, 131071, 262143, 262144, N - 1):
        row = np.empty((1, K), np.uint8)
        ctx._check(L.anima_d2h(ctx.h, row.ctypes.data, w.ptr + n * K, K))
        y, dy = product64(x64, from_e4m3(row) * np.repeat(sc[n // 128].astype(np.float64), 128))
        assert np.all(np.abs(got[:, n] - y[:, 0]) <= dy[:, 0] + U * np.abs(y[:, 0])), n
    for b in (w, scale, out):
        b.release()
    M, N, K = 70000, 32768, 16
    case(f"linear f8 far output M={M} N={N}")
    w, sc = f8_weight(14, N, K)
    q = random_e4m3(15, M, K)
    s = np.full((1, M), 0.01, np.float32)
    out = ctx.empty((M, N))
    ctx.linear(m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(sc)), M, out, xq=ctx.upload(q), xs=ctx.upload(s))
    for r in (0, 255, 65535, 65536, M - 1):
        row = np.empty(N, np.float32)
        ctx._check(L.anima_d2h(ctx.h, row.ctypes.data, out.ptr + r * N * 4, N * 4))
        y, dy = product64(rows64(q[r:r + 1], s[:, r:r + 1]), weight64(w, sc))
        assert np.all(np.abs(row - y[0]) <= dy[0] + U * np.abs(y[0])), r
    out.release()


# ------------------------------------------------------------------ gated feed-forward half


def check_f8_rows(got_q, got_s, h, dh):
    """e4m3 rows of values h known to dh: the scale is the largest magnitude's, every value is within half a
    step (2^-4 of it, 2^-10 of the scale) of a value within dh."""
    M, N = h.shape
    for b in range(got_s.shape[0]):
        v, d = np.abs(h[:, 128 * b:128 * b + 128]), dh[:, 128 * b:128 * b + 128]
        a = np.maximum(v.max(1), float(TINY))
        assert np.all(np.abs(got_s[b] * 448.0 - a) <= d.max(1) + 4 * U * a)
    s = np.repeat(got_s.T.astype(np.float64), 128, 1)[:, :N]
    err = np.abs(from_e4m3(got_q) * s - h)
    assert np.all(err <= dh + np.maximum(2.0 ** -4 * (np.abs(h) + dh), 2.0 ** -10 * s) * (1 + 8 * U))


GLU = [(1, 64, 16), (1, 4096, 1024), (3, 40, 176), (16, 272, 128), (33, 144, 1040), (64, 512, 256), (100, 1024, 384), (128, 128, 2048),
       (257, 272, 400), (512, 1040, 1024), (1030, 400, 144), (2100, 1296, 256)]


@pytest.mark.parametrize("M,F,K", GLU)
@pytest.mark.parametrize("kind,act,bias,fast", [("f8", "silu", False, True), ("f32", "gelu", True, False), ("f8", "none", True, True),
                                                ("f8", "silu", False, False)])
def test_glu(ctx, M, F, K, kind, act, bias, fast):
    case(f"linear_glu M={M} F={F} K={K} x={kind} {act} bias={bias} fast={fast}")
    m = amd()
    prec = m.PREC_BF16 if fast else m.PREC_FP32
    (wg, sg), (wu, su) = f8_weight(F, F, K), f8_weight(F + 1, F, K)
    args, x64 = inputs(ctx, M + 1, M, K, kind)
    bg, bu = randn(21, F).astype(np.float32), randn(22, F).astype(np.float32)
    G = m.weight(m.W_F8, F, K, ctx.upload(wg), scale=ctx.upload(sg), bias=ctx.upload(bg) if bias else None)
    Up = m.weight(m.W_F8, F, K, ctx.upload(wu), scale=ctx.upload(su), bias=ctx.upload(bu) if bias else None)
    g, dg = product64(x64, weight64(wg, sg), fast)
    u, du = product64(x64, weight64(wu, su), fast)
    if bias:
        g, u = g + bg, u + bu
    dg, du = dg + U * np.abs(g), du + U * np.abs(u)
    a, da = act64(g, act), act_error(g, act, dg)
    h = a * u
    dh = da * (np.abs(u) + du) + np.abs(a) * du + 2 * U * np.abs(h)
    out = Guarded(ctx, (M, F), np.float32)
    ctx.linear_glu(G, Up, M, act=act, out=out.ptr, precision=prec, **args)
    got = out.numpy()
    assert np.all(np.abs(got - h) <= dh) and np.linalg.norm(got - h) <= 4e-4 * np.linalg.norm(h)
    if F % 16 == 0:
        q, s = Guarded(ctx, (M, F), np.uint8), Guarded(ctx, (-(-F // 128), M), np.float32)
        ctx.linear_glu(G, Up, M, act=act, out_q=q.ptr, out_s=s.ptr, precision=prec, **args)
        check_f8_rows(q.numpy(), s.numpy(), h, dh)


@pytest.mark.parametrize("M,F,K", [(2, 30, 144), (80, 70, 272), (300, 390, 160)])
def test_glu_strides(ctx, M, F, K):
    """Gate and up as halves of one stacked matrix, odd widths, an output inside wider rows off 16 bytes."""
    case(f"linear_glu strides M={M} F={F} K={K}")
    m = amd()
    (wg, sg), (wu, su) = f8_weight(F, F, K), f8_weight(F + 1, F, K)
    stack, scales = ctx.upload(np.concatenate([wg, wu])), ctx.upload(np.concatenate([sg, su]))
    G = m.weight(m.W_F8, F, K, stack.ptr, scale=scales.ptr)
    Up = m.weight(m.W_F8, F, K, stack.ptr + F * K, scale=scales.ptr + 4 * sg.size)
    args, x64 = inputs(ctx, M + 1, M, K, "f8", ld=K + 16)
    ldc = F + 7
    out0 = randn(23, M * ldc + 3).astype(np.float32)
    out = Guarded(ctx, (M * ldc + 3,), np.float32, out0)
    ctx.linear_glu(G, Up, M, out=out.ptr + 12, ldc=ldc, **args)
    g, dg = product64(x64, weight64(wg, sg))
    u, du = product64(x64, weight64(wu, su))
    a, da = act64(g, "silu"), act_error(g, "silu", dg)
    got = out.numpy()[3:].reshape(M, ldc)
    assert np.all(np.abs(got[:, :F] - a * u) <= da * (np.abs(u) + du) + np.abs(a) * du + 2 * U * np.abs(a * u))
    assert np.array_equal(got[:, F:], out0[3:].reshape(M, ldc)[:, F:])


def test_glu_not_finite(ctx):
    case("linear_glu e4m3 rows with a NaN row")
    m = amd()
    for M in (5, 300):
        F, K = 256, 256
        (wg, sg), (wu, su) = f8_weight(1, F, K), f8_weight(2, F, K)
        G = m.weight(m.W_F8, F, K, ctx.upload(wg), scale=ctx.upload(sg))
        Up = m.weight(m.W_F8, F, K, ctx.upload(wu), scale=ctx.upload(su))
        x = randn(3, M * K).reshape(M, K).astype(np.float32)
        x[3, 7] = np.nan
        q, s = Guarded(ctx, (M, F), np.uint8), Guarded(ctx, (2, M), np.float32)
        ctx.linear_glu(G, Up, M, x=ctx.upload(x), out_q=q.ptr, out_s=s.ptr)
        v, sv = from_e4m3(q.numpy()), s.numpy()
        assert np.isnan(v[3]).all() and np.isnan(sv[:, 3]).all()
        assert np.isfinite(np.delete(v, 3, 0)).all() and np.isfinite(np.delete(sv, 3, 1)).all()


# ------------------------------------------------------------------ residual + norm


NORM = [(1, 4), (1, 1024), (3, 60), (5, 256), (7, 272), (9, 520), (200, 1040), (64, 2048), (33, 2064), (40, 4096), (6, 8192), (5, 8208), (3, 16384)]


@pytest.mark.parametrize("rows,C", NORM)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("parts", ["y", "", "y post gate w mod", "w", "y bf16 post", "y gate mod bf16"])
def test_residual_norm(ctx, rows, C, norm, parts):
    case(f"residual_norm rows={rows} C={C} {norm} [{parts}]")
    parts = parts.split()
    per = max(1, -(-rows // 3))
    groups, ldx, ldy, ldh, ldm = -(-rows // per), C + 8, C + 4, C + 12, 3 * C
    x0 = (randn(31, rows * ldx).reshape(rows, ldx) * 3 + 0.5).astype(np.float32)
    if rows > 2:
        x0[1] = 0
    y = randn(32, rows * ldy).reshape(rows, ldy).astype(np.float32)
    if rows > 2:
        y[1] = 0
    mod = randn(33, groups * ldm).reshape(groups, ldm).astype(np.float32)
    vec = (1 + 0.2 * randn(34, 2 * C).reshape(2, C)).astype(np.float32)
    d_mod, d_vec = ctx.upload(mod), ctx.upload(vec)
    eps, rs = 1e-5, 0.625
    kw = dict(norm=norm, eps=eps, res_scale=rs, ldx=ldx, group_rows=per, mod_ld=ldm, gate_ld=ldm)
    x64, dx = x0[:, :C].astype(np.float64), np.zeros((rows, C))
    g64 = np.repeat(mod.astype(np.float64), per, 0)[:rows]
    if "y" in parts:
        bits, vals = bf16(y)
        wide = "bf16" in parts
        kw.update(y=ctx.upload(bits if wide else y), ldy=ldy, y_bf16=wide)
        y = vals if wide else y
        y64 = y[:, :C].astype(np.float64)
        dy = np.zeros_like(y64)
        if "post" in parts:
            kw.update(post_w=d_vec.ptr)
            y64 = y64 / np.sqrt((y64 ** 2).mean(1, keepdims=True) + eps) * vec[0]
            dy = 24 * U * np.abs(y64)
        if "gate" in parts:
            kw.update(gate=d_mod.ptr + 8 * C)
            y64, dy = y64 * g64[:, 2 * C:], (dy + U * np.abs(y64)) * np.abs(g64[:, 2 * C:])
        x64 = x64 + rs * y64
        dx = rs * dy + U * np.abs(x64) + U * np.abs(y64)
    xg = Guarded(ctx, (rows, ldx), np.float32, x0)
    h, q = Guarded(ctx, (rows, ldh), np.float32), Guarded(ctx, (rows, C), np.uint8)
    s = Guarded(ctx, (-(-C // 128), rows), np.float32)
    if "w" in parts:
        kw.update(norm_w=d_vec.ptr + 4 * C)
    if "mod" in parts:
        kw.update(shift=d_mod.ptr, scale=d_mod.ptr + 4 * C)
    f8 = dict(q=q.ptr, s=s.ptr) if C % 16 == 0 else {}
    ctx.residual_norm(rows, C, xg.ptr, h=h.ptr, ldh=ldh, **f8, **kw)
    got_x, got_h = xg.numpy(), h.numpy()[:, :C]
    assert np.all(np.abs(got_x[:, :C] - x64) <= dx)
    assert np.array_equal(got_x[:, C:], x0[:, C:])
    mean = x64.mean(1, keepdims=True) if norm == "layer" else 0.0
    v = x64 - mean
    dv = dx + dx.mean(1, keepdims=True) + 40 * U * (np.abs(x64) + np.abs(x64).mean(1, keepdims=True))
    var = (v ** 2).mean(1, keepdims=True) + eps
    r = 1 / np.sqrt(var)
    # r's relative error: half of the sum's (32 roundings, and the terms' own), and four more roundings
    dr = (np.abs(v) * dv).mean(1, keepdims=True) / var + 24 * U
    f = (vec[1] if "w" in parts else 1.0) * ((1 + g64[:, C:2 * C]) if "mod" in parts else 1.0)
    sh = g64[:, :C] if "mod" in parts else 0.0
    h64 = v * r * f + sh
    dh = (dv * r + np.abs(v) * r * (dr + 8 * U)) * np.abs(f) + 4 * U * (np.abs(h64) + np.abs(sh))
    assert np.all(np.abs(got_h - h64) <= dh)
    if f8:  # the e4m3 rows of exactly these fp32 rows
        rq, rs_ = quant_ref(got_h)
        assert np.array_equal(s.numpy(), rs_) and np.array_equal(q.numpy(), rq)


def test_residual_norm_in_place_and_alone(ctx):
    """h over y, one kind of output at a time, x untouched without y."""
    case("residual_norm h over y; q alone; no y")
    rows, C = 37, 640
    x0 = randn(41, rows * C).reshape(rows, C).astype(np.float32)
    y0 = randn(42, rows * C).reshape(rows, C).astype(np.float32)
    xa, xb, ya = Guarded(ctx, x0.shape, np.float32, x0), Guarded(ctx, x0.shape, np.float32, x0), Guarded(ctx, x0.shape, np.float32, y0)
    h, yb = Guarded(ctx, x0.shape, np.float32), ctx.upload(y0)
    ctx.residual_norm(rows, C, xa.ptr, y=ya.ptr, h=ya.ptr)
    ctx.residual_norm(rows, C, xb.ptr, y=yb, h=h.ptr)
    assert np.array_equal(ya.numpy(), h.numpy()) and np.array_equal(xa.numpy(), xb.numpy())
    q, s = Guarded(ctx, x0.shape, np.uint8), Guarded(ctx, (5, rows), np.float32)
    ctx.residual_norm(rows, C, xb.ptr, q=q.ptr, s=s.ptr)
    ctx.residual_norm(rows, C, xb.ptr, h=h.ptr)
    assert np.array_equal(xa.numpy(), xb.numpy())
    rq, rs = quant_ref(h.numpy())
    assert np.array_equal(q.numpy(), rq) and np.array_equal(s.numpy(), rs)


# ------------------------------------------------------------------ as they are used


class Block:
    """A transformer block on e4m3 weights: norm, q/k/v, causal attention, output projection into the residual
    stream, norm, gated feed-forward half, down projection into the residual stream."""

    H, KH, HD, D, F = 4, 2, 128, 512, 1024

    def __init__(self, ctx, M):
        m = amd()
        self.ctx, self.M = ctx, M
        D, F, NQ = self.D, self.F, (self.H + 2 * self.KH) * self.HD
        self.host = {k: f8_weight(i, n, c, 0.7) for i, (k, n, c) in enumerate(
            [("qkv", NQ, D), ("o", D, self.H * self.HD), ("gate", F, D), ("up", F, D), ("down", D, F)])}
        self.keep = {k: (ctx.upload(w), ctx.upload(s)) for k, (w, s) in self.host.items()}
        self.w = {k: m.weight(m.W_F8, *self.host[k][0].shape, b[0], scale=b[1]) for k, b in self.keep.items()}
        self.n1, self.n2 = [(1 + 0.1 * randn(50 + i, D)).astype(np.float32) for i in range(2)]
        self.d_n1, self.d_n2 = ctx.upload(self.n1), ctx.upload(self.n2)
        self.x = ctx.empty((M, D))
        self.bufs()

    def bufs(self):
        ctx, M, D, F = self.ctx, self.M, self.D, self.F
        self.q1, self.s1 = ctx.empty((M, D), np.uint8), ctx.empty((D // 128, M))
        self.qkv = ctx.empty((M, (self.H + 2 * self.KH) * self.HD))
        self.a = ctx.empty((M, self.H * self.HD), np.uint16)
        self.q2, self.s2 = ctx.empty((M, self.H * self.HD), np.uint8), ctx.empty((self.H, M))
        self.y = ctx.empty((M, D))
        self.q3, self.s3 = ctx.empty((M, D), np.uint8), ctx.empty((D // 128, M))
        self.q4, self.s4 = ctx.empty((M, F), np.uint8), ctx.empty((F // 128, M))

    def run(self):
        ctx, m, M, D = self.ctx, amd(), self.M, self.D
        ld = (self.H + 2 * self.KH) * self.HD
        ctx.residual_norm(M, D, self.x, norm_w=self.d_n1, q=self.q1, s=self.s1)
        ctx.linear(self.w["qkv"], M, self.qkv, xq=self.q1, xs=self.s1)
        ctx.attention(q=self.qkv, k=self.qkv, v=self.qkv, o=self.a, B=1, Lq=M, Lk=M, H=self.H, D=self.HD, ldq=ld, ldk=ld, ldv=ld,
                      k_off=self.H * self.HD, v_off=(self.H + self.KH) * self.HD, group=self.H // self.KH, causal=1, o_bf16=True)
        ctx.quant_rows_f8(self.a, M, self.H * self.HD, self.q2, self.s2, bf16=True)
        ctx.linear(self.w["o"], M, self.y, xq=self.q2, xs=self.s2)
        ctx.residual_norm(M, D, self.x, y=self.y, norm_w=self.d_n2, q=self.q3, s=self.s3)
        ctx.linear_glu(self.w["gate"], self.w["up"], M, xq=self.q3, xs=self.s3, out_q=self.q4, out_s=self.s4)
        ctx.linear(self.w["down"], M, self.x, xq=self.q4, xs=self.s4, epilogue=m.EPI_RESID)


@pytest.mark.parametrize("M", [1, 43, 300])
def test_block(ctx, M):
    """Each step against 64 bits from what the step before left, and the whole in a replayed graph."""
    case(f"e4m3 block of {M} tokens")
    b = Block(ctx, M)
    D, HD, H, KH = b.D, b.HD, b.H, b.KH
    x0 = randn(60, M * D).reshape(M, D).astype(np.float32)
    b.x.write(x0)
    b.run()
    q1, s1 = b.q1.numpy(), b.s1.numpy()
    x64 = x0.astype(np.float64)
    h = x64 / np.sqrt((x64 ** 2).mean(1, keepdims=True) + 1e-6) * b.n1
    check_f8_rows(q1, s1, h, 64 * U * np.abs(h))
    y, dy = product64(rows64(q1, s1), weight64(*b.host["qkv"]))
    qkv = b.qkv.numpy()
    assert np.all(np.abs(qkv - y) <= dy + U * np.abs(y))
    q, k, v = [t.astype(np.float64) for t in (qkv[:, :H * HD], qkv[:, H * HD:(H + KH) * HD], qkv[:, (H + KH) * HD:])]
    o = np.empty((M, H * HD))
    for i in range(H):
        sc = q[:, HD * i:HD * i + HD] @ k[:, HD * (i // 2):HD * (i // 2) + HD].T / math.sqrt(HD)
        p = np.exp(np.where(np.tril(np.ones((M, M), bool)), sc, -np.inf) - sc.max(1, keepdims=True))
        o[:, HD * i:HD * i + HD] = p / p.sum(1, keepdims=True) @ v[:, HD * (i // 2):HD * (i // 2) + HD]
    a = torch.from_numpy(b.a.numpy().view(np.int16)).view(torch.bfloat16).float().numpy()
    assert np.linalg.norm(a - o) <= 1e-2 * np.linalg.norm(o)  # the bf16 attention's own bar
    rq, rs = quant_ref(a)
    assert np.array_equal(b.q2.numpy(), rq) and np.array_equal(b.s2.numpy(), rs)
    y, dy = product64(rows64(rq, rs), weight64(*b.host["o"]))
    x1, dx = x64 + y, dy + 2 * U * (np.abs(y) + np.abs(x64))
    r = 1 / np.sqrt((x1 ** 2).mean(1, keepdims=True) + 1e-6)
    h = x1 * r * b.n2
    dr = (np.abs(x1) * dx).mean(1, keepdims=True) * r * r
    q3, s3 = b.q3.numpy(), b.s3.numpy()
    check_f8_rows(q3, s3, h, (dx * r + np.abs(x1) * r * dr) * np.abs(b.n2) + 64 * U * np.abs(h))
    x64 = rows64(q3, s3)
    g, dg = product64(x64, weight64(*b.host["gate"]))
    u, du = product64(x64, weight64(*b.host["up"]))
    act, da = act64(g, "silu"), act_error(g, "silu", dg)
    q4, s4 = b.q4.numpy(), b.s4.numpy()
    check_f8_rows(q4, s4, act * u, da * (np.abs(u) + du) + np.abs(act) * du + 2 * U * np.abs(act * u))
    y, dy = product64(rows64(q4, s4), weight64(*b.host["down"]))
    assert np.all(np.abs(b.x.numpy() - (x1 + y)) <= dx + dy + 4 * U * (np.abs(x1) + np.abs(y)))

    # the same calls captured: replays with new inputs give the eager bits, eager work between them
    ctx.graph_begin()
    b.run()
    graph = ctx.graph_end()
    e = Block(ctx, M)
    for rep in range(3):
        x = randn(70 + rep, M * D).reshape(M, D).astype(np.float32)
        e.x.write(x)
        e.run()
        want = e.x.numpy()
        b.x.write(x)
        ctx.graph_launch(graph)
        assert np.array_equal(b.x.numpy(), want), rep
    ctx.graph_destroy(graph)


def test_two_contexts_and_two_graphs(ctx):
    """Calls of two contexts overlap, and two graphs that were captured with scratch of their own replay in turn."""
    m = amd()
    M, N, K = 200, 512, 1024
    case("two contexts, two graphs")
    w, scale = f8_weight(1, N, K)
    with m.Context(0) as other:
        want, runs = [], []
        for i, c in enumerate((ctx, other)):
            x = randn(80 + i, M * K).reshape(M, K).astype(np.float32)
            W = m.weight(m.W_F8, N, K, c.upload(w), scale=c.upload(scale))
            dx, out = c.upload(x), c.empty((M, N))
            c.linear(W, M, out, x=dx)
            want.append(out.numpy())
            runs.append((c, W, dx, out))
        for _ in range(20):
            for c, W, dx, out in runs:
                c.linear(W, M, out, x=dx)
        for r, (c, W, dx, out) in zip(want, runs):
            assert np.array_equal(out.numpy(), r)
    c, W, dx, out = runs[0]
    F = 256
    G = [m.weight(m.W_F8, F, K, ctx.upload(f8_weight(5 + i, F, K)[0]), scale=ctx.upload(f8_weight(5 + i, F, K)[1])) for i in range(2)]
    q, s = ctx.empty((M, F), np.uint8), ctx.empty((2, M))

    def glu():
        ctx.linear_glu(G[0], G[1], M, x=dx, out_q=q, out_s=s)

    glu()
    wq, wsc = q.numpy(), s.numpy()
    graphs = []
    for f in (lambda: ctx.linear(W, M, out, x=dx), glu):
        ctx.graph_begin()
        f()
        graphs.append(ctx.graph_end())
    for _ in range(3):
        ctx.zero(out, M * N)
        ctx.zero(s, 2 * M)
        for g in graphs + graphs[::-1]:
            ctx.graph_launch(g)
        assert np.array_equal(out.numpy(), want[0]) and np.array_equal(q.numpy(), wq) and np.array_equal(s.numpy(), wsc)
    for g in graphs:
        ctx.graph_destroy(g)


def test_refusals_leave_the_context_usable(ctx):
    m = amd()
    W = m.weight(m.W_F8, 64, 64, 0x10000, scale=0x10000)
    for f in (lambda: ctx.linear(W, 3, 0x10000, x=0x10004), lambda: ctx.linear(W, 3, 0x10000, xq=0x10000),
              lambda: ctx.linear_glu(W, W, 3, x=0x10000), lambda: ctx.residual_norm(3, 62, 0x10000, h=0x10000),
              lambda: ctx.quant_rows_f8(0x10000, 3, 60, 0x10000, 0x10000)):
        with pytest.raises(m.AnimaError):
            f()
    ctx.sync()
    # rows and products of nothing
    ctx.linear(W, 0, 0x10000, x=0x10000)
    ctx.linear_glu(W, W, 0, x=0x10000, out=0x10000)
    ctx.residual_norm(0, 64, 0x10000, h=0x10000)
    ctx.quant_rows_f8(0x10000, 0, 64, 0x10000, 0x10000)
    ctx.sync()


# ------------------------------------------------------------------ every kernel, as chosen


def sampled(M, seed):
    """Rows of the first, a middle and the last tile."""
    return np.unique(np.concatenate([np.arange(min(M, 20)), np.random.default_rng(seed).integers(0, M, 24), np.arange(max(M - 20, 0), M)]))


@pytest.mark.parametrize("fast", [True, False])
def test_linear_kernels(ctx, fast):
    """The five kernels of anima_linear, at sizes past their tiles' ends, into bf16 and gated fp32 rows; fp32 x
    quantized inside the product and before it."""
    m = amd()
    prec = m.PREC_BF16 if fast else m.PREC_FP32
    seen = set()
    for M, N, K in [(3, 514, 1040), (50, 1030, 2064), (517, 1316, 1424), (1499, 900, 528), (1501, 2004, 528), (3901, 4100, 400), (3333, 4104, 4112)]:
        case(f"linear f8 kernels M={M} N={N} K={K} fast={fast}")
        w, scale = f8_weight(N, N, K)
        W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale))
        w64, idx = weight64(w, scale), sampled(M, N)
        gate = randn(30, N).astype(np.float32)
        for kind in ("f8", "f32"):
            args, x64 = inputs(ctx, M, M, K, kind)
            y, dy = product64(x64[idx], w64, fast)
            out = Guarded(ctx, (M, N), np.float32, np.ones((M, N), np.float32))
            ran_f = ran(ctx, lambda: ctx.linear(W, M, out.ptr, epilogue=m.EPI_GATED, gate=ctx.upload(gate), precision=prec, **args))
            got, r = out.numpy()[idx], y * gate
            assert np.all(np.abs(got - (1 + r)) <= dy * np.abs(gate) + 2 * U * (1 + 2 * np.abs(r)))
            out = Guarded(ctx, (M, N), np.uint16)
            ctx.linear(W, M, out.ptr, out_bf16=True, precision=prec, **args)
            gb = torch.from_numpy(out.numpy()[idx].view(np.int16)).view(torch.bfloat16).double().numpy()
            assert np.all(np.abs(gb - y) <= dy * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(y))
            seen.add(tuple(sorted(ran_f)))
    names = {n for t in seen for n in t}
    assert {"gemm.f8.skinny", "gemm.f8.64x64", "gemm.f8.128x64", "gemm.f8.128x128", "gemm.f8.256x256", "quant.f8"} <= names
    assert ("gemm.f8.skinny",) in seen and ("gemm.f8.skinny", "quant.f8") in seen


@pytest.mark.parametrize("fast", [True, False])
def test_glu_kernels(ctx, fast):
    """The five kernels of anima_linear_glu, into fp32 and e4m3 rows (from the tile, or by a pass)."""
    m = amd()
    prec = m.PREC_BF16 if fast else m.PREC_FP32
    names = set()
    for M, F, K in [(3, 272, 1040), (517, 1040, 1040), (900, 4112, 272), (2101, 1296, 272), (1300, 8208, 528), (3333, 4112, 1040)]:
        (wg, sg), (wu, su) = f8_weight(F, F, K), f8_weight(F + 1, F, K)
        G, Up = m.weight(m.W_F8, F, K, ctx.upload(wg), scale=ctx.upload(sg)), m.weight(m.W_F8, F, K, ctx.upload(wu), scale=ctx.upload(su))
        args, x64 = inputs(ctx, M, M, K, "f8")
        idx = sampled(M, F)
        g, dg = product64(x64[idx], weight64(wg, sg), fast)
        u, du = product64(x64[idx], weight64(wu, su), fast)
        a, da = act64(g, "silu"), act_error(g, "silu", dg)
        h = a * u
        dh = da * (np.abs(u) + du) + np.abs(a) * du + 2 * U * np.abs(h)
        out = Guarded(ctx, (M, F), np.float32)
        q, s = Guarded(ctx, (M, F), np.uint8), Guarded(ctx, (-(-F // 128), M), np.float32)
        case(f"linear_glu kernels M={M} F={F} K={K} fast={fast}")
        n1 = ran(ctx, lambda: ctx.linear_glu(G, Up, M, act="silu", out=out.ptr, precision=prec, **args))
        n2 = ran(ctx, lambda: ctx.linear_glu(G, Up, M, act="silu", out_q=q.ptr, out_s=s.ptr, precision=prec, **args))
        print(n1, n2, flush=True)
        names |= n1 | n2
        assert np.all(np.abs(out.numpy()[idx] - h) <= dh)
        check_f8_rows(q.numpy()[idx], s.numpy()[:, idx], h, dh)
    assert names == {"glu.f8.skinny", "glu.f8.64x128", "glu.f8.128x128", "glu.f8.64x256", "glu.f8.256x256", "quant.f8"}


def test_quant_many_rows(ctx):
    """More blocks than one launch's whole waves of workgroups, an odd row count, both types."""
    m = amd()
    M, K = 70001, 272
    x = randn(31, 4096 * K).reshape(4096, K).astype(np.float32)
    x = np.tile(x, (-(-M // 4096), 1))[:M] * np.linspace(0.5, 2, M, dtype=np.float32)[:, None]
    for wide in (False, True):
        case(f"quant f8 many rows bf16={wide}")
        bits, val = bf16(x) if wide else (x, x)
        q, s = Guarded(ctx, (M, K), np.uint8), Guarded(ctx, (3, M), np.float32)
        ctx.quant_rows_f8(ctx.upload(bits), M, K, q.ptr, s.ptr, bf16=wide)
        rq, rs = quant_ref(val)
        assert np.array_equal(q.numpy(), rq) and np.array_equal(s.numpy(), rs)


@pytest.mark.parametrize("C", [132, 256, 272, 516, 1028, 1600, 2052, 4112, 8208, 16384])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_residual_norm_many_rows(ctx, C, norm):
    """The kernels of more rows than four per CU, rows that end inside a thread's stride, inside wider rows."""
    case(f"residual_norm many rows C={C} {norm}")
    m = amd()
    rows, ld, groups = 1031, C + 12, 5
    per = -(-rows // groups)
    x0, y = randn(70, rows * ld).reshape(rows, ld).astype(np.float32), randn(71, rows * C).reshape(rows, C).astype(np.float32)
    vec = (1 + 0.3 * randn(72, 2 * C)).reshape(2, C).astype(np.float32)
    mod = (0.5 * randn(73, groups * 3 * C)).reshape(groups, 3 * C).astype(np.float32)
    d_mod, x = ctx.upload(mod), Guarded(ctx, (rows, ld), np.float32, x0)
    h = Guarded(ctx, (rows, ld), np.float32, np.full((rows, ld), 7, np.float32))
    f8 = C % 16 == 0
    q, s = Guarded(ctx, (rows, C), np.uint8), Guarded(ctx, (-(-C // 128), rows), np.float32)
    ctx.residual_norm(rows, C, x.ptr, ldx=ld, y=ctx.upload(y), post_w=ctx.upload(vec[0]), gate=d_mod.ptr + 8 * C, gate_ld=3 * C, res_scale=0.5,
                      norm=norm, norm_w=ctx.upload(vec[1]), shift=d_mod.ptr, scale=d_mod.ptr + 4 * C, mod_ld=3 * C, group_rows=per,
                      h=h.ptr, ldh=ld, q=q.ptr if f8 else None, s=s.ptr if f8 else None)
    g64 = mod[np.arange(rows) // per].astype(np.float64)
    y64 = y.astype(np.float64)
    post = y64 / np.sqrt((y64 * y64).mean(1, keepdims=True) + 1e-6) * vec[0] * g64[:, 2 * C:]
    x64 = x0[:, :C] + 0.5 * post
    gx, gh = x.numpy(), h.numpy()
    # half of the sum's 44 roundings (41, the mean's two, eps), two of 1 / sqrt, three products; the addition
    dx = 28 * U * np.abs(post) + U * (np.abs(x64) + np.abs(post))
    assert np.all(np.abs(gx[:, :C] - x64) <= dx)
    assert np.array_equal(gx[:, C:], x0[:, C:]) and np.all(gh[:, C:] == 7)
    v = gx[:, :C].astype(np.float64)  # from here on the rows that the kernel wrote
    mean = v.mean(1, keepdims=True) if norm == "layer" else 0.0
    dv = 40 * U * (np.abs(v) + np.abs(v).mean(1, keepdims=True))
    v = v - mean
    var = (v * v).mean(1, keepdims=True) + 1e-6
    dr = (np.abs(v) * dv).mean(1, keepdims=True) / var + 24 * U
    f, sh = vec[1] * (1 + g64[:, C:2 * C]), g64[:, :C]
    ref = v / np.sqrt(var) * f + sh
    dh = (dv + np.abs(v) * (dr + 8 * U)) / np.sqrt(var) * np.abs(f) + 4 * U * (np.abs(ref) + np.abs(sh))
    assert np.all(np.abs(gh[:, :C] - ref) <= dh)
    if f8:
        rq, rs = quant_ref(gh[:, :C])
        assert np.array_equal(q.numpy(), rq) and np.array_equal(s.numpy(), rs)


def test_f8_fields_of_other_kinds(ctx):
    """precision and out_bf16 with another kind of weight are refused, before anything is written."""
    case("precision / out_bf16 with a bf16 weight")
    m = amd()
    W = m.weight(m.W_BF16, 32, 64, ctx.upload(np.zeros((32, 64), np.uint16)))
    x, out = ctx.upload(np.ones((4, 64), np.float32)), Guarded(ctx, (4, 32), np.float32, np.full((4, 32), 3, np.float32))
    for change in (dict(precision=m.PREC_FP32), dict(out_bf16=True)):
        with pytest.raises(m.AnimaError, match="f8 weights"):
            ctx.linear(W, 4, out.ptr, x=x, **change)
        assert np.all(out.numpy() == 3)
    ctx.linear(W, 4, out.ptr, x=x)
    assert np.all(out.numpy() == 0)


@pytest.mark.parametrize("M,N,K", [(1, 1, 16), (2, 3, 32), (1, 5, 144), (4099, 1, 16), (300, 2, 128)])
@pytest.mark.parametrize("kind", ["f8", "f32"])
def test_smallest(ctx, M, N, K, kind):
    case(f"smallest products M={M} N={N} K={K} x={kind}")
    m = amd()
    (w, sw), (u, su) = f8_weight(N, N, K), f8_weight(N + 9, N, K)
    args, x64 = inputs(ctx, M, M, K, kind)
    W, Up = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(sw)), m.weight(m.W_F8, N, K, ctx.upload(u), scale=ctx.upload(su))
    y, dy = product64(x64, weight64(w, sw), False)
    z, dz = product64(x64, weight64(u, su), False)
    out = Guarded(ctx, (M, N), np.float32)
    ctx.linear(W, M, out.ptr, precision=m.PREC_FP32, **args)
    assert np.all(np.abs(out.numpy() - y) <= dy + U * np.abs(y))
    out = Guarded(ctx, (M, N), np.float32)
    ctx.linear_glu(W, Up, M, act="none", out=out.ptr, precision=m.PREC_FP32, **args)
    assert np.all(np.abs(out.numpy() - y * z) <= dy * (np.abs(z) + dz) + np.abs(y) * dz + 3 * U * np.abs(y * z))


def test_widest(ctx):
    """The longest k of a product, and e4m3 rows as far apart as they may be."""
    m = amd()
    L = m.lib()
    M, N, K = 3, 20, 1 << 20
    case(f"linear f8 M={M} N={N} K={K}")
    w, scale = f8_weight(80, N, K)
    args, x64 = inputs(ctx, 81, M, K, "f8")
    out = Guarded(ctx, (M, N), np.float32)
    ctx.linear(m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale)), M, out.ptr, precision=m.PREC_FP32, **args)
    y, dy = product64(x64, weight64(w, scale), False)
    assert np.all(np.abs(out.numpy() - y) <= dy + U * np.abs(y))
    M, N, K, ld = 300, 1500, 272, 1 << 22
    case(f"linear f8 ldx={ld}")
    w, scale = f8_weight(82, N, K)
    q = random_e4m3(83, M, K)
    s = np.random.default_rng(84).uniform(0.5, 1.5, (3, M)).astype(np.float32) / 100
    x = ctx.empty(((M - 1) * ld + K,), np.uint8)
    for r in range(M):
        ctx._check(L.anima_h2d(ctx.h, x.ptr + r * ld, q[r].ctypes.data, K))
    W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale))
    y, dy = product64(rows64(q, s), weight64(w, scale), False)
    for rows in (5, M):
        out = Guarded(ctx, (rows, N), np.float32)
        ctx.linear(W, rows, out.ptr, xq=x, xs=ctx.upload(np.ascontiguousarray(s[:, :rows])), ldx=ld, precision=m.PREC_FP32)
        assert np.all(np.abs(out.numpy() - y[:rows]) <= dy[:rows] + U * np.abs(y[:rows]))
    x.release()


@pytest.mark.parametrize("M,N,K", [(100, 1300, 6000), (70, 1301, 8208), (513, 1024, 8192), (64, 4100, 4112)])
@pytest.mark.parametrize("fast", [True, False])
def test_linear_split(ctx, M, N, K, fast):
    """Products whose k loop is split over workgroups: every epilogue, replayed from a graph."""
    case(f"linear f8 split M={M} N={N} K={K} fast={fast}")
    m = amd()
    prec = m.PREC_BF16 if fast else m.PREC_FP32
    w, scale = f8_weight(N, N, K)
    bias, gate = randn(91, N).astype(np.float32), randn(92, N).astype(np.float32)
    add, out0 = randn(93, M * N).reshape(M, N).astype(np.float32), randn(94, M * N).reshape(M, N).astype(np.float32)
    W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale), bias=ctx.upload(bias))
    d_gate, d_add = ctx.upload(gate), ctx.upload(add)
    for kind in ("f8", "f32"):
        args, x64 = inputs(ctx, M + K, M, K, kind)
        y, dy = product64(x64, weight64(w, scale), fast)
        v = 0.75 * y + bias + add
        dv = 0.75 * dy + 3 * U * (np.abs(0.75 * y) + np.abs(bias) + np.abs(add))
        a, da = act64(v, "gelu"), act_error(v, "gelu", dv)
        for epi in (m.EPI_STORE, m.EPI_RESID, m.EPI_GATED):
            out = Guarded(ctx, (M, N), np.float32, out0)
            names = ran(ctx, lambda: ctx.linear(W, M, out.ptr, act="gelu", alpha=0.75, epilogue=epi, gate=d_gate, add=d_add, precision=prec, **args))
            assert "gemm.f8.join" in names, names
            r, dr = (a * gate, (da + U * np.abs(a)) * np.abs(gate)) if epi == m.EPI_GATED else (a, da)
            ref = r if epi == m.EPI_STORE else out0 + r
            assert np.all(np.abs(out.numpy() - ref) <= dr + 2 * U * (np.abs(r) + np.abs(ref)))
        eager = Guarded(ctx, (M, N), np.uint16)
        ctx.linear(W, M, eager.ptr, act="gelu", alpha=0.75, add=d_add, out_bf16=True, precision=prec, **args)
        bits = eager.numpy()
        gb = torch.from_numpy(bits.view(np.int16)).view(torch.bfloat16).double().numpy()
        assert np.all(np.abs(gb - a) <= (da + 2 * U * np.abs(a)) * (1 + 2.0 ** -8) + 2.0 ** -8 * np.abs(a))
        out = Guarded(ctx, (M, N), np.uint16)
        ctx.graph_begin()
        ctx.linear(W, M, out.ptr, act="gelu", alpha=0.75, add=d_add, out_bf16=True, precision=prec, **args)
        g = ctx.graph_end()
        for _ in range(3):
            ctx.linear(W, M, eager.ptr, act="gelu", alpha=0.75, add=d_add, out_bf16=True, precision=prec, **args)
            ctx.graph_launch(g)
            assert np.array_equal(out.numpy(), bits) and np.array_equal(eager.numpy(), bits)
        ctx.graph_destroy(g)


@pytest.mark.parametrize("tile,fast,M,N,K", [
    ("64x64", True, 372, 328, 4112), ("64x64", False, 502, 504, 2976), ("128x64", True, 786, 274, 5104), ("128x64", False, 326, 648, 4384),
    ("128x128", True, 131, 2097, 7792), ("128x128", False, 520, 775, 7056), ("256x256", True, 2400, 1707, 7136),
    ("256x256", False, 1233, 3316, 8000)])
def test_linear_split_tiles(ctx, tile, fast, M, N, K):
    """The k loop of every tile split over workgroups, in both precisions; the same bits on every call."""
    case(f"linear f8 split tile={tile} M={M} N={N} K={K} fast={fast}")
    m = amd()
    prec = m.PREC_BF16 if fast else m.PREC_FP32
    w, scale = f8_weight(N + K, N, K)
    bias, gate = randn(95, N).astype(np.float32), randn(96, N).astype(np.float32)
    out0 = randn(97, M * N).reshape(M, N).astype(np.float32)
    W = m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale), bias=ctx.upload(bias))
    args, x64 = inputs(ctx, M + K, M, K, "f8")
    y, dy = product64(x64, weight64(w, scale), fast)
    r, dr = (y + bias) * gate, (dy + U * np.abs(y + bias)) * np.abs(gate)
    d_gate, bits = ctx.upload(gate), None
    for _ in range(3):
        out = Guarded(ctx, (M, N), np.float32, out0)
        names = ran(ctx, lambda: ctx.linear(W, M, out.ptr, epilogue=m.EPI_GATED, gate=d_gate, precision=prec, **args))
        assert f"gemm.f8.{tile}" in names and "gemm.f8.join" in names, names
        got = out.numpy()
        assert np.all(np.abs(got - (out0 + r)) <= dr + 2 * U * (np.abs(r) + np.abs(out0 + r)))
        assert bits is None or np.array_equal(bits, got)
        bits = got


@pytest.mark.parametrize("M", [1, 300])
def test_silu_range(ctx, M):
    """The activation by itself: rows of zeros, so that a result is silu(bias).  Within 2^-22 (3/2 + |r| / 3) of itself from
    -87 to 0 and 1.3 2^-22 above (the roundings of its exponent, power, sum, reciprocal and product); below -87 within
    1.5e-36; an infinity stays, NaN too."""
    case(f"silu f8 M={M}")
    m = amd()
    N, K = 16384, 128
    r = np.concatenate([np.linspace(-120, 40, N - 1024), np.random.default_rng(6).normal(size=1020) * 3,
                        [np.inf, np.nan, 3e38, -3e38]]).astype(np.float32)
    zero = ctx.upload(np.zeros((M, K), np.float32))
    w, scale = f8_weight(1, N, K)
    weights = [m.weight(m.W_F8, N, K, ctx.upload(w), scale=ctx.upload(scale), bias=ctx.upload(b)) for b in (r, np.ones(N, np.float32))]
    lin, glu = Guarded(ctx, (M, N), np.float32), Guarded(ctx, (M, N), np.float32)
    ctx.linear(weights[0], M, lin.ptr, x=zero, act="silu", precision=m.PREC_FP32)
    ctx.linear_glu(weights[0], weights[1], M, x=zero, act="silu", out=glu.ptr, precision=m.PREC_FP32)
    r64 = r.astype(np.float64)
    fin, low = np.isfinite(r64), r64 < -87
    with np.errstate(all="ignore"):
        want = np.where(low, r64 * np.exp(np.maximum(r64, -700)), r64 / (1 + np.exp(-r64)))
        bound = np.where(low, 1.5e-36, 2.0 ** -22 * np.where(r64 < 0, 1.5 + np.abs(r64) / 3, 1.3) * np.abs(want))
    for got in (lin.numpy(), glu.numpy()):
        assert np.array_equal(got, np.broadcast_to(got[0], got.shape), equal_nan=True)
        off = np.abs(got[0][fin] - want[fin])
        assert (off <= bound[fin]).all(), r[fin][off > bound[fin]]
        assert got[0][-4] == np.inf and np.isnan(got[0][-3])
