"""Refusals of the 4-bit weights, the embedding rows and the prefix attention, without a device: the argument checks are
plain host code (csrc/q4_args.h, csrc/prefix_args.h), compiled here with the host compiler and driven through the
binding's own descriptors."""

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from helpers import PKG_DIR, amd

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")

SHIM = """
#include "prefix_args.h"
#include "q4_args.h"
using namespace anima;
extern "C" {
int t_wquant(const void* w, int b, int N, int K, int g, const uint8_t* q, const uint16_t* s, const uint16_t* z, char* m, size_t n) {
  return check_weight_quant_q4(w, b, N, K, g, q, s, z, Q4Msg{m, n}); }
int t_linear(const anima_linear_desc* d, char* m, size_t n) { return check_linear_q4(d, Q4Msg{m, n}); }
int t_embed(const anima_weight* w, const int32_t* ids, int64_t T, const float* f, const float* out, int64_t ldo, char* m, size_t n) {
  return check_embed_rows(w, ids, T, f, out, ldo, Q4Msg{m, n}); }
int t_prefix(const anima_prefix_attn_desc* d, int64_t* rows, int* longest, char* m, size_t n) {
  return check_attention_prefix(d, rows, longest, PrefixMsg{m, n}); }
int t_prepare(const anima_prefix_attn_desc* d, const void* out, int64_t bytes, char* m, size_t n) {
  return check_attention_prefix_prepare(d, out, bytes, PrefixMsg{m, n}); }
int64_t t_bytes(int h, int p, int prec) { return prefix_kv_bytes(h, p, prec); }
}
"""

P = 0x10000  # an aligned address; nothing is read


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    d = tmp_path_factory.mktemp("q4_args")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.t_bytes.restype = ctypes.c_int64
    return lib


def call(f, *args):
    buf = ctypes.create_string_buffer(256)
    return f(*args, buf, ctypes.c_size_t(256)), buf.value.decode()


def v(x):
    return ctypes.c_void_p(x)


I64 = ctypes.c_int64


@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"z": P}, 0), ({"g": 32}, 0), ({"g": 128, "K": 128}, 0), ({"N": 0}, -1), ({"K": 0}, -1), ({"K": 96}, -1),
    ({"g": 16}, -1), ({"g": 0}, -1), ({"g": -64}, -1), ({"g": 256, "K": 256}, -1), ({"bf16": 2}, -1), ({"w": 0}, -1),
    ({"q": 0}, -1), ({"s": 0}, -1), ({"w": P + 8}, -1), ({"q": P + 4}, -1), ({"s": P + 1}, -1), ({"z": P + 1}, -1),
    ({"N": 1 << 20, "K": 1 << 14}, -5), ({"N": (1 << 20) - 1, "K": 1 << 14}, 0)])
def test_weight_quant(checks, change, code):
    a = dict(dict(w=P, bf16=1, N=3, K=64, g=64, q=P, s=P, z=0), **change)
    rc, msg = call(checks.t_wquant, v(a["w"]), a["bf16"], a["N"], a["K"], a["g"], v(a["q"]), v(a["s"]), v(a["z"]))
    assert rc == code and (code == 0 or "anima_weight_quant_q4" in msg)


def weight(**kw):
    m = amd()
    a = dict(dict(kind=m.W_Q4, N=100, K=192, w=P, group=64, group_scale=P), **kw)
    return m.weight(**a)


@pytest.mark.parametrize("w,change,code", [
    ({}, {}, 0), ({"group_mid": P}, {}, 0), ({}, {"ldx": 196}, 0), ({"bias": P}, {"gate": P, "add": P}, 0), ({"group": 32}, {}, 0),
    ({}, {"out_bf16": 1, "precision": 0}, 0), ({}, {"precision": 1}, 0), ({"group": 128}, {}, -1), ({"group": 0}, {}, -1),
    ({"w": 0}, {}, -1), ({"group_scale": 0}, {}, -1), ({"w": P + 8}, {}, -1), ({"group_scale": P + 1}, {}, -1),
    ({"group_mid": P + 1}, {}, -1), ({"bias": P + 2}, {}, -1), ({}, {"x": 0}, -1), ({}, {"x": P + 4}, -1), ({}, {"ldx": 188}, -1),
    ({}, {"ldx": 194}, -1), ({}, {"xq": P}, -1), ({}, {"xs": P}, -1), ({}, {"precision": 2}, -1), ({}, {"out_bf16": 2}, -1),
    ({}, {"out_bf16": 1, "epilogue": 1}, -5), ({}, {"acc_out": P}, -5), ({}, {"out": P + 2}, -1), ({}, {"gate": P + 2}, -1),
    ({}, {"add": P + 1}, -1), ({}, {"M": (1 << 29) + 1}, -5), ({"N": (1 << 29) + 1}, {}, -5), ({"K": (1 << 20) + 64}, {}, -5),
    ({}, {"ldx": (1 << 22) + 4}, -5), ({}, {"ldx": 1 << 22}, 0)])
def test_linear(checks, w, change, code):
    W = weight(**w)
    a = dict(dict(M=5, x=P, out=P), **change)
    d = amd().LinearDesc(W=ctypes.pointer(W), **a)
    rc, msg = call(checks.t_linear, ctypes.byref(d))
    assert rc == code and (code == 0 or "anima_linear" in msg)


@pytest.mark.parametrize("w,change,code", [
    ({}, {}, 0), ({"kind": 0, "group": 0, "group_scale": 0}, {}, 0), ({"kind": 3, "K": 4}, {}, 0), ({}, {"T": 0, "out": 0}, 0),
    ({}, {"f": P, "ldo": 196}, 0), ({"kind": 0, "w": P + 8}, {}, 0), ({"kind": 1}, {}, -5), ({"kind": 5}, {}, -5), ({"kind": 4}, {}, -5),
    ({"kind": 9}, {}, -5), ({"kind": 0, "K": 6}, {}, -1), ({"N": 0}, {}, -1), ({"group": 48}, {}, -1), ({"group_scale": 0}, {}, -1),
    ({"w": 0}, {}, -1), ({"kind": 0, "w": 0}, {}, -1), ({"kind": 3, "w": P + 8}, {}, -1), ({"kind": 0, "w": P + 4}, {}, -1),
    ({}, {"ids": 0}, -1), ({}, {"ids": P + 2}, -1), ({}, {"out": 0}, -1), ({}, {"out": P + 8}, -1), ({}, {"f": P + 2}, -1),
    ({}, {"ldo": 188}, -1), ({}, {"ldo": 194}, -1), ({}, {"T": -1}, -1), ({}, {"T": 1 << 31}, -1)])
def test_embed(checks, w, change, code):
    a = dict(dict(ids=P, T=7, f=0, out=P, ldo=0), **change)
    rc, msg = call(checks.t_embed, ctypes.byref(weight(**w)), v(a["ids"]), I64(a["T"]), v(a["f"]), v(a["out"]), I64(a["ldo"]))
    assert rc == code and (code == 0 or "anima_embed_rows" in msg)


def test_embed_without_a_table(checks):
    assert call(checks.t_embed, None, v(P), I64(1), None, v(P), I64(0))[0] == -1


def prefix_desc(lens, **kw):
    d = dict(dict(P=100, H=6, D=128, group=3, q=P, ldq=1280, q_off=0, k=P, ldk=1280, k_off=768, v=P, ldv=1280, v_off=1024, o=P,
                  ldo=768, o_off=0, prefix_kv=P, prefix_kv_bytes=2 * 2 * 128 * 128 * 2, precision=0, causal=1), **kw)
    arr = np.asarray(lens, np.int32)
    out = amd().PrefixAttnDesc(B=d.pop("B", arr.size), len=d.pop("len", arr.ctypes.data), **d)
    out.keep = arr
    return out


NONE = {"P": 0, "prefix_kv": 0, "prefix_kv_bytes": 0}


@pytest.mark.parametrize("lens,change,code", [
    ([3, 0, 5], {}, 0), ([3], NONE, 0), ([0, 0], {"q": 0, "o": 0, "prefix_kv": 0}, 0), ([], {"len": 0}, 0), ([3], {"causal": 0}, 0),
    ([3], {"o_bf16": 1, "o": P + 8}, 0), ([3], {"rope_cs": P, "rope_sin_off": 103 * 64}, 0), ([3], {"group": 0, "H": 2,
     "prefix_kv_bytes": 2 * 2 * 128 * 128 * 2}, 0), ([3], {"precision": 1, "prefix_kv_bytes": 2 * 2 * 128 * 128 * 4}, 0),
    ([3], {"D": 64}, -5), ([3], {"B": -1}, -1), ([3], {"len": 0}, -1), ([3, -1], {}, -1), ([(1 << 22) + 1], {}, -1),
    ([1 << 22] * 65, {}, -5), ([1 << 22], {"H": 257, "group": 1, "ldq": 1 << 18}, -5), ([3], {"H": 0}, -1), ([3], {"group": 4}, -1), ([3], {"group": -1}, -1), ([3], {"H": 1 << 13, "group": 1}, -1),
    ([3], {"P": -1}, -1), ([3], {"P": (1 << 22) + 1}, -1), ([3], {"precision": 2}, -1), ([3], {"causal": 2}, -1), ([3], {"o_bf16": 2}, -1),
    ([3], {"precision": 1, "o_bf16": 1}, -1), ([3], {"q": 0}, -1), ([3], {"k": 0}, -1), ([3], {"v": 0}, -1), ([3], {"o": 0}, -1),
    ([3], {"ldq": 764}, -1), ([3], {"ldk": 1020}, -1), ([3], {"ldv": 1276}, -1), ([3], {"ldo": 764}, -1), ([3], {"ldq": 1282}, -1),
    ([3], {"q_off": 2}, -1), ([3], {"k_off": -4}, -1), ([3], {"ldq": (1 << 20) + 4}, -5), ([3], {"q": P + 8}, -1), ([3], {"o": P + 8}, -1),
    ([3], {"o_bf16": 1, "o": P + 4}, -1), ([3], {"q_norm": P + 4}, -1), ([3], {"k_norm": P + 4}, -1), ([3], {"prefix_kv": 0}, -1),
    ([3], {"prefix_kv": P + 8}, -1), ([3], {"P": 0}, -1), ([3], {"prefix_kv_bytes": 0}, -1), ([3], {"P": 129}, -1),
    ([3], {"precision": 1}, -1), ([3], {"rope_cs": P, "rope_sin_off": 102 * 64}, -1), ([3], {"rope_cs": P, "rope_sin_off": 110 * 64 + 4}, -1),
    ([3], {"rope_cs": P + 4, "rope_sin_off": 128 * 64}, -1), ([3], {"eps": -1.0}, -1), ([3], {"eps": float("nan")}, -1)])
def test_prefix(checks, lens, change, code):
    rows, longest = I64(), ctypes.c_int()
    rc, msg = call(checks.t_prefix, ctypes.byref(prefix_desc(lens, **change)), ctypes.byref(rows), ctypes.byref(longest))
    assert rc == code and (code == 0 or "anima_attention_prefix" in msg)
    if code == 0:
        assert (rows.value, longest.value) == (sum(lens), max(lens, default=0))


def test_prefix_without_a_descriptor(checks):
    rows, longest = I64(), ctypes.c_int()
    assert call(checks.t_prefix, None, ctypes.byref(rows), ctypes.byref(longest))[0] == -1


PREP = dict(NONE, q=0, ldq=0, o=0, ldo=0)
BYTES = 2 * 2 * 128 * 128 * 2


@pytest.mark.parametrize("lens,change,out,size,code", [
    ([100], {}, P, BYTES, 0), ([100], {"q_off": 3, "q_norm": 4, "o_bf16": 1}, P, BYTES, 0), ([100], {"precision": 1}, P, 2 * BYTES, 0),
    ([100], {"rope_cs": P, "rope_sin_off": 100 * 64}, P, BYTES, 0), ([129], {}, P, 3 * BYTES // 2, 0), ([100], {}, 0, BYTES, -1),
    ([100], {}, P + 8, BYTES, -1), ([100], {}, P, BYTES - 1, -1), ([100], {}, P, 0, -1), ([129], {}, P, BYTES, -1), ([0], {}, P, 0, -1),
    ([], {"len": 0}, P, 0, -1), ([50, 50], {}, P, BYTES, -1), ([100], {"P": 4}, P, BYTES, -1), ([100], {"prefix_kv": P}, P, BYTES, -1),
    ([100], {"k": 0}, P, BYTES, -1), ([100], {"v": 0}, P, BYTES, -1), ([100], {"ldk": 1020}, P, BYTES, -1), ([100], {"v": P + 4}, P, BYTES, -1),
    ([100], {"k_norm": P + 4}, P, BYTES, -1), ([100], {"rope_cs": P, "rope_sin_off": 99 * 64}, P, BYTES, -1),
    ([100], {"D": 64}, P, BYTES, -5), ([100], {"group": 4}, P, BYTES, -1), ([100], {"precision": 2}, P, BYTES, -1)])
def test_prepare(checks, lens, change, out, size, code):
    rc, msg = call(checks.t_prepare, ctypes.byref(prefix_desc(lens, **dict(PREP, **change))), v(out), I64(size))
    assert rc == code and (code == 0 or "anima_attention_prefix" in msg)


@pytest.mark.parametrize("p", [0, 1, 63, 64, 65, 1000, 1 << 22])
@pytest.mark.parametrize("prec", [0, 1])
def test_prefix_bytes(checks, p, prec):
    """The size the check asks for is anima_attention_kv_bytes'."""
    assert checks.t_bytes(5, p, prec) == (amd().Context.attention_kv_bytes(1, 5, p, prec) if p else 0)


def test_binding(monkeypatch):
    """What the Python binding takes as lengths, without a device (the library's own refusal is "null context")."""
    m = amd()
    ctx = m.Context.__new__(m.Context)
    ctx.h = None

    def go(lens):
        ctx.attention_prefix(q=P, k=P, v=P, o=P, lens=lens, H=2, ldq=256, ldk=256, ldv=256)

    for lens in ([1, 2], (np.int64(3),), np.asarray([4, 5]), np.asarray([4, 5], np.int32)[::2], np.asarray([7], np.int32), []):
        with pytest.raises(m.AnimaError, match="null context"):
            go(lens)
    for lens in ([1.5], ["3"], [None]):
        with pytest.raises(TypeError):
            go(lens)
    with pytest.raises(OverflowError):
        go([1 << 31])
    for W in (None, 5, b"x"):
        with pytest.raises(TypeError):
            ctx.embed_rows(W, P, 1, P)
