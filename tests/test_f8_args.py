"""Refusals of the e4m3 operators, without a device: the argument checks are plain host code (csrc/f8_args.h),
compiled here with the host compiler and driven through the binding's own descriptors."""

import ctypes
import os
import shutil
import subprocess

import pytest

from helpers import PKG_DIR, amd

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")

SHIM = """
#include "f8_args.h"
using namespace anima;
extern "C" {
int t_quant(const void* x, int b, int64_t M, int K, int64_t ldx, const uint8_t* q, const float* s, char* m, size_t n) {
  return check_quant_rows_f8(x, b, M, K, ldx, q, s, F8Msg{m, n}); }
int t_wquant(const void* w, int b, int N, int K, const uint8_t* q, const float* s, char* m, size_t n) {
  return check_weight_quant_f8(w, b, N, K, q, s, F8Msg{m, n}); }
int t_linear(const anima_linear_desc* d, char* m, size_t n) { return check_linear_f8(d, F8Msg{m, n}); }
int t_glu(const anima_glu_desc* d, char* m, size_t n) { return check_linear_glu(d, F8Msg{m, n}); }
int t_norm(const anima_resnorm_desc* d, char* m, size_t n) { return check_residual_norm(d, F8Msg{m, n}); }
}
"""

P = 0x10000  # an aligned address; nothing is read


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    d = tmp_path_factory.mktemp("f8_args")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(PKG_DIR, "csrc"),
                    str(d / "shim.cpp"), "-o", str(d / "shim.so")], check=True)
    return ctypes.CDLL(str(d / "shim.so"))


def call(f, *args):
    buf = ctypes.create_string_buffer(256)
    return f(*args, buf, ctypes.c_size_t(256)), buf.value.decode()


def v(x):
    return ctypes.c_void_p(x)


I64 = ctypes.c_int64


@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"M": 0, "x": 0}, 0), ({"ldx": 96}, 0), ({"M": -1}, -1), ({"K": 0}, -1), ({"K": 40}, -1), ({"ldx": 60}, -1),
    ({"ldx": 66}, -1), ({"bf16": 1, "ldx": 68}, -1), ({"bf16": 1, "ldx": 72}, 0), ({"bf16": 2}, -1), ({"x": 0}, -1),
    ({"q": 0}, -1), ({"s": 0}, -1), ({"x": P + 8}, -1), ({"q": P + 4}, -1), ({"s": P + 2}, -1)])
def test_quant_rows(checks, change, code):
    a = dict(dict(x=P, bf16=0, M=5, K=64, ldx=0, q=P, s=P), **change)
    rc, msg = call(checks.t_quant, v(a["x"]), a["bf16"], I64(a["M"]), a["K"], I64(a["ldx"]), v(a["q"]), v(a["s"]))
    assert rc == code and (code == 0 or "anima_quant_rows_f8" in msg)


@pytest.mark.parametrize("change,code", [({}, 0), ({"N": 0}, -1), ({"K": 24}, -1), ({"w": 0}, -1), ({"q": P + 1}, -1),
                                         ({"bf16": -1}, -1), ({"s": 0}, -1)])
def test_weight_quant(checks, change, code):
    a = dict(dict(w=P, bf16=1, N=3, K=16, q=P, s=P), **change)
    rc, msg = call(checks.t_wquant, v(a["w"]), a["bf16"], a["N"], a["K"], v(a["q"]), v(a["s"]))
    assert rc == code and (code == 0 or "anima_weight_quant_f8" in msg)


def weight(**kw):
    m = amd()
    a = dict(dict(kind=m.W_F8, N=100, K=160, w=P, scale=P), **kw)
    return m.weight(a["kind"], a["N"], a["K"], a["w"], scale=a["scale"], bias=a.get("bias"))


@pytest.mark.parametrize("w,change,code", [
    ({}, {}, 0), ({}, {"x": 0, "xq": P, "xs": P}, 0), ({}, {"ldx": 164}, 0), ({}, {"xq": P, "xs": P, "ldx": 176}, 0),
    ({"K": 168}, {}, -1), ({"K": (1 << 20) + 16}, {}, -1), ({"w": 0}, {}, -1), ({"w": P + 8}, {}, -1), ({"scale": 0}, {}, -1),
    ({}, {"x": 0}, -1), ({}, {"x": P + 4}, -1), ({}, {"ldx": 100}, -1), ({}, {"ldx": 162}, -1), ({}, {"xq": P}, -1),
    ({}, {"xq": P + 8, "xs": P}, -1), ({}, {"xq": P, "xs": P, "ldx": 168}, -1),
    ({}, {"xq": P, "xs": P, "ldx": (1 << 22) + 16}, -5), ({}, {"acc_out": P}, -5), ({}, {"precision": 1, "out_bf16": 1}, 0),
    ({}, {"precision": 2}, -1), ({}, {"out_bf16": 2}, -1), ({}, {"out_bf16": 1, "epilogue": 1}, -5), ({}, {"out": P + 2}, -1),
    ({}, {"out_bf16": 1, "out": P + 2}, 0), ({}, {"out_bf16": 1, "out": P + 1}, -1), ({"scale": P + 2}, {}, -1),
    ({"bias": P + 1}, {}, -1), ({}, {"xq": P, "xs": P + 2}, -1), ({}, {"gate": P + 2}, -1), ({}, {"add": P + 2}, -1)])
def test_linear(checks, w, change, code):
    m = amd()
    W = weight(**w)
    d = m.LinearDesc(**dict(dict(M=3, W=ctypes.pointer(W), x=P, out=P), **change))
    rc, msg = call(checks.t_linear, ctypes.byref(d))
    assert rc == code and (code == 0 or "anima_linear" in msg)


@pytest.mark.parametrize("g,u,change,code", [
    ({}, {}, {}, 0), ({"N": 96}, {"N": 96}, {"out": 0, "out_q": P, "out_s": P}, 0), ({}, {}, {"M": 0, "x": 0}, 0),
    ({}, {"N": 99}, {}, -1), ({}, {"K": 176}, {}, -1), ({"kind": 0}, {}, {}, -5), ({}, {"kind": 1}, {}, -5),
    ({}, {"w": P + 4}, {}, -1), ({}, {}, {"M": -2}, -1), ({}, {}, {"act": 3}, -1), ({}, {}, {"x": 0}, -1),
    ({}, {}, {"out": 0}, -1), ({}, {}, {"ldc": 99}, -1), ({}, {}, {"out_s": P}, -1), ({}, {}, {"out_q": P, "out_s": P}, -1),
    ({}, {}, {"out": 0, "out_q": P, "out_s": P}, -1),  # N = 100: rows of 100 bytes
    ({"N": 96}, {"N": 96}, {"out": 0, "out_q": P}, -1), ({"N": 96}, {"N": 96}, {"out": 0, "out_q": P + 8, "out_s": P}, -1),
    ({}, {"bias": P + 2}, {}, -1), ({}, {}, {"out": P + 2}, -1), ({"N": 96}, {"N": 96}, {"out": 0, "out_q": P, "out_s": P + 2}, -1)])
def test_glu(checks, g, u, change, code):
    m = amd()
    G, U = weight(**g), weight(**u)
    d = m.GluDesc(**dict(dict(M=3, gate=ctypes.pointer(G), up=ctypes.pointer(U), x=P, act=2, out=P), **change))
    rc, msg = call(checks.t_glu, ctypes.byref(d))
    assert rc == code and (code == 0 or "anima_linear_glu" in msg)


def test_glu_null(checks):
    m = amd()
    G = weight()
    assert call(checks.t_glu, v(0))[0] == -1
    assert call(checks.t_glu, ctypes.byref(m.GluDesc(M=1, gate=ctypes.pointer(G), x=P, out=P)))[0] == -1


@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"rows": 0, "x": 0, "h": 0}, 0), ({"y": P, "post_w": P, "gate": P, "shift": P, "scale": P, "q": P, "s": P}, 0),
    ({"cols": 16384}, 0), ({"rows": -1}, -1), ({"cols": 0}, -1), ({"cols": 66}, -1), ({"cols": 16388}, -1), ({"norm": 2}, -1),
    ({"eps": -1.0}, -1), ({"eps": float("nan")}, -1), ({"x": 0}, -1), ({"h": 0}, -1), ({"q": P}, -1), ({"s": P}, -1),
    ({"cols": 68, "q": P, "s": P}, -1), ({"post_w": P}, -1), ({"gate": P}, -1), ({"shift": P}, -1), ({"scale": P}, -1),
    ({"group_rows": -1}, -1), ({"ldx": 60}, -1), ({"ldy": 66}, -1), ({"ldh": 2}, -1), ({"mod_ld": 63}, -1), ({"gate_ld": 65}, -1),
    ({"x": P + 4}, -1), ({"y": P + 8}, -1), ({"y": P + 8, "y_bf16": 1}, 0), ({"y": P + 4, "y_bf16": 1}, -1), ({"y_bf16": 2}, -1), ({"norm_w": P + 4}, -1), ({"h": P + 8}, -1), ({"q": P, "s": P + 2}, -1)])
def test_residual_norm(checks, change, code):
    m = amd()
    d = m.ResNormDesc(**dict(dict(rows=3, cols=64, x=P, norm=0, eps=1e-6, h=P), **change))
    rc, msg = call(checks.t_norm, ctypes.byref(d))
    assert rc == code and (code == 0 or "anima_residual_norm" in msg)


@pytest.mark.parametrize("change,code", [
    ({}, 0), ({"ldy": 80, "ldh": 80}, 0), ({"ldy": 64}, 0), ({"ldh": 80}, -1), ({"ldy": 80}, -1), ({"y_bf16": 1}, -1),
    ({"rows": 1, "ldy": 80}, 0), ({"h": 0, "ldh": 80, "q": P, "s": P}, 0), ({"y": P + 64, "ldy": 80}, 0)])
def test_residual_norm_in_place(checks, change, code):
    """h may be y: the same fp32 rows; with other strides a row's h would be another row's y."""
    m = amd()
    d = m.ResNormDesc(**dict(dict(rows=3, cols=64, x=2 * P, y=P, norm=0, eps=1e-6, h=P), **change))
    rc, msg = call(checks.t_norm, ctypes.byref(d))
    assert rc == code and (code == 0 or "h may be" in msg)


def test_residual_norm_null(checks):
    assert call(checks.t_norm, v(0))[0] == -1


def test_null_context():
    L = amd().lib()
    assert L.anima_quant_rows_f8(None, None, 0, 1, 16, 0, None, None) == -1
    assert L.anima_weight_quant_f8(None, None, 0, 1, 16, None, None) == -1
    assert L.anima_linear_glu(None, None) == -1
    assert L.anima_residual_norm(None, None) == -1


@pytest.mark.parametrize("name", ["LinearDesc", "GluDesc", "ResNormDesc"])
def test_packed_descriptors(name):
    """The binding's packed descriptors are the bytes of the ctypes structs (whose offsets the library confirms)."""
    m = amd()
    cls = getattr(m, name)
    pack = {"LinearDesc": m._linear_desc, "GluDesc": m._glu_desc, "ResNormDesc": m._resnorm_desc}[name]
    values = [i + 0.25 if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
    d = cls.from_buffer_copy(pack(*values))
    for (f, t), v in zip(cls._fields_, values):
        got = getattr(d, f)
        if issubclass(t, ctypes._Pointer):
            got = ctypes.cast(got, ctypes.c_void_p).value
        assert got == v, f
