"""Batches of prompts on text encoders of every kind of weight, on the device: encodeBatch gives what encode gives of each prompt by
itself, but for roundings.

Tolerances (2-norm of a prompt's rows).  On bf16 weights: 1e-5 in fp32 precision and 1e-2 in bf16, as an encoding against 64 bits.
Quantized activations amplify what the two sides differ by: where they are d apart, d / s of the values go to the other side of a
rounding with steps of s and are s apart then, which is sqrt(d s) in the root mean square, more than d.  So 2^-20 becomes
sqrt(2^-20 0.09) = 3e-4 behind one product of e4m3 rows (steps of 2^-3 to 2^-4 of a value, 0.09), 0.005 behind the next, and the end is two
sides that round on their own: off by s / sqrt(12) each, sqrt(2) s / sqrt(12) from each other, 0.037 in e4m3 and 0.012 in int8 (steps of
a 127th of a row's largest value, 3.7 times its root mean square: 0.029).  Two layers have fourteen products whose errors add up as squares:
sqrt(14) of that, 0.14 and 0.044.  (A product of other rows or columns, or a key at another position, moves a row by its own size.)"""

import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from helpers import ROOT, report

NODE = shutil.which("node")
pytestmark = [pytest.mark.skipif(NODE is None, reason="node is not installed"), pytest.mark.gpu]


@pytest.mark.parametrize("kind", ["bf16", "f8", "i8", "w4", "unstacked", "mixed"])
def test_kinds(tmp_path, kind):
    rng = np.random.default_rng(19)
    head = [int(v) for v in rng.integers(0, 97, size=90)]
    prompts = [head + [int(v) for v in rng.integers(0, 97, size=n)] for n in (9, 0, 70, 1)]
    out = str(tmp_path / "k")
    (tmp_path / "case.json").write_text(json.dumps({"kind": kind, "layers": 2, "vocab": 97, "prompts": prompts, "keep": 66, "out": out}))
    print(f"[case] js batch kinds {kind}", flush=True)
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "run_kinds.mjs"), str(tmp_path / "case.json")], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0, r.stderr[-3000:]
    kinds = json.loads(r.stdout)
    want = {"bf16": "bf16", "f8": "f8", "i8": "i8", "w4": "w4", "unstacked": "w4"}
    assert all((f"q:{k}" in s and f"v:{k}" in s) if kind == "unstacked" else f"qkv:{k}" in s for s in kinds
               for k in [want.get(kind, "f8" if s is kinds[0] else "q4")]), kinds
    quantized = {"bf16": None, "f8": 0.14, "mixed": 0.14}.get(kind, 0.044)
    for prec, bar in (("fp32", quantized or 1e-5), ("bf16", quantized or 1e-2)):
        for i in range(len(prompts)):
            one, batch, kept = (np.fromfile(f"{out}.{prec}.{n}.{i}", np.float32).reshape(len(prompts[i]), 1024) for n in ("one", "batch", "kept"))
            assert np.isfinite(one).all() and one.any()
            assert report(f"{kind} {prec} batch {i}", batch, one)[0] <= bar
            assert report(f"{kind} {prec} kept {i}", kept, one)[0] <= bar
