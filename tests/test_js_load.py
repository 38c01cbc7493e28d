"""The addon loads where it cannot register for the end of the process: on the CPU, over a library of empty functions."""

import os
import re
import shutil
import subprocess

import pytest

from helpers import PKG_DIR, ROOT
from test_js_exit import CC, INCLUDE, NODE, STUB

pytestmark = pytest.mark.skipif(not (NODE and CC and os.path.exists(os.path.join(INCLUDE, "node_api.h"))), reason="node or its headers are not installed")


@pytest.mark.parametrize("on", ["undefined", "5", "() => { throw new Error('no listeners'); }"])
def test_load_without_a_listener(tmp_path, on):
    addon = os.path.join(PKG_DIR, "js", "addon.c")
    names = set(re.findall(r"\b(anima_\w+)\s*\(", open(addon).read()))
    (tmp_path / "stub.c").write_text("#include <stdlib.h>\n" + "\n".join(STUB.values()) + "\n" +
                                     "\n".join(f"long {n}(void) {{ return 0; }}" for n in sorted(names - set(STUB))))
    subprocess.run([CC, "-shared", "-fPIC", "-w", "-o", tmp_path / "libstub.so", tmp_path / "stub.c"], check=True)
    subprocess.run([CC, "-O1", "-fPIC", "-std=c11", "-I" + INCLUDE, "-I" + os.path.join(ROOT, "include"), "-DNODE_GYP_MODULE_NAME=anima",
                    "-DNAPI_VERSION=8", "-shared", "-o", tmp_path / "anima.node", addon, "-L" + str(tmp_path), "-lstub", "-Wl,-rpath,$ORIGIN"],
                   check=True)
    (tmp_path / "p.mjs").write_text(f"""
import Module from "module";
const on = process.on;
process.on = {on};
const n = Module.createRequire(import.meta.url)("./anima.node");
process.on = on;
const c = n.init(0);
n.release(n.allocHandle(c, 100));
n.destroy(c);
console.log("end");
""")
    r = subprocess.run([NODE, tmp_path / "p.mjs"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "end\n", (r.returncode, r.stderr[-500:])
