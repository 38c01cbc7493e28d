"""The end of a process that holds, has released and has dropped many device buffers: the addon on the CPU, over a library of
empty functions (its buffers from malloc)."""

import os
import re
import shutil
import subprocess

import pytest

from helpers import PKG_DIR, ROOT

NODE, CC = shutil.which("node"), shutil.which("gcc")
INCLUDE = "/usr/include/node"

pytestmark = pytest.mark.skipif(not (NODE and CC and os.path.exists(os.path.join(INCLUDE, "node_api.h"))), reason="node or its headers are not installed")

STUB = {"anima_init": "int anima_init(int d, void** c) { *c = malloc(16); return 0; }",
        "anima_alloc": "int anima_alloc(void* c, size_t n, void** p) { *p = malloc(64); return 0; }",
        "anima_free": "int anima_free(void* c, void* p) { free(p); return 0; }",
        "anima_destroy": "int anima_destroy(void* c) { free(c); return 0; }"}

# a collection that is under way when the program ends: old handles, then more of them in one turn of the event loop
PROGRAM = """
import Module from "module";
const n = Module.createRequire(import.meta.url)("./anima.node");
const c = n.init(0);
let keep = [];
for (let i = 0; i < COUNT; i++) {
  const h = n.allocHandle(c, 100);
  if (i % 3 === 1) n.release(h);
  if (i % 3 === 2) keep.push({ h, rest: new Array(20).fill(i) });
  if (keep.length > 20000) keep = keep.slice(10000);
}
n.destroy(c);
console.log("end");
"""


def test_exit_during_collection(tmp_path):
    addon = os.path.join(PKG_DIR, "js", "addon.c")
    names = set(re.findall(r"\b(anima_\w+)\s*\(", open(addon).read()))
    stub = tmp_path / "stub.c"
    stub.write_text("#include <stdlib.h>\n" + "\n".join(STUB.values()) + "\n" +
                    "\n".join(f"long {n}(void) {{ return 0; }}" for n in sorted(names - set(STUB))))
    subprocess.run([CC, "-shared", "-fPIC", "-w", "-o", tmp_path / "libstub.so", stub], check=True)
    subprocess.run([CC, "-O1", "-fPIC", "-std=c11", "-I" + INCLUDE, "-I" + os.path.join(ROOT, "include"), "-DNODE_GYP_MODULE_NAME=anima",
                    "-DNAPI_VERSION=8", "-shared", "-o", tmp_path / "anima.node", addon, "-L" + str(tmp_path), "-lstub", "-Wl,-rpath,$ORIGIN"],
                   check=True)
    for count in (3000, 60000, 111111, 150000, 200000):
        p = tmp_path / f"p{count}.mjs"
        p.write_text(PROGRAM.replace("COUNT", str(count)))
        for _ in range(3):
            r = subprocess.run([NODE, p], capture_output=True, text=True, timeout=60)
            assert r.returncode == 0 and r.stdout == "end\n", (count, r.returncode, r.stderr[-500:])
