"""What a batch of prompts keeps between its calls and its turns of the event loop, on the CPU: the native calls are recorded
instead of made."""

import pytest

from test_batch_js import NODE, RECORD, node

pytestmark = pytest.mark.skipif(NODE is None, reason="node is not installed")

# two-layer encoders of width 256, and a promise that is settled from outside
ENCODER = (RECORD + "const W = (N, K) => ({ kind: 'bf16', N, K, buf: ++last });"
           "const encoder = (Qwen3, layers) => { const te = new Qwen3(gpu, { hidden: 256, heads: 2, kvHeads: 1, headDim: 128, mlp: 256, theta: 1e6 });"
           " te.layers = Array.from({ length: layers }, () => ({ qkv: W(512, 256), o: W(256, 256), gate: W(256, 256), up: W(256, 256), down: W(256, 256),"
           "  ln1: tensor([256]), ln2: tensor([256]), qn: tensor([128]), kn: tensor([128]) }));"
           " te.norm = tensor([256]); te.embedRows = async (ids) => new Float32Array(ids.length * 256); return te; };"
           "const err = async (f) => { try { await f(); return ''; } catch (e) { return e.message; } };")


def test_prefix_of_another_encoder():
    """A kept prefix belongs to the encoder that made it: another one has other weights, and may have other layers."""
    got = node(ENCODER + "import('./qwen3.mjs').then(async ({ Qwen3 }) => {"
               "const a = encoder(Qwen3, 2), b = encoder(Qwen3, 2), c = encoder(Qwen3, 3), prefix = await a.keepPrefix([1, 2]);"
               "const go = (te) => err(() => te.encodeBatch([[1, 2, 3]], { prefix }));"
               "console.log(JSON.stringify([await go(a), await go(b), await go(c)])); })")
    assert got[0] == "" and all("another encoder" in e for e in got[1:]), got
