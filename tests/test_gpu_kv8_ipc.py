"""Hand-over of an 8-bit region to another process on the same GPU: the
destination exports its region, the source process maps and fills it."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

import hotseat_b200 as hs

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CTX = 16384  # an f32 region of the tiny model: 32 MiB, an 8-bit one 9

SOURCE = """
import json, sys
sys.path.insert(0, {root!r})
import numpy as np
import hotseat_b200 as hs
m = hs.Model.load({model!r}, max_ctx={ctx}, numeric=hs.NUMERIC_TC)
handle, block = bytes.fromhex(sys.argv[1]), int(sys.argv[2])
refused = []
try:
    hs.Kv.open_ipc(m, handle)
except hs.HotseatError as e:
    refused.append(e.code)
view = hs.Kv.open_ipc8(m, handle, block=block)
assert view.block == block and view.bytes == m.kv8(block=block).bytes
try:
    hs.Kv8Set([view])
except hs.HotseatError as e:
    refused.append(e.code)
kv, b = m.kv8(block=block), hs.Batch(m, 64)
prompt = (np.arange(40) * 7 + 3) % m.cfg.vocab
b.prefill(kv, prompt)
g = hs.Migration(kv, view, 40, 41, target_bytes=0)
for p in range(40, 50):
    b.forward([kv], [p], [p])
more = g.round(50, 51)
for p in range(50, 53):
    b.forward([kv], [p], [p])
rep = g.finish(53, 54)
other = m.kv8(block=16 if block == 1 else 1)
try:
    hs.Migration(kv, other, 53, 54)
except hs.HotseatError as e:
    refused.append(e.code)
view.close()
b.forward([kv], [9], [53])
print(json.dumps(dict(refused=refused, rounds=rep["n_rounds"], hash=kv.hash(54), logits=b.logits(0).tolist()[:50])))
"""


@pytest.mark.parametrize("block", [1, 16])
def test_a_process_hands_its_8_bit_cache_to_another(tiny_gguf, block):
    m = hs.Model.load(tiny_gguf, max_ctx=CTX, numeric=hs.NUMERIC_TC)
    dst, b = m.kv8(block=block), hs.Batch(m, 1)
    code = SOURCE.format(root=ROOT, model=tiny_gguf, ctx=CTX)
    r = subprocess.run([sys.executable, "-c", code, dst.ipc_handle().hex(), str(block)], cwd=ROOT, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-3000:]
    rec = json.loads([ln for ln in r.stdout.splitlines() if ln.startswith("{")][-1])
    # an f32 region over it, a set of a view, a hand-over between blocks
    assert rec["refused"] == [hs.HS_E_ARG, hs.HS_E_ARG, hs.HS_E_STATE]
    assert rec["rounds"] >= 2  # the copy of the prompt, and the ten steps after it
    b.forward([dst], [9], [53])
    assert dst.hash(54) == rec["hash"]
    assert np.array_equal(b.logits(0)[:50], np.float32(rec["logits"]))
