"""Paged attention whose copies do not come: each wait runs out, the call ends with WCB_PAGED_ABORTED in the status word, and the
device stays usable. A hook of the library (read once, so in a process of its own) makes every tile wait for bytes more than
its copies bring, and the waits short."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import sys
sys.path.insert(0, {pkg!r}); sys.path.insert(0, {tests!r})
import time, torch, wcb
import test_gpu_paged as t
# many rows (16-bit types, f32 over f16) on the tensor cores, few rows, both in one call; whole tiles and ragged ones
for act, cache in (("bf16", "bf16"), ("f16", "f16"), ("f32", "f16")):
    for dim in (64, 128):
        for q, kv in (([300], [2000]), ([1, 1, 2], [700, 65, 900]), ([1, 200, 130], [700, 1000, 130])):
            s = t.Step(q, kv, 8, 2, dim, act, cache, 64, seed=70)
            torch.cuda.synchronize()
            begin = time.time()
            s.attend()
            torch.cuda.synchronize()
            assert time.time() - begin < 2, time.time() - begin
            assert int(s.status.item()) & wcb.PAGED_ABORTED, (act, cache, dim, q)
# what brings nothing by bulk copy works as ever: an f32 cache on the tensor cores, pages of one token
s = t.Step([200], [900], 8, 2, 64, "f32", "f32", 16, seed=71)
s.attend()
s.check()
s = t.Step([1, 3], [300, 20], 8, 2, 64, "f16", "f16", 1, seed=72)
s.attend()
s.check()
print("every wait ended")
"""


def test_waits_end(gpu):
    here = os.path.dirname(os.path.abspath(__file__))
    code = CODE.format(pkg=os.path.join(os.path.dirname(here), "wasm-chord_b200"), tests=here)
    env = dict(os.environ, WCB_TEST_WITHHOLD_COPY="1")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and "every wait ended" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]
