"""Paged operators where CUDA cannot run: what a call reports. In a process without a visible device, so that the addresses below are
never dereferenced."""
import os
import subprocess
import sys

CODE = """
import sys
sys.path.insert(0, {pkg!r})
import wcb
A = 1 << 20
said = set()
for act, cache in ((wcb.KV_F32, wcb.KV_F32), (wcb.KV_F32, wcb.KV_F16), (wcb.KV_F32, wcb.KV_BF16), (wcb.KV_F16, wcb.KV_F16)):
    for q in (1, 500):  # few rows, many rows (the tensor cores)
        kv = wcb.PagedKV(A, A, cache, 8, 16, 4, 64)
        b = wcb.PagedBatch(A, A, A, 2, 2 * q, q, 4)
        for again in range(2):
            try:
                wcb.paged_attention_dev(kv, b, A, A + 4096, act, 8, 512, 512, A, 1 << 40)
                raise SystemExit("it ran")
            except wcb.WcbError as e:
                assert e.code == 5, e.code
                said.add(e.message)
print(len(said), "image" in said.pop())
"""


def test_every_kernel_says_that_there_is_no_device():
    here = os.path.dirname(os.path.abspath(__file__))
    code = CODE.format(pkg=os.path.join(os.path.dirname(here), "wasm-chord_b200"))
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, env=env)
    assert r.returncode == 0 and r.stdout.split() == ["1", "False"], r.stdout + r.stderr[-2000:]
