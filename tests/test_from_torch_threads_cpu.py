"""The first from_torch of a process on two threads at once, under an import hook that lets
other threads run: what is looked up once must not be waited for with the interpreter's
lock held."""
import subprocess
import sys

import pytest

CHILD = """
import builtins, threading, time
import torch
import tensorplay_amd as tp
plain = builtins.__import__
def hooked(name, *a, **k):
    if name == "torch":
        time.sleep(0.5)      # as a tracer's hook may: the other thread runs now
    return plain(name, *a, **k)
builtins.__import__ = hooked
got = [None, None]
def call(i):
    got[i] = tp.from_torch(torch.full((3,), float(i))).numpy().tolist()
threads = [threading.Thread(target=call, args=(i,)) for i in range(2)]
for t in threads: t.start()
for t in threads: t.join()
assert got == [[0.0] * 3, [1.0] * 3], got
print("ok")
"""


def test_first_calls_of_two_threads():
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", CHILD], capture_output=True, text=True, timeout=90)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
