"""Host tensors leave the HIP runtime alone: a process may make them and fork, or choose
its devices, before it asks for the first device tensor."""
import subprocess
import sys

SHIM = """
static int calls, devices;
extern "C" int hipGetDeviceCount(int* n) { ++calls; *n = devices; return devices ? 0 : 100; }
extern "C" int shim_calls() { return calls; }
extern "C" void shim_devices(int n) { devices = n; }
"""

CHILD = """
import ctypes, sys
shim = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)   # its hipGetDeviceCount comes first
import numpy as np
import tensorplay_amd as tp
before = shim.shim_calls()
t = tp.tensor(np.arange(6, dtype=np.float32).reshape(2, 3))
tp.empty([4, 4]).copy_(tp.empty([4, 4]))
assert t.transpose(0, 1).contiguous().numpy()[2, 1] == 5.0
assert shim.shim_calls() == before, "a host tensor asked for devices"
def refusal():
    try:
        tp.empty([2], device="rocm:0")
    except RuntimeError as e:
        return str(e)
assert "not available" in refusal() and shim.shim_calls() > before
shim.shim_devices(1)   # no device at first does not mean none later
assert not tp.rocm.is_available() or "not available" not in str(refusal())
assert tp.rocm.is_available()
print("ok")
"""


def test_host_tensors_do_not_ask_for_devices(tmp_path):
    src, lib = tmp_path / "shim.cpp", tmp_path / "libshim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-shared", "-fPIC", "-o", str(lib), str(src)], check=True)
    r = subprocess.run([sys.executable, "-c", CHILD, str(lib)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
