"""The large LDS of the product and of attention is asked for on every device that launches them,
and again after a failure. The runtime is a stand-in that counts: no GPU."""
import os
import subprocess
import sys

from conftest import ROOT

STUB = r"""
#include <cstddef>
struct Dim { unsigned x, y, z; };
static int device, asked, launched, refuse;
extern "C" {
int hipGetDevice(int* d) { *d = device; return 0; }
int hipFuncSetAttribute(const void*, int, int) { ++asked; return refuse; }
int __hipPushCallConfiguration(Dim, Dim, size_t, void*) { return 0; }
int __hipPopCallConfiguration(Dim*, Dim*, size_t*, void**) { return 0; }
int hipLaunchKernel(const void*, Dim, Dim, void**, size_t, void*) { ++launched; return 0; }
int hipGetLastError() { return 0; }
void stub_set(int d, int r) { device = d; refuse = r; }
int stub_asked() { return asked; }
int stub_launched() { return launched; }
}
"""

PROGRAM = r"""
import ctypes, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
from perm_amd import _lib
lib = ctypes.CDLL(_lib.LIB_PATH)
for name, (res, args) in _lib.SIGNATURES.items():
    f = getattr(lib, name)
    f.restype, f.argtypes = res, args
P = 1 << 20
cache = _lib.KvCacheDesc(P, P, P, P, 4, 2, 16, 64)
def matmul():
    return lib.cp_mx4_matmul(P, P, 64, P, P, 64, 64, P, 1, P, 1 << 40, None)
def attend():
    return lib.cp_kv_attention(ctypes.byref(cache), P, 256, 64, 1, 4096, 4, P, 1, 4096, P, P, 1, 0, 1.0, P, None, P,
                               1 << 40, None)
for call in (matmul, attend):
    a0 = stub.stub_asked()
    stub.stub_set(0, 1)
    first = call()
    assert first == _lib.CP_ERR_HIP, first  # refused: nothing is launched, and it is asked again
    stub.stub_set(0, 0)
    assert [call(), call()] == [0, 0] and stub.stub_asked() == a0 + 2
    stub.stub_set(3, 0)
    assert [call(), call()] == [0, 0] and stub.stub_asked() == a0 + 3
    stub.stub_set(0, 0)
    assert call() == 0 and stub.stub_asked() == a0 + 3
assert stub.stub_launched() >= 10
print("ok")
"""


def test_every_device_is_asked(tmp_path):
    src, so, prog = (tmp_path / n for n in ("stub.cpp", "stub.so", "prog.py"))
    src.write_text(STUB)
    prog.write_text(PROGRAM)
    subprocess.run(["g++", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    r = subprocess.run([sys.executable, str(prog), str(so), ROOT], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONDONTWRITEBYTECODE="1"))
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr
