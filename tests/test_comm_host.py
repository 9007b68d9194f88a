"""What an all-reduce, which writes its tensor in place, leaves of what the library knows of that tensor; without a device, and with
an NCCL that does nothing."""
import ctypes
import os
import subprocess
import sys

import numpy as np

from conftest import ROOT, cg

NCCL = """
int calls;
int ncclGetUniqueId(void* a) { return 0; }
int ncclCommInitRank(void* a, int n, ...) { return 0; }
int ncclCommDestroy(void* a) { return 0; }
int ncclAllReduce(const void* a, void* b, unsigned long n, int t, int o, void* c, void* s) { ++calls; return 0; }
int ncclAllGather(const void* a, void* b, unsigned long n, int t, void* c, void* s) { return 0; }
int ncclReduceScatter(const void* a, void* b, unsigned long n, int t, int o, void* c, void* s) { return 0; }
const char* ncclGetErrorString(int e) { return "none"; }
"""


def test_all_reduce_says_that_it_writes(tmp_path):
    """The rounded copy is dropped, none is kept again, a literal's value is forgotten, and what was recorded runs first (here: cannot).  In a
    process of its own, whose libnccl.so.2 is the one above."""
    cg.load_library()
    csrc, cuda = os.path.join(ROOT, "catgrad-rs_b200", "csrc"), os.environ.get("CUDA_HOME", "/usr/local/cuda")
    (tmp_path / "nccl.c").write_text(NCCL)
    subprocess.check_call(["gcc", "-fPIC", "-shared", str(tmp_path / "nccl.c"), "-o", str(tmp_path / "libnccl.so.2")])
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-I", csrc, "-I", f"{cuda}/include", os.path.join(ROOT, "tests", "comm_host.cpp"), "-o",
                           str(tmp_path / "comm_host.so"), cg.library_path(), f"-Wl,-rpath,{os.path.dirname(cg.library_path())}", "-L", f"{cuda}/lib64", "-lcudart"])
    env = {**os.environ, "LD_LIBRARY_PATH": f"{tmp_path}:{os.environ.get('LD_LIBRARY_PATH', '')}"}
    r = subprocess.run([sys.executable, __file__, str(tmp_path), cg.library_path()], env=env, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


def child(folder, library):
    L, lib, nccl = ctypes.CDLL(f"{folder}/comm_host.so"), ctypes.CDLL(library), ctypes.CDLL(f"{folder}/libnccl.so.2")
    vp = ctypes.c_void_p
    L.host_ctx.restype = L.host_tensor.restype = vp
    L.host_tensor.argtypes = [vp, ctypes.c_uint64, ctypes.c_int, ctypes.c_int, vp, vp]
    calls = ctypes.c_int.in_dll(nccl, "calls")

    def tensor(c, n):
        one = np.int64([n]), np.int64([1])
        t = vp(L.host_tensor(c, 1 << 40, 0, 1, one[0].ctypes.data, one[1].ctypes.data))
        L.host_known(t)
        return t

    c = vp(L.host_ctx())
    L.host_comm(c)
    t = tensor(c, 1)
    assert L.host_knows(t) == 1 | 2
    assert lib.cg_comm_all_reduce(c, t) == 0 and calls.value == 1
    assert L.host_knows(t) == 4
    # recorded mode: a call that is waiting runs first (without a device it fails, and nothing is reduced)
    assert lib.cg_set_option(c, b"lazy", ctypes.c_int64(1)) == 0
    t, out = tensor(c, 0), vp()
    assert lib.cg_neg(c, t, ctypes.byref(out)) == 0

    def pending():
        n = [ctypes.c_int64() for _ in range(3)]
        assert lib.cg_lazy_stats(c, *(ctypes.byref(x) for x in n)) == 0
        return n[2].value

    assert pending() == 1
    lib.cg_comm_all_reduce(c, t)
    assert pending() == 0
    # a recorded result itself, of this context and of another one
    assert lib.cg_neg(c, tensor(c, 0), ctypes.byref(out)) == 0 and pending() == 1
    other = vp(L.host_ctx())
    L.host_comm(other)
    before = calls.value
    assert lib.cg_comm_all_reduce(other, out) == 3 and calls.value == before and pending() == 1
    lib.cg_comm_all_reduce(c, out)
    assert pending() == 0


if __name__ == "__main__":
    child(*sys.argv[1:])
