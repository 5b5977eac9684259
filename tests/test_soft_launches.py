"""Every launch of the soft-correspondence entry points, judged on the CPU: the runtime's launch call is replaced by a recorder
(launch_recorder.c), so that the argument checks, plans and launchers run as they would on the card and nothing is started."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def recorder(tmp_path_factory):
    path = tmp_path_factory.mktemp("recorder") / "librecorder.so"
    subprocess.check_call(["gcc", "-O1", "-Wall", "-shared", "-fPIC", os.path.join(HERE, "launch_recorder.c"), "-o", str(path)])
    return str(path)


# In a process of its own: the recorder has to be there before the library.  The pointers stand for device memory, which the
# host side never reads.
CALLS = """
import ctypes, sys
rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
rec.recorder_fault.restype = ctypes.c_char_p
sys.path.insert(0, sys.argv[2])
from pose_estimation_amd import _abi
lib, at = _abi.lib, 1 << 30

def judged(name, rc, **call):
    if rc:
        print(name, call, "status", rc, lib.ispa_last_error().decode())
    if rec.recorder_fault():
        print(name, call, rec.recorder_fault().decode())
    launches = rec.recorder_launches()
    rec.recorder_clear()
    return launches

def forward(dtype, b, heads, d, dv, nq, cells, own, cap=0.0, falloff=None):
    need = lib.ispa_soft_match_workspace_bytes(dtype, b, heads, d, dv, nq, 1, cells)
    rc = lib.ispa_soft_match(at, at, at if own else None, dtype, b, heads, d, dv, nq, cells, 8, 1.0, cap, falloff, None, None, None, at,
                             None, at, at, need, None)
    return judged("forward", rc, dtype=dtype, b=b, heads=heads, d=d, dv=dv, nq=nq, cells=cells, own=own, cap=cap, falloff=falloff)

def backward(dtype, b, heads, d, dv, nq, cells, own, cap=0.0, falloff=None):
    need = lib.ispa_soft_match_backward_workspace_bytes(dtype, b, heads, d, dv, nq, cells)
    some = at if nq else None
    rc = lib.ispa_soft_match_backward(some, at, at if own else None, dtype, b, heads, d, dv, nq, cells, 8, 1.0, cap, falloff, None,
                                      None, None, some, some, some, None, some, at, at if own else None, at, need, None)
    return judged("backward", rc, dtype=dtype, b=b, heads=heads, d=d, dv=dv, nq=nq, cells=cells, own=own, cap=cap, falloff=falloff)
"""


def run(recorder, calls):
    done = subprocess.run([sys.executable, "-c", CALLS + calls, recorder, os.path.dirname(HERE)], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr
    *faults, last = done.stdout.splitlines()
    assert not faults, "\n".join(faults[:20])
    assert int(last) > 0                                     # launches that were recorded


def test_gradients_without_queries(recorder):
    run(recorder, """
n = 0
for dtype in (_abi.F32, _abi.BF16):
    for own in (False, True):
        for d in (16, 64, 128, 256):
            for cells in (1, 60, 4096):
                n += backward(dtype, 2, 1, d, d, 0, cells, own)
print(n)
""")


@pytest.mark.parametrize("own_first", [False, True])
def test_lds_of_every_kernel_form(recorder, own_first):
    """The same kernel serves calls with and without a value map, which take different amounts of LDS, in either order."""
    run(recorder, f"""
n = 0
for own in {(True, False) if own_first else (False, True)}:
    for dtype in (_abi.F32, _abi.BF16):
        for d in (16, 64, 128, 256):
            for nq in (1, 9, 64, 65, 500):
                for cap, falloff in ((0.0, None), (5.0, None), (0.0, at), (50.0, at)):
                    n += forward(dtype, 2, 1, d, d, nq, 4096, own, cap, falloff)
                    n += backward(dtype, 2, 1, d, d, nq, 4096, own, cap, falloff)
                    n += forward(dtype, 1, 2, d, d, nq, 60, own, cap, falloff) + backward(dtype, 1, 2, d, d, nq, 60, own, cap, falloff)
print(n)
""")
