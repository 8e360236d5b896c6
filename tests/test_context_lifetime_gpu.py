"""What the library keeps for a context does not outlive it: the status words of a driver-API context that is gone."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import ctypes as C
from tornadovm_b200.native import B200Native
from test_context_gpu import Driver
lib, drv, dev, status = B200Native.load(), Driver(), C.c_int(), C.c_int(-1)
drv.ok(drv.cu.cuInit(0), "cuInit")
drv.ok(drv.cu.cuDeviceGet(C.byref(dev), 0), "cuDeviceGet")
for turn in range(3):  # the first status of the process is asked for in a context that ends right after it
    ctx = C.c_void_p()
    drv.ok(drv.cu.cuCtxCreate_v2(C.byref(ctx), 0, dev.value), "cuCtxCreate")
    assert lib.tb200_device_status(C.byref(status)) == 0 and status.value == 0
    drv.ok(drv.cu.cuCtxDestroy_v2(ctx), "cuCtxDestroy")
drv.cu.cuCtxSetCurrent(None)
for _ in range(2):  # the primary context
    assert lib.tb200_device_status(C.byref(status)) == 0 and status.value == 0
print("alive")
"""


def test_status_after_the_context_that_asked_first_is_gone(lib):
    here = os.path.dirname(os.path.abspath(__file__))
    env = {**os.environ, "PYTHONPATH": os.pathsep.join((here, os.path.dirname(here), os.environ.get("PYTHONPATH", "")))}
    run = subprocess.run([sys.executable, "-c", CHILD], env=env, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.endswith("alive\n"), run.stderr[-2000:]
