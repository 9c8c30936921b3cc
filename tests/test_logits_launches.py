"""CPU tests of what the operators on logits launch: a host library with its own hipLaunchKernel, loaded in front of the HIP
runtime in a process of its own, notes every launch instead of making it."""

import json
import subprocess
import sys

import pytest

from distributions_amd import _lib
from distributions_amd._lib import BF16, F32, F64

RECORDER = r"""
#include <cstddef>
#include <cstdint>
struct dim { uint32_t x, y, z; };  // dim3
struct launch { uint32_t grid, block; uint64_t first; };  // workgroups, threads, the first 8 bytes of the arguments
extern "C" {
launch noted[64];
int count = 0;
dim pushed[2];
int __hipPushCallConfiguration(dim grid, dim block, size_t, void *) {
  pushed[0] = grid, pushed[1] = block;
  return 0;
}
int __hipPopCallConfiguration(dim *grid, dim *block, size_t *lds, void **stream) {
  *grid = pushed[0], *block = pushed[1], *lds = 0, *stream = nullptr;
  return 0;
}
int hipLaunchKernel(const void *, dim grid, dim block, void **args, size_t, void *) {
  if (count < 64) noted[count] = launch{grid.x, block.x, *(uint64_t *)args[0]};
  ++count;
  return 0;
}
int hipGetLastError() { return 0; }
}
"""

CALL = r"""
import ctypes, json, sys
sys.path.insert(0, sys.argv[3])
recorder = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
L = ctypes.CDLL(sys.argv[2])
from distributions_amd._lib import LogitAdjust
class Launch(ctypes.Structure):
    _fields_ = [("grid", ctypes.c_uint32), ("block", ctypes.c_uint32), ("first", ctypes.c_uint64)]
rows, k, dtype, bias_dtype, history = json.loads(sys.argv[4])
L.m355_logits_adjust_grad_workspace_bytes.restype = ctypes.c_size_t
L.m355_logits_adjust_grad_workspace_bytes.argtypes = [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
vp, i64, i32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int
L.m355_logits_adjust_grad.argtypes = [i64, i64, i32, vp, i64, vp, i64, ctypes.c_char_p, vp, vp, vp, ctypes.c_size_t, vp]
d = LogitAdjust()
for o, v in ((d.repetition, 1.0), (d.presence, 0.0), (d.frequency, 0.0), (d.temperature, 1.0)):
    o.scalar, o.div, o.mod = v, 1, 1
d.bias, d.bias_dtype = 4096, bias_dtype
if history:
    d.history, d.history_len, d.history_stride, d.history_dtype = 4096, 7, 7, 2
need = L.m355_logits_adjust_grad_workspace_bytes(rows, k, dtype)
rc = L.m355_logits_adjust_grad(rows, k, dtype, 4096, k, 4096, k, bytes(d), 4096, 4096, 8192 if need else None, need, None)
n = ctypes.c_int.in_dll(recorder, "count").value
noted = (Launch * 64).in_dll(recorder, "noted")
print(json.dumps([rc, need, [[e.grid, e.block, e.first] for e in noted[:n]]]))
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """rc, workspace bytes and [grid, threads, first argument's first word] per launch (the partial sums' address for the one that
    joins them) of an adjust_grad with a shared bias and
    exactly the workspace that is asked for."""
    where = tmp_path_factory.mktemp("recorder")
    (where / "recorder.cpp").write_text(RECORDER)
    so = str(where / "recorder.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-o", so, str(where / "recorder.cpp")], check=True)
    root = _lib._HERE.rsplit("/", 1)[0]

    def call(*case):
        p = subprocess.run([sys.executable, "-c", CALL, so, _lib.LIB_PATH, root, json.dumps(case)], capture_output=True, text=True,
                           timeout=120)
        assert p.returncode == 0, p.stderr
        return json.loads(p.stdout.splitlines()[-1])

    return call


@pytest.mark.parametrize("history", [False, True])
@pytest.mark.parametrize("dtype, bias", [(F32, F32), (F64, F64), (BF16, F32)])
def test_shared_bias_gradient_of_no_rows(launches, dtype, bias, history):
    """No rows: nothing but the fill of the bias' gradient runs, and it reads no workspace (none is asked for)."""
    k = 1000
    rc, need, made = launches(0, k, dtype, bias, history)
    assert rc == 0 and need == 0
    assert made == [[(k + 63) // 64, 256, 0]]
    assert launches(5, k, dtype, bias, history)[2] != made  # the recorder sees the others
