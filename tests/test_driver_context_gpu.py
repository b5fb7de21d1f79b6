"""The C ABI in a program of the driver API, with a context of its own current: the calls run in it and leave it current."""

import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = r"""
import ctypes as C
import torch
from oracle import block_oracle
from tests.block_helpers import U, assert_bounded, normal
from tests.test_feed_forward_gpu import bounds
from trifast_b200 import _lib

cuda = C.CDLL("libcuda.so.1")
def ok(rc):
    assert rc == 0, rc
ok(cuda.cuInit(0))
dev, ctx, now = C.c_int(), C.c_void_p(), C.c_void_p()
ok(cuda.cuDeviceGet(C.byref(dev), 0))
ok(cuda.cuCtxCreate_v2(C.byref(ctx), 0, dev))
lib = _lib.load()

def there(t):
    p = C.c_uint64()
    ok(cuda.cuMemAlloc_v2(C.byref(p), C.c_size_t(max(t.numel() * t.element_size(), 256))))
    ok(cuda.cuMemcpyHtoD_v2(p, C.c_void_p(t.data_ptr()), C.c_size_t(t.numel() * t.element_size())))
    return C.c_void_p(p.value)
def back(p, like):
    t = torch.empty_like(like)
    ok(cuda.cuCtxSynchronize())
    ok(cuda.cuMemcpyDtoH_v2(C.c_void_p(t.data_ptr()), C.c_uint64(p.value), C.c_size_t(t.numel() * t.element_size())))
    return t
def mine():
    ok(cuda.cuCtxGetCurrent(C.byref(now)))
    return now.value == ctx.value

x = normal(6, 7, 24, seed=1, device="cpu")
px, py = there(x), there(torch.zeros_like(x))
d = _lib.Dropout(outer=1, mid=1, inner=x.numel(), dtype=0, p=0.5, seed=3, offset=0)
ok(lib.trifast_dropout_add(C.byref(d), None, px, None, py, None))
assert torch.equal(back(py, x), torch.where(block_oracle.keep_mask(x.shape, 0.5, 3), 2 * x, torch.zeros_like(x))) and mine()

x = normal(64, 64, seed=1, device="cpu", dtype=torch.bfloat16)
w = [normal(64, 64, seed=2 + i, device="cpu", dtype=torch.bfloat16, std=0.125) for i in range(3)]
ff = _lib.FeedForward(64, 64, 64, 64, 64, 64, 1)
size = lib.trifast_feed_forward_workspace_bytes(C.byref(ff))
args = [there(t) for t in (x, *w, torch.zeros_like(x), torch.zeros(max(size, 1), dtype=torch.uint8))]
ok(lib.trifast_feed_forward(C.byref(ff), *args, C.c_size_t(size), None))
want, bound = bounds(torch.zeros_like(x), x, *w)
assert_bounded(back(args[4], x), want[0], bound[0], "y")
assert mine()
print("in its own context")
"""


@pytest.mark.gpu
def test_in_a_context_of_the_callers_own():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": ROOT})
    assert r.returncode == 0 and "in its own context" in r.stdout, r.stdout + r.stderr
