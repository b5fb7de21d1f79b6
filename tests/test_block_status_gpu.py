"""The device's status word: kernels read it in one place, where all threads of a block get one answer, so that they go
on or end together; with it set they write nothing and end."""

import ctypes as C
import os
import re

import pytest
import torch

from tests.block_helpers import normal

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trifast_b200", "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return f.read()


@pytest.mark.parametrize("name", ["ff_gemm.cu", "ff_fused.cu", "tc_bwd_d128.cu", "tc_bwd_db.cu", "tc_bwd_dkv.cu", "tc_bwd_dq.cu", "tc_bwd_fused.cu",
                                  "tc_fwd.cu", "tc_fwd_d128.cu"])
def test_status_is_read_once_a_block(name):
    """A thread that reads the word for itself may see it set where others of its block have not: it would leave them
    waiting at a barrier that counts on it."""
    direct = r"volatile unsigned int\*>\((p\.)?status"
    helper = source("common.cuh").split("bool block_gave_up(")[1].split("}")[0]
    assert "return __syncthreads_or(" in helper and re.search(direct, helper)
    assert "= block_gave_up(status, threadIdx.x == 0);" in source("ff_device.cuh") and not re.search(direct, source("ff_device.cuh"))
    text = source(name)
    if name == "tc_bwd_db.cu":     # (with clusters one thread hands what it has read to the others in shared memory)
        text, ours = re.subn(r"if \(kCluster\) \*skip = \*reinterpret_cast<volatile unsigned int\*>\(status\) != 0u;", "", text)
        assert ours == 1
    assert not re.search(direct, text)
    assert len(re.findall(r"__global__", text)) == len(re.findall(r"(device|block)_gave_up\((p\.)?status\)", text))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,hidden,dtype", [
    (300, 64, 64, torch.bfloat16), (100, 128, 96, torch.float16), (100, 136, 64, torch.bfloat16), (300, 136, 200, torch.bfloat16),
    (300, 264, 264, torch.float16), (40, 24, 64, torch.float32), (300, 136, 64, torch.float32)])
def test_every_product_after_a_kernel_that_gave_up(rows, width, hidden, dtype):
    """Forward and backward, one CTA a tile and pairs of them: nothing is written, the next call raises, the one after is right."""
    from trifast_b200 import _lib, gated_feed_forward
    lib = _lib.load()
    x, dy = normal(rows, width, seed=1, dtype=dtype), normal(rows, width, seed=5, dtype=dtype)
    w = [normal(*s, seed=2, dtype=dtype) for s in ((hidden, width), (hidden, width), (width, hidden))]
    want = gated_feed_forward(x, *w)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    ff = _lib.FeedForward(rows, width, width, width, hidden, width, _lib.DTYPE_CODE[dtype])
    sizes = [lib.trifast_feed_forward_workspace_bytes(C.byref(ff)), lib.trifast_feed_forward_backward_workspace_bytes(C.byref(ff))]
    ws = torch.zeros(max(*sizes, 1), dtype=torch.uint8, device="cuda")
    y, dx = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    dw = [torch.empty_like(t) for t in w]
    at = lambda *ts: [C.c_void_p(t.data_ptr()) for t in ts]
    _lib.check(lib.trifast_debug_wait_probe(1000, stream), "trifast_debug_wait_probe")
    _lib.check(lib.trifast_feed_forward(C.byref(ff), *at(x, *w, y, ws), sizes[0], stream), "trifast_feed_forward")
    _lib.check(lib.trifast_feed_forward_backward(C.byref(ff), *at(dy, x, *w, dx, *dw, ws), sizes[1], stream), "trifast_feed_forward_backward")
    torch.cuda.synchronize()
    assert (y == 7).all() and (dx == 7).all()
    with pytest.raises(RuntimeError, match="gave up"):
        gated_feed_forward(x, *w)
    assert torch.equal(gated_feed_forward(x, *w), want)


@pytest.mark.gpu
@pytest.mark.parametrize("n,d", [(64, 16), (128, 32), (200, 64), (384, 32), (128, 128)])
def test_attention_after_a_kernel_that_gave_up(n, d):
    """The backward's kernels end together too: the call after it raises, and the one after that is right."""
    from trifast_b200 import _lib, triangle_attention
    lib = _lib.load()
    q, k, v, do = (normal(1, 2, n, n, d, seed=s, dtype=torch.bfloat16) for s in range(4))
    b, m = normal(1, 2, n, n, seed=5, dtype=torch.bfloat16), torch.zeros(1, n, n, dtype=torch.bool, device="cuda")
    o, lse = torch.ops.trifast_b200.triangle_attention(q, k, v, b, m)
    grads = lambda: torch.ops.trifast_b200.triangle_attention_grads(do, q, k, v, b, o, lse, m)
    want = [t.clone() for t in grads()]
    torch.cuda.synchronize()
    _lib.check(lib.trifast_debug_wait_probe(1000, C.c_void_p(torch.cuda.current_stream().cuda_stream)), "trifast_debug_wait_probe")
    grads()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="gave up"):
        triangle_attention(q, k, v, b, m)
    assert all(torch.equal(a, b) for a, b in zip(grads(), want))
