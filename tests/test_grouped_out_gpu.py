"""A result written into the caller's tensor (out=) counts as an in-place change: a backward pass that saved
the earlier values is refused instead of using the new ones."""
import pytest
import torch

from gemm_b200 import ops

pytestmark = pytest.mark.gpu


def calls():
    x = torch.randn(16, 64, device="cuda").bfloat16()
    w = torch.randn(2, 64, 64, device="cuda").bfloat16()
    off = torch.tensor([0, 10, 16], dtype=torch.int32, device="cuda")
    q, qw = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    dense = ops.MxFp4(qw.codes[0], qw.scales[0])
    yield (16, 64), lambda out: ops.grouped_matmul(x, w, off, out=out)
    yield (16, 64), lambda out: ops.grouped_matmul_dx(x, w, off, out=out)
    yield (2, 64, 64), lambda out: ops.grouped_matmul_dw(x, x, off, out=out)
    yield (16, 64), lambda out: ops.matmul_mxfp4(q, dense, out=out)
    yield (16, 64), lambda out: ops.grouped_matmul_mxfp4(q, qw, off, out=out)


def test_saved_values_that_were_overwritten_are_noticed():
    for shape, call in calls():
        out = torch.ones(shape, device="cuda").bfloat16()
        leaf = torch.ones(shape, device="cuda").bfloat16().requires_grad_()
        loss = (out * leaf).sum()
        version = out._version
        assert call(out) is out and out._version == version + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        part = torch.zeros((3, *shape), device="cuda").bfloat16()
        version = part._version
        call(part[1])
        assert part._version == version + 1 and torch.equal(part[1], out)      # a view counts for its base
        with torch.inference_mode():
            mine = torch.zeros(shape, device="cuda").bfloat16()
            call(mine)
            call(out)
        assert torch.equal(mine, out)
