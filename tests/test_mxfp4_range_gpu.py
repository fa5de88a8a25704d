"""Every scale byte with every code: dequantised exactly where bf16 holds the value, Inf where it is 2^128 or
more, NaN for scale 255."""
import pytest
import torch

from gemm_b200 import ops

pytestmark = pytest.mark.gpu


def test_every_scale_and_code():
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    grid = torch.cat((grid, -grid))
    codes = (torch.arange(16, dtype=torch.uint8) | torch.arange(16, dtype=torch.uint8).flip(0) << 4).repeat(256, 1)
    scales = torch.zeros(2, 1, 32, 4, 4, dtype=torch.uint8)
    s = torch.arange(256)
    scales[s // 128, 0, s % 32, s % 128 // 32, 0] = s.to(torch.uint8)
    got = ops.dequantize_mxfp4(ops.MxFp4(codes.cuda(), scales.cuda())).cpu()
    value = torch.stack((grid[(codes % 16).long()], grid[(codes // 16).long()]), -1).flatten(-2)
    want = value * torch.exp2(s.double() - 127)[:, None]
    limit = 2.0 ** 128
    want = torch.where(want.abs() >= limit, torch.sign(want) * float("inf"), want)
    assert torch.isnan(got[255]).all()
    assert torch.equal(got[:255].double(), want[:255])
    assert torch.isfinite(got[:253]).all() and torch.isinf(got[253]).any() and torch.isinf(got[254]).any()
    # what the quantisation writes for the largest numbers there are
    top = torch.full((1, 32), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device="cuda")
    for x in (top, torch.full((1, 32), torch.finfo(torch.float32).max, device="cuda")):
        q = ops.quantize_mxfp4(x)
        assert int(q.scales.max()) == 252 and torch.isfinite(ops.dequantize_mxfp4(q)).all()
