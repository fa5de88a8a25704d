"""The exchange of partial sums between the CTAs that share a tile's contraction: many columns and many
tiles per cluster, so that each buffer is filled, read and freed again and again.

The operands are small whole numbers: every partial sum is a whole number below 2^24, exact in fp32 in
any order, so the result has to equal the exact one rounded once to bf16, each time.
"""
import pytest
import torch

from gemm_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[0, 2], ids=["narrow", "middle"])
def tiles(request):
    ops.set_tuning("grouped_kernel", request.param)
    yield request.param
    ops.set_tuning("grouped_kernel", -1)


def whole(*shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-4, 5, shape, generator=g, device="cuda").bfloat16()


@pytest.mark.parametrize("E,ROWS,wide", [(8, 117, 4104), (12, 30, 4104), (30, 5, 2056), (1, 13, 20008)])
@pytest.mark.parametrize("op", ["nt", "dx", "dw", "mx"])
def test_every_buffer_arrives_whole_and_is_read_before_it_is_filled_again(op, E, ROWS, wide, tiles):
    """Eight, four and two buffers; tiles of many and of one column group."""
    N, K = (1096, wide) if op == "dx" else (wide, 1096 if op != "mx" else 1088)
    T = E * ROWS
    off = torch.arange(0, T + 1, ROWS, dtype=torch.int32, device="cuda")
    x, w, dy = whole(T, K, seed=1), whole(E, N, K, seed=2), whole(T, N, seed=3)
    xd, wd, dyd = (t.double().view(E, -1, t.shape[-1]) for t in (x, w, dy))
    if op == "mx":
        qx, qw = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
        xd, wd = ops.dequantize_mxfp4(qx).double().view(E, ROWS, K), ops.dequantize_mxfp4(qw).double()
        call, want = lambda: ops.grouped_matmul_mxfp4(qx, qw, off), xd @ wd.transpose(1, 2)
    elif op == "nt":
        call, want = lambda: ops.grouped_matmul(x, w, off), xd @ wd.transpose(1, 2)
    elif op == "dx":
        call, want = lambda: ops.grouped_matmul_dx(dy, w, off), dyd @ wd
    else:
        call, want = lambda: ops.grouped_matmul_dw(dy, x, off), dyd.transpose(1, 2) @ xd
    assert float(want.abs().max()) < 2 ** 24
    want = want.bfloat16()
    for _ in range(20):
        got = call()
        assert torch.equal(got.view(want.shape), want)
    assert ops.device_status()[0] == 0
