"""Results that share memory with an operand are refused, in the layouts that the calls accept: rows inside
wider rows too.  The check itself runs on the CPU, against sets of addresses."""
import random

import pytest
import torch

from gemm_b200 import build, ops


@pytest.fixture(scope="module")
def share():
    build.build_extension()
    return ops._ext._share_memory


def addresses(t):
    base = torch.arange(t.untyped_storage().nbytes() // t.element_size())
    index = base.as_strided(t.shape, t.stride(), t.storage_offset()).flatten()
    size = t.element_size()
    return {int(i) * size + b for i in index for b in range(size)}


def test_views_of_one_padded_buffer(share):
    buf = torch.zeros(16, 128, dtype=torch.bfloat16)
    assert share(buf[:, :64], buf[:, :64]) and share(buf[:, :64], buf[:, :40])
    assert share(buf[:, 32:96], buf[:, :64]) and share(buf[:, :64], buf[:, 32:96])
    assert share(buf[3:], buf[:4, 100:]) and share(buf[:1, 8:16], buf[:, 15:20])
    assert not share(buf[:, :64], buf[:, 64:]) and not share(buf[:, 64:], buf[:, :64])
    assert not share(buf[:8, :64], buf[8:, :64]) and not share(buf[:8], buf[8:])
    assert not share(buf[:, 8:16], buf[3:4, 16:24]) and share(buf[:, 8:16], buf[3:4, 15:24])
    assert not share(buf[:, :64], torch.zeros(16, 64).bfloat16())
    stack = torch.zeros(4, 16, 128, dtype=torch.bfloat16)
    assert share(stack[:, :, :64], stack[2, :, 32:96]) and not share(stack[:, :, :64], stack[2, :, 64:])
    assert not share(stack[:2], stack[2:]) and not share(buf[:0], buf) and not share(buf, buf[:, :0])
    assert share(stack[:, 2:9, 8:64], stack[:, 2:9, 8:64])
    assert share(buf[:, :64], buf[:1, :64].expand(16, 64)) and share(buf.view(torch.uint8)[:, :1], buf)


def test_against_sets_of_addresses(share):
    rng = random.Random(1)

    def view(buf):
        rows, pitch = rng.randint(1, 6), rng.choice((12, 12, 12, 16, 7))
        width = rng.randint(1, pitch)
        offset = rng.randint(0, 60)
        if rng.random() < 0.25:
            return buf.as_strided((2, rows, width), (rng.choice((pitch * rows, 84)), pitch, 1), offset)
        if rng.random() < 0.1:
            return buf.as_strided((rows, width), (0, 1), offset)
        return buf.as_strided((rows, width), (pitch, 1), offset)

    exact = 0
    for _ in range(6000):
        buf = torch.zeros(256, dtype=torch.bfloat16)
        a, b = view(buf), view(buf)
        common = bool(addresses(a) & addresses(b))
        assert share(a, b) or not common                      # never passes what overlaps
        if a.dim() == b.dim() == 2 and 0 not in a.stride() + b.stride() and (
                a.stride(0) == b.stride(0) or a.shape[0] == 1 and b.shape[0] == 1):
            if share(a, b) != common:
                # rows wider than what is left of the period, past the other's first or last row
                assert share(a, b) and abs(a.storage_offset() - b.storage_offset()) % a.stride(0) != 0
            else:
                exact += 1
    assert exact > 1000


@pytest.mark.gpu
def test_pitched_results_over_an_operand_are_refused():
    off = torch.tensor([0, 10, 16], dtype=torch.int32, device="cuda")
    buf = torch.zeros(16, 192, device="cuda").bfloat16()
    w = torch.zeros(2, 64, 64, device="cuda").bfloat16()
    for f in (ops.grouped_matmul, ops.grouped_matmul_dx):
        for out in (buf[:, :64], buf[:, 32:96], buf[:, 56:120]):
            with pytest.raises(ValueError, match="share memory"):
                f(buf[:, :64], w, off, out=out)
        f(buf[:, :64], w, off, out=buf[:, 64:128])
        wide = torch.zeros(2, 64, 192, device="cuda").bfloat16()
        with pytest.raises(ValueError, match="share memory"):
            f(buf[:, :64], wide[:, :, :64], off, out=wide.view(128, 192)[8:24, :64])
        f(buf[:, :64], wide[:, :, :64], off, out=wide.view(128, 192)[8:24, 64:128])
        with pytest.raises(ValueError, match="share memory"):
            f(buf[:1, :64], w[:1], off[:2], out=buf[:1, :64])
        with pytest.raises(ValueError, match="share memory"):
            numbers = torch.zeros(64, dtype=torch.int64, device="cuda")
            f(buf[:1, :64], w[:1], numbers[8:10], out=numbers.view(torch.bfloat16)[:64].view(1, 64))
    dw = torch.zeros(2, 64, 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="share memory"):
        ops.grouped_matmul_dw(dw.view(64, 128)[:16, :64], buf[:, :64], off, out=dw)
    q = ops.quantize_mxfp4(buf[:, :64])
    with pytest.raises(ValueError, match="share memory"):
        ops.matmul_mxfp4(q, q, out=q.codes.view(torch.bfloat16))
    torch.cuda.synchronize()
    assert ops.device_status()[0] == 0
