"""MXFP4: conversion and products against a plain implementation in 64 bits.

Conversion is exact arithmetic (powers of two and one rounding to a grid), so codes, scales and
values are compared for equality.  A product of two codes and two scales is exact in fp32; the sum
of K of them is accumulated in fp32 and rounded once to bf16:
|y - exact| <= 2^-8 |exact| + 2 K 2^-23 sum |a b|.
"""
import pytest
import torch

from gemm_b200 import ops

pytestmark = pytest.mark.gpu
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def scale_bytes(q):
    """Scales as [.., rows, K/32]."""
    rows, blocks = q.codes.shape[-2], q.codes.shape[-1] // 16
    r = torch.arange(rows, device="cuda")[:, None]
    b = torch.arange(blocks, device="cuda")[None, :]
    return q.scales[..., r // 128, b // 4, r % 32, r % 128 // 32, b % 4]


def values(q):
    """What an MxFp4 stands for, in 64 bits."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float64, device="cuda")
    v = torch.stack((grid[(q.codes % 16).long()], grid[(q.codes // 16).long()]), -1).flatten(-2)
    s = scale_bytes(q).double()
    s = torch.where(s == 255, torch.full_like(s, float("nan")), torch.exp2(s - 127))
    return v * s.repeat_interleave(32, -1)


def plain_quantize(x):
    """(values, scale bytes) of x by the format's rule, in 64 bits."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1].double() - 3, torch.full_like(top, -127.0)).clamp(-127, 127)
    s = torch.exp2(e)[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    u = (b / s).abs()
    low, high = torch.bucketize(u, mid), torch.bucketize(u, mid, right=True)
    v = grid[torch.where(low % 2 == 0, low, high)] * s
    return torch.where(b < 0, -v, v).flatten(-2), (e + 127).to(torch.uint8)


def make(*shape, seed=1, dtype=torch.bfloat16, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    # block scales that differ along both axes, so that a misplaced one shows
    return (x * torch.exp2(torch.round(spread * torch.randn(*shape[:-1], shape[-1] // 32, 1, generator=g, device="cuda"))
                           ).expand(*shape[:-1], shape[-1] // 32, 32).flatten(-2)).to(dtype)


def assert_product(got, want, mag, K):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape and torch.isfinite(got).all()
    err = (got.double() - want).abs()
    bound = want.abs() * 2.0 ** -8 + 2 * K * 2.0 ** -23 * mag
    assert bool((err <= bound).all()), float((err - bound).max())
    assert ops.device_status()[0] == 0


@pytest.fixture(params=[-1, 0, 2, 1], ids=["auto", "narrow", "middle", "wide"])
def tiles(request):
    ops.set_tuning("grouped_kernel", request.param)
    yield request.param
    ops.set_tuning("grouped_kernel", -1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 32), (33, 64), (128, 128), (130, 160), (257, 416), (16, 8192),
                                   (3, 65, 96), (2, 128, 544)])
def test_conversion(shape, dtype):
    x = make(*shape, dtype=dtype, spread=8.0)
    q = ops.quantize_mxfp4(x)
    want, s = plain_quantize(x)
    assert torch.equal(scale_bytes(q), s)
    assert torch.equal(values(q), want)
    back = ops.dequantize_mxfp4(q)
    assert back.dtype == torch.bfloat16 and torch.equal(back.double(), want)
    # padding of the scale tiles is zero
    assert int(q.scales.long().sum()) == int(s.long().sum())


def test_ties_saturation_and_the_ends_of_the_range():
    rows = [
        [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0, 6.9, 7.0],   # scale 1
        [7.99, 5.01, 4.99, 0.2501, 0.2499, -0.75, 1.0, 0.0, -0.0, 2.0],
        [2.0 ** -126, 2.0 ** -127, 2.0 ** -128, 2.0 ** -129, -(2.0 ** -133)],  # subnormals
        [0.0, -0.0],
        [3.3e38, 1.0, -3.3e38, 2.0 ** 126],
        [2.0 ** -125, 2.0 ** -128],
    ]
    x = torch.zeros(len(rows), 32)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r, dtype=torch.float64).float()
    for dtype in (torch.float32, torch.bfloat16):
        xd = x.to(dtype).cuda()
        q = ops.quantize_mxfp4(xd)
        want, s = plain_quantize(xd)
        assert torch.equal(scale_bytes(q), s) and torch.equal(values(q), want)
        assert torch.equal(ops.dequantize_mxfp4(q).double(), want)


def test_infinities_and_nan_take_their_block_only():
    x = make(40, 128)
    x[3, 70], x[20, 5], x[39, 127] = float("nan"), float("inf"), -float("inf")
    q = ops.quantize_mxfp4(x)
    bad = torch.zeros(40, 4, dtype=torch.bool, device="cuda")
    bad[3, 2] = bad[20, 0] = bad[39, 3] = True
    assert torch.equal(scale_bytes(q) == 255, bad)
    back = ops.dequantize_mxfp4(q)
    assert torch.equal(torch.isnan(back), bad.repeat_interleave(32, -1))
    good = ~bad.repeat_interleave(32, -1)
    want = plain_quantize(torch.where(good, x, torch.zeros_like(x)))[0]
    assert torch.equal(back.double()[good], want[good])
    # and the rows of a product that they are in
    b = ops.quantize_mxfp4(make(72, 128, seed=2))
    y = ops.matmul_mxfp4(q, b)
    assert torch.equal(torch.isnan(y), bad.any(1)[:, None].expand(40, 72))


def test_strided_input():
    big = make(2, 70, 192)
    for view in (big[:, :, 64:160], big[:, 3:50, :64], big[:, ::2, 8:136], big[1, :, 32:64]):
        q = ops.quantize_mxfp4(view)
        want, s = plain_quantize(view)
        assert torch.equal(scale_bytes(q), s) and torch.equal(values(q), want)


@pytest.mark.parametrize("M,N,K", [(1, 1, 64), (1, 128, 128), (16, 128, 256), (33, 200, 192), (128, 72, 320),
                                   (129, 257, 448), (300, 1001, 2048), (257, 640, 8192), (1000, 130, 64)])
def test_product(M, N, K, tiles):
    a, b = ops.quantize_mxfp4(make(M, K)), ops.quantize_mxfp4(make(N, K, seed=2))
    va, vb = values(a), values(b)
    assert_product(ops.matmul_mxfp4(a, b), va @ vb.t(), va.abs() @ vb.abs().t(), K)


def test_product_of_every_scale_byte_and_code(tiles):
    """Scales from 2^-60 to 2^60 and codes drawn evenly; padding bytes of the scales are NaN."""
    g = torch.Generator(device="cuda").manual_seed(3)

    def raw(rows, K):
        codes = torch.randint(0, 256, (rows, K // 2), generator=g, device="cuda").to(torch.uint8)
        scales = torch.full((-(-rows // 128), -(-K // 128), 32, 4, 4), 255, dtype=torch.uint8, device="cuda")
        r = torch.arange(rows, device="cuda")[:, None]
        b = torch.arange(K // 32, device="cuda")[None, :]
        scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = \
            torch.randint(67, 188, (rows, K // 32), generator=g, device="cuda").to(torch.uint8)
        return ops.MxFp4(codes, scales)

    a, b = raw(70, 320), raw(136, 320)
    va, vb = values(a), values(b)
    assert_product(ops.matmul_mxfp4(a, b), va @ vb.t(), va.abs() @ vb.abs().t(), 320)


def test_rows_inside_a_wider_result(tiles):
    a, b = ops.quantize_mxfp4(make(40, 128)), ops.quantize_mxfp4(make(77, 128, seed=2))
    wide = torch.full((42, 80), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.matmul_mxfp4(a, b, out=wide[1:41, 1:78])
    assert torch.equal(wide[1:41, 1:78], ops.matmul_mxfp4(a, b))
    wide[1:41, 1:78] = 7.0
    assert (wide == 7).all()


def test_empty_operands():
    a, b = ops.quantize_mxfp4(make(0, 64)), ops.quantize_mxfp4(make(5, 64))
    assert ops.matmul_mxfp4(a, b).shape == (0, 5) and ops.matmul_mxfp4(b, a).shape == (5, 0)
    none = ops.quantize_mxfp4(torch.empty(5, 0, device="cuda"))
    assert ops.dequantize_mxfp4(none).shape == (5, 0)
    assert (ops.matmul_mxfp4(none, none) == 0).all()


COUNTS = {"one": [1], "short": [3, 0, 1, 7, 2], "edges": [127, 1, 129, 0, 255, 5], "long": [700, 0, 333],
          "many": [i % 4 for i in range(120)]}


@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS.keys())
@pytest.mark.parametrize("N,K", [(8, 64), (200, 448), (264, 1024)])
def test_grouped_product(counts, N, K, tiles):
    head, tail = 5, 9
    E, T = len(counts), head + sum(counts) + tail
    ends = [head]
    for c in counts:
        ends.append(ends[-1] + c)
    x = make(T, K)
    x[:head], x[T - tail:] = float("nan"), float("inf")       # rows of no group
    x, w = ops.quantize_mxfp4(x), ops.quantize_mxfp4(make(E, N, K, seed=2))
    off = torch.tensor(ends, dtype=torch.int32, device="cuda")
    got = ops.grouped_matmul_mxfp4(x, w, off)
    vx, vw = values(x), values(w)
    want = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(want)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        want[a:b], mag[a:b] = vx[a:b] @ vw[e].t(), vx[a:b].abs() @ vw[e].abs().t()
    assert_product(got, want, mag, K)
    mine = torch.full_like(got, 7.0)
    ops.grouped_matmul_mxfp4(x, w, off.long(), out=mine)
    assert (mine[:head] == 7).all() and (mine[T - tail:] == 7).all()
    assert torch.equal(mine[head:T - tail], got[head:T - tail])


def test_a_layer_captured_with_its_quantisation():
    """Quantise, multiply by group: replayed with other rows and other groups."""
    T, N, K, E = 90, 264, 320, 3
    w = ops.quantize_mxfp4(make(E, N, K, seed=2))
    x, off = make(T, K), torch.tensor([0, 90, 90, 90], dtype=torch.int32, device="cuda")
    y = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")

    def body():
        ops.grouped_matmul_mxfp4(ops.quantize_mxfp4(x), w, off, out=y)

    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for seed, ends in ((5, [0, 30, 30, 90]), (6, [0, 1, 89, 90])):
        x.copy_(make(T, K, seed=seed))
        off.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        eager = ops.grouped_matmul_mxfp4(ops.quantize_mxfp4(x), w, off)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        vx, vw = values(ops.quantize_mxfp4(x)), values(w)
        want = torch.cat([vx[a:b] @ vw[e].t() for e, (a, b) in enumerate(zip(ends, ends[1:]))])
        mag = torch.cat([vx[a:b].abs() @ vw[e].abs().t() for e, (a, b) in enumerate(zip(ends, ends[1:]))])
        assert_product(y, want, mag, K)


def test_refusals_on_the_device():
    a, b = ops.quantize_mxfp4(make(10, 64)), ops.quantize_mxfp4(make(12, 128))
    with pytest.raises(ValueError):                     # K differs
        ops.matmul_mxfp4(a, b)
    with pytest.raises(ValueError):                     # K % 32
        ops.quantize_mxfp4(torch.zeros(4, 40, device="cuda"))
    with pytest.raises(TypeError):
        ops.quantize_mxfp4(torch.zeros(4, 64, device="cuda").half())
    with pytest.raises(ValueError):                     # strided along K
        ops.quantize_mxfp4(torch.zeros(64, 64, device="cuda").t())
    with pytest.raises(TypeError):
        ops.matmul_mxfp4(a.codes, b)
    with pytest.raises(ValueError):                     # scales of another shape
        ops.matmul_mxfp4(ops.MxFp4(a.codes, a.scales[:, :, :16]), a)
    with pytest.raises(TypeError):
        ops.matmul_mxfp4(ops.MxFp4(a.codes, a.scales.int()), a)
    odd = ops.quantize_mxfp4(make(10, 96))
    with pytest.raises(ops.NeoGemmError):               # K % 64
        ops.matmul_mxfp4(odd, odd)
    with pytest.raises(ops.NeoGemmError):               # rows that do not start on 16 bytes
        ops.quantize_mxfp4(torch.zeros(4, 104, device="cuda")[:, 2:66])
    with pytest.raises(ValueError):
        ops.grouped_matmul_mxfp4(a, a, torch.tensor([0, 10], dtype=torch.int32, device="cuda"))


def test_tensors_of_more_than_2_31_values():
    """Conversion there and back, and a product whose result passes 32 bits."""
    x = make(64, 8192)
    big = x.repeat(4200, 1)                      # 2.2e9 values
    q = ops.quantize_mxfp4(big)
    want = ops.dequantize_mxfp4(ops.quantize_mxfp4(x))
    back = ops.dequantize_mxfp4(q)
    assert big.numel() > 2 ** 31 and torch.equal(back[-64:], want) and torch.equal(back[:64], want)
    del big, back, q
    a, b = ops.quantize_mxfp4(make(33000, 64)), ops.quantize_mxfp4(make(65536, 64, seed=2))
    c = ops.matmul_mxfp4(a, b)
    va, vb = values(ops.MxFp4(a.codes, a.scales))[-9:], values(b)
    assert c.numel() > 2 ** 31
    assert_product(c[-9:], va @ vb.t(), va.abs() @ vb.abs().t(), 64)
