"""What the grouped and MXFP4 layers accept and refuse: the same under fake tensors (tracing) and in earnest,
and in every layout of their input."""
import pytest
import torch

from gemm_b200 import build, ops, torch_ops


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_extension()


def bf16(*shape):
    return torch.empty(shape, dtype=torch.bfloat16)


def grouped_cases():
    """(exception, message, arguments); the first is a call that passes."""
    off = torch.empty(3, dtype=torch.int32)
    x, w = bf16(4, 16), bf16(2, 24, 16)
    yield None, "", (x, w, off)
    yield None, "", (bf16(16, 4).t(), w, off.long())
    yield None, "", (bf16(4, 18)[:, 1:13], bf16(2, 24, 16)[:, :, :12], off)
    yield None, "", (bf16(4, 0), bf16(2, 24, 0), off)
    yield None, "", (bf16(4, 12), bf16(1, 1, 12), off[:2])
    yield ValueError, "K mismatch", (x, bf16(2, 24, 8), off)
    yield ValueError, "offsets", (x, w, off[:2])
    yield ValueError, r"x\[T, K\]", (x.view(2, 2, 16), w, off)
    yield TypeError, "bfloat16", (x.float(), w, off)
    yield TypeError, "bfloat16", (x, w.half(), off)
    yield TypeError, "int32 or int64", (x, w, off.float())
    yield ValueError, "multiples of 8", (bf16(4, 12), bf16(2, 24, 12), off)
    yield ValueError, "multiples of 8", (x, bf16(2, 16, 24).transpose(1, 2), off)
    yield ValueError, "multiples of 8", (x, bf16(2, 24, 24)[:, :, 4:20], off)
    yield ValueError, "matrix per group", (x, bf16(1, 24, 16).expand(2, 24, 16), off)
    yield ValueError, "multiples of 8", (x, bf16(2, 1, 16).expand(2, 24, 16), off)
    yield ValueError, "at most 1024", (x, bf16(1025, 1, 16), torch.empty(1026, dtype=torch.int32))


def mxfp4_cases():
    def held(*lead, n=40, k=64):
        return (torch.empty(*lead, n, k // 2, dtype=torch.uint8),
                torch.empty(*lead, -(-n // 128), -(-k // 128), 32, 4, 4, dtype=torch.uint8))

    codes, scales = held()
    x = bf16(3, 64)
    yield None, "", (x, codes, scales)
    yield None, "", (bf16(2, 3, 68)[:, :, 3:67].float(), codes, scales)
    yield None, "", (bf16(64), codes, scales)
    yield None, "", (bf16(0, 64), codes, scales)
    yield ValueError, "multiple of 64", (bf16(3, 96), *held(k=96))
    yield ValueError, "K mismatch", (bf16(3, 128), codes, scales)
    yield ValueError, "2 dimensions", (x, *held(2))
    yield TypeError, "uint8", (x, codes.int(), scales)
    yield TypeError, "uint8", (x, codes, scales.int())
    yield TypeError, "bfloat16 or float32", (x.half(), codes, scales)
    yield ValueError, "scales of codes", (x, codes, held(n=200)[1])
    yield ValueError, "contiguous", (x, torch.empty(32, 40, dtype=torch.uint8).t(), scales)
    off = torch.empty(3, dtype=torch.int64)
    yield None, "", (x, *held(2), off)
    yield ValueError, "multiple of 64", (bf16(3, 32), *held(2, k=32), off)
    yield ValueError, "offsets", (x, *held(2), off[:2])
    yield TypeError, "int32 or int64", (x, *held(2), off.double())
    yield ValueError, "3 dimensions", (bf16(1, 3, 64), *held(2), off)
    yield ValueError, "at most 1024", (x, *held(1025, n=1), torch.empty(1026, dtype=torch.int32))


def call(arguments):
    if len(arguments) == 4:
        return torch.ops.neogemm.mxfp4_grouped_linear(*arguments)
    return (torch.ops.neogemm.mxfp4_linear if arguments[1].dtype in (torch.uint8, torch.int32)
            else torch.ops.neogemm.grouped_linear)(*arguments)


@pytest.mark.parametrize("cases", [grouped_cases, mxfp4_cases])
def test_fake_tensors_are_refused_like_real_ones(cases):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        for exception, message, arguments in cases():
            if exception is None:
                assert call(arguments).dtype == torch.bfloat16
            else:
                with pytest.raises(exception, match=message):
                    call(arguments)
    for exception, message, arguments in cases():
        if exception is not None:              # before the device of the tensors is looked at
            with pytest.raises(exception, match=message):
                call(arguments)


def test_layers_refuse_what_their_kernels_refuse():
    for k in (32, 96, 100):
        with pytest.raises(ValueError, match="multiple of 64"):
            torch_ops.NeoLinearMxFp4(torch.zeros(8, k))
    with pytest.raises(ValueError, match="multiple of 64"):
        torch_ops.NeoLinearMxFp4(torch.zeros(64))
    with pytest.raises(ValueError, match="multiple of 8"):
        torch_ops.NeoGroupedLinear(2, 12, 16)
    with pytest.raises(ValueError, match="at most 1024"):
        torch_ops.NeoGroupedLinear(1025, 8, 8)


def layouts(x):
    """The matrix x as views of other memory."""
    rows, width = x.shape
    yield "contiguous", x.clone()
    for offset in (1, 4, 8):
        wide = torch.full((rows, width + 2 * offset + 3), float("nan"), dtype=x.dtype, device=x.device)
        yield f"columns from {offset}", wide[:, offset:offset + width].copy_(x)
    yield "transposed", x.t().contiguous().t()
    yield "every other row", x.repeat_interleave(2, 0)[::2]
    yield "every other column", x.repeat_interleave(2, 1)[:, ::2]
    flat = torch.full((rows * width + 4,), float("nan"), dtype=x.dtype, device=x.device)
    yield "from 8 bytes on", flat[8 // x.element_size():][:rows * width].view(rows, width).copy_(x)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_layout_gives_the_same_bits(K, dtype):
    g = torch.Generator(device="cuda").manual_seed(K)
    T, E, N = 37, 3, 40
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    w = torch.randn(E, N, K, generator=g, device="cuda").bfloat16()
    off = torch.tensor([0, 11, 11, 37], dtype=torch.int32, device="cuda")
    dense, grouped = torch_ops.NeoLinearMxFp4(w[0]), torch_ops.NeoLinearMxFp4(w)
    y, z = dense(x), grouped(x, off)
    for name, view in layouts(x):
        assert torch.equal(view, x)
        assert torch.equal(dense(view), y) and torch.equal(grouped(view, off), z), name
    # the one row and the batch in more dimensions
    assert torch.equal(dense(x[0]), dense(x[:1])[0]) and dense(x[:0]).shape == (0, N)
    assert torch.equal(dense(x[:36].view(3, 4, 3, K).transpose(0, 2)), y[:36].view(3, 4, 3, N).transpose(0, 2))


@pytest.mark.gpu
def test_every_layout_of_a_trained_layer():
    g = torch.Generator(device="cuda").manual_seed(2)
    T, E, N, K = 37, 3, 40, 12
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    w = torch.randn(E, N, 16, generator=g, device="cuda").bfloat16()[:, :, :K].requires_grad_()   # pitch 16
    off = torch.tensor([0, 11, 11, 37], dtype=torch.int32, device="cuda")
    dy = torch.randn(T, N, generator=g, device="cuda").bfloat16()
    want = None
    for name, view in layouts(x):
        view.requires_grad_()
        y = torch.ops.neogemm.grouped_linear(view, w, off)
        got = (y.detach(), *torch.autograd.grad(y, (view, w), dy))
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
    xd, wd, ranges = x.double(), w.detach().double(), ((0, 11), (11, 11), (11, 37))
    ref = torch.cat([xd[a:b] @ wd[e].t() for e, (a, b) in enumerate(ranges)])
    mag = torch.cat([xd[a:b].abs() @ wd[e].abs().t() for e, (a, b) in enumerate(ranges)])
    # one rounding (2^-8) of an fp32 sum of K products
    assert bool(((want[0].double() - ref).abs() <= ref.abs() * 2.0 ** -8 + 2 * K * 2.0 ** -23 * mag).all())


@pytest.mark.gpu
def test_weights_in_every_layout_are_held_alike():
    w = torch.randn(2, 40, 128, device="cuda").bfloat16()
    want = torch_ops.NeoLinearMxFp4(w)
    flat = torch.zeros(w.numel() + 4, device="cuda").bfloat16()
    for view in (w.transpose(1, 2).contiguous().transpose(1, 2), w.repeat(1, 1, 2)[:, :, 128:],
                 flat[4:].view(w.shape).copy_(w), w.transpose(0, 1).contiguous().transpose(0, 1)):
        got = torch_ops.NeoLinearMxFp4(view)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    with pytest.raises(ops.NeoGemmError):      # the operators themselves read rows from 16 bytes on
        ops.quantize_mxfp4(flat[4:].view(w.shape))
