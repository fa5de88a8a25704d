"""The grouped and MXFP4 products as layers: shapes without a GPU, gradients, and a run of them
together - a router's sorted rows through an expert block, trained in bf16 and served in 4 bits."""
import pytest
import torch

from gemm_b200 import build, ops, torch_ops


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_extension()


def test_fake_implementations_give_shapes_without_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(10, 64, dtype=torch.bfloat16)
        w = torch.empty(3, 40, 64, dtype=torch.bfloat16)
        off = torch.empty(4, dtype=torch.int32)
        y = torch.ops.neogemm.grouped_linear(x, w, off)
        assert y.shape == (10, 40) and y.dtype == torch.bfloat16
        codes, scales = torch.empty(40, 32, dtype=torch.uint8), torch.empty(1, 1, 32, 4, 4, dtype=torch.uint8)
        z = torch.ops.neogemm.mxfp4_linear(x.float().view(2, 5, 64), codes, scales)
        assert z.shape == (2, 5, 40) and z.dtype == torch.bfloat16
        stack = torch.empty(3, 40, 32, dtype=torch.uint8), torch.empty(3, 1, 1, 32, 4, 4, dtype=torch.uint8)
        assert torch.ops.neogemm.mxfp4_grouped_linear(x, *stack, off).shape == (10, 40)


def test_layers_refuse():
    x, w, off = torch.zeros(4, 8).bfloat16(), torch.zeros(2, 16, 8).bfloat16(), torch.zeros(3, dtype=torch.int32)
    for bad in ((x, w[:, :, :4], off), (x, w, off[:2]), (x.view(2, 2, 8), w, off), (x.float(), w, off)):
        with pytest.raises(Exception):
            torch.ops.neogemm.grouped_linear(*bad)
    with pytest.raises(Exception):
        torch.ops.neogemm.mxfp4_linear(x, torch.zeros(4, 8, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4))


def sorted_rows(T, E, seed):
    """A router's choice: (order, offsets) of T rows over E groups."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    choice = torch.randint(0, E, (T,), generator=g, device="cuda")
    order = torch.argsort(choice, stable=True)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = torch.cumsum(torch.bincount(choice, minlength=E), 0)
    return order, offsets


@pytest.mark.gpu
@pytest.mark.parametrize("T,N", [(1, 40), (77, 40), (300, 37)])
def test_gradients_of_the_layer(T, N):
    """Against the formulas in 64 bits; dy is handed over as autograd finds it (expanded, odd widths)."""
    E, K = 4, 72
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T + 3, K, generator=g, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(E, N, K, generator=g, device="cuda") / K ** 0.5).bfloat16().requires_grad_()
    _, off = sorted_rows(T, E, 5)
    y = torch.ops.neogemm.grouped_linear(x, w, off)
    assert (y[T:] == 0).all()
    ends = off.tolist()
    for dy in (torch.randn(T + 3, N, generator=g, device="cuda").bfloat16(),
               torch.ones((), device="cuda").bfloat16().expand(T + 3, N),
               torch.randn(N, T + 3, generator=g, device="cuda").bfloat16().t()):
        dx, dw = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
        assert (dx[T:] == 0).all() and dx.dtype == dw.dtype == torch.bfloat16
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            d, xe, we = dy[a:b].double(), x[a:b].detach().double(), w[e].detach().double()
            for got, want, mag, depth in ((dx[a:b], d @ we, d.abs() @ we.abs(), N),
                                          (dw[e], d.t() @ xe, d.abs().t() @ xe.abs(), b - a)):
                bound = want.abs() * 2.0 ** -8 + 2 * max(depth, 1) * 2.0 ** -23 * mag
                assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.gpu
def test_gradients_against_differences():
    """<dy, f(x + h v) - f(x - h v)> / 2h of the layer in exact arithmetic equals <dx, v>: f is linear, so
    the plain product of the perturbation gives the difference without rounding."""
    T, E, N, K = 50, 3, 24, 40
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(E, N, K, generator=g, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(T, N, generator=g, device="cuda").bfloat16()
    _, off = sorted_rows(T, E, 2)
    dx, dw = torch.autograd.grad(torch.ops.neogemm.grouped_linear(x, w, off), (x, w), dy)
    v = torch.randn(T, K, generator=g, device="cuda").double()
    u = torch.randn(E, N, K, generator=g, device="cuda").double()
    group = torch.repeat_interleave(torch.arange(E, device="cuda"), off[1:] - off[:-1])
    by_x = torch.einsum("tn,tnk,tk->", dy.double(), w.detach().double()[group], v)
    by_w = torch.einsum("tn,tnk,tk->", dy.double(), u[group], x.detach().double())
    # each gradient value is rounded once (2^-8 of it) on top of its fp32 sum
    for got, direction, want in ((dx, v, by_x), (dw, u, by_w)):
        bound = float((got.double().abs() * direction.abs()).sum()) * (2.0 ** -8 + 2.0 ** -14)
        assert abs(float((got.double() * direction).sum() - want)) <= bound


@pytest.mark.gpu
def test_an_expert_block_trained_and_then_served_in_four_bits():
    """Route, sort, up-projection, activation, down-projection, back to the rows' order: one training
    step's gradients against the same block in 64 bits, then the block with MXFP4 weights against the
    products of the dequantised tensors."""
    T, E, D, H = 200, 5, 128, 192
    torch.manual_seed(3)
    up, down = (torch_ops.NeoGroupedLinear(E, a, b, device="cuda") for a, b in ((D, H), (H, D)))
    x = torch.randn(T, D, device="cuda").bfloat16().requires_grad_()
    order, off = sorted_rows(T, E, 7)
    back = torch.argsort(order)

    def block(first, second):
        h = torch.nn.functional.silu(first(x[order], off))
        return second(h, off)[back]

    dy = torch.randn(T, D, device="cuda").bfloat16()
    y = block(up, down)
    grads = torch.autograd.grad(y, (x, up.weight, down.weight), dy)

    xd, ud, dd = (t.detach().double().requires_grad_() for t in (x, up.weight, down.weight))
    ends, parts = off.tolist(), []
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        parts.append(torch.nn.functional.silu(xd[order][a:b] @ ud[e].t()) @ dd[e].t())
    want = torch.cat(parts)[back]
    wanted = torch.autograd.grad(want, (xd, ud, dd), dy.double())
    # five roundings to bf16 of at most 2^-8 lie on the longest path (product, activation, their two
    # gradients, the result), uncorrelated over the sums: compared in norm
    for got, ref in zip((y.detach(), *grads), (want.detach(), *wanted)):
        assert float((got.double() - ref).norm() / ref.norm()) < 5 * 2.0 ** -8

    with torch.no_grad():
        up4, down4 = torch_ops.NeoLinearMxFp4(up.weight), torch_ops.NeoLinearMxFp4(down.weight)
        served = block(up4, down4)

        def value(t):
            return ops.dequantize_mxfp4(ops.quantize_mxfp4(t)).double()

        parts = []
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            h = (value(x[order])[a:b] @ value(up.weight)[e].t()).bfloat16()
            parts.append(value(torch.nn.functional.silu(h)) @ value(down.weight)[e].t() if b > a else h.new_zeros(0, D))
        ref = torch.cat([p.double() for p in parts])[back]
        # h may differ by one rounding, which moves few codes by one step of a quarter at most
        assert float((served.double() - ref).norm() / ref.norm()) < 2.0 ** -6
    assert ops.device_status()[0] == 0


@pytest.mark.gpu
def test_a_dense_layer_in_four_bits():
    torch.manual_seed(4)
    w = torch.randn(72, 128, device="cuda")
    layer = torch_ops.NeoLinearMxFp4(w)
    x = torch.randn(3, 7, 128, device="cuda")
    y = layer(x)
    a = ops.dequantize_mxfp4(ops.quantize_mxfp4(x.view(21, 128))).double()
    b = ops.dequantize_mxfp4(ops.MxFp4(layer.codes, layer.scales)).double()
    bound = (a @ b.t()).abs() * 2.0 ** -8 + 2 * 128 * 2.0 ** -23 * (a.abs() @ b.abs().t())
    assert y.shape == (3, 7, 72) and bool(((y.view(21, 72).double() - a @ b.t()).abs() <= bound).all())
    with pytest.raises(ValueError):
        torch_ops.NeoLinearMxFp4(torch.randn(2, 72, 128, device="cuda"))(x)


@pytest.mark.gpu
def test_a_training_step_captured_into_a_graph():
    """Forward and both gradients, replayed with other rows, weights and groups."""
    T, E, N, K = 120, 4, 64, 96
    x = torch.randn(T, K, device="cuda").bfloat16().requires_grad_()
    w = torch.randn(E, N, K, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(T, N, device="cuda").bfloat16()
    off = torch.tensor([0, 30, 30, 100, 120], dtype=torch.int32, device="cuda")

    def step():
        y = torch.ops.neogemm.grouped_linear(x, w, off)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
        w.copy_(torch.randn_like(w))
    off.copy_(torch.tensor([0, 1, 64, 65, 120], dtype=torch.int32))
    graph.replay()
    again = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, again))


@pytest.mark.gpu
def test_calls_from_a_fresh_host_thread():
    """A thread that has made no CUDA call yet, as autograd's is in a backward pass."""
    import threading
    x, w = torch.randn(9, 64, device="cuda").bfloat16(), torch.randn(2, 24, 64, device="cuda").bfloat16()
    off = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    q = ops.MxFp4(*ops.quantize_mxfp4(x))
    want = ops.grouped_matmul(x, w, off), ops.matmul_mxfp4(q, q)
    torch.cuda.synchronize()
    got = []

    def work():
        got.append((ops.grouped_matmul(x, w, off), ops.matmul_mxfp4(q, q)))
        torch.cuda.synchronize()

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert got and all(torch.equal(a, b) for a, b in zip(got[0], want))
