"""Products grouped by expert against a plain implementation in 64 bits.

Tolerance (derived, not fitted).  A result is a sum of D products of bf16 values - each exact in
fp32 - accumulated in fp32 and rounded once to bf16.  D roundings of at most 2^-23 (the tensor
core may truncate: one unit in the last place) relative to partial sums bounded by S = sum |a b|, and
one rounding of at most 2^-8 relative to the result:  |y - exact| <= 2^-8 |exact| + 2 D 2^-23 S.
"""
import pytest
import torch

from gemm_b200 import ops

pytestmark = pytest.mark.gpu
NAN = float("nan")


def offsets_of(counts, head=0, dtype=torch.int32):
    ends = [head]
    for c in counts:
        ends.append(ends[-1] + c)
    return ends, torch.tensor(ends, dtype=dtype, device="cuda")


def make(counts, N, K, head=0, tail=0, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = head + sum(counts) + tail

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).bfloat16()

    return normal(T, K), normal(len(counts), N, K, scale=K ** -0.5), normal(T, N)


def plain(op, ends, x, w, dy):
    """(result, sum of magnitudes) in 64 bits."""
    x, w, dy = x.double(), w.double(), dy.double()
    E, N, K = w.shape
    shape = {"nt": (x.shape[0], N), "dx": (x.shape[0], K), "dw": (E, N, K)}[op]
    out = torch.zeros(shape, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if op == "nt":
            out[a:b], mag[a:b] = x[a:b] @ w[e].t(), x[a:b].abs() @ w[e].t().abs()
        elif op == "dx":
            out[a:b], mag[a:b] = dy[a:b] @ w[e], dy[a:b].abs() @ w[e].abs()
        else:
            out[e], mag[e] = dy[a:b].t() @ x[a:b], dy[a:b].t().abs() @ x[a:b].abs()
    return out, mag


def assert_close(got, want, mag, depth):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    bound = want.abs() * 2.0 ** -8 + 2 * max(depth, 1) * 2.0 ** -23 * mag
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= bound).all()), float((err - bound).max())
    assert ops.device_status()[0] == 0


def call(op, x, w, dy, offsets, out=None):
    if op == "nt":
        return ops.grouped_matmul(x, w, offsets, out=out)
    if op == "dx":
        return ops.grouped_matmul_dx(dy, w, offsets, out=out)
    return ops.grouped_matmul_dw(dy, x, offsets, out=out)


@pytest.fixture(params=[-1, 0, 2, 1], ids=["auto", "narrow", "middle", "wide"])
def tiles(request):
    ops.set_tuning("grouped_kernel", request.param)
    yield request.param
    ops.set_tuning("grouped_kernel", -1)


COUNTS = {
    "one row": [1],
    "one row of many groups": [0, 0, 1, 0],
    "empty batch rows": [0, 0, 0],
    "edges of a k-block": [63, 64, 65, 1, 0, 127, 128, 129],
    "edges of a tile": [255, 0, 256, 257, 31, 33],
    "long": [700, 3, 0, 513],
    "many": [i % 5 for i in range(150)],
}


@pytest.mark.parametrize("op", ["nt", "dx", "dw"])
@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS.keys())
@pytest.mark.parametrize("N,K", [(8, 8), (136, 72), (264, 520)])
def test_groups(op, counts, N, K, tiles):
    x, w, dy = make(counts, N, K, head=3, tail=5)
    ends, off = offsets_of(counts, head=3)
    got = call(op, x, w, dy, off)
    want, mag = plain(op, ends, x, w, dy)
    depth = {"nt": K, "dx": N, "dw": max(counts)}[op]
    assert_close(got, want, mag, depth)


@pytest.mark.parametrize("op", ["nt", "dx", "dw"])
def test_a_long_contraction_and_more_tiles_than_processors(op, tiles):
    counts = [301, 0, 77, 1000]
    x, w, dy = make(counts, 2056, 1544)
    ends, off = offsets_of(counts, dtype=torch.int64)
    want, mag = plain(op, ends, x, w, dy)
    assert_close(call(op, x, w, dy, off), want, mag, 2056)


@pytest.mark.parametrize("N", [1, 7, 129, 1001])
def test_odd_widths_of_the_result(N, tiles):
    """Rows of Y that do not start on 16 bytes; guard columns stay as they were."""
    counts, K = [5, 0, 40], 136
    x, w, dy = make(counts, N, K)
    ends, off = offsets_of(counts)
    want, mag = plain("nt", ends, x, w, dy)
    assert_close(ops.grouped_matmul(x, w, off), want, mag, K)
    wide = torch.full((45, N + 3), NAN, dtype=torch.bfloat16, device="cuda")
    ops.grouped_matmul(x, w, off, out=wide[:, 1:N + 1])
    assert_close(wide[:, 1:N + 1], want, mag, K)
    assert torch.isnan(wide[:, 0]).all() and torch.isnan(wide[:, N + 1:]).all()


@pytest.mark.parametrize("op", ["nt", "dx", "dw"])
def test_strided_operands(op, tiles):
    """Rows inside wider rows, matrices inside wider and more distant matrices, surrounded by NaN."""
    counts, N, K = [70, 0, 9, 130], 100, 50
    x0, w0, dy0 = make(counts, N, K, seed=4)
    ends, off = offsets_of(counts)
    x = torch.full((209, 72), NAN, dtype=torch.bfloat16, device="cuda")[:, 8:8 + K]
    dy = torch.full((209, 112), NAN, dtype=torch.bfloat16, device="cuda")[:, 8:8 + N]
    w = torch.full((4, N + 4, 64), NAN, dtype=torch.bfloat16, device="cuda")[:, 2:2 + N, 8:8 + K]
    x.copy_(x0), dy.copy_(dy0), w.copy_(w0)
    want, mag = plain(op, ends, x, w, dy)
    assert_close(call(op, x, w, dy, off), want, mag, 209)


@pytest.mark.parametrize("op", ["nt", "dx"])
def test_rows_of_no_group(op, tiles):
    """Zero in a fresh result, untouched in the caller's; what the inputs hold there is not used."""
    counts, N, K = [20, 0, 70], 200, 136
    x, w, dy = make(counts, N, K, head=37, tail=300)
    for t in (x, dy):
        t[:37], t[127:] = NAN, float("inf")
    ends, off = offsets_of(counts, head=37)
    fresh = call(op, x, w, dy, off)
    assert (fresh[:37] == 0).all() and (fresh[127:] == 0).all()
    want, mag = plain(op, ends, x[:127], w, dy[:127])
    assert_close(fresh[37:127], want[37:], mag[37:], 200)
    mine = torch.full_like(fresh, 7.0)
    assert call(op, x, w, dy, off, out=mine) is mine
    assert (mine[:37] == 7).all() and (mine[127:] == 7).all()
    assert torch.equal(mine[37:127], fresh[37:127])


def test_a_neighbours_infinities_stay_with_the_neighbour(tiles):
    counts, N, K = [30, 70, 33, 5], 136, 72
    x, w, dy = make(counts, N, K)
    ends, off = offsets_of(counts)
    clean = {op: call(op, x, w, dy, off) for op in ("nt", "dx", "dw")}
    x[30:100], dy[30:100], w[3] = NAN, float("inf"), NAN
    for op in ("nt", "dx"):
        got = call(op, x, w, dy, off)
        assert torch.equal(got[:30], clean[op][:30]) and torch.equal(got[100:133], clean[op][100:133])
        assert torch.isnan(got[133:]).all()
    got = call("dw", x, w, dy, off)
    assert torch.equal(got[[0, 2, 3]], clean["dw"][[0, 2, 3]]) and torch.isnan(got[1]).all()


@pytest.mark.parametrize("op", ["nt", "dx", "dw"])
def test_lengths_of_zero(op, tiles):
    off = torch.zeros(4, dtype=torch.int32, device="cuda")
    x, w, dy = make([0, 0, 0], 16, 24)
    got = call(op, x, w, dy, off)
    assert (got == 0).all() and got.shape == ((0, 16), (0, 24), (3, 16, 24))[("nt", "dx", "dw").index(op)]
    # no groups at all: every row belongs to none
    x, dy = torch.ones(5, 24, device="cuda").bfloat16(), torch.ones(5, 16, device="cuda").bfloat16()
    got = call(op, x, w[:0], dy, off[:1])
    assert (got == 0).all() and got.numel() == (80, 120, 0)[("nt", "dx", "dw").index(op)]
    # a contraction of length zero
    if op != "dw":
        off = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
        w0 = torch.empty((1, 16, 0) if op == "nt" else (1, 0, 24), dtype=torch.bfloat16, device="cuda")
        got = call(op, x[:, :0], w0, dy[:, :0], off)
        assert (got == 0).all() and got.numel() == (80, 120)[("nt", "dx").index(op)]


def test_results_are_the_same_bits_each_time_and_one_kernel_treats_rows_alike(tiles):
    counts, N, K = [100, 28, 0, 64], 512, 776
    x, w, dy = make(counts, N, K)
    _, off = offsets_of(counts)
    for op in ("nt", "dx", "dw"):
        a = call(op, x, w, dy, off)
        for _ in range(3):
            assert torch.equal(a, call(op, x, w, dy, off))
    if tiles >= 0:
        one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        alone = ops.grouped_matmul(x[100:101], w[1:2], one)
        assert torch.equal(alone[0], ops.grouped_matmul(x, w, off)[100])


def test_a_captured_graph_replays_with_other_groups_beside_eager_calls():
    N, K, T = 264, 328, 190
    x, w, dy = make([190, 0, 0], N, K)
    _, off = offsets_of([190, 0, 0])
    static = off.clone()
    y, dx = torch.zeros(T, N, device="cuda").bfloat16(), torch.zeros(T, K, device="cuda").bfloat16()
    dw = torch.zeros(3, N, K, device="cuda").bfloat16()

    def body():
        ops.grouped_matmul(x, w, static, out=y)
        ops.grouped_matmul_dx(dy, w, static, out=dx)
        ops.grouped_matmul_dw(dy, x, static, out=dw)

    body()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    for counts in ([64, 63, 63], [0, 190, 0], [1, 0, 189]):
        ends, now = offsets_of(counts)
        static.copy_(now)
        graph.replay()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            eager = call("dw", x, w, dy, off)
        torch.cuda.synchronize()
        for op, got in (("nt", y), ("dx", dx), ("dw", dw)):
            want, mag = plain(op, ends, x, w, dy)
            assert_close(got, want, mag, 330)
        want, mag = plain("dw", [0, 190, 190, 190], x, w, dy)
        assert_close(eager, want, mag, 190)


def test_two_streams_at_once():
    """Nothing is shared between calls: no workspace, no counters."""
    counts = [200, 56, 0, 300]
    x, w, dy = make(counts, 776, 1032)
    _, off = offsets_of(counts)
    want = {op: call(op, x, w, dy, off) for op in ("nt", "dx", "dw")}
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(8):
        for s, op in zip(streams, want):
            with torch.cuda.stream(s):
                got.append((op, call(op, x, w, dy, off)))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[op]) for op, t in got)


@pytest.mark.parametrize("bad", [[0, 40, 20, 60], [-5, 10, 20, 60], [0, 10, 20, 61], [0, 1 << 40, 20, 60],
                                 [70, 80, 90, 100]])
def test_offsets_out_of_order_or_range_are_clamped_and_reported(bad, tiles):
    x, w, dy = make([60, 0, 0], 72, 40)
    off = torch.tensor(bad, dtype=torch.int64, device="cuda")
    guard = torch.full((62, 72), 7.0, dtype=torch.bfloat16, device="cuda")
    try:
        ops.grouped_matmul(x, w, off, out=guard[1:61])
        torch.cuda.synchronize()
        assert (guard[0] == 7).all() and (guard[61] == 7).all()
        status = ops.device_status()
        assert status[0] == 6 and status[3] == 4
        with pytest.raises(ops.NeoGemmError):
            ops.grouped_matmul_dw(dy, x, off)
    finally:
        ops.clear_device_status()
    ends, good = offsets_of([20, 30, 10])
    want, mag = plain("nt", ends, x, w, dy)
    assert_close(ops.grouped_matmul(x, w, good), want, mag, 40)


def test_refusals_on_the_device():
    x, w, dy = make([10, 6], 24, 16)
    _, off = offsets_of([10, 6])
    with pytest.raises(ValueError):                      # groups differ
        ops.grouped_matmul(x, w, off[:2])
    with pytest.raises(ValueError):                      # K differs
        ops.grouped_matmul(dy, w, off)
    with pytest.raises(ValueError):
        ops.grouped_matmul_dx(x, w, off)
    with pytest.raises(ValueError):                      # rows differ
        ops.grouped_matmul_dw(dy[:5], x, off)
    with pytest.raises(TypeError):
        ops.grouped_matmul(x, w, off.float())
    with pytest.raises(ValueError):
        ops.grouped_matmul(x, w, off.cpu())
    with pytest.raises(TypeError):
        ops.grouped_matmul(x.float(), w, off)
    with pytest.raises(TypeError):
        ops.grouped_matmul(x, w.half(), off)
    with pytest.raises(ValueError):                      # strided along K
        ops.grouped_matmul(x, w.transpose(1, 2), off)
    with pytest.raises(ValueError):                      # result of another shape
        ops.grouped_matmul(x, w, off, out=torch.empty(16, 25, device="cuda").bfloat16())
    with pytest.raises(ValueError):
        ops.grouped_matmul_dw(dy, x, off, out=torch.empty(2, 16, 24, device="cuda").bfloat16())
    with pytest.raises(ops.NeoGemmError):                # row pitch of 12 elements
        ops.grouped_matmul(torch.empty(16, 12, device="cuda").bfloat16(),
                           torch.empty(2, 24, 12, device="cuda").bfloat16(), off)
    with pytest.raises(ops.NeoGemmError):                # base not on 16 bytes
        ops.grouped_matmul(torch.empty(16, 24, device="cuda").bfloat16()[:, 1:17], w, off)
    with pytest.raises(ops.NeoGemmError):                # too many groups
        ops.grouped_matmul(x, torch.empty(1025, 8, 16, device="cuda").bfloat16(),
                           torch.zeros(1026, dtype=torch.int32, device="cuda"))
    assert ops.device_status()[0] == 0


def test_results_that_share_memory_with_an_operand_and_one_matrix_for_all_are_refused():
    x = torch.randn(16, 64, device="cuda").bfloat16()
    w = torch.randn(2, 64, 64, device="cuda").bfloat16()
    _, off = offsets_of([10, 6])
    for f in (ops.grouped_matmul, ops.grouped_matmul_dx):
        with pytest.raises(ValueError, match="share memory"):
            f(x, w, off, out=x)
        with pytest.raises(ValueError, match="share memory"):
            f(x, w, off, out=w.view(128, 64)[8:24])
        with pytest.raises(ValueError, match="matrix per group"):
            f(x, w[:1].expand(2, 64, 64), off)
    with pytest.raises(ValueError, match="share memory"):
        ops.grouped_matmul_dw(w.view(128, 64)[:16], x, off, out=w)
    q = ops.quantize_mxfp4(x)
    with pytest.raises(ValueError, match="share memory"):
        ops.matmul_mxfp4(q, q, out=q.codes.view(torch.bfloat16)[:, :16])
    # Other columns of the same rows are fine.
    both = torch.zeros(16, 128, device="cuda").bfloat16()
    both[:, :64] = x
    ops.grouped_matmul(both[:, :64], w, off, out=both[:, 64:])
    assert torch.equal(both[:, 64:], ops.grouped_matmul(x, w, off)) and torch.equal(both[:, :64], x)
    assert ops.device_status()[0] == 0


def test_as_many_groups_as_there_may_be(tiles):
    counts = [0] * 1024
    for e, c in ((0, 1), (31, 2), (32, 1), (33, 3), (500, 17), (1022, 1), (1023, 40)):
        counts[e] = c
    N, K = 40, 72
    x, w, dy = make(counts, N, K, tail=2)
    ends, off = offsets_of(counts)
    for op, depth in (("nt", K), ("dx", N), ("dw", 40)):
        want, mag = plain(op, ends, x, w, dy)
        assert_close(call(op, x, w, dy, off), want, mag, depth)


@pytest.mark.parametrize("op", ["nt", "dx", "dw"])
def test_results_of_more_than_2_31_values(op):
    """Offsets past 32 bits: the last rows and the last matrix are where they belong."""
    g = torch.Generator(device="cuda").manual_seed(8)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").bfloat16()

    if op == "dw":
        E, N, K, T = 34, 8192, 8192, 70
        dy, x = normal(T, N), normal(T, K)
        off = torch.tensor([0] * 33 + [3, T], dtype=torch.int32, device="cuda")
        out = ops.grouped_matmul_dw(dy, x, off)
        assert out.numel() > 2 ** 31 and (out[:32, ::1000, ::1000] == 0).all()
        want = dy[3:, -40:].double().t() @ x[3:, -50:].double()
        mag = dy[3:, -40:].double().abs().t() @ x[3:, -50:].double().abs()
        assert_close(out[33, -40:, -50:], want, mag, T)
        return
    wide, deep, T = 65536, 64, 33000
    w = normal(2, wide, deep) if op == "nt" else normal(2, deep, wide)
    r = normal(T, deep)
    off = torch.tensor([0, 10, T], dtype=torch.int64, device="cuda")
    out = ops.grouped_matmul(r, w, off) if op == "nt" else ops.grouped_matmul_dx(r, w, off)
    assert out.numel() > 2 ** 31
    m = w[1].double().t() if op == "nt" else w[1].double()
    assert_close(out[-20:], r[-20:].double() @ m, r[-20:].double().abs() @ m.abs(), deep)
