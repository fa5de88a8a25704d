"""Offsets that descend or leave the batch: clamped to [0, T] and to the largest index in front of them, so
that no row belongs to two groups, and recorded.  Results have to be those of the clamped offsets, bit for
bit, in every product, for either integer type and with the groups in registers (up to 32) and in shared
memory (more)."""
import pytest
import torch

from gemm_b200 import ops

pytestmark = pytest.mark.gpu
T, N, K = 300, 72, 128


def bad_offsets(groups, kind):
    good = [T * e // groups for e in range(groups + 1)]
    if kind == "descending":
        return good[::-1]
    if kind == "alternating":
        return [0 if e % 2 == 0 else T for e in range(groups + 1)]
    if kind == "one lower":
        return good[:groups // 2] + [good[1] - 3] + good[groups // 2 + 1:]
    if kind == "one higher":
        return good[:groups // 2] + [T - 5] + good[groups // 2 + 1:]
    if kind == "below and above":
        return [-7] + good[1:-1] + [T + 1000]
    if kind == "at the seams":      # across the 32 groups that a warp holds at a time
        return [good[e] if e % 32 else good[max(e - 40, 0)] - 1 for e in range(groups)] + [T]
    assert kind == "the last behind"
    return good[:-1] + [5]


KINDS = ["descending", "alternating", "one lower", "one higher", "below and above", "at the seams",
         "the last behind"]


def clamped(ends):
    out, top = [], 0
    for e in ends:
        top = max(top, min(max(e, 0), T))
        out.append(top)
    return out


@pytest.fixture(params=[-1, 0, 2, 1], ids=["auto", "narrow", "middle", "wide"])
def tiles(request):
    ops.set_tuning("grouped_kernel", request.param)
    yield request.param
    ops.set_tuning("grouped_kernel", -1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("groups", [1, 2, 32, 33, 100, 1000])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_results_are_those_of_the_clamped_offsets(groups, kind, dtype, tiles):
    ends = bad_offsets(groups, kind)
    right = clamped(ends)
    g = torch.Generator(device="cuda").manual_seed(groups)
    x, dy = (torch.randn(T, n, generator=g, device="cuda").bfloat16() for n in (K, N))
    w = torch.randn(groups, N, K, generator=g, device="cuda").bfloat16()
    qx, qw = ops.quantize_mxfp4(x), ops.quantize_mxfp4(w)
    bad, good = (torch.tensor(o, dtype=dtype, device="cuda") for o in (ends, right))
    calls = (lambda o: ops.grouped_matmul(x, w, o), lambda o: ops.grouped_matmul_dx(dy, w, o),
             lambda o: ops.grouped_matmul_dw(dy, x, o), lambda o: ops.grouped_matmul_mxfp4(qx, qw, o))
    for i, call in enumerate(calls):
        want = call(good)
        assert torch.isfinite(want).all()
        try:
            got = call(bad)
            torch.cuda.synchronize()
            status = ops.device_status()
            if ends != right:
                assert status[0] == 6 and status[3] == 4, i
                with pytest.raises(ops.NeoGemmError):
                    call(good)
        finally:
            ops.clear_device_status()
        assert torch.equal(got, want), i
    # and in 64 bits, once
    y = torch.zeros(T, N, dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(zip(right, right[1:])):
        y[a:b] = x[a:b].double() @ w[e].double().t()
    got = ops.grouped_matmul(x, w, good).double()
    # one rounding to bf16 (2^-8) on top of an fp32 sum of K terms (2^-23 each, of sums below max |x| |w| K)
    assert bool(((got - y).abs() <= y.abs() * 2.0 ** -8 + 2 * K * 2.0 ** -23 *
                 (x.double().abs().amax() * w.double().abs().amax() * K)).all())
