"""What the grouped and MXFP4 layers accept and refuse: the same under fake tensors (tracing) and in earnest."""
import pytest
import torch

from gemm_b200 import build, torch_ops


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
