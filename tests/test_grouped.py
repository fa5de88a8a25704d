"""CPU: the refusals of the grouped and MXFP4 products, at the C ABI and at the Python face, before a
device is touched."""
import pytest
import torch

from gemm_b200 import _lib, build, ops

OK, BAD_ARG, UNSUPPORTED = 0, 1, 2


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_extension()


@pytest.fixture(scope="module")
def memory():
    """(a 16-byte aligned host address that no call may get as far as using, its owner)"""
    buf = torch.zeros(4096, dtype=torch.int64)
    assert buf.data_ptr() % 16 == 0
    return buf.data_ptr(), buf


def rows_call(fn, p, **change):
    a = dict(R=p, W=p, out=p, offsets=p, wide=0, groups=2, T=8, N=16, K=24, ldr=24, ldw=24, stack=16 * 24,
             ldo=16, zero_rest=0)
    if fn is _lib.lib.neogemm_grouped_dx:
        a.update(ldr=16, ldo=24)
    a.update(change)
    return fn(a["R"], a["W"], a["out"], a["offsets"], a["wide"], a["groups"], a["T"], a["N"], a["K"], a["ldr"],
              a["ldw"], a["stack"], a["ldo"], a["zero_rest"], None)


@pytest.mark.parametrize("name", ["neogemm_grouped_nt", "neogemm_grouped_dx"])
def test_rows_products_refuse(name, memory):
    p, _ = memory
    fn = getattr(_lib.lib, name)
    for bad in (dict(T=-1), dict(N=-1), dict(K=-8), dict(groups=-1), dict(out=None), dict(R=None), dict(W=None),
                dict(offsets=None), dict(ldr=8), dict(ldw=16), dict(ldo=8), dict(stack=-8)):
        assert rows_call(fn, p, **bad) == BAD_ARG, bad
    for bad in (dict(ldr=28), dict(ldw=28), dict(stack=388), dict(R=p + 2), dict(W=p + 8), dict(out=p + 1),
                dict(offsets=p + 2), dict(offsets=p + 4, wide=1), dict(groups=1025), dict(T=1 << 31),
                dict(N=1 << 40, ldo=1 << 40), dict(K=1 << 31), dict(ldr=1 << 62), dict(stack=1 << 62),
                dict(ldw=1 << 40), dict(ldo=1 << 60)):
        assert rows_call(fn, p, **bad) in (UNSUPPORTED, BAD_ARG), bad
    # nothing to do
    assert rows_call(fn, p, T=0) == OK
    assert rows_call(fn, p, groups=0, offsets=None) == OK
    assert rows_call(fn, p, **(dict(N=0) if name.endswith("nt") else dict(K=0))) == OK


def test_dw_refuses(memory):
    p, _ = memory

    def call(**change):
        a = dict(dy=p, x=p, out=p, offsets=p, wide=0, groups=2, T=8, N=16, K=24, lddy=16, ldx=24)
        a.update(change)
        return _lib.lib.neogemm_grouped_dw(a["dy"], a["x"], a["out"], a["offsets"], a["wide"], a["groups"], a["T"],
                                           a["N"], a["K"], a["lddy"], a["ldx"], None)

    for bad in (dict(T=-1), dict(groups=-1), dict(out=None), dict(dy=None), dict(x=None), dict(offsets=None),
                dict(lddy=8), dict(ldx=16)):
        assert call(**bad) == BAD_ARG, bad
    for bad in (dict(lddy=20), dict(ldx=28), dict(dy=p + 2), dict(x=p + 8), dict(out=p + 1), dict(offsets=p + 1),
                dict(groups=1025)):
        assert call(**bad) == UNSUPPORTED, bad
    assert call(groups=0, offsets=None) == OK and call(N=0) == OK and call(K=0) == OK


def test_mxfp4_conversion_refuses(memory):
    p, _ = memory
    q, d = _lib.lib.neogemm_mxfp4_quantize, _lib.lib.neogemm_mxfp4_dequantize
    assert q(p, 0, p, p, 1, 4, 48, 48, 0, None) == UNSUPPORTED          # K % 32
    assert q(p, 0, p, p, 1, -4, 64, 64, 0, None) == BAD_ARG
    assert q(None, 0, p, p, 1, 4, 64, 64, 0, None) == BAD_ARG
    assert q(p, 0, None, p, 1, 4, 64, 64, 0, None) == BAD_ARG
    assert q(p, 0, p, p, 1, 4, 64, 32, 0, None) == BAD_ARG              # pitch below K
    assert q(p + 2, 0, p, p, 1, 4, 64, 64, 0, None) == UNSUPPORTED
    assert q(p, 0, p, p, 1, 4, 64, 68, 0, None) == UNSUPPORTED          # rows not on 16 bytes
    assert q(p, 0, p, p, 2, 4, 64, 64, 260, None) == UNSUPPORTED
    assert q(p, 0, p, p + 8, 1, 4, 64, 64, 0, None) == UNSUPPORTED
    assert q(p, 0, p, p, 1 << 31, 1 << 31, 64, 64, 0, None) == UNSUPPORTED
    assert d(p, p, p, 1, 4, 40, None) == UNSUPPORTED
    assert d(p, p, None, 1, 4, 64, None) == BAD_ARG
    assert d(p, p, p + 2, 1, 4, 64, None) == UNSUPPORTED
    for n in ((0, 4, 64), (1, 0, 64), (1, 4, 0)):
        assert q(None, 0, None, None, *n, n[2], 0, None) == OK and d(None, None, None, *n, None) == OK


def test_mxfp4_products_refuse(memory):
    p, _ = memory
    f, g = _lib.lib.neogemm_mxfp4_nt, _lib.lib.neogemm_grouped_mxfp4_nt
    assert f(p, p, p, p, p, 4, 8, 96, 8, None) == UNSUPPORTED           # K % 64
    assert f(p, p, p, p, p, -4, 8, 64, 8, None) == BAD_ARG
    assert f(p, p, p, p, None, 4, 8, 64, 8, None) == BAD_ARG
    assert f(p, None, p, p, p, 4, 8, 64, 8, None) == BAD_ARG
    assert f(p, p, p, p, p, 4, 8, 64, 4, None) == BAD_ARG               # short pitch
    assert f(p, p, p + 8, p, p, 4, 8, 64, 8, None) == UNSUPPORTED
    assert f(p, p, p, p, p + 1, 4, 8, 64, 8, None) == UNSUPPORTED
    assert f(None, None, None, None, None, 0, 8, 64, 8, None) == OK
    assert g(p, p, p, p, p, None, 0, 2, 4, 8, 64, 8, 0, None) == BAD_ARG
    assert g(p, p, p, p, p, p, 0, 2000, 4, 8, 64, 8, 0, None) == UNSUPPORTED
    assert g(p, p, p, p, p, p, 0, 2, 4, 8, 80, 8, 0, None) == UNSUPPORTED


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-GPU behaviour")
def test_valid_calls_fail_loudly_without_a_gpu(memory):
    p, _ = memory
    assert rows_call(_lib.lib.neogemm_grouped_nt, p) not in (OK, BAD_ARG)
    assert _lib.lib.neogemm_mxfp4_nt(p, p, p, p, p, 4, 8, 64, 8, None) not in (OK, BAD_ARG)
    assert _lib.lib.neogemm_mxfp4_quantize(p, 0, p, p, 1, 4, 64, 64, 0, None) not in (OK, BAD_ARG)


def test_python_face_refuses_cpu_tensors_and_other_things():
    x, w = torch.zeros(4, 8).bfloat16(), torch.zeros(2, 8, 8).bfloat16()
    off = torch.zeros(3, dtype=torch.int32)
    q = ops.MxFp4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8))
    for f in (lambda: ops.grouped_matmul(x, w, off), lambda: ops.grouped_matmul_dx(x, w, off),
              lambda: ops.grouped_matmul_dw(x, x, off), lambda: ops.quantize_mxfp4(x),
              lambda: ops.dequantize_mxfp4(q), lambda: ops.matmul_mxfp4(q, q),
              lambda: ops.grouped_matmul_mxfp4(q, q, off)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        ops.grouped_matmul(x, w, [0, 2, 4])
    with pytest.raises(TypeError):
        ops.matmul_mxfp4(x, x)
    with pytest.raises(TypeError):
        ops.dequantize_mxfp4(None)


def test_extension_and_ctypes_share_one_library(tmp_path):
    """Also when the library file is replaced between the two loads (a rebuild in a running session)."""
    import subprocess
    import sys
    script = """
import os, shutil, sys, torch
from gemm_b200 import _lib
path = str(_lib.LIB_PATH)
copy = sys.argv[1]
shutil.copy2(path, copy)          # another file of the same name takes its place, then the first returns
os.replace(copy, path)
import neoGEMM
maps = {line.split()[-1] + line.split()[4] for line in open('/proc/self/maps') if 'libneogemm' in line}
assert len({m.replace(' (deleted)', '') for m in maps}) == 1, maps
print('one')
"""
    target = _lib.LIB_PATH.with_name("libneogemm.replaced.so")
    out = subprocess.run([sys.executable, "-c", script, str(target)], cwd=str(build.ROOT), capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "one", out.stderr[-500:]
