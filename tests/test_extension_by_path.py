"""The grouped and MXFP4 calls use the extension built beside the package, whatever else is called neoGEMM."""
import subprocess
import sys

import pytest

from gemm_b200 import build


@pytest.fixture(scope="module", autouse=True)
def extension():
    build.build_extension()


CALL = """
import torch
from gemm_b200 import ops
try:
    ops.grouped_matmul(torch.zeros(4, 8).bfloat16(), torch.zeros(2, 8, 8).bfloat16(), torch.zeros(3, dtype=torch.int32))
except ValueError as e:
    assert "CUDA" in str(e), e
"""


def run(script, *paths):
    head = f"import sys\nsys.path[:0] = {[str(p) for p in paths]!r}\n"
    out = subprocess.run([sys.executable, "-c", head + script + "\nprint('done')"], cwd="/", capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "done", out.stderr[-800:]


@pytest.mark.parametrize("first", ["", "import neoGEMM\n"])
def test_another_module_of_the_same_name(tmp_path, first):
    (tmp_path / "neoGEMM.py").write_text("def neoGemmV1(A, B, C):\n    return 'other'\n")
    run(first + CALL + "import neoGEMM\nassert neoGEMM.neoGemmV1(0, 0, 0) == 'other'\n", tmp_path, build.ROOT)


@pytest.mark.parametrize("first", ["", "import torch, neoGEMM\n"])
def test_beside_an_import_of_the_extension_itself(first):
    run(first + CALL + """
import neoGEMM
assert neoGEMM.grouped_matmul.__doc__ == ops._ext.grouped_matmul.__doc__
before = list(sys.path)
ops._ext.quantize_mxfp4
assert sys.path == before
assert len({line.split()[-1] for line in open('/proc/self/maps') if 'neoGEMM' in line}) == 1
""", build.ROOT)
