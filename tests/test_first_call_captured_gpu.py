"""The grouped and MXFP4 calls allocate nothing per call and may be captured from the first call on: also
when that is the process's first call into the library, which sets up the device's state and loads the
kernel."""
import subprocess
import sys

import pytest

from gemm_b200 import build

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
import torch
from gemm_b200 import ops
which = sys.argv[1]
off = torch.tensor([0, 30, 64], dtype=torch.int32, device="cuda")
one = torch.ones(64, 64, device="cuda").bfloat16()
w = torch.ones(2, 64, 64, device="cuda").bfloat16()
codes = torch.full((64, 32), 0x22, dtype=torch.uint8, device="cuda")          # ones
scales = torch.full((1, 1, 32, 4, 4), 127, dtype=torch.uint8, device="cuda")
q = ops.MxFp4(codes, scales)
stack = ops.MxFp4(codes.expand(2, 64, 32).contiguous(), scales.expand(2, 1, 1, 32, 4, 4).contiguous())
calls = {"rows": lambda: ops.grouped_matmul(one, w, off), "dx": lambda: ops.grouped_matmul_dx(one, w, off),
         "dw": lambda: ops.grouped_matmul_dw(one, one, off), "quantize": lambda: ops.quantize_mxfp4(one),
         "dequantize": lambda: ops.dequantize_mxfp4(q), "mx": lambda: ops.matmul_mxfp4(q, q),
         "grouped mx": lambda: ops.grouped_matmul_mxfp4(q, stack, off)}
want = {"rows": 64, "dx": 64, "mx": 64, "grouped mx": 64, "dequantize": 1}
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls[which]()
graph.replay()
torch.cuda.synchronize()
if which == "dw":
    assert (out[0] == 30).all() and (out[1] == 34).all()
elif which == "quantize":
    assert torch.equal(ops.dequantize_mxfp4(out), one)
else:
    assert (out == want[which]).all()
assert ops.device_status()[0] == 0
print("captured")
"""


@pytest.mark.parametrize("which", ["rows", "dw", "quantize", "grouped mx"])
def test_the_first_call_of_a_process_inside_a_capture(which):
    out = subprocess.run([sys.executable, "-c", SCRIPT, which], cwd=str(build.ROOT), capture_output=True,
                         text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "captured", out.stderr[-800:]
