"""What the device says of the clusters it holds (tests/csrc/loop_parts_probe.cu)."""
import ctypes
import subprocess
import sys

import pytest

from dscuda_b200.library import ROOT, build_directory

pytestmark = pytest.mark.gpu


def test_counts_of_the_device(gpu):
    lib = ctypes.CDLL(str(build_directory() / "libdscuda_test_probes.so"))
    counts = (ctypes.c_int * 17)()
    assert lib.dscuda_test_cluster_counts(200 * 1024, 8, counts) == 0
    assert counts[1] == 148 and 2 <= counts[2] <= 74 and counts[8] >= 1 and all(c == 0 for c in counts[9:])
    assert all(counts[n + 1] <= counts[n] for n in range(1, 8))
    # 16 is not portable: the kernel does not allow it, so the answer is none, and no error stays behind
    assert lib.dscuda_test_cluster_counts(200 * 1024, 16, counts) == 0 and counts[16] == 0
    assert lib.dscuda_test_per_device() == 0


def test_the_first_call_of_a_process_is_captured(gpu):
    """The device is asked inside the capture then."""
    program = """
import torch
from dscuda_b200 import flash
g = torch.Generator(device="cuda").manual_seed(1)
query, dout = (torch.randn(1, 700, 4, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
key, value = (torch.randn(1, 900, 2, 128, device="cuda", generator=g).bfloat16() for _ in range(2))
out, lse, grads = torch.empty_like(query), torch.empty(1, 4, 700, device="cuda"), [torch.empty_like(x) for x in (query, key, value)]
workspaces = flash.cross_forward_workspace(1, 700, 900, 4, 2), flash.cross_backward_workspace(1, 700, 900, 4, 2)
def step():
    flash.cross_forward(query, key, value, 0.1, None, workspaces[0], out, lse)
    flash.cross_backward(dout, out, lse, query, key, value, 0.1, None, workspaces[1], grads)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    step()
graph.replay()
torch.cuda.synchronize()
kept = [x.clone() for x in (out, lse, *grads)]
for x in (out, lse, *grads):
    x.zero_()
step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(kept, (out, lse, *grads))) and bool(torch.isfinite(kept[0].float()).all())
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", program], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]
