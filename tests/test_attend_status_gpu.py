"""``attend_status`` asks for the tcgen05 shared-prefix kernel's flag once that kernel was launched, and not before."""

from __future__ import annotations

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

# In a process of its own: nothing else may have launched the kernel. The knob makes the next launch's wait run out.
_SCRIPT = """
import time, torch
from veloxquant_mlx_b200 import VQLibraryError, kernels

def cost():
    torch.cuda.synchronize()
    best = 1e9
    for _ in range(20):
        t = time.perf_counter()
        for _ in range(20):
            kernels.attend_status()
        best = min(best, (time.perf_counter() - t) / 20)
    return best * 1e6

z = torch.zeros(1, 1, 256, 128, device="cuda", dtype=torch.float16)
rows = kernels.KiviRows(k_res=z, v_res=z.clone())
q = torch.zeros(40, 1, 1, 128, device="cuda", dtype=torch.float16)
kernels.attend_status()
kernels.kivi_shared_prefix_attend(q, rows, None, 0.1, variant=1)
before = cost()
graph = torch.cuda.CUDAGraph()
kernels.tune("shared_wait_test", 1)
with torch.cuda.graph(graph):   # the launch is only recorded: a replay raises the flag
    kernels.kivi_shared_prefix_attend(q, rows, None, 0.1, variant=2)
kernels.attend_status()
for _ in range(2):
    graph.replay()
    try:
        kernels.attend_status()
        raise SystemExit("the flag was not reported")
    except VQLibraryError as e:
        assert "TIMEOUT" in str(e) and "shared" in str(e)
    kernels.attend_status()
print("us", before, cost())
"""


def test_the_flag_is_asked_for_after_a_launch_only():
    run = subprocess.run([sys.executable, "-c", _SCRIPT], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    before, after = map(float, run.stdout.split("us")[-1].split())
    print(f"attend_status: {before:.1f} us before the kernel's first launch, {after:.1f} us behind it")
    assert before < after  # one device synchronisation and one copy from the device less
