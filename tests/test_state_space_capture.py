"""Every call may be its process's first, and captured: nothing has been set up by an eager one."""
import os
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import sys
import torch
import fastaf_kernel_b200 as fk
which, P = sys.argv[1], int(sys.argv[2])
dev = torch.device("cuda", 0)
g = torch.Generator(device=dev).manual_seed(0)
bf16 = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)
T, H = 4133, 2                                             # few long prompts: cut, with a workspace
x, dt, B, C, A_log = bf16(T, H, P), bf16(T, H), bf16(T, 1, 128), bf16(T, 1, 128), torch.zeros(H, device=dev)
cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
w, state = torch.randn(64, 4, device=dev), torch.randn(T, H, P, 128, device=dev)[:3].clone()
rows = bf16(T, 64)
calls = dict(
    ssm_prefill=lambda: fk.ssm_prefill(x, dt, A_log, B, C, None, None, None, cu),
    ssm_recurrent=lambda: fk.ssm_prefill(x, dt, A_log, B, C, None, None, None, cu, method="recurrent"),
    ssm_decode=lambda: fk.ssm_decode(x[:3, None], dt[:3, None], A_log, B[:3, None], C[:3, None], None, None, state),
    conv_prefill=lambda: fk.conv_prefill(rows, w, None, None, cu),
    conv_decode=lambda: fk.conv_decode(rows, w, None, None))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = calls[which]()
graph.replay()
want = calls[which]()
torch.cuda.synchronize()
fk.device_status()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("the same")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("which,P", [("ssm_prefill", 128), ("ssm_prefill", 64), ("ssm_recurrent", 64), ("ssm_decode", 128),
                                     ("conv_prefill", 64), ("conv_decode", 64)])
def test_the_first_call_may_be_captured(which, P):
    r = subprocess.run([sys.executable, "-c", CHILD, which, str(P)], cwd=REPO, capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=REPO))
    assert r.returncode == 0 and "the same" in r.stdout, r.stderr[-2000:]
