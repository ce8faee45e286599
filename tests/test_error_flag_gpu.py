"""The flag that kernels report errors through, in a process whose first call is captured into a graph."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import torch, surfb200
from surfb200.ops import _lib, delta as DR, gemm as G, rl as R
r = lambda *s: torch.randn(*s, device="cuda")
tokens = lambda n: (r(n, 2, 16), r(n, 2, 16), r(n, 2, 16), r(n, 2), r(n, 2), -torch.ones(2, device="cuda"))
state, z, row = r(3, 2, 16, 16), r(5, 3000), r(5)
good, answers = tokens(3), torch.zeros(5, dtype=torch.int32, device="cuda")
calls = dict(step=lambda: DR.gated_delta_step(*good, state), policy=lambda: R.policy_loss(z, answers, row, row))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    calls["%s"]()
G.check_error_flag("cuda")
DR.gated_delta_step(*tokens(1), state, slots=torch.tensor([7], dtype=torch.int32, device="cuda"))
graph.replay()
try:
    G.check_error_flag("cuda")
except _lib.KernelError as e:
    assert "state slot" in str(e)
else:
    raise SystemExit("the replay cleared what another call had reported")
graph.replay()
G.check_error_flag("cuda")
"""


@pytest.mark.parametrize("first", ["step", "policy"])
def test_a_replay_keeps_what_was_reported(first):
    r = subprocess.run([sys.executable, "-c", SCRIPT % first], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
