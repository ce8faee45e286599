"""What the delta rule keeps for its gradient: sizes whose values the blocks' warps do not divide, among few and
many heads of sequences, with the memory about the kept states left as it was."""
import pytest
import torch

from surfb200.ops import delta as DR
from test_delta_gpu import BF, F32, INNER, NAMES, call, make, oracle, rel

pytestmark = pytest.mark.gpu

GUARD = 4096                                            # numbers before and behind what is kept


@pytest.fixture
def guarded(monkeypatch):
    """``saved`` of the forward calls in a buffer with GUARD numbers of 7 on both sides, which must stay, and 7 at
    first itself."""
    new_empty, bufs = torch.Tensor.new_empty, []

    def inside(self, size, **kw):
        if not isinstance(size, tuple) or len(size) != 5:          # the kept states alone have five axes
            return new_empty(self, size, **kw)
        n = torch.Size(size).numel()
        bufs.append(torch.full((n + 2 * GUARD,), 7.0, device=self.device))
        return bufs[-1][GUARD:GUARD + n].view(size)

    monkeypatch.setattr(torch.Tensor, "new_empty", inside)
    yield
    assert bufs
    for buf in bufs:
        assert bool((buf[:GUARD] == 7.0).all()) and bool((buf[-GUARD:] == 7.0).all())


def kept(c):
    """The states before every 16 tokens, by the definition in 64 bits, of rows without lengths."""
    x = [t.double() for t in c["tokens"]]
    s, out = c["state"].double(), []
    for lo in range(0, x[0].shape[1], DR.TILE):
        out.append(s)
        part = [t[:, lo:lo + DR.TILE] for t in x]
        reset = None if c["reset"] is None else c["reset"][:, lo:lo + DR.TILE]
        s = DR.gated_delta_reference(*part, c["A"].double(), dt_bias=c["dt_bias"].double(), state=s, reset=reset)[1]
    return torch.stack(out, 1)                          # [B, tiles, H, V, K]


HEADS = [(40, 1), (30, 2), (20, 4), (147, 1), (37, 4), (128, 4)]           # rows, value heads


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,h", HEADS)
@pytest.mark.parametrize("nv", [40, 48, 72, 80, 96, 104, 112])
def test_values_that_the_warps_do_not_divide(guarded, nv, rows, h, dtype):
    """Tolerances of what is 32-bit: three planes of 2^-24 each for either type of token (test_delta_gpu's of 32-bit
    tokens); states kept are final states of shorter rows."""
    nk = {0: 32, 1: 64, 2: 128}[(nv // 8 + rows) % 3]
    c = make(rows, 21, 1, h, nk, nv, dtype, reset=0.05, seed=nv + rows)
    out, final, want = oracle(c)
    r, d = call(c)
    half = torch.finfo(dtype).eps / 2
    assert rel(r.out, out) < half + INNER[dtype]
    assert rel(r.final, final) < INNER[F32]
    states = r.saved[..., :nk]
    assert rel(states, kept(c)) < INNER[F32]
    for n, x in zip(NAMES, d):
        assert rel(x, want[n]) < 2 * INNER[dtype] + (half if n not in ("A", "dt_bias", "state") else 0), n


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nk", [32, 64, 128])
@pytest.mark.parametrize("rows,nv", [(128, 96), (50, 72), (74, 33), (80, 47), (37, 100), (60, 65), (147, 48), (300, 111)])
def test_kept_states_end_with_their_head(guarded, rows, nv, nk, dtype):
    """Ragged rows: tiles past a row's length are not written, nor is anything about them."""
    c = make(rows, 50, 1, 1, nk, nv, dtype, reset=0.1, ragged=True, seed=nv)
    out, final, want = oracle(c)
    r, d = call(c)
    half = torch.finfo(dtype).eps / 2
    assert rel(r.out, out) < half + INNER[dtype] and rel(r.final, final) < INNER[F32]
    tiles = (c["lengths"][:, None] + DR.TILE - 1) // DR.TILE
    unwritten = torch.arange(r.saved.shape[1], device="cuda")[None] >= tiles
    assert bool((r.saved[unwritten] == 7.0).all())
    for n, x in zip(NAMES, d):
        assert rel(x, want[n]) < 2 * INNER[dtype] + (half if n not in ("A", "dt_bias", "state") else 0), n


def test_a_core_of_such_heads_runs():
    """Four heads of 96 values: two warps of each head's second block lie behind the last value."""
    from surfb200.models import memory as M
    cfg = M.MemoryConfig(dim=384, core="delta", heads=4, keys=32)
    r = M.train_recall(2, envs=128, length=20, cfg=cfg, act_steps=2)
    assert all(torch.isfinite(torch.tensor(r["loss"])))
