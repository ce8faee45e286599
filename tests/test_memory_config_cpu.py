"""Configurations of the memory core that no network can be made of are refused by name."""
import pytest

from surfb200.models import memory as M


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=-4), dict(heads=2), dict(dim=0), dict(heads=16, dim=8), dict(keys=0), dict(keys=-8)])
def test_heads_of_the_delta_core(bad):
    with pytest.raises(ValueError, match="heads must be a positive multiple of 4"):
        M.MemoryNet(M.MemoryConfig(core="delta", **bad))


def test_the_scan_core_takes_no_notice_of_them():
    assert M.MemoryNet(M.MemoryConfig(dim=32, heads=0, keys=0)).cfg.core == "scan"
