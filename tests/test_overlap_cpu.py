"""Outputs whose elements share memory with one another are refused, and no others."""
import itertools

import numpy as np
import pytest
import torch

from surfb200.ops import _lib


@pytest.mark.parametrize("shape,strides,bad", [
    ((4, 8), (8, 1), False), ((4, 8), (9, 1), False), ((4, 8), (5, 1), True), ((4, 8), (7, 1), True), ((4, 1), (0, 1), True),
    ((1, 8), (0, 1), False), ((0, 8), (0, 1), False), ((2, 4, 2, 8), (64, 8, 16, 1), True), ((2, 3, 4, 8), (8, 64, 16, 1), False),
    ((2, 3), (3, 2), False), ((2, 4), (3, 2), False), ((3, 4), (3, 2), True), ((5, 6, 2), (6, 1, 30), False), ((3, 1 << 20), (1 << 30, 1), False),
    ((1 << 12, 1 << 12), ((1 << 12) - 1, 1), True), ((), (), False),
])
def test_elements_that_share_memory(shape, strides, bad):
    t = torch.empty(400).as_strided(shape, strides) if max((sum((n - 1) * s for n, s in zip(shape, strides)), 0)) < 400 else \
        torch.empty(1, device="meta").expand(1)
    if t.device.type == "meta":
        class Far:                                      # such views are larger than any memory here: their layout alone is read
            def __init__(self):
                self.shape, self._s = torch.Size(shape), strides

            def stride(self): return self._s
            def numel(self): return int(np.prod(shape))
            def is_contiguous(self): return False
            def data_ptr(self): return 1 << 20
            def element_size(self): return 4
        t = Far()
    assert _lib.overlaps_itself(t) == bad


def test_against_the_elements_themselves():
    gen = np.random.default_rng(0)
    buf = torch.empty(4000)
    for _ in range(400):
        shape = gen.integers(1, 5, gen.integers(1, 5)).tolist()
        strides = gen.integers(0 if gen.random() < 0.2 else 1, 40, len(shape)).tolist()
        seen = [sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, shape))]
        assert _lib.overlaps_itself(buf.as_strided(shape, strides)) == (len(set(seen)) < len(seen)), (shape, strides)


def test_such_outputs_are_refused():
    buf = torch.zeros(400)
    for out in (buf.as_strided((4, 8), (5, 1)), buf.as_strided((2, 4, 2, 8), (64, 8, 16, 1)), buf[:8].expand(4, 8)):
        for inputs, in_place in (({}, ()), (dict(x=out), ("x",))):
            with pytest.raises(ValueError, match="out has elements that share memory"):
                _lib.require_apart("op", "out", out, inputs, in_place)
    _lib.require_apart("op", "out", buf.as_strided((4, 8), (9, 1)), dict(x=buf[100:]))
