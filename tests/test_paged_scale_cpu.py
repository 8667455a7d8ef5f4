"""CPU test of the paged attention's largest scale: what overflows f32 together with the
factor from e to 2 would make NaN of scores of zero (0 times infinity)."""
from __future__ import annotations

import numpy as np
import pytest

from mote_b200 import _native
from tests.test_paged_cpu import attend


@pytest.fixture(scope="module")
def lib():
    return _native.lib()


def test_scales_next_to_the_largest(lib):
    largest = float(np.finfo(np.float32).max)
    assert attend(lib, tokens=0, scale=largest / 1.45) == 0
    assert attend(lib, tokens=0, scale=largest / 1.44) == 1
    assert attend(lib, tokens=0, scale=largest) == 1
    assert attend(lib, tokens=0, scale=1e-45) == 0
