"""cos/sin tables of positions with several axes, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from mote_b200 import errors, ops  # noqa: E402
from mote_b200.context import CudaContext  # noqa: E402
from mote_b200.types import DType, RopeAxes, plain  # noqa: E402
from tests._paged_cache import get, put  # noqa: E402


@pytest.fixture(scope="module")
def ctx():
    return CudaContext(0)


def angles(positions, sections, theta, order):
    pairs, out, used = sum(sections), [], [0] * len(sections)
    for j in range(pairs):
        if order is RopeAxes.Interleaved:
            a = j % len(sections)
            a = a if j // len(sections) < sections[a] else 0
        else:
            a = next(i for i in range(len(sections)) if j < sum(sections[:i + 1]))
        e = used[a] / sections[a] if order is RopeAxes.Own else j / pairs
        used[a] += 1
        out.append(positions[a].astype(np.float64) * np.float64(theta) ** -e)
    assert tuple(used) == tuple(sections)
    return np.stack(out, 1)


def tables(ctx, positions, sections, theta, order):
    shape = (positions.shape[1], sum(sections))
    c, s = (put(ctx, np.full(shape, np.nan, np.float32)) for _ in range(2))
    ops.rope_cos_sin_axes_f32(ctx, put(ctx, positions), c, s, sections, theta, order)
    return get(ctx, c, np.float32), get(ctx, s, np.float32)


def check(got, want, largest):
    """Half a step of what is left of the angle (at most half a quarter turn:
    2^-26 quarter turns, 2^-25.3 in the angle), two steps of a sine below 1
    (2^-23), and the frequency's own error: exp2 and its argument of up to 20
    bits before the point are off by 2^-47 of it together."""
    assert np.abs(got - want).max() <= 2.0 ** -25.3 + 2.0 ** -23 + largest * 2.0 ** -47


@pytest.mark.parametrize("order", list(RopeAxes))
@pytest.mark.parametrize("tokens,sections", [
    (1, (16, 24, 24)), (7, (1,)), (37, (24, 20, 20)), (300, (32, 32)), (5, (1, 1, 1)),
    (19, (33, 32, 32, 31)), (2500, (11, 10, 10)), (129, (64, 0, 0)), (64, (0, 5))])
def test_tables(ctx, order, tokens, sections):
    if order is RopeAxes.Interleaved and any(
            n and a + len(sections) * (n - 1) >= sum(sections) for a, n in enumerate(sections) if a):
        with pytest.raises(errors.CudaError):  # an axis would not find its pairs
            tables(ctx, np.zeros((len(sections), tokens), np.int32), sections, 1e4, order)
        return
    rng = np.random.default_rng(tokens)
    positions = rng.integers(0, 4000, (len(sections), tokens)).astype(np.int32)
    theta = [1e4, 5e5][tokens % 2]
    want = angles(positions, sections, theta, order)
    c, s = tables(ctx, positions, sections, theta, order)
    check(c, np.cos(want), 4000)
    check(s, np.sin(want), 4000)


def test_far_and_negative_positions(ctx):
    """Positions up to 2^20, where f32 angles would be off by 2^-4, and below 0."""
    rng = np.random.default_rng(3)
    positions = rng.integers(-(1 << 20), 1 << 20, (3, 500)).astype(np.int32)
    positions[:, :4] = [[1 << 20] * 4, [-(1 << 20)] * 4, [0] * 4]
    want = angles(positions, (16, 24, 24), 1e6, RopeAxes.Sections)
    c, s = tables(ctx, positions, (16, 24, 24), 1e6, RopeAxes.Sections)
    check(c, np.cos(want), 1 << 20)
    check(s, np.sin(want), 1 << 20)


def test_farthest_positions_stay_on_the_circle(ctx):
    """2^31 - 1 and -2^31: the product in 64 bits is off by 2^-22 of a radian."""
    positions = np.array([[2 ** 31 - 1, -2 ** 31]], np.int32)
    c, s = tables(ctx, positions, (64,), 1e4, RopeAxes.Sections)
    want = angles(positions, (64,), 1e4, RopeAxes.Sections)
    check(c, np.cos(want), 2.0 ** 31)
    check(s, np.sin(want), 2.0 ** 31)


def test_one_axis_is_the_plain_table(ctx):
    """One axis: the tables of rope_cos_sin_f32, which rounds a cosine taken in 64 bits once."""
    positions = np.random.default_rng(0).integers(0, 100000, (1, 777)).astype(np.int32)
    c, s = tables(ctx, positions, (64,), 5e5, RopeAxes.Sections)
    c1, s1 = (ctx.empty(plain((777, 64), DType.F32)) for _ in range(2))
    ops.rope_cos_sin_f32(ctx, put(ctx, positions[0]), c1, s1, 5e5)
    for got, other in ((c, c1), (s, s1)):
        check(got, get(ctx, other, np.float32).astype(np.float64), 100000)
