"""Beam search's selection (batch_beam.select) where its sums lose most: long rows of equal logits, thousands of beams,
scores below every float."""
import math

import numpy as np
import pytest
import torch

from tests.test_beam_gpu import check
from tests.util import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu

# Heights of the one logit of 64 in a row's first tile that stand out; all others are 0.  Added up one after the other in float, their sums are off in one direction, by 1.7e-6 of
# 248320 terms and 1e-5 of four million.
HEIGHTS = [0.00830078125, 0.030029296875, 0.53125, 1.234375]


def standing(dev, V, height):
    """a row [V] and log sum exp of it"""
    x = torch.zeros(V, dtype=BF16, device=dev)
    x[0:512:8] = height
    return x, math.log((V - 64) + 64 * math.exp(height))


def bound(height):
    """of log sum exp: an exponential (2^-23 of it) of an argument of `height` log2 e (2^-24 of it, the constant's own rounding 2^-26), sums of 32 in float (eight in a row: 4.5 times 2^-24
    of what they come to, then two), the rest in double"""
    return 2 ** -23 + height * 1.4427 * (2 ** -24 + 2 ** -26) + (4.5 + 2) * 2 ** -24


@pytest.mark.parametrize("height", HEIGHTS)
@pytest.mark.parametrize("V", [248320, (1 << 22) + 77])
def test_sums_of_many_beams(dev, V, height):
    """4096 rows, each of which one wavefront sums up; the beams' scores are such that hardly more than the error of the sum is left"""
    import qwen_tailor_amd as qt
    x, lse = standing(dev, V, height)
    G = 4096
    scores = torch.full((G, 1), lse, device=dev)                 # (float32 of it)
    want = float(scores[0, 0].double()) + height - lse
    s, w, t = qt.batch_beam.select(x.expand(G, 1, V), scores, 2)
    assert int(w.abs().max()) == 0 and t.tolist() == [[0, 8]] * G
    err = float((s.double() - want).abs().max())
    assert err <= bound(height) + 2 ** -24 * abs(want), f"{err:.2e}"


def test_order_of_two_beams(dev):
    """candidates of two beams a little further apart than the sums are off: the order is that of the definition"""
    import qwen_tailor_amd as qt
    V, G = 248320, 2048
    (a, la), (b, lb) = standing(dev, V, HEIGHTS[0]), standing(dev, V, HEIGHTS[1])
    least = bound(HEIGHTS[0]) + bound(HEIGHTS[1])
    x = torch.stack([a, b]).expand(G, 2, V)
    sa = np.float32(12.0)
    gap = lambda sb: (float(sb) + HEIGHTS[1] - lb) - (float(sa) + HEIGHTS[0] - la)  # noqa: E731
    steps = [np.float32(sa + k * 2.0 ** -20) for k in range(-40000, 40000)]
    near = [s for s in steps if 1.05 * least < abs(gap(s)) < 1.05 * least + 2e-6]
    assert any(gap(s) > 0 for s in near) and any(gap(s) < 0 for s in near)
    sb = [near[g % len(near)] for g in range(G)]
    scores = torch.tensor(np.stack([np.full(G, sa), np.array(sb, np.float32)], 1), device=dev)
    _, w, t = qt.batch_beam.select(x, scores, 1)
    assert w.flatten().tolist() == [int(gap(s) > 0) for s in sb]
    assert not bool(t.any())


@pytest.mark.parametrize("G,W,V,dtype", [(700, 3, 9000, torch.bfloat16), (4500, 1, 5000, torch.float32), (1030, 1, 20001, torch.float16)])
def test_thousands_of_beams(dev, G, W, V, dtype):
    g = torch.Generator(dev).manual_seed(G)
    x = torch.empty((G, W, V), dtype=dtype, device=dev).normal_(0.0, 2.5, generator=g)
    check(x, torch.empty((G, W), device=dev).uniform_(-12.0, -2.0, generator=g), 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rising_rows(dev, dtype):
    """logits that rise by hundreds along the row, and a row whose first part is masked with the type's lowest value: the reference point of the sums has to follow"""
    V = 30000
    up = torch.arange(V, device=dev) * 0.02
    low = torch.where(torch.arange(V, device=dev) < 25000, torch.finfo(dtype).min, up % 7)
    x = torch.stack([up, up.flip(0), low, low.flip(0)])[None].to(dtype)
    check(x, torch.tensor([[-1.0, -2.0, -600.0, -3.0]], device=dev), 6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_below_every_float(dev, dtype):
    """a score that float32 gives out as -inf is no candidate: its place gets -inf, -1, -1 like any that is left over"""
    import qwen_tailor_amd as qt
    big = torch.finfo(dtype).max
    x = torch.full((1, 2, 700), -big, dtype=dtype, device=dev)
    x[0, 0, 300], x[0, 1, 5], x[0, 1, 699] = big, 0.0, -1.0
    s, w, t = qt.batch_beam.select(x, torch.tensor([[-1.0, -2.0]], device=dev), 5)
    assert w[0, :3].tolist() == [0, 1, 1] and t[0, :3].tolist() == [300, 5, 699]
    lse = math.log(1 + math.exp(-1.0))
    assert float((s[0, :3].cpu().double() - torch.tensor([-1.0, -2.0 - lse, -3.0 - lse], dtype=torch.float64)).abs().max()) <= 1e-6
    # of the second beam the others are at -big, which a float holds; those of the first at -2 big are none
    assert w[0, 3:].tolist() == [1, 1] and t[0, 3:].tolist() == [0, 1] and bool((s[0, 3:] == -big).all())
    s, w, t = qt.batch_beam.select(x[:, :1], torch.tensor([[-1.0]], device=dev), 3)
    assert w.tolist() == [[0, -1, -1]] and t.tolist() == [[300, -1, -1]] and s.tolist() == [[-1.0, -math.inf, -math.inf]]
