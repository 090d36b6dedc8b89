"""CPU checks that the bounds on a whole call's distance hold for the kernels' arithmetic and show a part that is missing."""
import pytest
import torch

import paged_norms as N
from helpers import randn_half
from oracle import paged_oracle as P

T = [300, 777, 64]


def setup(e4m3, group, scale):
    c = N.plain_cache(T, 2, 128, 16, e4m3, seed=601)
    q = torch.stack([P.rope(randn_half((2 * group, 128), 602 + b), T[b], 128, 10000.0) for b in range(3)])
    return c, q, N.exact(q, c, c["table"], T, range(3), scale)


@pytest.mark.parametrize("group", [1, 8])
def test_e4m3_parts(group):
    scale = 128 ** -0.5
    c, q, want = setup(True, group, scale)
    at = lambda *parts: N.off(N.emulated(q, c, c["table"], T, scale, "e4m3", *parts), want)  # noqa: E731
    assert at(3, 4) < N.SPLIT
    assert at(2, 4) > N.SPLIT and at(3, 3) > N.SPLIT


@pytest.mark.parametrize("group", [1, 8])
def test_fp16_parts(group):
    """Scores of a wider spread: there one fp16 rounding of the queries is more than the result's own."""
    c, q, want = setup(False, group, N.WIDE)
    at = lambda parts: N.off(N.emulated(q, c, c["table"], T, N.WIDE, "fp16", parts), want)  # noqa: E731
    assert at(2) < N.SPLIT < at(1)


def test_parts_are_exact():
    """Four cut e5m2 parts are the fp16 weight, from the largest down to the last bit of the subnormal ones."""
    w = torch.cat([torch.rand(20000, dtype=torch.float64) * 2.0 ** torch.randint(-24, 16, (20000,)),
                   torch.tensor([0.0, 2.0 ** -24, 2.0 ** -14, 1.0, 2.0 ** 13, 2.0 ** 15.75], dtype=torch.float64)])
    assert torch.equal(N.e5m2_parts(w, 4), w.half().double())
    assert not torch.equal(N.e5m2_parts(w, 3), w.half().double())
