"""What AdamW's moments in 8 bits keep of gradients that change, step after step beside float32
moments, for both roundings of their codes (the kernels equal these formulas bit for bit:
tests/test_gpu_adamw_codes.py)."""

from __future__ import annotations

import functools
import math

import pytest
import torch

import adamw_plain as plain

BETAS = (0.9, 0.999)
HALF = 3000  # steps before and after the change


THEN = (0.4, 0.1, 0.01, 0.0)  # one block for each


@functools.cache
def _moments(rounding: str) -> dict:
    """In each block element 0 has gradient 1 throughout, the others 0.1 and after HALF steps the block's.
    Returns the others' moments at the end, and what they are in float64, by the second gradient."""
    b1, b2 = BETAS
    n = 256 * len(THEN)
    m, ms = torch.zeros(n, dtype=torch.int8), torch.zeros(len(THEN))
    v, vs = torch.zeros(n, dtype=torch.uint8), torch.zeros(len(THEN))
    exact = torch.zeros(2, len(THEN), dtype=torch.float64)
    for t in range(1, 2 * HALF + 1):
        g = torch.full((len(THEN),), 0.1) if t <= HALF else torch.tensor(THEN)
        grad = g.repeat_interleave(256)
        grad[::256] = 1.0
        exact[0] = b1 * exact[0] + (1 - b1) * g.double()
        exact[1] = b2 * exact[1] + (1 - b2) * g.double() ** 2
        m, ms = plain.encode(plain.decode(m, ms, False) * b1 + grad * (1 - b1), False, rounding, t, 0)
        v, vs = plain.encode(plain.decode(v, vs, True) * b2 + (grad * grad) * (1 - b2), True, rounding, t, 0)
    m, v = (plain.decode(c, s, second).view(-1, 256)[:, 1:].double() for c, s, second in ((m, ms, False), (v, vs, True)))
    return {g: (m[i], v[i], exact[0, i].item(), exact[1, i].item()) for i, g in enumerate(THEN)}


def test_nearest_codes_lose_small_changes():
    """The known error of rounding to the nearest code while the block's largest element holds."""
    m, v, em, ev = _moments("nearest")[0.4]
    assert abs(math.sqrt(ev) - 0.39) < 0.01 and ((v.sqrt() - 0.101).abs() < 0.002).all()  # a second moment that does not rise
    m, v, em, ev = _moments("nearest")[0.0]
    assert em < 1e-100 and ((m - (9 / 127) ** 2).abs() < 1e-6).all()  # code 9, for good
    assert math.sqrt(ev) < 0.025 and ((v.sqrt() - 0.1).abs() < 0.002).all()


@pytest.mark.parametrize("then", [0.4, 0.1, 0.01])
def test_unbiased_codes_follow_changes(then):
    """Means of 255 elements. A second moment takes about (4th root of the change) x 80 single codes of 4 / c of
    it at random times: from 0.1 to 0.4 and back to rest 77 codes of 0.025 to 0.05, to 0.01 (where the old gradient's
    0.05 of v is still most of it) 43 of 0.05 to 0.1, so that one element's relative deviation is at most
    sqrt(43) x 0.08 = 0.5, the mean's a sixteenth of that; five of those are 0.16. The first moment is within a code
    or two of its value, at most 2 / c = 0.16 of it at c = 12.7: the mean's five deviations are 0.05."""
    m, v, em, ev = _moments("unbiased")[then]
    assert abs(v.mean().item() / ev - 1) < 0.16 and abs(m.mean().item() / em - 1) < 0.05


def test_unbiased_codes_forget():
    m, v, em, ev = _moments("unbiased")[0.0]
    assert not m.any() and abs(v.mean().item() / ev - 1) < 0.16


def test_an_unbiased_second_moment_is_not_rounded_to_zero():
    x = torch.full((256,), 1e-14)
    x[0], x[1] = 1.0, 0.0
    code, scale = plain.encode(x, True, "unbiased", 5, 1)
    assert code[0] == 255 and code[1] == 0 and (code[2:] == 1).all() and scale == 1


def test_random_words():
    """Mean 1/2 and variance 1/12 over a million elements within five deviations, no correlation of neighbours,
    of steps, of tensors or of the two moments."""
    n = 1 << 20
    u = plain.uniforms(7, 0, n, False).double()
    assert abs(u.mean() - 0.5) < 5 * (n * 12) ** -0.5 and abs(u.var() - 1 / 12) < 5 * (180 * n) ** -0.5
    others = [u.roll(1), plain.uniforms(8, 0, n, False), plain.uniforms(7, 1, n, False), plain.uniforms(7, 0, n, True)]
    for w in others:
        assert abs(((u - 0.5) * (w.double() - 0.5)).mean() * 12) < 5 * n ** -0.5
