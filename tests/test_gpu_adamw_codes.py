"""AdamW against its formula in elementary float32 operations, bit for bit, and its moments in 8 bits:
both roundings of the codes, and blocks that are not finite."""

from __future__ import annotations

import pytest
import torch

import adamw_plain as plain
import gru_qat_amd as G
import test_gpu_adamw as adamw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 1e20])
def test_a_block_that_is_not_finite_is_nan_as_a_whole(dev, bad):
    """1e20 leaves the first moment finite and makes the second infinite."""
    s = adamw._make([700], 8, bits=8)
    s["grads"][0][300] = bad
    adamw._run(s, 2)
    m, v = (G.adamw_dequantize_state(s[k + "s"][0], s[k + "_scales"][0]).cpu() for k in ("exp_avg", "exp_avg_sq"))
    assert v[256:512].isnan().all() and v[:256].isfinite().all() and v[512:].isfinite().all()
    assert m[:256].isfinite().all() and m[512:].isfinite().all()
    assert m[256:512].isfinite().all() if bad == 1e20 else m[256:512].isnan().all()


MOMENTS = [(32, "nearest"), (8, "nearest"), (8, "unbiased")]


@pytest.mark.parametrize("bits,rounding", MOMENTS, ids=str)
@pytest.mark.parametrize("kind", adamw.KINDS, ids=lambda k: f"{k[0]}-{k[1]}-{k[2]}".replace("torch.", ""))
def test_steps_equal_the_plain_formula_bit_for_bit(dev, kind, bits, rounding):
    """Parameters, masters, moments, codes and scales after each of five steps, among them blocks that end
    early, tensors without elements, a block of zeros, and the steps that a step count of more than 32 bits gives."""
    s = adamw._make([1, 3, 255, 256, 257, 0, 2049, 6001], 21, *kind[:2], bits=bits, master=kind[2])
    s["grads"][6][256:512] = 0
    for k in ("exp_avgs", "exp_avg_sqs"):
        s[k][6][256:512] = 0
    ref = {k: None if v is None else [t.cpu().clone() for t in v] for k, v in s.items()}
    hyper = dict(lr=0.02, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    for step, scale in ((1, None), (2, 0.25), (3, None), (1000, None), (2 ** 33 + 5, None)):
        plain.step_(ref, step, **hyper, rounding=rounding, grad_scale=scale)
        adamw._run(s, step, **hyper, rounding=rounding,
                   grad_scale=None if scale is None else torch.tensor(scale, device=dev))
        for k, v in s.items():
            for i, t in enumerate(v or ()):
                assert torch.equal(t.cpu(), ref[k][i]), (k, i, step)


@pytest.mark.parametrize("n", [300, 70000])
def test_more_tensors_than_a_launch_keep_their_random_words(dev, n):
    """A tensor's words go by its place in the list, not by its launch (48 tensors) or its workgroup."""
    s = adamw._make([5] * 60 + [n], 22, bits=8)
    ref = {k: None if v is None else [t.cpu().clone() for t in v] for k, v in s.items()}
    plain.step_(ref, 4, **adamw.HYPER, rounding="unbiased")
    adamw._run(s, 4, rounding="unbiased")
    for k in ("params", "exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales"):
        assert all(torch.equal(t.cpu(), r) for t, r in zip(s[k], ref[k])), k


def test_the_optimizer_follows_a_gradient_that_ends(dev):
    """Where gradients end beside one that does not, updates end: within 200 steps no first moment is left
    (0.9^200 of it is 1e-9 of a code). With codes rounded to the nearest they never do."""
    def drift(**kw):
        w = torch.nn.Parameter(torch.zeros(256, device=dev))
        opt = G.AdamW([w], lr=1e-3, weight_decay=0.0, state_bits=8, **kw)
        for t in range(600):
            w.grad = torch.full((256,), 0.1 if t < 200 else 0.0, device=dev)
            w.grad[0] = 1.0
            if t == 400:
                before = w.detach().clone()
            opt.step()
        return (w.detach() - before)[1:].abs(), opt.state[w]

    moved, state = drift()
    assert not moved.any() and not state["exp_avg"][1:].any()
    moved, _ = drift(state_rounding="nearest")
    assert (moved > 200 * 1e-3 * 0.03).all()  # 5 % of the learning rate a step


def test_refusals(dev):
    s = adamw._make([4], 1, bits=8)
    for bad in ("up", None, 1, []):
        with pytest.raises(ValueError, match="rounding"):
            adamw._run(s, 1, rounding=bad)
    with pytest.raises(ValueError, match="rounding"):
        G.AdamW([torch.nn.Parameter(torch.zeros(3, device=dev))], state_bits=8, state_rounding="stochastic")
