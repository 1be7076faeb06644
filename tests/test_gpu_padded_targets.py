"""Rows of padding in token_logprobs: what their logits hold does not reach the gradients."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G
import sequence_plain as P

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
ODD = (float("nan"), float("inf"), -float("inf"))


def _rows(V, dtype, dev):
    g = torch.Generator().manual_seed(V)
    x = (2 * torch.randn(12, V, generator=g)).to(dtype).to(dev)
    tokens = torch.randint(0, V, (12,), generator=g).to(dev)
    return x, tokens, torch.randn(12, generator=g).to(dev), torch.randn(12, generator=g).to(dev)


# a row in one part and in several, whole accesses and not
@pytest.mark.parametrize("V", [130, 301, 9000, 40001])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("entropy", ["none", "masked"])
def test_odd_logits_of_padding_send_no_gradient(dev, V, dtype, entropy):
    x, tokens, dl, de = _rows(V, dtype, dev)
    for k, odd in enumerate(ODD):
        x[k], x[3 + k, V // 2] = odd, odd
    tokens[:6] = -1
    tokens[6] = V  # out of range: NaN, and no gradient
    x[6] = float("nan")
    leaf = x.clone().requires_grad_(True)
    lp, h, _, _ = G.token_logprobs(leaf, tokens)
    assert (lp[:6] == 0).all() and lp[6].isnan()
    masked = torch.where(torch.arange(12, device=dev) < 7, 0.0, de)
    outs, grads = ((lp, h), (dl, masked)) if entropy == "masked" else ((lp,), (dl,))
    dx, = torch.autograd.grad(outs, leaf, grads)
    assert (dx[:7] == 0).all()
    keep = slice(7, None)
    want = P.token_logprobs(x[keep], tokens[keep], 0, dl[keep], masked[keep] if entropy == "masked" else None)[4]
    p = torch.softmax(x[keep].double().cpu(), -1)
    hot = torch.nn.functional.one_hot(tokens[keep].cpu(), V)
    # logits are below 10, log probabilities and the entropy below 20; exp is off by 8 units at an argument off by 2 of 10
    size = (p + hot) * (dl[keep].cpu().double().abs() + 40 * de[keep].cpu().double().abs())[:, None]
    P.assert_within(dx[keep], want, size, V // 64 + 64 + 8 + 20, "dx")


def test_a_row_without_a_gradient(dev):
    """Zeros from the loss in a row whose token counts: no gradient, also of NaN logits; a gradient of either makes it NaN."""
    x, tokens, dl, de = _rows(70, F32, dev)
    x[2:5, 3] = float("nan")
    leaf = x.clone().requires_grad_(True)
    lp, h, _, _ = G.token_logprobs(leaf, tokens)
    dl[2], de[2], dl[3], de[4] = 0.0, 0.0, 0.0, 0.0
    dx, = torch.autograd.grad((lp, h), leaf, (dl, de))
    assert (dx[2] == 0).all() and dx[3].isnan().any() and dx[4].isnan().any()
    assert dx[[0, 1, 5, 6, 7, 8, 9, 10, 11]].isfinite().all()


@pytest.mark.parametrize("padded", [0, 3, 11])
def test_the_loss_over_targets_that_count(dev, padded):
    """What the documents call the loss is the cross entropy that leaves padding out, with its gradient."""
    x, tokens, _, _ = _rows(301, F32, dev)
    tokens[:padded] = -1
    leaf = x.clone().requires_grad_(True)
    lp = G.token_logprobs(leaf, tokens)[0]
    loss = -lp.sum() / (tokens >= 0).sum()
    dx, = torch.autograd.grad(loss, leaf)
    ref = x.double().cpu().requires_grad_(True)
    want = torch.nn.functional.cross_entropy(ref, tokens.cpu(), ignore_index=-1)
    dref, = torch.autograd.grad(want, ref)
    # a loss of some 8, log probabilities up to 20: 12 sums and V / 64 + 64 roundings of them
    assert abs(loss.item() - want.item()) < (301 // 64 + 64 + 12) * 2.0 ** -24 * 20
    hot = torch.nn.functional.one_hot(tokens.clamp(min=0).cpu(), 301) * (tokens >= 0).cpu()[:, None]
    size = (torch.softmax(x.double().cpu(), -1) * (tokens >= 0).cpu()[:, None] + hot) / (12 - padded)
    P.assert_within(dx, dref, size, 301 // 64 + 64 + 8 + 20, "dx")
