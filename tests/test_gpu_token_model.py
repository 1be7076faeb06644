"""The operators over sequences of tokens together: a selective layer against its formula, and a model of
tokens trained with AdamW and served token by token."""

from __future__ import annotations

import pytest
import torch

import gru_qat_amd as G

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def _layer(layer, x, reset):
    """A selective layer in float64 on the CPU, step by step, from its parameters p (a dict)."""
    p = {k: v for k, v in layer.items()}
    T, B, _ = x.shape
    H, N, R, W = p["D"].shape[0], p["A_log"].shape[1], p["weight_d"].shape[1], p["weight_c"].shape[1]
    h, z = (x @ p["weight_i"].t()).chunk(2, -1)
    A = -torch.exp(p["A_log"])
    state, past, out = x.new_zeros(B, H, N), x.new_zeros(B, W - 1, H), []
    for t in range(T):
        if reset is not None:
            keep = ~reset[t][:, None, None]
            state, past = state * keep, past * keep
        window = torch.cat([past, h[t][:, None]], 1)
        past = window[:, 1:]
        u = torch.nn.functional.silu((window * p["weight_c"].t()).sum(1) + p["bias_c"])
        d, b, c = (u @ p["weight_x"].t()).split([R, N, N], -1)
        dt = torch.nn.functional.softplus(d @ p["weight_d"].t() + p["bias_d"])
        state = torch.exp(dt[..., None] * A) * state + (dt * u)[..., None] * b[:, None]
        y = (state * c[:, None]).sum(-1) + p["D"] * u
        out.append((y * torch.nn.functional.silu(z[t])) @ p["weight_o"].t() + x[t])
    return torch.stack(out)


def _gated(p, x, reset):
    gi = x @ p["weight_g"].t() + p["bias_g"]
    H = gi.shape[-1] // 2
    h, out = x.new_zeros(x.shape[1], H), []
    for t in range(x.shape[0]):
        z, n = torch.sigmoid(gi[t, :, :H]), torch.tanh(gi[t, :, H:])
        if reset is not None:
            h = h * ~reset[t][:, None]
        h = z * h + (1 - z) * n
        out.append(h @ p["weight_o"].t() + p["bias_o"] + x[t])
    return torch.stack(out)


def _model(dev, dtype=F32, batch_first=False, V=101, size=24):
    torch.manual_seed(0)
    layers = [G.SelectiveLayer(size, 40, states=5, batch_first=batch_first, device=dev, dtype=dtype),
              G.GatedLinearLayer(size, 36, batch_first=batch_first, device=dev, dtype=dtype),
              G.SelectiveLayer(size, 48, taps=3, rank=4, batch_first=batch_first, device=dev, dtype=dtype)]
    return G.TokenModel(V, size, layers, device=dev, dtype=dtype)


def _double(model, tokens, targets, reset):
    """(logprobs, the parameters' gradients of the mean loss) of the model in float64 on the CPU."""
    leaves = {k: v.detach().cpu().double().requires_grad_(True) for k, v in model.named_parameters()}
    of = lambda k: {n.split(".", 2)[2]: v for n, v in leaves.items() if n.startswith(f"layers.{k}.")}
    w = leaves["weight"]
    y = torch.where((tokens >= 0)[..., None], model.scale * w[tokens.clamp(min=0)], 0.0)
    y = _layer(of(2), _gated(of(1), _layer(of(0), y, reset), reset), reset)
    logp = torch.log_softmax(y @ w.t(), -1).gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    logp = torch.where(targets >= 0, logp, 0.0)
    (-logp.mean()).backward()
    return logp.detach(), {k: v.grad for k, v in leaves.items()}


def _tokens(T, B, V, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    tokens, targets = torch.randint(0, V, (T, B), generator=g), torch.randint(0, V, (T, B), generator=g)
    tokens[T // 2:, 1] = -1  # a short row, padded
    targets[T // 2:, 1] = -1
    reset = torch.rand(T, B, generator=g) < 0.05
    return tokens.to(dev), targets.to(dev), reset.to(dev)


@pytest.mark.parametrize("batch_first", [False, True])
def test_model_and_gradients_against_their_formulas(dev, batch_first):
    """float32: three layers of a few hundred roundings of 2^-24 each, on terms of a few times the results'
    size: 2^-13 of the largest element covers them, and no mistake in a formula."""
    T, B, V = 45, 3, 101
    model = _model(dev, batch_first=batch_first)
    tokens, targets, reset = _tokens(T, B, V, dev)
    flip = (lambda t: t.t()) if batch_first else (lambda t: t)
    logp, entropy, _, best = model(flip(tokens), flip(targets), reset=flip(reset), top=3)
    (-logp.mean()).backward()
    want, grads = _double(model, tokens.cpu(), targets.cpu(), reset.cpu())
    assert (flip(logp).detach().cpu().double() - want).abs().max() < 2.0 ** -13 * want.abs().max()
    assert (flip(logp)[T // 2:, 1] == 0).all() and (entropy > 0).all() and best.shape == (*flip(tokens).shape, 3)
    for k, p in model.named_parameters():
        d = (p.grad.cpu().double() - grads[k]).abs().max()
        assert d < 2.0 ** -13 * grads[k].abs().max(), (k, d, grads[k].abs().max())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_tokens_one_by_one(dev, dtype):
    """Serving gives what the whole sequence gives, with rows of the caches in any order and empty rows."""
    T, B, V = 20, 3, 101
    model = _model(dev, dtype)
    tokens, _, _ = _tokens(T, B, V, dev, seed=1)
    tokens = tokens.clamp(min=0)
    with torch.no_grad():
        _, _, whole, _ = model(tokens, tokens, top=4)
    states = model.new_states(7)
    slots = torch.tensor([5, -1, 0, 3], dtype=torch.int32, device=dev)
    rows = [0, 2, 3]
    for t in range(T):
        batch = torch.full((4,), -1, device=dev)
        batch[rows] = tokens[t]
        lp, ids = model.step(batch, states, slots, top=4)
        assert ids.dtype == torch.int64 and lp.shape == (4, 4)
        # float32: other orders of sums. bfloat16: units of 2^-8 of activations of a few units, three layers
        assert (lp[rows] - whole[t]).abs().max() < (2.0 ** -13 if dtype == F32 else 0.25) * whole[t].abs().max()


def test_prompt_then_tokens(dev):
    """A prompt's states are the caches that single tokens continue."""
    T, B, V = 18, 2, 101
    model = _model(dev)
    tokens = _tokens(T, B, V, dev, seed=2)[0].clamp(min=0)
    with torch.no_grad():
        y, states = model.hidden(tokens[:11])
        full, _ = model.hidden(tokens)
        _, _, want, ids = model(tokens, tokens, top=2)
        rest, _ = model.hidden(tokens[11:], states)
    assert (rest - full[11:]).abs().max() < 2.0 ** -13 * full.abs().max()
    for t in range(11, T):
        lp, best = model.step(tokens[t], states, top=2)
        assert (lp - want[t]).abs().max() < 2.0 ** -13 * want[t].abs().max()


@pytest.mark.parametrize("dtype,bits", [(F32, 32), (BF16, 8)])
def test_a_few_steps_of_training(dev, dtype, bits):
    """Loss, backward and update run together, and repeat bit for bit."""

    def run():
        model = _model(dev, dtype)
        opt = G.AdamW(model.parameters(), lr=1e-3, state_bits=bits)
        tokens, targets, reset = _tokens(64, 4, 101, dev, seed=3)
        for _ in range(4):
            opt.zero_grad()
            logp, entropy, _, _ = model(tokens, targets, reset=reset)
            (-logp.mean() - 0.01 * entropy.mean()).backward()
            assert all(p.grad.isfinite().all() for p in model.parameters())
            opt.step()
        return [p.detach().clone() for p in model.parameters()]

    a, b = run(), run()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
