"""Trains a stack of gated linear layers and serves it token by token.

The task: from a stream of random vectors, some of which open a new sequence, give at every
step the mean of the vectors since then, weighted towards the recent ones (a moving average
that starts anew). One batch row holds many sequences, so training uses the scan's resets.

    python examples/gated_linear.py [--steps N] [--dtype f32|bf16] [--state-bits 8|32]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gru-triton_amd"))

import gru_qat_amd as G  # noqa: E402


def batch(T, B, size, generator, dev):
    x = torch.randn(T, B, size, generator=generator, device=dev)
    reset = torch.rand(T, B, generator=generator, device=dev) < 1 / 32
    want = torch.empty_like(x)
    h = torch.zeros(B, size, device=dev)
    for t in range(T):
        h = 0.9 * torch.where(reset[t][:, None], 0.0, h) + 0.1 * x[t]
        want[t] = h
    return x, reset, 5.0 * want


def train(steps=200, dtype=torch.float32, state_bits=32, T=96, B=16, size=32, hidden=96, layers=2, dev="cuda", say=print):
    g = torch.Generator(device=dev).manual_seed(0)
    torch.manual_seed(0)
    model = torch.nn.ModuleList([G.GatedLinearLayer(size, hidden, device=dev, dtype=dtype) for _ in range(layers)])
    head = torch.nn.Parameter(torch.eye(size, device=dev, dtype=dtype))
    params = [*model.parameters(), head]
    opt = G.AdamW(params, lr=5e-3, weight_decay=0.0, state_bits=state_bits)
    data = [batch(T, B, size, g, dev) for _ in range(8)]
    losses = []
    for k in range(steps):
        x, reset, want = data[k % len(data)]
        y = x.to(dtype)
        for layer in model:
            y, _ = layer(y, reset=reset)
        y = G.linear_act(y, head)
        loss = (y.float() - want).square().mean()
        for p in params:
            p.grad = None
        loss.backward()
        norm = torch.stack([p.grad.float().square().sum() for p in params]).sum().sqrt()
        for group in opt.param_groups:
            group["lr"] = 5e-3 * (1 - k / steps)
        opt.step(grad_scale=torch.clamp(1.0 / norm, max=1.0))  # clipped, without asking the device
        losses.append(loss.detach())
        if say and (k % 50 == 0 or k == steps - 1):
            say(f"step {k}: loss {loss.item():.4f}")
    return model, head, data, [v.item() for v in losses]


@torch.no_grad()
def serve(model, head, x, dtype):
    """The sequences of x [T, B, size], a token at a time; each request's states are rows of the layers' caches."""
    T, B, _ = x.shape
    slots = torch.randperm(2 * B, device=x.device)[:B].to(torch.int32)
    states = [torch.zeros(2 * B, layer.hidden, device=x.device) for layer in model]
    out = []
    for t in range(T):
        y = x[t].to(dtype)
        for layer, state in zip(model, states):
            y = layer.step(y, state, slots)
        out.append(G.linear_act(y, head))
    return torch.stack(out)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--dtype", choices=("f32", "bf16"), default="f32")
    ap.add_argument("--state-bits", type=int, choices=(8, 32), default=32)
    a = ap.parse_args()
    dtype = torch.float32 if a.dtype == "f32" else torch.bfloat16
    model, head, data, losses = train(a.steps, dtype, a.state_bits)
    x = data[0][0]
    y = x.to(dtype)
    with torch.no_grad():
        for layer in model:
            y, _ = layer(y)
        whole = G.linear_act(y, head)
    served = serve(model, head, x, dtype)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; token by token, the outputs differ by at most "
          f"{(served.float() - whole.float()).abs().max().item():.2e}")
