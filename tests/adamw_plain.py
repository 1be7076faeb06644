"""AdamW's step in elementary float32 operations, each rounded in the order in which the
kernels' documents write them, with moments in 32 bits or as codes of 8 bits."""

from __future__ import annotations

import numpy as np
import torch

BLOCK, TINY, GOLDEN = 256, 2.0 ** -120, 0x9E3779B9
LEVELS = {"exp_avg": 127, "exp_avg_sq": 255}


def _sqrt(x: torch.Tensor) -> torch.Tensor:
    """Correctly rounded: torch's own on the CPU is an ulp off here and there."""
    return torch.from_numpy(np.sqrt(x.numpy()))


def mix(x: torch.Tensor) -> torch.Tensor:
    """On 32-bit words held in int64."""
    low = 0xFFFFFFFF
    x = ((x ^ x >> 16) * 0x6A09E667) & low
    x = ((x ^ x >> 15) * 0xBB67AE85) & low
    return x ^ x >> 16


def uniforms(step: int, tensor: int, n: int, second: bool) -> torch.Tensor:
    word = torch.tensor([step & 0xFFFFFFFF])
    key = mix((mix(word) + tensor * GOLDEN + (step >> 32)) & 0xFFFFFFFF)
    e = torch.arange(n)
    w = mix((key + e * GOLDEN + (e >> 32)) & 0xFFFFFFFF)
    if second:
        w = (w * GOLDEN) & 0xFFFFFFFF
    return (w >> 8).float() * 2.0 ** -24


def _blocks(x: torch.Tensor) -> torch.Tensor:
    pad = torch.zeros(-(-x.numel() // BLOCK) * BLOCK, dtype=x.dtype)
    pad[:x.numel()] = x
    return pad.view(-1, BLOCK)


def decode(code: torch.Tensor, scale: torch.Tensor, second: bool) -> torch.Tensor:
    c = _blocks(code.float())
    if second:
        v = (c * c) * (c * c) * (scale * (1.0 / 255 ** 4))[:, None]
    else:
        v = c * c.abs() * (scale * (1.0 / 127 ** 2))[:, None]
    return v.reshape(-1)[:code.numel()]


def encode(x: torch.Tensor, second: bool, rounding: str, step: int, tensor: int):
    n, levels = x.numel(), 255.0 if second else 127.0
    b = _blocks(x)
    most = b.abs().amax(1)
    none = most < TINY
    inv = torch.where(none, torch.zeros_like(most), 1.0 / torch.where(none, torch.ones_like(most), most))
    part = b.abs() * inv[:, None]
    root = _sqrt(_sqrt(part)) if second else _sqrt(part)
    if rounding == "nearest":
        c = torch.clamp(torch.round(root * levels), max=levels)
    else:
        lo = torch.clamp(torch.floor(root * levels), max=levels - 1)
        up = lo + 1
        below, above = ((lo * lo) * (lo * lo), (up * up) * (up * up)) if second else (lo * lo, up * up)
        at = part * (levels ** 4 if second else levels ** 2)
        u = _blocks(uniforms(step, tensor, n, second))
        c = lo + (u * (above - below) < at - below).float()
        c = torch.where(b.abs() == most[:, None], torch.full_like(c, levels), c)
        if second:
            c = torch.where(b > 0, c.clamp(min=1), c)
        c = torch.where(none[:, None], torch.zeros_like(c), c)
    if not second:
        c = torch.where(b < 0, -c, c)
    code = c.reshape(-1)[:n].to(torch.uint8 if second else torch.int8)
    return code, torch.where(none, torch.zeros_like(most), most)


def step_(s: dict, step: int, lr, betas, eps, weight_decay, rounding="nearest", grad_scale=None) -> None:
    """On lists of CPU tensors by the names of ``adamw_step``'s arguments (None where not used), in place."""
    b1, b2 = betas
    c1, c2 = 1 - b1 ** step, 1 - b2 ** step
    bits8 = s["exp_avg_scales"] is not None
    for i, param in enumerate(s["params"]):
        if param.numel() == 0:
            continue
        g = s["grads"][i].float()
        if grad_scale is not None:
            g = g * grad_scale
        p = (s["masters"] or s["params"])[i].float()
        m, v = s["exp_avgs"][i], s["exp_avg_sqs"][i]
        if bits8:
            m, v = decode(m, s["exp_avg_scales"][i], False), decode(v, s["exp_avg_sq_scales"][i], True)
        m = m * b1 + g * (1 - b1)
        v = v * b2 + (g * g) * (1 - b2)
        p = p * (1 - lr * weight_decay) - m / (_sqrt(v) * c2 ** -0.5 + eps) * (lr / c1)
        if s["masters"] is not None:
            s["masters"][i].copy_(p)
        param.copy_(p)
        if not bits8:
            s["exp_avgs"][i].copy_(m)
            s["exp_avg_sqs"][i].copy_(v)
            continue
        for key, x in (("exp_avg", m), ("exp_avg_sq", v)):
            code, scale = encode(x, key == "exp_avg_sq", rounding, step, i)
            s[key + "s"][i].copy_(code)
            s[key + "_scales"][i].copy_(scale)
