"""Plain 64-bit restatement (CPU, numpy) of the decoder-layer operators:
per-token quantisation, the scaled int8 product and the quantised K/V cache
with the attention over it."""
import math

import numpy as np
import torch

HALF_STEP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.float16, torch.bfloat16)}


def rounding(want, tol, dtype):
    """Bound after one rounding to dtype of a value within tol of want: half a
    step relative to the value, and below the smallest normal number, where
    steps stop shrinking, half a step there (f16: 2^-14 * 2^-10 / 2 = 2^-25)."""
    return tol + HALF_STEP[dtype] * (np.abs(want) + tol + torch.finfo(dtype).tiny)


def quantize_per_token(x: np.ndarray):
    """x f64 [rows, K] (values of the input type) -> (q int8, scale f32)."""
    q = np.zeros(x.shape, np.int8)
    scale = np.zeros(x.shape[0], np.float32)
    for r, row in enumerate(x):
        if not np.isfinite(row).all():
            scale[r] = np.nan
            continue
        scale[r] = np.float32(np.abs(row).max(initial=0.0) / 127)
        if scale[r] > 0:
            q[r] = np.clip(np.rint(row / np.float64(scale[r])), -127, 127).astype(np.int8)
    return q, scale


def scaled_product(q, q_scale, w, w_scale, bias=None, residual=None):
    acc = q.astype(np.int64) @ w.astype(np.int64)
    out = acc * q_scale.astype(np.float64)[:, None] * w_scale.astype(np.float64)
    if bias is not None:
        out = out + bias.astype(np.float64)
    if residual is not None:
        out = out + residual
    return acc, out


def round_bf16(x: float, up: bool) -> float:
    """x rounded up or down to bf16 (8 significant bits, subnormals below 2^-126)."""
    if x == 0.0 or not math.isfinite(x):
        return x
    unit = 2.0 ** (max(math.frexp(x)[1], -125) - 8)
    return (math.ceil(x / unit) if up else math.floor(x / unit)) * unit


BF16_MAX = float(torch.finfo(torch.bfloat16).max)


def cached_values(x: np.ndarray, bits: int, group: int) -> np.ndarray:
    """What the cache stands for after x [..., D] (f64) was written, in 64 bits."""
    out = np.empty(x.shape)
    top = (1 << bits) - 1
    flat, res = x.reshape(-1, group), out.reshape(-1, group)
    for i, row in enumerate(flat):
        if not np.isfinite(row).all():
            res[i] = np.nan
            continue
        low = max(round_bf16(float(row.min()), False), -BF16_MAX)
        step = round_bf16((float(row.max()) - low) / top, True)
        code = np.clip(np.rint((row - low) / step), 0, top) if step > 0 else np.zeros(group)
        res[i] = code * step + low
    return out


def attention(q, k, v, scale):
    """q [n, heads, D] are the last n of len(k) positions; k, v [len, kv_heads, D]; all f64."""
    n, hq, _ = q.shape
    length, hk = k.shape[0], k.shape[1]
    out = np.zeros(q.shape)
    for i in range(n):
        last = length - n + i
        if last < 0:
            continue
        for h in range(hq):
            s = k[:last + 1, h // (hq // hk)] @ q[i, h] * scale
            p = np.exp(s - s.max())
            out[i, h] = p @ v[:last + 1, h // (hq // hk)] / p.sum()
    return out


def attention_tolerance(q, k, v, scale, dtype, want):
    """Bound of |out - want|: the output's rounding, plus what 32-bit scores,
    exponentials and sums cost.  A score of D products in 32 bits is off by
    about sqrt(D) * 2^-24 of sum |q k| (four times that is allowed, the
    matrix units add in less than full f32 rounding), a weight by twice its
    score's error plus 2^-20 for the exponential and the split weights, and a
    sum of n weighted values by sqrt(n) * 2^-23 of the largest."""
    dim = q.shape[-1]
    grow = np.abs(q).max() * np.abs(k).max() * dim * abs(scale)
    score = 4 * math.sqrt(dim) * 2.0 ** -24 * grow
    top = np.abs(v).max()
    tol = top * (4 * score + 2.0 ** -20 + math.sqrt(k.shape[0]) * 2.0 ** -23)
    if dtype == torch.bfloat16:
        tol += top * 2.0 ** -11   # weights rounded once to 11 bits beside an 8-bit output
    return rounding(want, tol, dtype)
