"""How far a sparse (or dense) decode's outputs may be from the exact ones, case by case.

An absolute tolerance from max |v| says nothing about outputs that average thousands of tokens.
With exact weights w (softmax, sum 1) over the n attended tokens of a query head, the kernels'
output differs from w v by
  * the rounding of each weight to the 16-bit type, relative errors of at most u that are
    independent from token to token: by Hoeffding above 7 u sqrt(sum w^2 v^2) with a
    probability of 2 exp(-24.5) = 5e-11 an element;
  * for fp16, weights below 2^-14 of the running maximum, which are rounded to multiples of
    2^-24: at most 2^-25 sum |v| / L, L the sum of the weights relative to the maximum;
  * fp32 sums of d products in a logit, each step off by 2^-24 of the partial sum: taken as 4
    standard deviations, 4 sqrt(d) 2^-24 sum |q k| scale, once for the weight and once for
    the sum of all of them;
  * fp32 sums over the tokens, 4 sqrt(n) 2^-24 sum w |v|;
  * the output's rounding, u |w v|.
fp32 caches have no rounding to 16 bits (u = 0, and 2^-24 for the output).
"""
import math

import numpy as np
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 0.0}


def head_output(q, k, v, scale):
    """Exact outputs [G, d] of queries q [G, d] over tokens k, v [n, d], with their weights."""
    x = q @ k.T * scale
    w = np.exp(x - x.max(-1, keepdims=True))
    total = w.sum(-1, keepdims=True)
    return w / total @ v, w / total, total


def head_bound(q, k, v, scale, dt):
    ref, w, total = head_output(q, k, v, scale)
    u, n, d = UNIT[dt], *k.shape
    mean = w @ np.abs(v)
    bound = 7 * u * np.sqrt(w ** 2 @ v ** 2)
    if dt == torch.float16:
        bound += 2.0 ** -25 * np.abs(v).sum(0) / total
    logit = 4 * math.sqrt(d) * 2.0 ** -24 * (np.abs(q) @ np.abs(k).T).max(-1, keepdims=True) * scale
    bound += (2 * logit + 4 * math.sqrt(n) * 2.0 ** -24) * mean
    return ref, bound + max(u, 2.0 ** -24) * np.abs(ref)


def tokens_of(p, s, pages):
    """(block, offset) of the tokens of sequence s in these pages, in order."""
    bs = p["bs"]
    t = (np.asarray(pages)[:, None] * bs + np.arange(bs)).reshape(-1)
    t = t[t < p["lens"][s]]
    return p["tables"][s][t // bs], t % bs


def attention_bound(p, selected, scale=None):
    """Exact output [S, H, d] over the pages selected [S, Hkv, n] (-1 = none) and how far each
    element may be off. p: a problem of make_sparse."""
    S, H, d = p["q"].shape
    Hkv = p["k"].shape[1]
    G, scale = H // Hkv, scale or 1 / math.sqrt(d)
    ref, bound = np.zeros((S, H, d)), np.zeros((S, H, d))
    for s in range(S):
        for h in range(Hkv):
            pages = selected[s, h][selected[s, h] >= 0]
            if not len(pages):
                continue
            b, o = tokens_of(p, s, pages)
            rows = slice(h * G, (h + 1) * G)
            ref[s, rows], bound[s, rows] = head_bound(p["q"][s, rows], p["k"][b, h, o],
                                                      p["v"][b, h, o], scale, p["dt"])
    return ref, bound
