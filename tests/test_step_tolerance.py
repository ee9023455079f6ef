"""The bounds of step_util.py tell a right output from one that lost a part: checked on the
CPU for the cases that the GPU tests run (those with the most tokens an output, whose values
are the smallest), with outputs that attend to too little."""
import math

import numpy as np
import pytest
import torch

from step_util import head_bound, head_output, tokens_of
from test_gpu_step import BF16, F16, F32, O, make_sparse

# (seed, lens, H, Hkv, d, block size, pages): see test_gpu_step_edges.py
LONG = [(13, [140000, 90], 2, 1, 64, 16, 8100), (13, [140000, 90], 2, 1, 64, 16, 8300),
        (31, [70000, 33333], 8, 2, 64, 16, 600), (32, [20000], 4, 1, 128, 32, 65),
        (33, [3000, 700], 16, 1, 128, 16, 13)]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{c[1][0]}-{c[6]}")
def test_bounds_reject_outputs_that_lost_a_part(case, dt):
    seed, lens, H, Hkv, d, bs, num_pages = case
    p = make_sparse(seed, lens, H, Hkv, d, bs, dt)
    G, scale = H // Hkv, 1 / math.sqrt(d)
    for s in range(len(lens)):
        total = -(-lens[s] // bs)
        if total <= num_pages:
            continue
        # any num_pages pages will do: what is bounded does not depend on the choice
        pages = np.sort(np.random.default_rng(seed).permutation(total)[:num_pages])
        b, o = tokens_of(p, s, pages)
        q, k, v = p["q"][s, :G], p["k"][b, 0, o], p["v"][b, 0, o]
        ref, bound = head_bound(q, k, v, scale, dt)

        def rejected(out):
            return bool((np.abs(out - ref) > bound).any())

        def without(lo, hi):  # pages lo .. hi - 1 of the list lost
            keep = np.ones(len(k), bool)
            keep[lo * bs:hi * bs] = False
            return head_output(q, k[keep], v[keep], scale)[0]

        # the exact output rounded once is inside, with room for the kernel's own errors
        once = torch.from_numpy(ref).to(dt).double().numpy()
        assert not rejected(once) and (np.abs(once - ref) <= 0.9 * bound).all()
        assert rejected(np.zeros_like(ref))
        ctas = 8
        for r in range(ctas):  # a CTA's share of the pages
            assert rejected(without(num_pages * r // ctas, num_pages * (r + 1) // ctas)), r
        assert rejected(without(num_pages // 2, num_pages))      # a list cut short
        parts = [head_output(q, k[i::ctas], v[i::ctas], scale)[0] for i in range(ctas)]
        wrong = sum(parts) / ctas * 1.02                          # a wrong weight in the join
        assert rejected(wrong)
        assert rejected(head_output(q, k, np.roll(v, 1, 0), scale)[0])  # V of the next token


def test_bounds_follow_the_weights():
    """One token: the rounding of the output alone; equal weights of n tokens: 1 / sqrt(n)."""
    q = np.zeros((1, 64))
    v = np.ones((4096, 64))
    for dt, u in ((BF16, 2.0 ** -8), (F16, 2.0 ** -11)):
        _, one = head_bound(q, v[:1], v[:1], 0.125, dt)
        _, many = head_bound(q, v, v, 0.125, dt)
        assert np.allclose(one, 8 * u, rtol=2e-2)
        assert np.allclose(many, (1 + 7 / 64) * u, rtol=6e-2)
