"""Continuous batching over a paged KV cache with the serving-step operators.

Requests with random prompts arrive, are planned into steps (prompt chunks and decode
tokens together), written into the cache, and decoded with sparse attention; finished ones
give their blocks back. Lengths, block tables, positions and slots never leave the GPU. One
attention layer with random weights stands for the model; the sparse outputs of the last
step are compared with the dense decode over the same cache.

    python examples/serving_step.py [--steps 64] [--requests 32] [--pages 32]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "flash-kernel-engine_b200"))
import flash_engine as fe  # noqa: E402


class Layer:
    """QKV projection with QK norm and rotary embedding over a paged cache with page boxes."""

    def __init__(self, hidden, heads, kv_heads, d, num_blocks, block_size, max_pos, gen):
        kw = dict(device="cuda", dtype=torch.bfloat16)
        self.heads, self.bs = heads, block_size
        self.w_qkv = torch.randn((hidden, (heads + 2 * kv_heads) * d), generator=gen, **kw)
        self.w_qkv /= hidden ** 0.5
        self.w_out = torch.randn((heads * d, hidden), generator=gen, **kw) / (heads * d) ** 0.5
        self.q_norm, self.k_norm = (torch.full((d,), 1.5, **kw) for _ in range(2))
        inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda") / d)
        angle = torch.arange(max_pos, device="cuda")[:, None] * inv
        self.rope = (angle.cos(), angle.sin())
        self.kc, self.vc = (torch.zeros((num_blocks, kv_heads, block_size, d), **kw)
                            for _ in range(2))
        self.bounds = fe.new_page_bounds(num_blocks, kv_heads, d, "cuda")

    def append(self, x, plan):
        return fe.paged_qkv_append(x @ self.w_qkv, self.kc, self.vc, plan.positions, plan.slots,
                                   self.heads, self.bs, q_weight=self.q_norm,
                                   k_weight=self.k_norm, rope=self.rope, interleaved=False,
                                   page_bounds=self.bounds)

    def decode(self, q, tables, lens, pages):
        """Output rows and chosen pages of one query a request."""
        out, chosen = fe.sparse_paged_attention(q, self.kc, self.vc, self.bounds, tables, lens,
                                                pages, self.bs)
        return out.flatten(1) @ self.w_out, out, chosen


def serve(steps=64, requests=32, pages=32, seed=0, heads=32, kv_heads=8, d=128, block_size=16,
          max_len=4096, prompt=(64, 1500), tokens_per_step=1024, quiet=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    hidden, width = 512, max_len // block_size
    num_blocks = requests * width // 2
    layer = Layer(hidden, heads, kv_heads, d, num_blocks, block_size, max_len, gen)
    i32 = dict(dtype=torch.int32, device="cuda")
    tables = torch.zeros((requests, width), **i32)
    ring, state = torch.arange(num_blocks, **i32), torch.tensor([0, num_blocks], **i32)
    lens, left = torch.zeros(requests, **i32), torch.zeros(requests, dtype=torch.int64)
    finished = torch.zeros(requests, dtype=torch.bool, device="cuda")
    served, spans = 0, []
    for step in range(steps):
        # rows without a request get one: a prompt, and how many steps it may decode
        new = torch.ones(requests, dtype=torch.int32)
        for r in range(requests):
            if left[r] == 0:
                new[r] = int(torch.randint(*prompt, (1,), generator=host))
                left[r] = int(torch.randint(8, 48, (1,), generator=host))
        begin = torch.cuda.Event(enable_timing=True)
        end = torch.cuda.Event(enable_timing=True)
        begin.record()
        plan = fe.plan_paged_step(lens, new.cuda(), tables, ring, state, block_size,
                                  max_tokens=tokens_per_step, finished=finished)
        x = torch.randn((tokens_per_step, hidden), generator=gen, device="cuda",
                        dtype=torch.bfloat16)
        q = layer.append(x, plan)
        last = (plan.cu_seqlens[1:] - 1).clamp(min=0).long()  # each request's newest token
        y, out, chosen = layer.decode(q[last], tables, plan.context_lens, pages)
        end.record()
        spans.append((begin, end))
        # requests the step did not serve keep waiting: their prompt comes again
        got = (plan.cu_seqlens[1:] > plan.cu_seqlens[:-1]).cpu()
        served += int(plan.free_state[3])
        left[(new > 1) & ~got] = 0
        left[got] -= 1
        lens, state, finished = plan.context_lens, plan.free_state, (left == 0).cuda()
    dense = fe.paged_attention(q[last], layer.kc, layer.vc, tables, lens, block_size)
    held = (lens + block_size - 1) // block_size
    share = float(chosen.ge(0).sum()) / max(1, int(held.sum()) * kv_heads)
    diff = float((out.float() - dense.float()).norm() / dense.float().norm())
    errors = fe.device_errors()
    ms = sorted(a.elapsed_time(b) for a, b in spans[1:])
    if not quiet:
        print(f"{steps} steps, {served} tokens, {ms[len(ms) // 2]:.3f} ms a step (median); "
              f"{100 * share:.0f}% of the pages attended, {100 * diff:.1f}% from the dense "
              f"output; device errors {errors}")
    return {"tokens": served, "share": share, "diff": diff, "errors": errors,
            "lens": lens, "tables": tables, "finite": bool(torch.isfinite(y).all())}


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--pages", type=int, default=32)
    a = ap.parse_args()
    serve(a.steps, a.requests, a.pages)
