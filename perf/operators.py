"""Measured cases of the paged serving-step operators.

A serving step over a paged KV cache runs four operators in a row:

* ``plan``    -- from request lengths on the GPU: blocks taken from and given back to a
  ring of free blocks, block tables, positions and cache slots of the step's tokens;
* ``append``  -- per-head RMS norm of queries and keys, the rotary embedding, and the
  write of K and V into their cache slots, in one pass over the QKV projection;
* ``bounds``  -- an int8 bounding box of the keys of every page that the step filled;
* ``sparse``  -- decode attention of one query token per sequence over the pages that the
  boxes rank highest for it.

Each has a plain form in elementary torch operations (32-bit arithmetic, rounded once) and
a 64-bit form written apart from it (``exact``). The box of a page is, per KV head and
channel, the largest and smallest key value in units of 2^e, rounded outwards to whole
numbers, with the smallest e for which they lie within [-127, 127]; the query is rounded
to whole numbers in the same way. A page's score is then an upper bound of its largest
q.k in exact arithmetic, so the chosen pages do not depend on the order of a sum.
"""
import math

import torch

own = False

BF16, F16, F32 = "bf16", "fp16", "fp32"
_T = {BF16: torch.bfloat16, F16: torch.float16, F32: torch.float32}
_MIN_EXP = -120  # smallest box exponent: 2^-e stays finite


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step's bookkeeping for the serving-mix batch: a token per request,
        # a few requests finished and their rows taken by new ones
        {"name": "plan decode 256", "op": "plan", "seqs": 256, "tokens": 256, "bs": 16,
         "ctx": 4096, "width": 2048, "prompts": 0, "finished": 9, "free": 1000},
        # a large step: thousands of requests, some of them with chunks of their prompts
        {"name": "plan mixed 4096", "op": "plan", "seqs": 4096, "tokens": 65536, "bs": 32,
         "ctx": 8192, "width": 1024, "prompts": 61, "finished": 203, "free": 4000},
        # a single stream's decode step, where latency counts
        {"name": "append one token", "op": "append", "tokens": 1, "heads": 32, "kv": 8, "d": 128,
         "bs": 16, "dtype": BF16, "pairs": "adjacent", "pad": 0},
        # a decode step of 256 requests, 64 query heads, the halves of a head rotated
        {"name": "append decode 256", "op": "append", "tokens": 256, "heads": 64, "kv": 8,
         "d": 128, "bs": 16, "dtype": F16, "pairs": "halves", "pad": 0},
        # a chunk of prompts, the throughput case
        {"name": "append prompt 8192", "op": "append", "tokens": 8192, "heads": 32, "kv": 8,
         "d": 128, "bs": 16, "dtype": BF16, "pairs": "halves", "pad": 0},
        # fp32 with one KV head a query head, an odd count, rows of a wider projection
        {"name": "append odd 1237 fp32", "op": "append", "tokens": 1237, "heads": 12, "kv": 12,
         "d": 64, "bs": 32, "dtype": F32, "pairs": "adjacent", "pad": 64},
        # the boxes of four 131072-token contexts, made once when the prompts are in
        {"name": "bounds 4 x 131072", "op": "bounds", "seqs": 4, "new": 131072, "kv": 8, "d": 128,
         "bs": 16, "dtype": BF16},
        # a ragged chunk of prompts, pages that start and end inside it
        {"name": "bounds ragged 37", "op": "bounds", "seqs": 37, "new": 411, "kv": 4, "d": 64,
         "bs": 32, "dtype": F16},
        # one short sequence: the latency of the call
        {"name": "sparse one 2000", "op": "sparse", "seqs": 1, "ctx_lo": 2000, "ctx": 2000,
         "heads": 32, "kv": 8, "d": 128, "bs": 16, "pages": 32, "dtype": BF16},
        # one very long sequence, 64 query heads
        {"name": "sparse one 500003", "op": "sparse", "seqs": 1, "ctx_lo": 500003, "ctx": 500003,
         "heads": 64, "kv": 8, "d": 128, "bs": 16, "pages": 256, "dtype": F16},
        # the long-context decode batch: four contexts of 131072 tokens
        {"name": "sparse 4 x 131072", "op": "sparse", "seqs": 4, "ctx_lo": 131072, "ctx": 131072,
         "heads": 32, "kv": 8, "d": 128, "bs": 16, "pages": 256, "dtype": BF16},
        # a decode batch of 64 mixed contexts
        {"name": "sparse batch 64", "op": "sparse", "seqs": 64, "ctx_lo": 512, "ctx": 16384,
         "heads": 32, "kv": 8, "d": 128, "bs": 16, "pages": 64, "dtype": BF16},
    ]


def _log(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = min(hi, max(lo, n))
    return n + 1 if n == 3072 and n < hi else n


def draw(rng):
    op = rng.choice(["plan", "append", "append", "bounds", "sparse", "sparse"])
    bs = rng.choice([16, 32])
    if op == "plan":
        seqs = _log(rng, 1, 4096)
        ctx = _log(rng, 1, 16384)
        prompts = min(rng.choice([0, _log(rng, 1, 64)]), seqs)
        tokens = seqs if prompts == 0 else _log(rng, max(seqs, 16), 65536)
        longest = 1 if prompts == 0 else 2 * tokens // prompts
        width = (ctx + longest) // bs + 2
        seqs = max(prompts, 1, min(seqs, 4096 * 1024 // width))
        return {"op": op, "seqs": seqs, "tokens": max(tokens, seqs), "bs": bs, "ctx": ctx,
                "width": width, "prompts": prompts, "finished": rng.randint(0, seqs // 8),
                # some steps run out of free blocks
                "free": int((tokens / bs + seqs) * rng.uniform(0.3, 2)) + 1}
    dtype = rng.choice([BF16, BF16, F16, F32])
    d = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 4, 7, 8])
    if op == "append":
        if (heads + 2 * kv) * d == 3072:
            d = 128 if d == 64 else 64
        return {"op": op, "tokens": _log(rng, 1, 8192 if dtype != F32 else 4096), "heads": heads,
                "kv": kv, "d": d, "bs": bs, "dtype": dtype,
                "pairs": rng.choice(["adjacent", "halves"]), "pad": rng.choice([0, 0, 8, 136])}
    if op == "bounds":
        seqs = _log(rng, 1, 64)
        return {"op": op, "seqs": seqs, "new": _log(rng, 64, 262144 // seqs), "kv": kv,
                "d": d, "bs": bs, "dtype": dtype}
    seqs = _log(rng, 1, 128)
    ctx = _log(rng, 64, max(512, 393216 // seqs // (2 if dtype == F32 else 1)))
    # the chosen pages of a step hold no more than the listed batch's
    most = 64 * 8 * 64 * 16 * 128 // (seqs * kv * bs * d * (2 if dtype == F32 else 1))
    return {"op": op, "seqs": seqs, "ctx_lo": rng.randint(1, ctx), "ctx": ctx, "heads": heads,
            "kv": kv, "d": d, "bs": bs, "pages": _log(rng, 2, min(256, most)), "dtype": dtype}


# ----------------------------------------------------------------------------- the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda", dtype=torch.int32)


def _tables(g, ctx_blocks, width, num_blocks):
    """Block tables whose first ctx_blocks[s] entries of row s are blocks of a random
    permutation, and the permutation's blocks that no row holds."""
    perm = torch.randperm(num_blocks, generator=g, device="cuda").to(torch.int32)
    ends = torch.cumsum(ctx_blocks.long(), 0)
    j = torch.arange(width, device="cuda")
    at = (ends - ctx_blocks)[:, None] + j[None, :]
    held = j[None, :] < ctx_blocks[:, None]
    table = torch.where(held, perm[at.clamp(max=num_blocks - 1)], -1).to(torch.int32).contiguous()
    return table, perm, int(ends[-1])


def _prepare_plan(c, g):
    n, bs = c["seqs"], c["bs"]
    ctx = _ints(g, 0, c["ctx"], n)
    new = torch.ones(n, dtype=torch.int32, device="cuda")
    if c["prompts"]:
        # a few prompt chunks that share what the decode tokens leave of the step
        share = max(1, (c["tokens"] - n) // c["prompts"])
        rows = torch.randperm(n, generator=g, device="cuda")[:c["prompts"]]
        new[rows] = _ints(g, max(1, share // 2), share + share // 4, c["prompts"])
    finished = torch.zeros(n, dtype=torch.bool, device="cuda")
    finished[torch.randperm(n, generator=g, device="cuda")[:c["finished"]]] = True
    held = (ctx + bs - 1) // bs
    spare = c["free"]
    num_blocks = n * ((c["ctx"] + bs - 1) // bs) + spare  # others hold what is left
    table, perm, at = _tables(g, held, c["width"], num_blocks)
    head = int(torch.randint(0, num_blocks, (1,), generator=g, device="cuda"))
    ring = torch.full((num_blocks,), -1, dtype=torch.int32, device="cuda")
    ring[(head + torch.arange(spare, device="cuda")) % num_blocks] = perm[at:at + spare]
    state = torch.tensor([head, spare], dtype=torch.int32, device="cuda")
    t = c["tokens"]
    i32 = dict(dtype=torch.int32, device="cuda")
    return {"ctx": ctx, "new": new, "finished": finished, "table": table, "ring": ring,
            "free": state, "bs": bs, "out": (torch.empty(n, **i32), torch.empty(n + 1, **i32),
                                   torch.empty(t, **i32),
                                   torch.empty(t, dtype=torch.int64, device="cuda"),
                                   torch.empty(4, **i32))}


def _rope_tables(n, d):
    inv = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    a = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return a.cos().float(), a.sin().float()


def _prepare_append(c, g):
    t, h, kv, d, bs, dt = c["tokens"], c["heads"], c["kv"], c["d"], c["bs"], _T[c["dtype"]]
    wide = torch.randn((t, (h + 2 * kv) * d + c["pad"]), generator=g, device="cuda").to(dt)
    # chunks of a few prompts (up to 1024 tokens each) and single decode tokens
    lens, left = [], t
    while left:
        n = min(left, 1 if t <= 512 else 1024)
        lens.append(n)
        left -= n
    start = _ints(g, 0, 4000, len(lens)).tolist()
    pos, page, num_blocks = [], [], 0
    for a, n in zip(start, lens):
        p = torch.arange(a, a + n)
        pos.append(p)
        page.append(p // bs - a // bs + num_blocks)
        num_blocks += (n + bs - 2) // bs + 1  # at most; some stay another request's
    pos, page = torch.cat(pos).cuda(), torch.cat(page).cuda()
    slots = torch.randperm(num_blocks, generator=g, device="cuda")[page] * bs + pos % bs
    cos, sin = _rope_tables(max(a + n for a, n in zip(start, lens)), d)
    w = [(1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) for _ in range(2)]
    return {"qkv": wide[:, :(h + 2 * kv) * d], "pos": pos.to(torch.int32), "slots": slots,
            "cos": cos, "sin": sin, "qw": w[0], "kw": w[1], "heads": h, "kv": kv, "d": d,
            "bs": bs, "pairs": c["pairs"], "eps": 1e-6,
            "kc": torch.zeros((num_blocks, kv, bs, d), dtype=dt, device="cuda"),
            "vc": torch.zeros((num_blocks, kv, bs, d), dtype=dt, device="cuda"),
            "q": torch.empty((t, h, d), dtype=dt, device="cuda")}


def _keys(g, num_blocks, kv, bs, d, dt):
    """Keys whose pages differ: a common direction per page and head, and noise."""
    page = torch.randn((num_blocks, kv, 1, d), generator=g, device="cuda", dtype=dt)
    k = torch.randn((num_blocks, kv, bs, d), generator=g, device="cuda", dtype=dt)
    return k.mul_(0.8).add_(page, alpha=0.6)


def _prepare_bounds(c, g):
    n, bs, kv, d, dt = c["seqs"], c["bs"], c["kv"], c["d"], _T[c["dtype"]]
    new = c["new"]
    start = _ints(g, 0, 0 if new >= 65536 else 5 * bs, n).long()
    blocks = (start + new + bs - 1) // bs
    width = (new + bs - 1) // bs + 5
    num_blocks = n * width
    table, _, _ = _tables(g, blocks, width, num_blocks)
    pos = start[:, None] + torch.arange(new, device="cuda")[None, :]
    slots = (torch.gather(table.long(), 1, pos // bs) * bs + pos % bs).reshape(-1).contiguous()
    return {"kc": _keys(g, num_blocks, kv, bs, d, dt), "slots": slots, "bs": bs,
            "values": torch.zeros((num_blocks, kv, 2, d), dtype=torch.int8, device="cuda"),
            "scales": torch.ones((num_blocks, kv), dtype=torch.float32, device="cuda")}


def _prepare_sparse(c, g):
    n, bs, kv, h, d, dt = c["seqs"], c["bs"], c["kv"], c["heads"], c["d"], _T[c["dtype"]]
    ctx = _ints(g, c["ctx_lo"], c["ctx"], n)
    blocks = (ctx + bs - 1) // bs
    num_blocks = int(blocks.long().sum())
    width = (c["ctx"] + bs - 1) // bs
    table, _, _ = _tables(g, blocks, width, num_blocks)
    kc = _keys(g, num_blocks, kv, bs, d, dt)
    vc = torch.randn((num_blocks, kv, bs, d), generator=g, device="cuda", dtype=dt)
    values = torch.empty((num_blocks, kv, 2, d), dtype=torch.int8, device="cuda")
    scales = torch.empty((num_blocks, kv), dtype=torch.float32, device="cuda")
    for at in range(0, num_blocks, 8192):
        values[at:at + 8192], scales[at:at + 8192] = _boxes(kc[at:at + 8192])
    q = (1.5 * torch.randn((n, h, d), generator=g, device="cuda")).to(dt)
    return {"q": q, "kc": kc, "vc": vc, "values": values, "scales": scales,
            "table": table.clamp(min=0), "ctx": ctx, "pages": c["pages"], "bs": bs,
            "out": torch.empty_like(q),
            "sel": torch.empty((n, kv, c["pages"]), dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    g = _gen(seed)
    state = {"plan": _prepare_plan, "append": _prepare_append, "bounds": _prepare_bounds,
             "sparse": _prepare_sparse}[case["op"]](case, g)
    state["op"] = case["op"]
    return state


# ------------------------------------------------------------------------ the plain forms
def _plain_plan(s):
    bs = s["bs"]
    ctx, ring, table = s["ctx"].long(), s["ring"], s["table"]
    num_blocks, width, cap = ring.numel(), table.shape[1], s["out"][2].numel()
    head, count = s["free"][0].long(), s["free"][1].long()
    fin = s["finished"]
    j = torch.arange(width, device=ctx.device)[None, :]
    # finished requests give their blocks back, row by row
    back = torch.where(fin, (ctx + bs - 1) // bs, 0)
    at = torch.cumsum(back, 0) - back
    give = (j < back[:, None])
    dest = torch.where(give, (head + count + at[:, None] + j) % num_blocks, num_blocks)
    freed = torch.cat([ring, ring[:1]]).index_put((dest,), table)[:num_blocks]
    # requests are served in order until one does not fit
    ctx = torch.where(fin, 0, ctx)
    new = s["new"].long().clamp(min=0)
    have = (ctx + bs - 1) // bs
    need = (ctx + new + bs - 1) // bs - have
    fits = (torch.cumsum(new, 0) <= cap) & (torch.cumsum(need, 0) <= count) & \
        (ctx + new <= width * bs)
    served = torch.cumprod(fits.long(), 0)
    new, need = new * served, need * served
    pop = torch.cumsum(need, 0) - need
    take = (j >= have[:, None]) & (j < (have + need)[:, None])
    src = (head + pop[:, None] + (j - have[:, None]).clamp(min=0)) % num_blocks
    table.copy_(torch.where(take, ring[src], table))
    ring.copy_(freed)
    cu = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    t = torch.arange(cap, device=ctx.device)
    seq = torch.searchsorted(cu[1:], t, right=True).clamp(max=len(ctx) - 1)
    live = t < cu[-1]
    pos = torch.where(live, ctx[seq] + t - cu[seq], -1)
    block = table[seq, (pos.clamp(min=0) // bs).clamp(max=width - 1)].long()
    slots = torch.where(live, block * bs + pos % bs, -1)
    taken = need.sum()
    free = torch.stack([(head + taken) % num_blocks, count - taken + back.sum(), served.sum(),
                        cu[-1]])
    return {"ctx": (ctx + new).int(), "cu": cu.int(), "pos": pos.int(), "slots": slots,
            "free": free.int(), "table": table, "ring": ring}


def _rms(x, w, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()


def _rotate(x, cos, sin, pairs):
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs == "adjacent" else x.chunk(2, -1)
    y0, y1 = a * cos - b * sin, a * sin + b * cos
    return torch.stack([y0, y1], -1).flatten(-2) if pairs == "adjacent" else \
        torch.cat([y0, y1], -1)


def _plain_append(s):
    h, kv, d, bs = s["heads"], s["kv"], s["d"], s["bs"]
    dt = s["qkv"].dtype
    q, k, v = s["qkv"].float().unflatten(1, (h + 2 * kv, d)).split([h, kv, kv], 1)
    cos, sin = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]
    q = _rotate(_rms(q, s["qw"], s["eps"]), cos, sin, s["pairs"]).to(dt)
    k = _rotate(_rms(k, s["kw"], s["eps"]), cos, sin, s["pairs"]).to(dt)
    at = (s["slots"] // bs, slice(None), s["slots"] % bs)
    s["kc"][at] = k
    s["vc"][at] = v.to(dt)
    return {"q": q, "kc": s["kc"], "vc": s["vc"]}


def _exponent(amax):
    """The smallest e with amax <= 127 * 2^e, at least _MIN_EXP."""
    m, e = torch.frexp(amax)
    return (e - 7 + (m > 127 / 128).int()).clamp(min=_MIN_EXP)


def _boxes(k):
    """int8 boxes [n, kv, 2, d] and scales [n, kv] of keys [n, kv, bs, d]."""
    k = k.float()
    hi, lo = k.amax(2), k.amin(2)
    e = _exponent(torch.maximum(hi.abs(), lo.abs()).amax(-1))
    inv = torch.ldexp(torch.ones_like(e, dtype=torch.float32), -e)[..., None]
    box = torch.stack([(hi * inv).ceil(), (lo * inv).floor()], 2)
    return box.to(torch.int8), torch.ldexp(torch.ones_like(e, dtype=torch.float32), e)


def _plain_bounds(s):
    bs = s["bs"]
    full = s["slots"][s["slots"] % bs == bs - 1] // bs
    v, e = _boxes(s["kc"][full])
    s["values"][full], s["scales"][full] = v, e
    return {"values": s["values"], "scales": s["scales"]}


def _plain_sparse(s, first=1, last=1):
    q, kc, bs, want = s["q"], s["kc"], s["bs"], s["pages"]
    n, h, d = q.shape
    kv, width = kc.shape[1], s["table"].shape[1]
    g = h // kv
    table, ctx = s["table"].long(), s["ctx"].long()
    pages = (ctx + bs - 1) // bs
    # score of every page: the largest bound over the group's heads
    qf = q.float()
    e = _exponent(qf.abs().amax(-1))
    one = torch.ones_like(e, dtype=torch.float32)
    qi = torch.round(qf * torch.ldexp(one, -e)[..., None])
    qi = torch.stack([qi.clamp(min=0), qi.clamp(max=0)], 2).view(n, kv, g, 2 * d)
    box = s["values"][table].float().view(n, width, kv, 2 * d)
    # whole numbers below 2^24: every order of this sum is exact
    dot = torch.einsum("skgc,spkc->skgp", qi, box)
    score = (dot * torch.ldexp(one, e).view(n, kv, g, 1)).amax(2)
    score = score * s["scales"][table].permute(0, 2, 1)
    j = torch.arange(width, device=q.device)
    there = (j < pages[:, None])[:, None]
    score = torch.where(there, score, -math.inf).expand(n, kv, width)
    keep = (there[:, 0] & ((j < first) | (j >= (pages - last)[:, None])))[:, None]
    # by (kept, score), ties to the lower page
    order = torch.sort(score, dim=-1, descending=True, stable=True)[1]
    kept = torch.gather(keep.expand(n, kv, width), 2, order)
    order = torch.gather(order, 2, torch.sort(kept.int(), dim=-1, descending=True, stable=True)[1])
    order = order[..., :want]
    if order.shape[-1] < want:
        order = torch.nn.functional.pad(order, (0, want - order.shape[-1]), value=width)
    count = pages.clamp(max=want)[:, None, None]
    r = torch.arange(want, device=q.device)
    sel = torch.sort(torch.where(r < count, order, width), -1)[0]
    live = sel < width
    # attention over the chosen pages
    phys = torch.gather(table, 1, sel.clamp(max=width - 1).view(n, -1)).view(n, kv, want)
    head = torch.arange(kv, device=q.device)[None, :, None]
    kk = kc[phys, head].float().view(n, kv, want * bs, d)
    vv = s["vc"][phys, head].float().view(n, kv, want * bs, d)
    token = (sel[..., None] * bs + torch.arange(bs, device=q.device)).view(n, kv, -1)
    seen = (token < ctx[:, None, None]) & live.repeat_interleave(bs, -1)
    logit = torch.einsum("skgd,sktd->skgt", qf.view(n, kv, g, d), kk) / math.sqrt(d)
    logit = logit.masked_fill(~seen[:, :, None], -math.inf)
    p = torch.exp(logit - logit.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.einsum("skgt,sktd->skgd", p, vv).reshape(n, h, d).to(q.dtype)
    return {"out": out, "sel": torch.where(live, sel, -1).int()}


def _engine():
    import os
    import sys
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "flash-kernel-engine_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import flash_engine
    return flash_engine


_fe = None


def run(s):
    global _fe
    op = s["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "bounds": _plain_bounds,
                "sparse": _plain_sparse}[op](s)
    if _fe is None:
        _fe = _engine()
    if op == "plan":
        r = _fe.plan_paged_step(s["ctx"], s["new"], s["table"], s["ring"], s["free"],
                                s["bs"], finished=s["finished"], out=s["out"])
        return {"ctx": r.context_lens, "cu": r.cu_seqlens, "pos": r.positions, "slots": r.slots,
                "free": r.free_state, "table": s["table"], "ring": s["ring"]}
    if op == "append":
        q = _fe.paged_qkv_append(s["qkv"], s["kc"], s["vc"], s["pos"], s["slots"], s["heads"],
                                 s["bs"], q_weight=s["qw"], k_weight=s["kw"], eps=s["eps"],
                                 rope=(s["cos"], s["sin"]),
                                 interleaved=s["pairs"] == "adjacent", out=s["q"])
        return {"q": q, "kc": s["kc"], "vc": s["vc"]}
    if op == "bounds":
        _fe.update_page_bounds(s["kc"], (s["values"], s["scales"]), s["slots"], s["bs"])
        return {"values": s["values"], "scales": s["scales"]}
    out, sel = _fe.sparse_paged_attention(s["q"], s["kc"], s["vc"], (s["values"], s["scales"]),
                                          s["table"], s["ctx"], s["pages"], s["bs"],
                                          out=s["out"], selected=s["sel"])
    return {"out": out, "sel": sel}


# ---------------------------------------------------------------------- 64-bit definitions
def _exact_append(c, s):
    """Each token by itself from the definition, pairs as complex numbers."""
    h, kv, d, bs = s["heads"], s["kv"], s["d"], s["bs"]
    x = s["qkv"].double().reshape(-1, h + 2 * kv, d)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()][:, None]

    def head(y, w):
        y = y / torch.sqrt(torch.square(y).sum(-1, keepdim=True) / d + s["eps"]) * w.double()
        if s["pairs"] == "adjacent":
            z = torch.view_as_complex(y.reshape(*y.shape[:-1], d // 2, 2).contiguous()) * turn
            return torch.view_as_real(z).reshape(y.shape)
        z = torch.complex(y[..., :d // 2], y[..., d // 2:]) * turn
        return torch.cat([z.real, z.imag], -1)

    out = {"q": head(x[:, :h], s["qw"])}
    for name, rows in (("kc", head(x[:, h:h + kv], s["kw"])), ("vc", x[:, h + kv:])):
        cache = s[name].double().transpose(1, 2).reshape(-1, kv, d)
        cache[s["slots"]] = rows
        out[name] = cache.view(-1, bs, kv, d).transpose(1, 2).contiguous()
    return out


def _exact_sparse(c, s):
    """Sequence by sequence and KV head by KV head."""
    import numpy as np
    n, h, d = s["q"].shape
    kv, bs, want = c["kv"], c["bs"], c["pages"]
    g = h // kv
    out = torch.zeros((n, h, d), dtype=torch.float64, device="cuda")
    ctx = s["ctx"].tolist()
    scales = s["scales"].double()
    for i in range(n):
        np_ = -(-ctx[i] // bs)
        if np_ == 0:
            continue
        rows = s["table"][i, :np_].long()
        for k in range(kv):
            q = s["q"][i, k * g:(k + 1) * g].double()
            top = q.abs().amax(1).cpu().numpy()
            unit = np.where(top > 0, top, 1.0) / 127
            unit = 2.0 ** np.maximum(np.ceil(np.log2(unit)), _MIN_EXP)
            unit = torch.from_numpy(unit).cuda()[:, None]
            qi = torch.round(q / unit) * unit
            box = s["values"][rows, k].double() * scales[rows, k][:, None, None]
            best = torch.zeros(np_, dtype=torch.float64, device="cuda") - math.inf
            for a in range(g):
                best = torch.maximum(best, torch.where(qi[a] > 0, box[:, 0] * qi[a],
                                                       box[:, 1] * qi[a]).sum(-1))
            best = best.cpu().numpy()
            best[0] = best[-1] = np.inf
            rank = np.lexsort((np.arange(np_), -best))
            chosen = torch.from_numpy(np.sort(rank[:want])).cuda()
            tok = (chosen[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1)
            keep = tok < ctx[i]
            kk = s["kc"][rows[chosen], k].reshape(-1, d)[keep].double()
            vv = s["vc"][rows[chosen], k].reshape(-1, d)[keep].double()
            p = torch.softmax((q @ kk.T) / math.sqrt(d), -1)
            out[i, k * g:(k + 1) * g] = p @ vv
    return {"out": out, "sel": None}


def exact(case, seed):
    op = case["op"]
    if op == "plan":
        return None
    s = prepare(case, seed)
    if op == "append":
        return _exact_append(case, s)
    if op == "sparse":
        return _exact_sparse(case, s)
    # the scales, as powers of two; the boxes themselves are whole numbers
    full = torch.unique(s["slots"][(s["slots"] + 1) % s["bs"] == 0] // s["bs"])
    scales = s["scales"].double()
    for at in range(0, len(full), 4096):
        top = s["kc"][full[at:at + 4096]].abs().amax((2, 3)).double()
        scales[full[at:at + 4096]] = torch.exp2(torch.ceil(torch.log2(top / 127)))
    return {"values": None, "scales": scales}


# -------------------------------------------------------------------------------- the work
def work(case):
    c = case
    op = c["op"]
    if op == "plan":
        # lengths and flags in, lengths and offsets out; position and slot of every token;
        # a table entry and a ring entry of every block that changes hands
        moved = c["tokens"] / c["bs"] + c["finished"] * c["ctx"] / 2 / c["bs"] + c["seqs"] / c["bs"]
        return {"bytes": c["seqs"] * (4 + 4 + 1 + 4 + 4) + c["tokens"] * 12 + moved * 8,
                "flops": 0}
    elt = 4 if c["dtype"] == F32 else 2
    d, kv, bs = c["d"], c["kv"], c["bs"]
    if op == "append":
        rows = c["tokens"] * (c["heads"] + 2 * kv)
        return {"bytes": 2 * rows * d * elt + c["tokens"] * (12 + 4 * d),
                "flops": c["tokens"] * (c["heads"] + kv) * d * 7}
    if op == "bounds":
        pages = c["seqs"] * (c["new"] // bs)
        return {"bytes": c["seqs"] * c["new"] * 8 + pages * kv * (bs * d * elt + 2 * d + 4),
                "flops": pages * kv * bs * d * 2}
    ctx = c["seqs"] * (c["ctx_lo"] + c["ctx"]) / 2
    pages = ctx / bs
    some = c["seqs"] * min(c["pages"], (c["ctx_lo"] + c["ctx"]) / 2 / bs)
    return {"bytes": pages * (kv * (2 * d + 4) + 4) + some * kv * 2 * bs * d * elt +
            2 * c["seqs"] * c["heads"] * d * elt + some * kv * 4,
            "flops": pages * c["heads"] * 4 * d + some * bs * c["heads"] * 4 * d}
