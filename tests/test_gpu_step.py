"""The serving-step operators (flash_engine/step.py) on the GPU, against the 64-bit oracle
of oracle/step_oracle.py.

Tolerances. The append computes in fp32 (errors of a few 2^-24 of the result, and of the
rotation's summands, which stay below 16 here) and rounds once: its output lies between the
roundings of the exact value less and plus that error. The attention rounds the softmax
weights and the output to bf16 / fp16, u = 2^-8 / 2^-11 each: 2 u max|v| at the worst, with
|v| <= 5.5 here; half of that is allowed, since the weights' errors are as often up as down.
Whole numbers (plans, boxes, chosen pages) are equal.
"""
import numpy as np
import pytest
import torch

from gpu_util import cuda, host
from oracle import step_oracle as O

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ATTN_ATOL = {BF16: 5.5 * 2.0 ** -8, F16: 5.5 * 2.0 ** -11, F32: 2e-5}


def fe():
    import flash_engine
    return flash_engine


def rounded(x, dt):
    """float64 values that dt holds."""
    return torch.from_numpy(np.ascontiguousarray(x)).to(dt).double().numpy()


def assert_rounds_to(got, ref, dt, what):
    """got (a tensor of dt) is ref up to dt's rounding and the fp32 arithmetic before it."""
    got = got.double().cpu().numpy()
    err = np.abs(ref) * 8 * 2.0 ** -24 + 16 * 8 * 2.0 ** -24
    bad = (got < rounded(ref - err, dt)) | (got > rounded(ref + err, dt))
    assert not bad.any(), (what, int(bad.sum()), float(np.abs(got - ref).max()))


# ------------------------------------------------------------------------------- the plan
def run_plan(ctx, new, tables, ring, head, count, bs, max_tokens, finished=None):
    t, r = cuda(tables), cuda(ring)
    step = fe().plan_paged_step(cuda(np.array(ctx, np.int32)), cuda(np.array(new, np.int32)), t, r,
                                cuda(np.array([head, count], np.int32)), bs,
                                max_tokens=max_tokens,
                                finished=None if finished is None else cuda(np.array(finished)))
    return step, t, r


def check_plan(ctx, new, tables, ring, head, count, bs, max_tokens, finished=None):
    ref = O.plan(ctx, new, tables, ring, head, count, bs, max_tokens, finished)
    step, t, r = run_plan(ctx, new, tables, ring, head, count, bs, max_tokens, finished)
    for name in ("context_lens", "cu_seqlens", "positions", "slots"):
        np.testing.assert_array_equal(getattr(step, name).cpu().numpy(), ref[name], name)
    np.testing.assert_array_equal(step.free_state.cpu().numpy(), ref["state"])
    np.testing.assert_array_equal(t.cpu().numpy(), ref["tables"])
    np.testing.assert_array_equal(r.cpu().numpy(), ref["ring"])
    return ref


def make_plan(seed, S, bs, width, spare, max_ctx):
    """Requests over a permutation of the blocks, the rest in a ring with a random head."""
    g = np.random.default_rng(seed)
    ctx = g.integers(0, max_ctx + 1, S)
    held = -(-ctx // bs)
    nb = int(held.sum()) + spare
    perm = g.permutation(nb).astype(np.int32)
    tables = np.full((S, width), -7, np.int32)
    at = 0
    for s in range(S):
        tables[s, :held[s]] = perm[at:at + held[s]]
        at += held[s]
    head = int(g.integers(0, nb))
    ring = np.full(nb, -5, np.int32)
    ring[(head + np.arange(spare)) % nb] = perm[at:]
    return g, ctx, tables, ring, head, spare


@pytest.mark.parametrize("S,bs", [(1, 16), (3, 1), (31, 7), (33, 16), (300, 32), (1500, 16)])
@pytest.mark.parametrize("mode", ["decode", "chunks", "finished"])
def test_plan(S, bs, mode):
    g, ctx, tables, ring, head, count = make_plan(S * 10 + bs, S, bs, 64 // bs + 70, 3 * S + 90,
                                                  60)
    new = np.ones(S, int) if mode == "decode" else g.integers(0, 40, S)
    fin = g.random(S) < 0.3 if mode == "finished" else None
    ref = check_plan(ctx, new, tables, ring, head, count, bs, int(new.sum()) + 11, fin)
    assert fe().device_errors() == 0
    assert mode != "decode" or ref["state"][2] == S


def test_plan_stops_at_the_first_request_that_does_not_fit():
    bs = 4
    g, ctx, tables, ring, head, count = make_plan(5, 40, bs, 30, 25, 60)
    new = g.integers(0, 12, 40)
    total = int(new.sum())
    # too few blocks; too few tokens; a row that is too short, before requests that fit
    a = check_plan(ctx, new, tables, ring, head, 9, bs, total)
    b = check_plan(ctx, new, tables, ring, head, count, bs, 77)
    new2 = np.ones(40, int)
    new2[17] = 130
    c = check_plan(ctx, new2, tables, ring, head, count, bs, 400)
    assert 0 < a["state"][2] < 40 and 0 < b["state"][2] < 40 and c["state"][2] == 17


def test_plan_edges():
    bs = 16
    z = np.zeros((0, 4), np.int32)
    check_plan([], [], z, np.arange(3, dtype=np.int32), 2, 3, bs, 5)             # no request
    one = np.full((1, 4), -1, np.int32)
    ring = np.arange(3, dtype=np.int32)
    check_plan([0], [0], one, ring, 0, 3, bs, 0)                                 # no token
    check_plan([0], [-4], one, ring, 0, 3, bs, 3)                                # negative = 0
    check_plan([0], [48], one, ring, 1, 3, bs, 48)                               # every block
    check_plan([0], [49], one, ring, 1, 3, bs, 49)                               # one too many
    big = 2 ** 31 - 1                                                            # no overflow
    check_plan([0, big, 5, 0], [big, big, big, 1], np.full((4, 4), -1, np.int32), ring, 1, 3, bs,
               20)
    check_plan([0, 0, 0, 0, 0], [4] * 5, np.full((5, 4), -1, np.int32),
               np.arange(5, dtype=np.int32), 4, 5, bs, 20)                       # the ring wraps
    assert fe().device_errors() == 0


def test_plan_reports_a_ring_that_overflows():
    from flash_engine import _lib
    tables = np.array([[0, 1, 2, -1]], np.int32)
    run_plan([48], [0], tables, np.arange(4, dtype=np.int32), 0, 2, 16, 4, [True])
    assert fe().device_errors() == _lib.ERR_BAD_BLOCK


def test_plan_over_many_steps_loses_no_block():
    """Requests come, grow and go; held and free blocks stay a partition of all blocks."""
    bs, S, nb, width, cap = 8, 24, 400, 30, 96
    g = np.random.default_rng(0)
    ctx = np.zeros(S, int)
    tables, ring = cuda(np.full((S, width), -1, np.int32)), cuda(g.permutation(nb).astype(np.int32))
    state = cuda(np.array([7, nb, 0, 0], np.int32))
    lens = cuda(np.zeros(S, np.int32))
    m_tables, m_ring, m_state = tables.cpu().numpy(), ring.cpu().numpy(), [7, nb]
    for k in range(40):
        fin = (g.random(S) < 0.15) & (ctx > 0)
        new = np.where(g.random(S) < 0.2, g.integers(1, 40, S), 1)
        new = np.where(fin & (g.random(S) < 0.5), 0, new)
        ref = O.plan(ctx, new, m_tables, m_ring, m_state[0], m_state[1], bs, cap, fin)
        step = fe().plan_paged_step(lens, cuda(new.astype(np.int32)), tables, ring, state, bs,
                                    max_tokens=cap, finished=cuda(fin))
        lens, state = step.context_lens, step.free_state
        np.testing.assert_array_equal(step.slots.cpu().numpy(), ref["slots"], f"step {k}")
        np.testing.assert_array_equal(state.cpu().numpy(), ref["state"])
        ctx, m_tables, m_ring = ref["context_lens"].astype(int), ref["tables"], ref["ring"]
        m_state = [int(ref["state"][0]), int(ref["state"][1])]
        held = [int(m_tables[s, j]) for s in range(S) for j in range(-(-ctx[s] // bs))]
        free = [int(m_ring[(m_state[0] + i) % nb]) for i in range(m_state[1])]
        assert sorted(held + free) == list(range(nb))
    np.testing.assert_array_equal(tables.cpu().numpy(), m_tables)
    assert fe().device_errors() == 0


def test_plan_largest_request_count():
    S, bs = 16384, 16
    g, ctx, tables, ring, head, count = make_plan(9, S, bs, 8, S, 100)
    check_plan(ctx, np.ones(S, int), tables, ring, head, count, bs, S + 5, g.random(S) < 0.05)


# ------------------------------------------------------------------------------ the append
def vllm_k(k):
    """flat [n, Hkv, bs, d] -> x-packed [n, Hkv, d/8, bs, 8]."""
    n, h, bs, d = k.shape
    return np.ascontiguousarray(k.reshape(n, h, bs, d // 8, 8).transpose(0, 1, 3, 2, 4))


def vllm_v(v):
    return np.ascontiguousarray(v.transpose(0, 1, 3, 2))


def check_append(seed, T, H, Hkv, d, dt, bs=16, rotary=None, interleaved=True, weights="same",
                 layout="flat", pad=0, holes=False, start=0):
    g = np.random.default_rng(seed)
    nb = T // bs + 3
    wide = rounded(g.standard_normal((T, (H + 2 * Hkv) * d + pad)), dt)
    pos = (start + g.integers(0, 50, T)).astype(np.int32)
    slots = g.permutation(nb * bs)[:T].astype(np.int64)
    if holes:
        pos[T // 2:] = np.where(g.random(T - T // 2) < 0.5, -1, pos[T // 2:])
        slots[::3] = -1
    kc = rounded(g.standard_normal((nb, Hkv, bs, d)), dt)
    vc = rounded(g.standard_normal((nb, Hkv, bs, d)), dt)
    qw = kw = cos = sin = None
    if weights is not None:
        wdt = dt if weights == "same" else F32
        qw, kw = (rounded(1 + 0.3 * g.standard_normal(d), wdt) for _ in range(2))
    if rotary:
        a = g.uniform(-3, 3, (start + 50, rotary // 2))
        cos, sin = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)
    flat = wide[:, :(H + 2 * Hkv) * d]
    q, k, v = O.qkv_append(flat, H, Hkv, d, kc, vc, pos, slots, bs, qw, kw, 1e-6, cos, sin,
                           interleaved)
    vl = layout == "vllm"
    dk, dv = cuda(vllm_k(kc) if vl else kc, dt), cuda(vllm_v(vc) if vl else vc, dt)
    got = fe().paged_qkv_append(
        cuda(wide, dt)[:, :(H + 2 * Hkv) * d], dk, dv, cuda(pos), cuda(slots), H, bs,
        q_weight=None if qw is None else cuda(qw, wdt),
        k_weight=None if kw is None else cuda(kw, wdt),
        rope=None if cos is None else (cuda(cos), cuda(sin)), interleaved=interleaved,
        kv_layout=layout)
    assert got.shape == (T, H, d)
    assert_rounds_to(got, q, dt, "q")
    assert_rounds_to(dk, vllm_k(k) if vl else k, dt, "k")
    assert_rounds_to(dv, vllm_v(v) if vl else v, dt, "v")


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("T,H,Hkv,d", [(1, 32, 8, 128), (5, 7, 1, 64), (64, 28, 4, 128),
                                       (67, 12, 12, 64), (9, 4, 2, 256), (300, 16, 2, 128)])
def test_append(dt, interleaved, T, H, Hkv, d):
    check_append(T + d, T, H, Hkv, d, dt, rotary=d, interleaved=interleaved)
    assert fe().device_errors() == 0


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("kw", [
    dict(d=80, rotary=80), dict(d=96, rotary=32), dict(d=128, rotary=64),       # generic path
    dict(d=128, rotary=64, interleaved=False), dict(d=33, rotary=None), dict(d=1, rotary=None),
    dict(d=128, rotary=None), dict(d=128, rotary=128, weights=None),            # vector path
    dict(d=64, rotary=64, weights="fp32"), dict(d=64, rotary=None, weights=None),
    dict(d=128, rotary=128, pad=1), dict(d=128, rotary=128, pad=136),           # row strides
    dict(d=64, rotary=64, holes=True), dict(d=48, rotary=48, holes=True),
    dict(d=128, rotary=128, bs=5), dict(d=128, rotary=128, start=70000)])
def test_append_options(dt, kw):
    check_append(3, 41, 6, 2, dt=dt, **kw)
    assert fe().device_errors() == 0


@pytest.mark.parametrize("dt", [BF16, F16])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_append_vllm_layout(dt, d):
    check_append(4, 37, 8, 2, d, dt, rotary=d, layout="vllm", interleaved=False)


def test_append_many_tokens_spread_over_the_gpu():
    check_append(6, 2500, 5, 1, 64, BF16, rotary=64)


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("kw", [
    dict(H=6, Hkv=2, d=128, rotary=128, holes=True), dict(H=5, Hkv=3, d=64, rotary=64, pad=16),
    dict(H=6, Hkv=2, d=128, rotary=None, interleaved=False),
    dict(H=4, Hkv=4, d=256, rotary=256, weights=None, interleaved=False),
    dict(H=2, Hkv=1, d=128, rotary=128, weights="fp32", bs=7),
    dict(H=6, Hkv=2, d=128, rotary=64, interleaved=False), dict(H=40, Hkv=8, d=256, rotary=256),
    dict(H=3, Hkv=1, d=128, rotary=128, layout="vllm")])
def test_append_many_tokens(dt, kw):
    """More than four tokens an SM: the ring of token rows, and what it does not take."""
    if dt == F32 and "layout" in kw:
        pytest.skip("the fp32 cache takes the flat layout")
    check_append(7, 643, dt=dt, **kw)
    assert fe().device_errors() == 0


def test_append_norm_of_zero_and_of_large_rows():
    """An all-zero head stays zero, and a row whose squares pass bf16 stays finite."""
    d, bs = 128, 16
    qkv = np.zeros((2, 3 * d))
    qkv[1] = 3e4 * np.sign(np.random.default_rng(0).standard_normal(3 * d))
    qkv = rounded(qkv, F32)
    k, v = np.zeros((1, 1, bs, d)), np.zeros((1, 1, bs, d))
    pos, slots, w = np.array([0, 1], np.int32), np.array([0, 1], np.int64), np.ones(d)
    q, rk, _ = O.qkv_append(qkv, 1, 1, d, k, v, pos, slots, bs, w, w)
    dk, dv = cuda(k, F32), cuda(v, F32)
    got = fe().paged_qkv_append(cuda(qkv, F32), dk, dv, cuda(pos), cuda(slots), 1, bs,
                                q_weight=cuda(w, F32), k_weight=cuda(w, F32))
    assert_rounds_to(got, q, F32, "q")
    assert_rounds_to(dk, rk, F32, "k")


def test_append_flags_positions_and_slots_out_of_range():
    from flash_engine import _lib
    d, bs, nb = 64, 16, 2
    g = np.random.default_rng(0)
    for bad_pos, bad_slot in ((9, 0), (0, nb * bs), (0, 2 ** 40)):
        qkv = cuda(g.standard_normal((3, 4 * d)), BF16)
        kc, vc = (torch.zeros((nb, 1, bs, d), dtype=BF16, device="cuda") for _ in range(2))
        pos = cuda(np.array([1, bad_pos, 2], np.int32))
        slots = cuda(np.array([1, bad_slot, 2], np.int64))
        t = torch.ones((9, d // 2), device="cuda")
        q = fe().paged_qkv_append(qkv, kc, vc, pos, slots, 2, bs, rope=(t, t))
        assert fe().device_errors() == _lib.ERR_BAD_BLOCK
        assert (kc[0, 0, 1] != 0).any() and (vc[0, 0, 2] != 0).any()
        assert int((kc != 0).any(-1).sum()) == 2 and (q[1] == 0).all() == (bad_pos == 9)


# ------------------------------------------------------------------------------- the boxes
@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs,layout", [(16, "flat"), (32, "flat"), (16, "vllm")])
@pytest.mark.parametrize("Hkv", [1, 3])
def test_bounds(dt, d, bs, layout, Hkv):
    if dt == F32 and layout == "vllm":
        pytest.skip("the fp32 cache takes the flat layout")
    g = np.random.default_rng(d + bs)
    nb = 70
    k = rounded(g.standard_normal((nb, Hkv, bs, d)) * 2.0 ** g.integers(-12, 9, (nb, Hkv, 1, 1)), dt)
    k[3], k[4, 0] = 0, -1.5
    # the exponent's edge: the largest value exactly 127 * 2^e, and the next one above it
    k[5] = np.clip(k[5], -1, 1)
    k[5, :, 2, 7] = 127 / 64
    k[6] = np.clip(k[6], -1, 1)
    k[6, :, 2, 7] = 127.5 / 64
    special = {8: np.nan, 9: np.inf, 10: -np.inf}
    for b, x in special.items():
        k[b, 0, bs - 1, d - 1] = x
    closed = np.sort(g.permutation(nb)[:50])
    closed = np.union1d(closed, [3, 4, 5, 6, 8, 9, 10])
    slots = [b * bs + bs - 1 for b in closed] + [b * bs + int(g.integers(0, bs - 1))
                                                 for b in range(nb)] + [-1, -1]
    slots = np.array(slots, np.int64)[g.permutation(len(slots))]
    v, s = O.boxes(k)
    pb = fe().new_page_bounds(nb, Hkv, d, "cuda")
    pb.values.fill_(99)
    pb.scales.fill_(-1)
    dk = cuda(vllm_k(k) if layout == "vllm" else k, dt)
    fe().update_page_bounds(dk, pb, cuda(slots), bs, kv_layout=layout)
    gv, gs = pb.values.cpu().numpy(), pb.scales.cpu().numpy()
    np.testing.assert_array_equal(gv[closed], v[closed])
    np.testing.assert_array_equal(gs[closed], s[closed])
    rest = np.setdiff1d(np.arange(nb), closed)
    assert (gv[rest] == 99).all() and (gs[rest] == -1).all()
    assert fe().device_errors() == 0


@pytest.mark.parametrize("dt,tiny,huge", [(BF16, 2.0 ** -133, 3.3895e38), (F16, 2.0 ** -24, 65504.0),
                                          (F32, 2.0 ** -149, 3.4028234e38)])
def test_bounds_of_the_smallest_and_largest_values(dt, tiny, huge):
    k = np.zeros((2, 1, 16, 64))
    k[0, 0, 3, 5], k[0, 0, 4, 6] = tiny, -tiny
    k[1, 0, 3, 5], k[1, 0, 4, 6] = huge, -huge
    k = rounded(k, dt)
    assert np.isfinite(k).all() and (k != 0).sum() == 4
    v, s = O.boxes(k)
    pb = fe().update_page_bounds(cuda(k, dt), fe().new_page_bounds(2, 1, 64, "cuda"),
                                 cuda(np.array([15, 31], np.int64)), 16)
    np.testing.assert_array_equal(pb.values.cpu().numpy(), v)
    np.testing.assert_array_equal(pb.scales.cpu().numpy(), s)


def test_bounds_flag_slots_out_of_range():
    from flash_engine import _lib
    k = torch.zeros((2, 1, 16, 64), dtype=BF16, device="cuda")
    pb = fe().new_page_bounds(2, 1, 64, "cuda")
    pb.scales.fill_(-1)
    fe().update_page_bounds(k, pb, cuda(np.array([47, 15], np.int64)), 16)
    assert fe().device_errors() == _lib.ERR_BAD_BLOCK
    assert pb.scales[:, 0].tolist() == [2.0 ** -7, -1]


# -------------------------------------------------------------------- the sparse attention
def make_sparse(seed, lens, H, Hkv, d, bs, dt, spread=1.0):
    g = np.random.default_rng(seed)
    lens = np.asarray(lens)
    pages = -(-lens // bs)
    width, nb = max(1, int(pages.max())), int(pages.sum()) + 3
    perm = g.permutation(nb).astype(np.int32)
    tables = np.zeros((len(lens), width), np.int32)
    at = 0
    for s, n in enumerate(pages):
        tables[s, :n] = perm[at:at + n]
        at += n
    k = rounded(0.8 * g.standard_normal((nb, Hkv, bs, d)) +
                0.6 * spread * g.standard_normal((nb, Hkv, 1, d)), dt)
    v = np.clip(rounded(g.standard_normal((nb, Hkv, bs, d)), dt), -5.5, 5.5)
    q = rounded(1.5 * g.standard_normal((len(lens), H, d)), dt)
    return dict(q=q, k=k, v=v, tables=tables, lens=lens.astype(np.int32), bs=bs, dt=dt)


def check_sparse(p, num_pages, first=1, last=1, layout="flat", scale=None, stream=None,
                 values_scales=None):
    v, s = values_scales or O.boxes(p["k"])
    ref, sel = O.sparse_attention(p["q"], p["k"], p["v"], v, s, p["tables"], p["lens"], p["bs"],
                                  num_pages, first, last, scale)
    dt, vl = p["dt"], layout == "vllm"
    args = (cuda(p["q"], dt), cuda(vllm_k(p["k"]) if vl else p["k"], dt),
            cuda(vllm_v(p["v"]) if vl else p["v"], dt), (cuda(v), cuda(s)), cuda(p["tables"]),
            cuda(p["lens"]), num_pages, p["bs"], scale)
    kw = dict(keep_first=first, keep_last=last, kv_layout=layout)
    if stream is None:
        out, got = fe().sparse_paged_attention(*args, **kw)
    else:
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            out, got = fe().sparse_paged_attention(*args, **kw)
        stream.synchronize()
    np.testing.assert_array_equal(got.cpu().numpy(), sel)
    err = np.abs(host(out).astype(np.float64) - ref)
    assert np.isfinite(host(out)).all() and err.max(initial=0) <= ATTN_ATOL[dt], err.max()
    assert fe().device_errors() == 0
    return out, got


LENS = [0, 1, 15, 16, 17, 200, 333, 512, 31, 32, 33, 1000]


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("H,Hkv,d,bs", [(32, 8, 128, 16), (7, 1, 64, 32), (16, 1, 128, 16),
                                        (4, 4, 64, 16), (24, 1, 64, 16), (6, 3, 128, 32)])
@pytest.mark.parametrize("num_pages", [2, 5, 13])
def test_sparse(dt, H, Hkv, d, bs, num_pages):
    check_sparse(make_sparse(H + d, LENS, H, Hkv, d, bs, dt), num_pages)


@pytest.mark.parametrize("dt", [BF16, F16])
def test_sparse_vllm_layout(dt):
    check_sparse(make_sparse(1, LENS, 8, 2, 64, 16, dt), 6, layout="vllm")


@pytest.mark.parametrize("first,last,num_pages", [(0, 1, 1), (0, 1, 4), (3, 2, 5), (2, 9, 12),
                                                  (0, 4, 33), (33, 20, 55), (0, 50, 60)])
@pytest.mark.parametrize("lens", [LENS, [3000, 2999]])
def test_sparse_kept_pages(first, last, num_pages, lens):
    check_sparse(make_sparse(2, lens, 8, 2, 64, 16, BF16), num_pages, first, last)


@pytest.mark.parametrize("S,Hkv,ctx", [(1, 1, 9001), (2, 1, 70000), (1, 8, 20000), (3, 2, 33333)])
@pytest.mark.parametrize("num_pages", [2, 65, 600])
def test_sparse_long(S, Hkv, ctx, num_pages):
    """Few rows with many pages: a row's pages are shared by a cluster of CTAs."""
    g = np.random.default_rng(ctx)
    lens = [ctx] + [int(x) for x in g.integers(1, ctx, S - 1)]
    check_sparse(make_sparse(S + ctx, lens, 4 * Hkv, Hkv, 64, 16, BF16), num_pages)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_sparse_longest(dt):
    """More pages than a row's scores fit in shared memory."""
    p = make_sparse(11, [700001], 4, 1, 64, 16, dt)
    check_sparse(p, 40)


@pytest.mark.parametrize("H,Hkv,d,bs", [(16, 4, 128, 16), (36, 4, 64, 32)])
def test_sparse_many_rows(H, Hkv, d, bs):
    g = np.random.default_rng(H)
    check_sparse(make_sparse(12, g.integers(0, 700, 45), H, Hkv, d, bs, BF16), 5)


def test_sparse_more_sequences_than_a_score_launch_takes():
    g = np.random.default_rng(15)
    check_sparse(make_sparse(15, g.integers(0, 80, 4099), 2, 1, 64, 16, BF16), 2)


def test_sparse_many_pages_chosen():
    """A list longer than the attention's shared memory holds goes through the paged decode."""
    check_sparse(make_sparse(13, [140000, 90], 2, 1, 64, 16, BF16), 8300)
    check_sparse(make_sparse(13, [140000, 90], 2, 1, 64, 16, BF16), 8100)


@pytest.mark.parametrize("ctx", [900, 40000])
def test_sparse_ties_go_to_the_lower_page(ctx):
    """Equal scores: a zero query, pages that repeat, and few different scores."""
    p = make_sparse(3, [ctx, ctx // 2], 8, 2, 64, 16, BF16)
    q0 = dict(p, q=np.zeros_like(p["q"]))
    check_sparse(q0, 9)
    same = dict(p, k=np.broadcast_to(p["k"][:1], p["k"].shape).copy())
    check_sparse(same, 10)
    few = dict(p, k=p["k"][np.arange(len(p["k"])) % 3])
    check_sparse(few, 21)


def test_sparse_ties_in_a_long_row():
    """More equal scores than the registers of a CTA hold."""
    p = make_sparse(14, [150001], 2, 1, 64, 16, BF16)
    check_sparse(dict(p, q=np.zeros_like(p["q"])), 9)
    few = dict(p, k=p["k"][np.arange(len(p["k"])) % 3])
    check_sparse(few, 33)
    check_sparse(p, 33, 20, 12)


def test_sparse_scores_below_zero():
    """Keys that point away from the query: all scores negative, the nearest to zero win."""
    p = make_sparse(4, [700, 650], 2, 1, 64, 16, F32)
    p["k"] = rounded(-np.abs(p["k"]), F32)
    p["q"] = rounded(np.abs(p["q"]) + 0.1, F32)
    check_sparse(p, 7)


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_sparse_scale(scale):
    check_sparse(make_sparse(5, [500, 90], 4, 2, 128, 16, F32), 6, scale=scale)


def test_sparse_reads_nothing_outside_the_chosen_pages():
    """NaN in every page that is not chosen, in the last page's unused rows and in blocks of
    other sequences changes nothing."""
    p = make_sparse(6, [610, 77, 300], 8, 2, 64, 16, BF16)
    vs = O.boxes(p["k"])
    out, got = check_sparse(p, 5, values_scales=vs)
    used = np.zeros(p["k"].shape[:3], bool)
    for s in range(3):
        for h in range(2):
            for j in got[s, h].tolist():
                for o in range(16):
                    if j >= 0 and j * 16 + o < p["lens"][s]:
                        used[p["tables"][s, j], h, o] = True
    for name in "kv":
        p[name] = np.where(used[..., None], p[name], np.nan)
    out2, _ = fe().sparse_paged_attention(
        cuda(p["q"], BF16), cuda(p["k"], BF16), cuda(p["v"], BF16), (cuda(vs[0]), cuda(vs[1])),
        cuda(p["tables"]), cuda(p["lens"]), 5, 16)
    assert torch.equal(out, out2)


def test_sparse_always_takes_pages_with_non_finite_keys():
    p = make_sparse(7, [400], 4, 1, 64, 16, BF16)
    for j in (5, 17):
        p["k"][p["tables"][0, j], 0, 3, 3] = np.inf
    v, s = O.boxes(p["k"])
    _, got = fe().sparse_paged_attention(
        cuda(p["q"], BF16), cuda(p["k"], BF16), cuda(p["v"], BF16), (cuda(v), cuda(s)),
        cuda(p["tables"]), cuda(p["lens"]), 4, 16)
    assert got[0, 0].tolist() == [0, 5, 17, 24]
    # a query with a NaN ranks nothing: the lowest pages, and a NaN output as the dense one's
    p["q"][0, 1, 0] = np.nan
    out, got = fe().sparse_paged_attention(
        cuda(p["q"], BF16), cuda(p["k"], BF16), cuda(p["v"], BF16), (cuda(v), cuda(s)),
        cuda(p["tables"]), cuda(p["lens"]), 4, 16)
    assert got[0, 0].tolist() == [0, 1, 2, 24] and torch.isnan(out[0, 1]).all()
    fe().device_errors()


@pytest.mark.parametrize("dt", [BF16, F32])
def test_sparse_with_all_pages_is_the_dense_decode(dt):
    p = make_sparse(8, LENS, 8, 2, 128, 16, dt)
    v, s = O.boxes(p["k"])
    args = cuda(p["q"], dt), cuda(p["k"], dt), cuda(p["v"], dt)
    bt, lens = cuda(p["tables"]), cuda(p["lens"])
    out, _ = fe().sparse_paged_attention(*args, (cuda(v), cuda(s)), bt, lens, 64, 16)
    dense = fe().paged_attention(*args, bt, lens, 16)
    assert float((out.float() - dense.float()).abs().max()) <= 2 * ATTN_ATOL[dt]


def test_sparse_flags_a_block_out_of_range():
    from flash_engine import _lib
    p = make_sparse(9, [300], 4, 1, 64, 16, BF16)
    v, s = O.boxes(p["k"])
    for bad in (-3, len(p["k"]), 2 ** 30):
        t = p["tables"].copy()
        t[0, 0] = bad  # always chosen
        fe().sparse_paged_attention(
            cuda(p["q"], BF16), cuda(p["k"], BF16), cuda(p["v"], BF16), (cuda(v), cuda(s)),
            cuda(t), cuda(p["lens"]), 4, 16)
        assert fe().device_errors() == _lib.ERR_BAD_BLOCK


def test_offsets_past_32_bits():
    """The operators at the end of a cache of more than 2^32 bytes and 2^31 elements give what
    they give in a small one."""
    H, Hkv, d, bs, T = 8, 4, 128, 16, 75
    small, nb = 5, 262144 + 500
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn((T, (H + 2 * Hkv) * d), device="cuda", generator=g).to(BF16)
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    order = torch.tensor([3, 0, 4, 2, 1], device="cuda")
    q = qkv[:, :H * d].view(T, H, d)[-1:].contiguous()
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    got = []
    for blocks in (small, nb):
        # the big cache is not cleared: only the blocks in use are looked at
        kc, vc = (torch.empty((blocks, Hkv, bs, d), dtype=BF16, device="cuda") for _ in range(2))
        table = order + blocks - small
        kc[-small:], vc[-small:] = 0, 0
        pb = fe().new_page_bounds(blocks, Hkv, d, "cuda")
        slots = table[pos.long() // bs] * bs + pos.long() % bs
        qa = fe().paged_qkv_append(qkv, kc, vc, pos, slots, H, bs, page_bounds=pb)
        out, sel = fe().sparse_paged_attention(q, kc, vc, pb, table.int().view(1, -1), lens, 3, bs)
        got.append([x.clone() for x in (qa, kc[-small:], vc[-small:], pb.values[-small:],
                                        pb.scales[-small:], out, sel)])
        del kc, vc
    assert nb * Hkv * bs * d > 2 ** 31
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert fe().device_errors() == 0


def test_sparse_on_another_stream_and_repeated():
    p = make_sparse(10, [3000, 100], 8, 2, 64, 16, BF16)
    a = check_sparse(p, 9, stream=torch.cuda.Stream())
    b = check_sparse(p, 9)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# --------------------------------------------------------------------------- all together
def test_step_in_a_cuda_graph():
    """plan -> append (with boxes) -> sparse attention captured once and replayed: ten decode
    steps give what the same calls give outside a graph."""
    F = fe()
    S, H, Hkv, d, bs, nb, width = 5, 8, 2, 64, 16, 80, 16
    g = torch.Generator(device="cuda").manual_seed(0)

    def world():
        w = dict(tables=torch.full((S, width), -1, dtype=torch.int32, device="cuda"),
                 ring=torch.arange(nb, dtype=torch.int32, device="cuda"),
                 state=torch.tensor([0, nb, 0, 0], dtype=torch.int32, device="cuda"),
                 lens=torch.zeros(S, dtype=torch.int32, device="cuda"),
                 kc=torch.zeros((nb, Hkv, bs, d), dtype=BF16, device="cuda"),
                 vc=torch.zeros((nb, Hkv, bs, d), dtype=BF16, device="cuda"),
                 pb=F.new_page_bounds(nb, Hkv, d, "cuda"),
                 new=torch.tensor([31, 0, 33, 7, 48], dtype=torch.int32, device="cuda"),
                 qkv=torch.zeros((128, (H + 2 * Hkv) * d), dtype=BF16, device="cuda"))
        return w

    w_q = 1 + torch.randn(d, device="cuda", generator=g) * 0.1
    a = torch.arange(width * bs, device="cuda")[:, None] * 0.01 * torch.arange(1, d // 2 + 1,
                                                                             device="cuda")
    rope = (a.cos(), a.sin())

    def step(w):
        plan = F.plan_paged_step(w["lens"], w["new"], w["tables"], w["ring"], w["state"], bs,
                                 max_tokens=w["qkv"].shape[0])
        q = F.paged_qkv_append(w["qkv"], w["kc"], w["vc"], plan.positions, plan.slots, H, bs,
                               q_weight=w_q, k_weight=w_q, rope=rope, page_bounds=w["pb"])
        last = (plan.cu_seqlens[1:] - 1).clamp(min=0).long()
        out, sel = F.sparse_paged_attention(q[last], w["kc"], w["vc"], w["pb"], w["tables"],
                                            plan.context_lens, 3, bs)
        w["lens"].copy_(plan.context_lens)
        w["state"].copy_(plan.free_state)
        return out, sel

    data = [torch.randn((128, (H + 2 * Hkv) * d), device="cuda", generator=g).to(BF16)
            for _ in range(11)]
    eager, graphed = world(), world()
    for w in (eager, graphed):  # the prompts, outside the graph
        w["qkv"].copy_(data[10])
        step(w)
        w["new"].copy_(torch.tensor([1, 1, 1, 0, 1], dtype=torch.int32))
    before = {k: v.clone() for k, v in graphed.items() if isinstance(v, torch.Tensor)}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graphed)  # warm-up of the capture stream
    torch.cuda.synchronize()
    for k, v in before.items():
        graphed[k].copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, sel = step(graphed)
    for x in data[:10]:
        for w in (eager, graphed):
            w["qkv"].copy_(x)
        ref, rsel = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(sel, rsel)
    for k in before:
        assert torch.equal(eager[k], graphed[k]), k
    assert F.device_errors() == 0


def test_serving_example_runs():
    """The example's loop, small: with as many pages as the longest request has, the sparse
    decode is the dense one; with fewer it attends to fewer and stays near."""
    import os
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    sys.path.insert(0, os.path.join(root, "examples"))
    try:
        import serving_step
    finally:
        sys.path.pop(0)
    kw = dict(steps=14, requests=6, heads=8, kv_heads=2, d=64, max_len=512, prompt=(20, 200),
              tokens_per_step=256, quiet=True)
    whole = serving_step.serve(pages=32, **kw)
    few = serving_step.serve(pages=3, **kw)
    assert whole["errors"] == 0 and few["errors"] == 0 and whole["finite"] and few["finite"]
    assert whole["tokens"] == few["tokens"] > 14 * 3
    assert whole["share"] == 1 and whole["diff"] < 2 ** -7
    assert few["share"] < 0.9 and few["diff"] < 1
