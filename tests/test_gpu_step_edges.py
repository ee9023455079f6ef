"""Edges of the serving-step operators on the GPU: inputs that no kernel of the framework
wrote, refusals, orders of launches, and outputs too small for an absolute tolerance."""
import numpy as np
import pytest
import torch

from gpu_util import cuda
from step_util import attention_bound
from test_gpu_step import BF16, F16, F32, O, fe, make_sparse, vllm_k, vllm_v
from test_step_tolerance import LONG

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------------- scales nobody wrote
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("ctx", [900, 9000, 150001])
def test_sparse_pages_with_nan_scales_rank_as_infinite_ones(dt, ctx):
    """Far more pages with NaN scales than are chosen: the first of them, num_pages in all."""
    p = make_sparse(ctx, [ctx], 4, 1, 64, 16, dt)
    v, s = O.boxes(p["k"])
    pages = -(-ctx // 16)
    s[p["tables"][0, 3:pages - 5], 0] = np.array([0x7fffffff, 0xffffffff, 0x7fc00000],
                                                 np.uint32).view(np.float32)[
        np.arange(pages - 8) % 3]
    for first, last, num_pages in ((1, 1, 4), (2, 3, 9), (0, 1, 40)):
        out, got = fe().sparse_paged_attention(
            cuda(p["q"], dt), cuda(p["k"], dt), cuda(p["v"], dt), (cuda(v), cuda(s)),
            cuda(p["tables"]), cuda(p["lens"]), num_pages, 16, keep_first=first, keep_last=last)
        rest = num_pages - first - last
        want = list(range(first)) + list(range(3, 3 + rest)) + list(range(pages - last, pages))
        assert got[0, 0].tolist() == want
        assert torch.isfinite(out).all() and fe().device_errors() == 0


# ------------------------------------------------------------------------------- refusals
def test_plan_refuses_outputs_that_share_memory_with_inputs_or_one_another():
    """Some CTAs would read lengths that others have written over. Nothing is launched."""
    S, cap = 6, 6
    i32 = dict(dtype=torch.int32, device="cuda")
    lens, new = torch.full((S,), 5, **i32), torch.ones(S, **i32)
    table, ring = torch.zeros((S, 2), **i32), torch.arange(9, **i32)
    state, finished = torch.tensor([0, 9, 0, 0], **i32), torch.zeros(S, dtype=torch.bool,
                                                                     device="cuda")
    out = lambda: [torch.empty(S, **i32), torch.empty(S + 1, **i32),  # noqa: E731
                   torch.empty(cap, **i32), torch.empty(cap, dtype=torch.int64, device="cuda"),
                   torch.empty(4, **i32)]
    wide = torch.empty(64, **i32)  # outputs that overlap in part
    part = [wide[:S], wide[S - 1:2 * S], wide[20:20 + cap], wide[28:28 + 2 * cap].view(torch.int64),
            wide[60:]]
    flags = torch.zeros(4 * S, dtype=torch.bool, device="cuda")
    cases = [(0, lens), (0, new), (2, new), (2, lens), (4, state), (0, table.view(-1)[:S]),
             (1, ring[:S + 1]), (4, ring[2:6]), (3, table.view(torch.int64).view(-1)),
             (0, flags.view(torch.int32))]
    before = [x.clone() for x in (lens, new, table, ring, state)]

    def plan(o, fin=finished):
        return fe().plan_paged_step(lens, new, table, ring, state, 16, finished=fin, out=tuple(o))

    for k, t in cases:
        o = out()
        o[k] = t
        with pytest.raises(ValueError, match="inputs"):
            plan(o, flags[:S] if t.data_ptr() == flags.data_ptr() else finished)
    for o in (part, (lambda o: [o[0], o[1], o[0], o[3], o[4]])(out())):
        with pytest.raises(ValueError, match="overlap"):
            plan(o)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (lens, new, table, ring, state)))
    # neighbours in one buffer share nothing
    part[1] = wide[S:2 * S + 1]
    assert plan(part).positions.tolist() == [5] * S
    assert fe().device_errors() == 0


def test_append_refuses_page_bounds_before_it_writes():
    """A call that is refused for its boxes has left queries and caches as they were."""
    c, bf = dict(device="cuda"), dict(dtype=BF16, device="cuda")

    def attempt(d, bs, bounds, error, Hkv=2, shift=0):
        store = torch.zeros(4 * Hkv * bs * d + 8, **bf)
        kc = store[shift:shift + 4 * Hkv * bs * d].view(4, Hkv, bs, d)
        vc = torch.zeros((4, Hkv, bs, d), **bf)
        q = torch.zeros((5, 4, d), **bf)
        qkv = torch.randn((5, (4 + 2 * Hkv) * d), **c).to(BF16)
        i = torch.arange(5, **c)
        with pytest.raises(error):
            fe().paged_qkv_append(qkv, kc, vc, i.int(), i, 4, bs, page_bounds=bounds, out=q)
        torch.cuda.synchronize()
        assert not kc.any() and not vc.any() and not q.any()

    good = lambda d: fe().new_page_bounds(4, 2, d, "cuda")  # noqa: E731
    b = good(64)
    attempt(64, 16, (b.values[:, :1].contiguous(), b.scales), ValueError)
    attempt(64, 16, (b.values, b.scales[:3]), ValueError)
    attempt(64, 16, (b.values.int(), b.scales), ValueError)
    attempt(64, 16, (b.values.transpose(1, 2), b.scales), ValueError)
    attempt(64, 16, b.values, ValueError)
    attempt(64, 16, (b.values.cpu(), b.scales), TypeError)
    attempt(96, 16, good(96), RuntimeError)      # what the boxes do not take
    attempt(64, 8, good(64), RuntimeError)
    attempt(64, 16, good(64), RuntimeError, shift=4)
    assert fe().device_errors() == 0


def test_sparse_scale_that_fp32_does_not_hold_is_refused():
    """It would be 0 there, which the C entry takes as 1 / sqrt(d)."""
    p = make_sparse(21, [60], 4, 2, 64, 16, BF16)
    v, s = O.boxes(p["k"])
    args = (cuda(p["q"], BF16), cuda(p["k"], BF16), cuda(p["v"], BF16), (cuda(v), cuda(s)),
            cuda(p["tables"]), cuda(p["lens"]), 4, 16)
    for scale in (1e-60, 0.0, -0.0, -1e-60, float("nan"), -1.0):
        with pytest.raises(ValueError):
            fe().sparse_paged_attention(*args, scale)
    # the smallest ones that it does hold: equal weights, and not the default scale
    tiny, _ = fe().sparse_paged_attention(*args, 2.0 ** -149)
    assert torch.equal(tiny, fe().sparse_paged_attention(*args, 1e-30)[0])
    assert not torch.equal(tiny, fe().sparse_paged_attention(*args)[0])
    assert fe().device_errors() == 0


# ------------------------------------------------------------ lengths near the end of 32 bits
def test_plan_with_the_largest_blocks_and_lengths():
    big = 2 ** 31 - 1
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def plan(ctx, new, tables, bs, finished=None, max_tokens=2):
        t, ring = i(tables), i([0, 1, 2, 5])
        s = fe().plan_paged_step(i(ctx), i(new), t, ring, i([0, 3]), bs, max_tokens=max_tokens,
                                 finished=None if finished is None else
                                 torch.tensor(finished, device="cuda"))
        return [x.tolist() for x in s] + [t.tolist(), ring.tolist()]

    # blocks of 2^31 - 1 tokens: the token goes to the row's own block
    assert plan([2], [1], [[3]], big) == [[3], [0, 1], [2, -1], [3 * big + 2, -1], [0, 3, 1, 1],
                                          [[3]], [0, 1, 2, 5]]
    # a finished row of them gives its block back and takes a new one
    assert plan([7], [2], [[3]], big, [True]) == [[2], [0, 2], [0, 1], [0, 1], [1, 3, 1, 2], [[0]],
                                                  [0, 1, 2, 3]]
    # a row with room for 2^31 tokens: a length ends at 2^31 - 1
    assert plan([big - 1], [1], [[3, 2]], 2 ** 30) == [
        [big], [0, 1], [big - 1, -1], [2 * 2 ** 30 + 2 ** 30 - 2, -1], [0, 3, 1, 1], [[3, 2]],
        [0, 1, 2, 5]]
    full = plan([big], [1], [[3, 2]], 2 ** 30)
    assert full[0] == [big] and full[1] == [0, 0] and full[2] == [-1, -1]
    assert full[4] == [0, 3, 0, 0] and full[5] == [[3, 2]]
    assert fe().device_errors() == 0


def test_append_refuses_an_out_that_overlaps_qkv_or_the_caches():
    T, H, Hkv, d, bs = 3, 4, 2, 64, 16
    store = torch.zeros(4096 * 8, dtype=BF16, device="cuda")
    wide = store[:T * 1000].view(T, 1000)
    qkv = wide[:, :(H + 2 * Hkv) * d]
    kc, vc = (store[at:at + 4 * Hkv * bs * d].view(4, Hkv, bs, d) for at in (8192, 20480))
    i = torch.arange(T, device="cuda")
    at = lambda x: store[x:x + T * H * d].view(T, H, d)  # noqa: E731
    app = lambda out: fe().paged_qkv_append(qkv, kc, vc, i.int(), i, H, bs, out=out)  # noqa: E731
    for x in (0, 2000, 2 * 1000 + (H + 2 * Hkv) * d - 1, 8192, 16000, 20480 - 1, 20480 + 8191):
        with pytest.raises(ValueError, match="overlap"):
            app(at(x))
    for x in (2 * 1000 + (H + 2 * Hkv) * d, 16384, 20480 - T * H * d, 20480 + 8192):
        app(at(x))
    assert fe().device_errors() == 0


# ------------------------------------------------------------------- launches right in a row
@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("between", [False, True])
def test_dense_decode_right_behind_the_plan(dt, between):
    """plan -> dense decode -> plan -> .. on one stream with nothing between them (or with an
    append and a sparse attention): every decode attends to the lengths and tables of its
    own step."""
    from oracle import attention_oracle as A
    bs, S, H, Hkv, d, nb, width, steps = 16, 7, 8, 2, 64, 160, 16, 12
    g = np.random.default_rng(5)
    k, v = (torch.from_numpy(g.standard_normal((nb, Hkv, bs, d))).cuda().to(dt) for _ in range(2))
    q = [torch.from_numpy(g.standard_normal((S, H, d))).cuda().to(dt) for _ in range(steps)]
    new = g.integers(1, 20, (steps, S)).astype(np.int32)
    new[0] = g.integers(1, 60, S)
    fin = g.random((steps, S)) < 0.25
    fin[0] = False
    cap = int(new.sum(1).max())
    qkv = torch.randn((cap, (H + 2 * Hkv) * d), device="cuda").to(dt)
    pb = fe().new_page_bounds(nb, Hkv, d, "cuda")
    dnew, dfin = [cuda(x) for x in new], [cuda(x) for x in fin]
    tables, ring = cuda(np.zeros((S, width), np.int32)), cuda(np.arange(nb, dtype=np.int32))
    lens, state = cuda(np.zeros(S, np.int32)), cuda(np.array([3, nb, 0, 0], np.int32))
    kw = dict(dtype=torch.int32, device="cuda")
    bufs = [(torch.empty(S, **kw), torch.empty(S + 1, **kw), torch.empty(cap, **kw),
             torch.empty(cap, dtype=torch.int64, device="cuda"), torch.empty(4, **kw))
            for _ in range(steps)]
    outs = [torch.empty_like(x) for x in q]
    # what each step's decode reads: its own lengths and tables, and the caches as they are then
    want, m_tables, m_ring, m_state = [], np.zeros((S, width), np.int32), ring.cpu().numpy(), [3, nb]
    m_lens = np.zeros(S, int)
    for i in range(steps):
        r = O.plan(m_lens, new[i], m_tables, m_ring, m_state[0], m_state[1], bs, cap, fin[i])
        assert r["state"][2] == S
        m_lens, m_tables, m_ring = r["context_lens"].astype(int), r["tables"], r["ring"]
        m_state = [int(r["state"][0]), int(r["state"][1])]
        want.append((m_tables, m_lens.astype(np.int32), r["positions"], r["slots"]))
    caches = [(k.clone(), v.clone())]
    if between:
        for i in range(steps - 1):
            kk, vv = (x.clone() for x in caches[-1])
            fe().paged_qkv_append(qkv, kk, vv, cuda(want[i][2]), cuda(want[i][3]), H, bs)
            caches.append((kk, vv))
    torch.cuda.synchronize()
    for i in range(steps):
        s = fe().plan_paged_step(lens, dnew[i], tables, ring, state, bs, finished=dfin[i],
                                 out=bufs[i])
        fe().paged_attention(q[i], k, v, tables, s.context_lens, bs, out=outs[i])
        if between:
            fe().paged_qkv_append(qkv, k, v, s.positions, s.slots, H, bs, page_bounds=pb)
            fe().sparse_paged_attention(q[i], k, v, pb, tables, s.context_lens, 3, bs)
        lens, state = s.context_lens, s.free_state
    torch.cuda.synchronize()
    f64 = lambda x: x.double().cpu().numpy()  # noqa: E731
    for i in range(steps):
        kk, vv = caches[i if between else 0]
        ref = A.paged_attention_gqa(f64(q[i]), f64(kk), f64(vv), want[i][0], want[i][1])
        err = np.abs(f64(outs[i]) - ref).max()
        assert err <= (2e-2 if dt == BF16 else 1e-3), (i, err)
    np.testing.assert_array_equal(tables.cpu().numpy(), want[-1][0])
    assert fe().device_errors() == 0


# ------------------------------------------------- outputs, to within what their sums allow
def check_outputs(p, num_pages, first=1, last=1, layout="flat"):
    """Chosen pages equal, every output within the bound of step_util.py."""
    v, s = O.boxes(p["k"])
    S, Hkv, G = len(p["lens"]), p["k"].shape[1], p["q"].shape[1] // p["k"].shape[1]
    sel = np.full((S, Hkv, num_pages), -1, np.int32)
    for i in range(S):
        for h in range(Hkv):
            pages = O.select(p["q"][i, h * G:(h + 1) * G], v[:, h], s[:, h], p["tables"][i],
                             p["lens"][i], p["bs"], num_pages, first, last)
            sel[i, h, :len(pages)] = pages
    dt, vl = p["dt"], layout == "vllm"
    out, got = fe().sparse_paged_attention(
        cuda(p["q"], dt), cuda(vllm_k(p["k"]) if vl else p["k"], dt),
        cuda(vllm_v(p["v"]) if vl else p["v"], dt), (cuda(v), cuda(s)), cuda(p["tables"]),
        cuda(p["lens"]), num_pages, p["bs"], keep_first=first, keep_last=last, kv_layout=layout)
    np.testing.assert_array_equal(got.cpu().numpy(), sel)
    ref, bound = attention_bound(p, sel)
    over = np.abs(out.double().cpu().numpy() - ref) / np.maximum(bound, 1e-300)
    assert (over <= 1).all(), float(over.max())
    assert fe().device_errors() == 0


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("case", LONG, ids=lambda c: f"{c[1][0]}-{c[6]}")
def test_sparse_outputs_of_many_pages(case, dt):
    """A CTA's share, a join weight or the end of the list lost would show (see
    test_step_tolerance.py)."""
    check_outputs(make_sparse(*case[:6], dt), case[6])


@pytest.mark.parametrize("layout", ["flat", "vllm"])
@pytest.mark.parametrize("dt", [BF16, F16])
def test_sparse_outputs_of_many_pages_in_both_layouts(dt, layout):
    check_outputs(make_sparse(34, [9000, 5000], 8, 2, 64, 16, dt), 200, layout=layout)


@pytest.mark.parametrize("dt", [BF16, F32])
@pytest.mark.parametrize("H,Hkv,d,bs", [
    (9, 9, 64, 16), (12, 12, 128, 16), (32, 32, 128, 16), (40, 40, 64, 32),  # one head a group
    (64, 16, 64, 16), (80, 10, 128, 16),                                     # and more
    (64, 4, 128, 16), (48, 3, 128, 32), (128, 8, 128, 16),  # query rows that shrink the group
    (80, 2, 128, 16), (130, 2, 64, 16)])                    # more heads than a fused call takes
def test_sparse_more_kv_heads_than_a_score_cta_takes(dt, H, Hkv, d, bs):
    """The scores of several groups of KV heads, the last one not full."""
    check_outputs(make_sparse(H + Hkv, [700, 31, 1500, 0, 6 * bs + 1], H, Hkv, d, bs, dt), 6)


@pytest.mark.parametrize("H,Hkv", [(9, 9), (64, 16)])
def test_sparse_more_kv_heads_over_long_rows(H, Hkv):
    check_outputs(make_sparse(40 + Hkv, [20000, 3001], H, Hkv, 64, 16, BF16), 40, 2, 3)


# --------------------------------------------------------------- arguments made for the call
@pytest.mark.parametrize("T", [64, 1024])
def test_append_with_rope_tables_that_live_as_long_as_the_call(T):
    """rope may be any pair, an iterator of fresh tensors too: the queries' memory must not be
    that of a table that was let go before the kernel ran."""
    H, Hkv, d, bs = 8, 2, 128, 16
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn((T, (H + 2 * Hkv) * d), device="cuda", generator=g).to(BF16)
    angle = torch.rand((T * H, d // 2), device="cuda", generator=g)  # a table like out
    tables = [angle.cos(), angle.sin()]
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    slots = torch.arange(T, device="cuda")
    cache = lambda: torch.zeros((T // bs, Hkv, bs, d), dtype=BF16, device="cuda")  # noqa: E731
    app = lambda rope: fe().paged_qkv_append(qkv, cache(), cache(), pos, slots, H, bs,  # noqa: E731
                                             rope=rope)
    want = app(tuple(tables))
    assert tables[0].nbytes == want.nbytes
    for _ in range(20):
        assert torch.equal(app(x.clone() for x in tables), want)
    assert torch.equal(app(tables), want)
