"""What the serving-step operators refuse, before any GPU work: the C entries by status, the
Python operators by exception (the GPU cases with CUDA tensors of wrong shapes and types).

The C entries are called with addresses that are nobody's: where a GPU is present, a missing
check would send a kernel there. These run without one, where it shows as another status."""
import pytest
import torch

no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="calls with invalid addresses")
AT = 1 << 16  # aligned, not mapped


def lib():
    from flash_engine import _lib
    return _lib.lib


@no_gpu
def test_plan_entry_refuses():
    def call(S=1, maxb=4, nb=8, bs=16, mt=4, null=None):
        p = [AT] * 11
        if null is not None:
            p[null] = None
        return lib().fe_plan_paged_step(*p, S, maxb, nb, bs, mt, None)
    assert call() not in (0, 1)  # accepted, and no device
    assert call(null=2) not in (0, 1)  # finished may be NULL
    for i in (0, 1, 3, 4, 5, 6, 7, 8, 9, 10):
        assert call(null=i) == 1, i
    for kw in (dict(S=-1), dict(S=16385), dict(maxb=-1), dict(nb=0), dict(nb=2 ** 30), dict(bs=0),
               dict(mt=-1), dict(mt=2 ** 30)):
        assert call(**kw) == 1, kw


@no_gpu
def test_append_entry_refuses():
    def call(stride=1000, eps=1e-6, cos=None, sin=None, rd=64, rmax=8, T=1, H=4, Hkv=1, d=64,
             bs=16, nb=4, dt=0, lay=0, null=None):
        p = [AT] * 6
        if null is not None:
            p[null] = None
        return lib().fe_paged_qkv_append(p[0], stride, *p[1:], None, None, 0, eps, cos, sin, rd,
                                         rmax, 1, T, H, Hkv, d, bs, nb, dt, lay, None)
    assert call() not in (0, 1)
    for i in range(6):
        assert call(null=i) == 1, i
    for kw in (dict(stride=383), dict(eps=-1.0), dict(eps=float("nan")), dict(cos=16),
               dict(sin=16), dict(cos=16, sin=16, rd=65), dict(cos=16, sin=16, rd=66),
               dict(cos=16, sin=16, rd=0), dict(cos=16, sin=16, rmax=0), dict(T=-1), dict(H=0),
               dict(Hkv=0), dict(d=0), dict(bs=0), dict(nb=0), dict(dt=3), dict(dt=-1),
               dict(lay=2), dict(lay=1, dt=2), dict(lay=1, d=60)):
        assert call(**kw) == 1, kw
    assert call(T=0) == 0


@no_gpu
def test_bounds_entry_refuses():
    def call(k=AT, v=AT, s=AT, slots=AT, T=1, Hkv=1, d=64, bs=16, nb=4, dt=0, lay=0):
        return lib().fe_update_page_bounds(k, v, s, slots, T, Hkv, d, bs, nb, dt, lay, None)
    assert call() not in (0, 1)
    for kw in (dict(k=AT + 8), dict(v=AT + 4), dict(s=AT + 2), dict(k=None), dict(v=None),
               dict(s=None), dict(slots=None), dict(T=-1), dict(Hkv=0), dict(d=96), dict(bs=8), dict(nb=0),
               dict(dt=3), dict(lay=2), dict(lay=1, bs=32), dict(lay=1, dt=2)):
        assert call(**kw) == 1, kw
    assert call(T=0) == 0


@no_gpu
def test_sparse_entry_refuses():
    lib_ws = (1 << 64) - 1

    def call(S=1, H=8, Hkv=2, d=64, bs=16, maxb=8, nb=8, k=4, first=1, last=1, dt=0, lay=0,
             ws=None, n=lib_ws, at=None, to=None):
        p = [AT] * 10
        if at is not None:
            p[at] = to
        return lib().fe_sparse_paged_attention(*p, S, H, Hkv, d, bs, maxb, nb, k, first, last, 0.0,
                                               dt, lay, ws, n, None)
    assert call() not in (0, 1)
    for i in range(10):
        assert call(at=i) == 1, i
    for kw in (dict(S=-1), dict(H=7), dict(Hkv=0), dict(d=96), dict(bs=8), dict(maxb=0),
               dict(nb=0), dict(k=1), dict(first=-1), dict(last=0), dict(first=4, last=1),
               dict(dt=3), dict(lay=2), dict(lay=1, bs=32), dict(lay=1, dt=2),
               dict(at=1, to=AT + 8), dict(at=2, to=AT + 8), dict(at=4, to=AT + 8),
               dict(at=5, to=AT + 2), dict(at=0, to=AT + 2), dict(at=0, to=AT + 4, dt=2),
               dict(S=2 ** 30), dict(nb=2 ** 30), dict(H=2 * 129), dict(n=0), dict(ws=AT, n=5)):
        assert call(**kw) == 1, kw
    assert call(S=0) == 0
    scratch = lib().fe_sparse_paged_attention_scratch_ints
    assert scratch(3, 2, 64, 9) >= 60 + 6 * 64 and scratch(3, 2, 5000, 9) >= 60 + 6 * 5000
    assert scratch(-1, 2, 8, 9) == scratch(1, 0, 8, 9) == scratch(1, 1, 0, 9) == 0


def test_operators_have_no_cpu_fallback():
    import flash_engine as F
    z = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: F.plan_paged_step(z, z, z.view(4, 1), z, z, max_tokens=4),
                 lambda: F.paged_qkv_append(torch.zeros(1, 256), z, z, z, z, 2),
                 lambda: F.update_page_bounds(z, (z, z), z),
                 lambda: F.sparse_paged_attention(z, z, z, (z, z), z, z, 4)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
def test_operators_check_shapes_and_types():
    import flash_engine as F
    c = dict(device="cuda")
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, **c)  # noqa: E731
    lens, tab, ring, st = i(3), i(3, 4), i(9), i(2)
    ok = F.plan_paged_step(lens, lens, tab, ring, st, max_tokens=4)
    for bad in (lambda: F.plan_paged_step(lens, i(2), tab, ring, st, max_tokens=4),
                lambda: F.plan_paged_step(lens, lens, tab, ring, i(1), max_tokens=4),
                lambda: F.plan_paged_step(lens, lens, tab, ring, st),
                lambda: F.plan_paged_step(lens, lens, tab.t(), ring, st, max_tokens=4),
                lambda: F.plan_paged_step(lens, lens, tab, ring, st, max_tokens=4,
                                          finished=i(3)),
                lambda: F.plan_paged_step(lens, lens, tab, ring, st, max_tokens=5, out=ok),
                lambda: F.plan_paged_step(ok.context_lens, lens, tab, ring, st, out=ok)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        F.plan_paged_step(lens.long(), lens, tab, ring, st, max_tokens=4)
    with pytest.raises(RuntimeError):
        F.plan_paged_step(lens, lens, tab, ring, st, 0, max_tokens=4)

    kc = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16, **c)
    qkv = torch.zeros((5, 8 * 64), dtype=torch.bfloat16, **c)
    pos, slots = i(5), torch.zeros(5, dtype=torch.int64, **c)
    app = lambda q=qkv, k=kc, v=kc, p=pos, s=slots, h=4, **kw: F.paged_qkv_append(  # noqa: E731
        q, k, v, p, s, h, **kw)
    app()
    w = torch.ones(64, **c)
    for bad in (lambda: app(h=5), lambda: app(v=kc.half()), lambda: app(p=pos[:4]),
                lambda: app(s=slots.int()), lambda: app(q=qkv.t()), lambda: app(k=kc[:, :, :8]),
                lambda: app(q_weight=w[:32]), lambda: app(q_weight=w.half()),
                lambda: app(q_weight=w, k_weight=w.bfloat16()),
                lambda: app(rope=(torch.ones(9, 33, **c),) * 2),
                lambda: app(out=torch.zeros(5, 4, 64, **c)), lambda: app(kv_layout="vllm")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        app(q=qkv.double())

    pb = F.new_page_bounds(4, 2, 64, "cuda")
    with pytest.raises(ValueError):
        F.update_page_bounds(kc, (pb.values[:, :1], pb.scales), slots)
    with pytest.raises(ValueError):
        F.update_page_bounds(kc, pb, slots.int())
    with pytest.raises(RuntimeError):
        k8 = torch.zeros((4, 2, 8, 64), dtype=torch.bfloat16, **c)
        F.update_page_bounds(k8, pb, slots, 8)

    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, **c)
    att = lambda q=q, k=kc, b=pb, t=tab, n=lens, m=3, **kw: F.sparse_paged_attention(  # noqa: E731
        q, k, kc, b, t, n, m, **kw)
    att()
    for bad in (lambda: att(m=1), lambda: att(keep_last=0), lambda: att(keep_first=3),
                lambda: att(q=q[0]), lambda: att(q=q[:, :3].contiguous()), lambda: att(scale=-1.0),
                lambda: att(b=(pb.values, pb.scales[:3])), lambda: att(t=tab[:2]),
                lambda: att(out=q[:2]), lambda: att(selected=i(3, 2, 2)),
                lambda: att(workspace=torch.zeros(8, **c))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        att(q=q.half())
    torch.cuda.synchronize()
    assert F.device_errors() == 0
