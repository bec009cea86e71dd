"""Norm and rotation of new heads with the cache write, against the formulas in 64 bits.

Tolerances.  Per element the kernel works in fp32 on inputs taken as exact: the
root mean square costs at most (D + 4) half steps of 2^-24 (a sum of D squares,
the product with 1 / D, the root and the quotient), the two products with it and
the weight one each, the rotation two products and a sum of size |a| + |b|: below
(D + 10) 2^-24 (|a| + |b|).  The store adds half a step of its type, and the
scaled store another 2^-24 for the quotient.  Below a type's normal range half a
step is absolute: 2^-25 for fp16, 2^-10 for e4m3."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8, "fp8": 2.0**-4}
LEAST = {"f32": 0.0, "f16": 2.0**-25, "bf16": 0.0, "fp8": 2.0**-10}
TOP = {"fp8": 448.0}


def table(rows, rot, dtype=torch.float64):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    return torch.cat([a.cos(), a.sin()], 1).to(dtype)


def turned(x, w, cs, pos, rot, pairs, eps):
    """(value, size that its error scales with) in 64 bits."""
    x = x.double().cpu()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().cpu()
    size = x.abs()
    if rot:
        inside = (pos >= 0) & (pos < cs.shape[0])
        t = cs.double().cpu()[pos.clamp(0, cs.shape[0] - 1)][:, None]
        t = torch.where(inside[:, None, None], t, float("nan"))
        c, s = t[..., :rot // 2], t[..., rot // 2:]
        ia = torch.arange(0, rot, 2) if pairs else torch.arange(rot // 2)
        ib = ia + 1 if pairs else ia + rot // 2
        a, b = x[..., ia], x[..., ib]
        x, size = x.clone(), size.clone()
        x[..., ia], x[..., ib] = a * c - b * s, b * c + a * s
        size[..., ia] = size[..., ib] = a.abs() + b.abs()
    return x, size


def near(got, want, size, D, to, scaled):
    want = want.clamp(-TOP.get(to, np.inf), TOP.get(to, np.inf))
    tol = (D + 10 + (1 if scaled else 0)) * 2.0**-24 * size
    tol = tol + HALF[to] * (want.abs() + tol) + LEAST[to]
    got = got.double().cpu()
    ok = ((got - want).abs() <= tol) | (got.isnan() & want.isnan())
    assert ok.all(), (int((~ok).sum()), (got - want)[~ok][:4], tol[~ok][:4])


def check(pa, dev, T, H, HKV, D, BS, *, rot, pairs=False, act="bf16", kv="bf16", norm=True, ks=1.0, vs=1.0, out=None,
          wt=None, tt="f32", slots=None, pos=None, packed=True, seed=0, i32=False, in_place=False, eps=1e-6):
    print("rope", T, H, HKV, D, rot, pairs, act, kv, flush=True)
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    qkv = torch.randn((T, H + 2 * HKV, D), generator=g).to(DT[act]).to(dev)
    q, k, v = qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:]
    if not packed:  # head-major sources
        q, k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    qw = kw = None
    if norm:
        qw, kw = ((torch.randn(D, generator=g) * 0.2 + 1).to(DT[wt or act]).to(dev) for _ in range(2))
    rows = 500
    cs = table(rows, rot).to(DT[tt]).to(dev)
    NB = -(-T // BS) + 2
    it = torch.int32 if i32 else torch.int64
    slots = torch.from_numpy(rng.permutation(NB * BS)[:T]) if slots is None else torch.tensor(slots)
    pos = torch.from_numpy(rng.integers(0, rows, T)) if pos is None else torch.tensor(pos)
    kc, vc = (torch.randn((NB, BS, HKV, D), generator=g).to(DT[kv]).to(dev) for _ in range(2))
    k0, v0 = kc.clone(), vc.clone()
    want_q, size_q = turned(q, qw, cs, pos, rot, pairs, eps)
    want_k, size_k = turned(k, kw, cs, pos, rot, pairs, eps)
    kh, vh = k.clone(), v.clone()
    o = pa.qk_norm_rope_write_kv(q, k, v, kc, vc, slots.to(it).to(dev), cs, pos.to(it).to(dev), q_weight=qw,
                                 k_weight=kw, eps=eps, interleaved=pairs, k_scale=ks, v_scale=vs,
                                 out_dtype=DT[out] if out else None, out=q if in_place else None)
    assert (o is q) == in_place and o.dtype == (DT[out] if out else DT[act])
    near(o, want_q, size_q, D, out or act, False)
    used = (slots >= 0) & (slots < NB * BS)
    at = slots[used].to(dev)
    f = lambda c: c.flatten(0, 1)  # noqa: E731
    near(f(kc.float())[at], (want_k / ks)[used], (size_k / abs(ks))[used], D, kv, ks != 1)
    near(f(vc.float())[at], (vh.double().cpu() / vs)[used], torch.zeros_like(want_k)[used], D, kv, vs != 1)
    rest = torch.ones(NB * BS, dtype=torch.bool, device=dev)
    rest[at] = False
    for c, c0 in ((kc, k0), (vc, v0)):
        assert torch.equal(f(c.view(torch.uint8))[rest], f(c0.view(torch.uint8))[rest])
    assert torch.equal(k, kh) and torch.equal(v, vh)


@pytest.mark.parametrize("T", [1, 2, 33, 700])
@pytest.mark.parametrize("H,HKV,D,rot,pairs", [(12, 12, 64, 64, False), (32, 8, 128, 128, False), (8, 1, 128, 32, True),
                                               (4, 2, 256, 256, False), (5, 5, 32, 16, False), (3, 1, 80, 48, True),
                                               (6, 2, 96, 96, False), (2, 2, 16, 16, True), (7, 1, 208, 64, False)])
def test_shapes(pa, dev, T, H, HKV, D, rot, pairs):
    check(pa, dev, T, H, HKV, D, 16, rot=rot, pairs=pairs)


@pytest.mark.parametrize("act", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kv,ks,vs", [("f16", 1, 1), ("bf16", 1, 1), ("f32", 0.5, 3.0), ("fp8", 1 / 16, 1 / 16),
                                      ("fp8", 1, 1), ("fp8", -0.37, 0.011), ("f16", 1, 0.3)])
def test_types(pa, dev, act, kv, ks, vs):
    check(pa, dev, 40, 8, 2, 64, 8, rot=64, act=act, kv=kv, ks=ks, vs=vs, seed=3)
    check(pa, dev, 600, 24, 4, 64, 8, rot=32, pairs=True, act=act, kv=kv, ks=ks, vs=vs, norm=False, seed=4)


def test_options(pa, dev):
    base = dict(rot=64, act="bf16", kv="f16")
    check(pa, dev, 37, 8, 2, 64, 16, out="f32", wt="f32", tt="bf16", **base)
    check(pa, dev, 37, 8, 2, 64, 16, out="f16", wt="f16", tt="f16", i32=True, **base)
    check(pa, dev, 37, 8, 2, 64, 16, packed=False, **base)
    check(pa, dev, 37, 8, 2, 64, 16, in_place=True, **base)
    check(pa, dev, 900, 24, 8, 64, 16, in_place=True, **base)
    check(pa, dev, 37, 8, 2, 64, 16, eps=0.5, **base)
    check(pa, dev, 37, 8, 2, 64, 16, **{**base, "rot": 0})  # the norm and the write alone


def test_padding(pa, dev):
    """Padding tokens write no cache row, positions outside the table make NaN, other tokens are not touched."""
    slots = [5, -1, 7, 48, 1 << 40, 0, -(1 << 33)]
    check(pa, dev, 7, 8, 2, 64, 16, rot=64, slots=slots)
    check(pa, dev, 7, 8, 2, 64, 16, rot=32, kv="fp8", pos=[0, -1, 499, 500, 1 << 40, 3, 7])
    check(pa, dev, 7, 8, 2, 64, 16, rot=64, kv="bf16", pos=[0, -1, 499, 500, 9, 3, 7], i32=True, pairs=True)


def test_non_finite_rows_stay_alone(pa, dev):
    """Inf and NaN in one head reach that head's results only."""
    T, H, HKV, D = 6, 8, 2, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((T, n, D), generator=g).bfloat16().to(dev) for n in (H, HKV, HKV))
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    cs, pos, slots = table(64, 64, torch.float32).to(dev), torch.arange(T, device=dev), torch.arange(T, device=dev)

    def call(q, k, v):
        kc, vc = (torch.zeros((2, 4, HKV, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
        return pa.qk_norm_rope_write_kv(q, k, v, kc, vc, slots, cs, pos, q_weight=w, k_weight=w), kc, vc

    print("non-finite", flush=True)
    want = call(q, k, v)
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    q2[2, 3, 5], k2[4, 1, 9], v2[0, 0, 0] = float("nan"), float("inf"), float("-inf")
    got = call(q2, k2, v2)
    keep = torch.ones((T, H), dtype=torch.bool, device=dev)
    keep[2, 3] = False
    assert torch.equal(got[0][keep], want[0][keep]) and got[0][2, 3].isnan().all()
    kg, kw_ = got[1].flatten(0, 1), want[1].flatten(0, 1)
    keep = torch.ones((8, HKV), dtype=torch.bool, device=dev)
    keep[4, 1] = False
    assert torch.equal(kg[keep], kw_[keep]) and kg[4, 1].isnan().any()
    vg, vw = got[2].flatten(0, 1), want[2].flatten(0, 1)
    assert vg[0, 0, 0] == float("-inf") and torch.equal(vg.flatten()[1:], vw.flatten()[1:])


def test_write_equals_write_kv(pa, dev):
    """Without norm and rotation the cache holds what write_kv writes, bit for bit."""
    g = torch.Generator().manual_seed(2)
    for act, kv, s in (("bf16", "bf16", 1.0), ("f32", "fp8", 0.07), ("f16", "f32", 1.0)):
        q, k, v = (torch.randn((50, n, 64), generator=g).to(DT[act]).to(dev) for n in (4, 2, 2))
        a, b, c, d = (torch.zeros((4, 16, 2, 64), dtype=DT[kv], device=dev) for _ in range(4))
        slots = torch.randperm(64, generator=g)[:50].to(dev)
        cs, pos = torch.zeros((1, 0), device=dev), torch.zeros(50, dtype=torch.int64, device=dev)
        print("as write_kv", act, kv, flush=True)
        o = pa.qk_norm_rope_write_kv(q, k, v, a, b, slots, cs, pos, k_scale=s, v_scale=s)
        pa.write_kv(c, d, k, v, slots, s, s)
        assert torch.equal(o, q)
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8))
        assert torch.equal(b.view(torch.uint8), d.view(torch.uint8))


def test_captured_and_on_a_stream(pa, dev):
    T, H, HKV, D = 9, 8, 2, 128
    q, k, v = (torch.randn((T, n, D), device=dev).bfloat16() for n in (H, HKV, HKV))
    kc, vc = (torch.zeros((4, 16, HKV, D), dtype=torch.bfloat16, device=dev) for _ in range(2))
    cs, pos = table(64, D, torch.float32).to(dev), torch.arange(T, device=dev)
    slots = torch.arange(T, device=dev)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    call = lambda: pa.qk_norm_rope_write_kv(q, k, v, kc, vc, slots, cs, pos, q_weight=w, k_weight=w)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    print("capture", flush=True)
    with torch.cuda.graph(graph):
        out = call()
    for step in range(3):
        q.normal_()
        k.normal_()
        slots.copy_(torch.randperm(64)[:T])
        kc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), kc.clone()
        kc.zero_()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], kc)


def test_python_paths_agree(pa, dev, monkeypatch, tmp_path):
    """Without the operator library, on copies and views: the same results and refusals."""
    import sys
    ops = sys.modules[pa.paged_attention.__module__]
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((9, n, 64), generator=g).bfloat16().to(dev) for n in (4, 2, 2))
    w = torch.randn(64, generator=g).to(dev)
    cs = table(32, 32, torch.float32).to(dev)
    pos, slots = torch.arange(9), torch.arange(9, dtype=torch.int16) * 3

    def calls():
        kc, vc = (torch.zeros((3, 16, 2, 64), dtype=torch.float8_e4m3fn, device=dev) for _ in range(2))
        odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=dev)[1:].view(q.shape).copy_(q)  # not 16-byte aligned
        wide = k.repeat_interleave(2, 2)[..., ::2]                                              # last dim strided
        a = pa.qk_norm_rope_write_kv(odd, wide, v, kc, vc, slots, cs, pos, q_weight=w, k_weight=w, k_scale=0.5)
        b = pa.qk_norm_rope_write_kv(q, k, v, kc, vc, slots.to(dev) + 1, cs, pos.to(dev), out_dtype=torch.float32)
        return [a, b, kc.view(torch.uint8), vc.view(torch.uint8)]

    def refusals():
        kc = torch.zeros((3, 16, 2, 64), dtype=torch.bfloat16, device=dev)
        with pytest.raises(RuntimeError, match="key must be on CUDA"):
            pa.qk_norm_rope_write_kv(q, k.cpu(), v, kc, kc.clone(), slots, cs, pos)
        with pytest.raises(RuntimeError, match=r"q must be \[T, H, D\]"):
            pa.qk_norm_rope_write_kv(q[0], k, v, kc, kc.clone(), slots, cs, pos)
        with pytest.raises(RuntimeError, match="16-byte aligned"):
            pa.qk_norm_rope_write_kv(q, k, v, kc.transpose(2, 3), kc.clone(), slots, cs, pos)
        with pytest.raises(RuntimeError, match="positions must have 9 entries"):
            pa.qk_norm_rope_write_kv(q, k, v, kc, kc.clone(), slots, cs, pos[:8])

    print("python paths", flush=True)
    want = calls()
    refusals()
    monkeypatch.setattr(ops, "_ops", None)
    monkeypatch.setattr(ops, "_torch_path", lambda: tmp_path / "none.so")
    for x, y in zip(calls(), want):
        assert x.dtype == y.dtype and torch.equal(x, y)
    refusals()


def test_more_heads_than_one_launch(pa, dev):
    """2^21 tokens of 40 heads, taken in two launches: as calls of their parts."""
    T, H, HKV, D, BS = (1 << 21) + 7, 40, 1, 16, 16
    qkv = torch.randn((T, H + 2 * HKV, D), device=dev, dtype=torch.bfloat16)
    q, k, v = qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:]
    w = (torch.randn(D, device=dev) * 0.2 + 1).bfloat16()
    cs = table(500, D, torch.float32).to(dev)
    pos, slots = torch.arange(T, device=dev) % 500, torch.arange(T, device=dev).flip(0)
    new = lambda: [torch.zeros((T // BS + 1, BS, HKV, D), dtype=torch.bfloat16, device=dev) for _ in range(2)]  # noqa: E731
    a, b = new(), new()
    print("two launches", T, flush=True)
    got = pa.qk_norm_rope_write_kv(q, k, v, *a, slots, cs, pos, q_weight=w, k_weight=w)
    for i in range(0, T, 1 << 19):
        s = slice(i, i + (1 << 19))
        part = pa.qk_norm_rope_write_kv(q[s], k[s], v[s], *b, slots[s], cs, pos[s], q_weight=w, k_weight=w)
        assert torch.equal(got[s], part)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[1].flatten(0, 1)[:T].any(-1).any(-1).all()
