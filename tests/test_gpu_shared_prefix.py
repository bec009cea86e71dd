"""Attention over shared prefixes against softmax attention in 64 bits.

Tolerances, per element, with w the exact weights, A = sum w |v| and n attended keys:
  * a score's error is at most e_s = scale sum |q||k| ((D + 8) 2^-24 + split), split being
    what a q of another type than the tiles' loses in two 16-bit pieces (2^-22 of
    fp16's, 2^-16 of bf16's), plus 2^-23 of the score for its scaling; a weight's
    relative error is twice that (the sum has it too);
  * exponentials, fp32 sums of n weights and products and the merge of states: (2 n + 64)
    2^-24, relative to A;
  * the weights' rounding: half a step of the tiles' type where out is a 16-bit type,
    the two-piece residue (its square) where it is fp32;
  * the store: half a step of out's type of the value (2^-25 absolute for small fp16)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def case(B, H, HKV, D, BS, starts, prefix, ctx, *, S=1, kv="f16", q="f16", seed=0, dev=None, extra=3, share=True):
    """Inputs on the CPU: pages of a group agree up to the last whole page of its prefix."""
    g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    pages = [-(-max(n, 0) // BS) for n in ctx]
    for gi in range(len(prefix)):  # the first of a group holds the whole prefix, whatever its context
        if starts[gi] < starts[gi + 1]:
            pages[starts[gi]] = max(pages[starts[gi]], -(-max(prefix[gi], 0) // BS))
    MB = max(pages + [1])
    NB = sum(pages) + extra
    perm, at = rng.permutation(NB), 0
    bt = np.full((B, MB), -12345, np.int32)  # entries that nothing may read
    for b in range(B):
        bt[b, :pages[b]] = perm[at:at + pages[b]]
        at += pages[b]
    if share:
        for gi, P in enumerate(prefix):
            for b in range(starts[gi] + 1, starts[gi + 1]):
                bt[b, :min(max(P, 0) // BS, pages[b])] = bt[starts[gi], :min(max(P, 0) // BS, pages[b])]
    mul = 16.0 if kv == "fp8" else 1.0
    k, v = ((torch.randn((NB, BS, HKV, D), generator=g) * mul).to(DT[kv]) for _ in range(2))
    qq = torch.randn((B, S, H, D), generator=g).to(DT[q])
    i = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=qq if S > 1 else qq[:, 0], k=k, v=v, bt=torch.from_numpy(bt), ctx=i(ctx), starts=i(starts),
                prefix=i(prefix), kvs=1 / 16 if kv == "fp8" else 1.0, S=S, tile={"fp8": "bf16" if q == "bf16" else "f16"}.get(kv, kv),
                qt=q)


def exact(c, scale):
    """(out, A, e_s, n) in 64 bits, [B, S, H, D] and [B, S, H]."""
    q = c["q"].double().reshape(c["q"].shape[0], c["S"], *c["q"].shape[-2:])
    B, S, H, D = q.shape
    NB, BS, HKV, _ = c["k"].shape
    G = H // HKV
    out, A = torch.zeros_like(q), torch.zeros_like(q)
    es, count = torch.zeros((B, S, H), dtype=torch.float64), torch.zeros((B, S, H), dtype=torch.float64)
    starts, prefix, bt, maxctx = c["starts"].tolist(), c["prefix"].tolist(), c["bt"].long(), c["bt"].shape[1] * BS
    broken = any(a > b for a, b in zip(starts, starts[1:])) or min(starts) < 0 or max(starts) > B
    for b in range(B):
        n = int(c["ctx"][b])
        gi = next((i for i in range(len(prefix)) if starts[i] <= b < starts[i + 1]), None)
        P = 0 if gi is None else max(prefix[gi], 0)
        if broken or n > maxctx or (P > maxctx and n > 0):
            out[b] = float("nan")
            if not broken and n <= 0:
                out[b] = 0
            continue
        if n <= 0:
            continue
        tok = torch.arange(n)
        row = torch.where(tok < P, starts[gi] if gi is not None else b, b)
        page = bt[row, tok // BS]
        gone = (page < 0) | (page >= NB)
        page = page.clamp(0, NB - 1)
        k = c["k"].double()[page, tok % BS] * c["kvs"]
        v = c["v"].double()[page, tok % BS] * c["kvs"]
        k[gone] = float("nan")
        for s in range(S):
            m = n - S + s + 1
            if m <= 0:
                continue
            for h in range(H):
                kk, vv = k[:m, h // G], v[:m, h // G]
                z = (kk @ q[b, s, h]) * scale
                w = torch.softmax(z, 0)
                live = w.isnan() | (w != 0)
                out[b, s, h], A[b, s, h] = w[live] @ vv[live], w[live] @ vv[live].abs()
                es[b, s, h] = (kk.abs() @ q[b, s, h].abs()).max() * abs(scale)
                count[b, s, h] = m
    return out, A, es, count


def check(pa, dev, c, out="f32", scale=None, wr=None, **kw):
    D = c["q"].shape[-1]
    scale = D**-0.5 if scale is None else scale
    t = {n: c[n].to(dev) for n in ("q", "k", "v", "bt", "ctx", "starts", "prefix")}
    print("shared", tuple(c["q"].shape), tuple(c["k"].shape), c["starts"].tolist()[:9], c["prefix"].tolist()[:8],
          str(c["k"].dtype), c["qt"], out, flush=True)
    got = pa.paged_attention_shared_prefix(t["q"], t["k"], t["v"], t["bt"], t["ctx"], t["starts"], t["prefix"], scale,
                                           out_dtype=DT[out], k_scale=c["kvs"], v_scale=c["kvs"], **kw)
    assert got.shape == c["q"].shape and got.dtype == DT[out]
    want, A, es, n = exact(c, scale)
    got = got.double().cpu().reshape(want.shape)
    split = 0.0 if c["qt"] == c["tile"] else (2.0**-22 if c["tile"] == "f16" else 2.0**-16)
    e = es * ((D + 8) * 2.0**-24 + split + 2.0**-23)
    wr = wr if wr is not None else HALF[c["tile"]] if out != "f32" else HALF[c["tile"]] ** 2
    rel = 2 * e + (2 * n + 64) * 2.0**-24 + wr
    tol = A * rel[..., None]
    tol = tol + HALF[out] * (want.abs() + tol) + (2.0**-25 if out == "f16" else 0)
    ok = ((got - want).abs() <= tol) | (got.isnan() & want.isnan()) | (got == want)
    if not ok.all():
        bad = (~ok).nonzero()
        raise AssertionError(f"{len(bad)} of {ok.numel()} off, first at {bad[0].tolist()}: {got[~ok][:4]} for {want[~ok][:4]}, "
                             f"tolerance {tol[~ok][:4]}; rows {sorted({tuple(x[:2].tolist()) for x in bad})[:8]}")
    return got


RAGGED = dict(starts=[0, 4, 4, 9, 10], prefix=[70, 33, 128, 5],
              ctx=[71, 300, 70, 20, 129, 128, 1, 0, 200, 260, 40, 17])  # (the last two in no group)


@pytest.mark.parametrize("H,HKV,D", [(12, 12, 64), (8, 2, 128), (8, 1, 128), (16, 4, 64), (6, 2, 32), (4, 2, 256),
                                     (40, 2, 64)])
@pytest.mark.parametrize("kv,q,out", [("f16", "f16", "f16"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f32"),
                                      ("bf16", "f32", "f32"), ("fp8", "bf16", "bf16"), ("fp8", "f16", "f32"),
                                      ("fp8", "f32", "f16"), ("bf16", "f16", "f32"), ("f16", "bf16", "f16")])
def test_ragged_groups(pa, dev, H, HKV, D, kv, q, out):
    check(pa, dev, case(12, H, HKV, D, 16, kv=kv, q=q, seed=H + D, **RAGGED), out)


@pytest.mark.parametrize("BS", [1, 5, 8, 16, 32, 48])
def test_page_sizes(pa, dev, BS):
    check(pa, dev, case(12, 8, 2, 64, BS, kv="bf16", q="bf16", seed=BS, **RAGGED), "bf16")
    check(pa, dev, case(12, 8, 2, 128, BS, kv="fp8", q="bf16", seed=BS, S=3, **RAGGED), "f32")


@pytest.mark.parametrize("S", [2, 3, 17, 64])
@pytest.mark.parametrize("H,HKV,D,kv", [(8, 2, 64, "f16"), (4, 4, 128, "bf16"), (8, 1, 128, "fp8")])
def test_several_rows(pa, dev, S, H, HKV, D, kv):
    """Causal rows of a chunk, some of them before the prefix's end or the sequence's start."""
    q = "f16" if kv == "fp8" else kv
    check(pa, dev, case(12, H, HKV, D, 16, kv=kv, q=q, S=S, seed=S, **RAGGED), "f32")


def test_lone_sequences(pa, dev):
    for B, ctx in ((1, [1]), (1, [400]), (3, [5, 0, 77])):
        check(pa, dev, case(B, 12, 12, 64, 16, [0], [], ctx), "f32")
        check(pa, dev, case(B, 12, 12, 64, 16, [0, B], [0], ctx), "f32")
        check(pa, dev, case(B, 12, 12, 64, 16, [0, B], [-4], ctx), "f32")
    check(pa, dev, case(1, 8, 2, 128, 16, [0, 1], [1], [1], kv="bf16", q="bf16"), "bf16")
    check(pa, dev, case(2, 8, 2, 128, 16, [0, 2], [1], [2, 1], kv="bf16", q="bf16"), "bf16")


def test_long_prefixes_over_the_whole_grid(pa, dev):
    """Units cut over many work-groups; several row blocks a group."""
    rng = np.random.default_rng(1)
    B, prefix = 40, [3001, 1500]
    ctx = [prefix[b >= 30] + int(x) for b, x in enumerate(rng.integers(0, 400, B))]
    check(pa, dev, case(B, 16, 4, 64, 16, [0, 30, 40], prefix, ctx, kv="bf16", q="bf16"), "bf16")
    check(pa, dev, case(B, 4, 1, 128, 16, [0, 30, 40], prefix, ctx, kv="f16", q="f16"), "f32")


def test_many_sequences(pa, dev):
    """More sequences and groups than the work-group has threads."""
    rng = np.random.default_rng(2)
    B = 1024
    starts = sorted([0, B] + [int(x) for x in rng.integers(0, B + 1, 300)])
    prefix = [int(x) for x in rng.integers(0, 40, len(starts) - 1)]
    ctx = [int(x) for x in rng.integers(0, 60, B)]
    check(pa, dev, case(B, 2, 1, 32, 16, starts, prefix, ctx, kv="f16", q="f16"), "f16")


def test_as_decode_and_prefill(pa, dev):
    """The same tables without shared prefixes, through the other entry points."""
    c = case(9, 8, 2, 128, 16, [0, 5, 9], [200, 64], [230, 210, 500, 201, 350, 64, 65, 300, 90], kv="bf16", q="bf16")
    t = {n: c[n].to(dev) for n in ("q", "k", "v", "bt", "ctx", "starts", "prefix")}
    print("as decode", flush=True)
    a = (t["q"], t["k"], t["v"], t["bt"].clamp(min=0), t["ctx"])
    # (own pages hold the prefix's last tokens too: copy them from the first of the group)
    for g, (lo, hi) in enumerate(((0, 5), (5, 9))):
        P = int(c["prefix"][g])
        for b in range(lo + 1, hi):
            if P % 16:
                for x in (a[1], a[2]):
                    x[a[3][b, P // 16], :P % 16] = x[a[3][lo, P // 16], :P % 16]
    got = pa.paged_attention_shared_prefix(*a, t["starts"], t["prefix"], 0.1)
    want = pa.paged_attention_v3(*a, 0.1, 0)
    assert (got - want).abs().max() < 2e-5  # (two roundings of about 2^-17 of values below 1)
    q4 = torch.randn((9, 6, 8, 128), device=dev).bfloat16()
    got = pa.paged_attention_shared_prefix(q4, *a[1:], t["starts"], t["prefix"], 0.1)
    want = pa.paged_attention_prefill(q4, *a[1:], 0.1)
    assert (got - want).abs().max() < 4e-5


def test_unreadable_pages(pa, dev):
    """A page outside the cache makes NaN of the rows that attend it, and of no other."""
    for H, S in ((8, 1), (40, 1), (8, 5)):
        c = case(9, H, 2, 64, 16, [0, 5, 9], [100, 64], [130, 101, 40, 300, 120, 64, 65, 90, 200], S=S, kv="f16", q="f16",
                 share=False)
        c["bt"][0, 3] = c["k"].shape[0]      # tokens 48 .. 63 of the first group's prefix
        c["bt"][1, 2] = -1                   # under the prefix in a row that is not the group's first: not read
        c["bt"][3, 17] = 1 << 30             # tokens 272 .. 287 of sequence 3
        c["bt"][8, 5] = -(1 << 31)           # tokens 80 .. 95 of sequence 8
        got = check(pa, dev, c, "f32").reshape(9, S, -1)
        assert got[0].isnan().all() and got[8].isnan().all() and not got[2].isnan().any() and not got[6].isnan().any()


def test_lengths_past_the_table(pa, dev):
    c = case(6, 8, 2, 64, 16, [0, 3, 6], [100, 64], [130, 101, 40, 64, 65, 90])
    top = c["bt"].shape[1] * 16
    for ctx, prefix in (([130, top + 1, 40, 64, 65, 90], [100, 64]), ([130, 101, 40, 2**31 - 1, -5, 90], [100, 64]),
                        ([130, 101, 0, -(2**31), 65, 90], [2**31 - 1, 64]), ([130, 101, 40, 64, 65, 90], [100, top + 1])):
        c["ctx"], c["prefix"] = torch.tensor(ctx, dtype=torch.int32), torch.tensor(prefix, dtype=torch.int32)
        check(pa, dev, c, "f16")


def test_unusable_groups(pa, dev):
    c = case(6, 8, 2, 64, 16, [0, 3, 6], [100, 64], [130, 101, 40, 64, 65, 90])
    for starts in ([0, 4, 3], [-1, 3, 6], [0, 3, 7], [2**31 - 1, 0, 6]):
        c["starts"] = torch.tensor(starts, dtype=torch.int32)
        assert check(pa, dev, c, "f32").isnan().all()


@pytest.mark.parametrize("kv", ["f16", "bf16", "fp8"])
@pytest.mark.parametrize("H,S", [(8, 1), (40, 1), (8, 6)])
def test_non_finite_masked_keys(pa, dev, kv, H, S):
    """Infinities and NaN in keys that a row does not attend leave it as it is: behind the contexts, in
    pages nobody holds, and in keys that other rows of the same tile do attend."""
    q = "f16" if kv == "fp8" else kv
    ctx = [130, 101, 40, 300, 120, 64, 65, 90, 200]
    c = case(9, H, 2, 64, 16, [0, 5, 9], [100, 64], ctx, S=S, kv=kv, q=q, share=False)
    k, v = c["k"].float(), c["v"].float()
    odd = float("nan") if kv == "fp8" else float("inf")
    used = torch.zeros(k.shape[:2], dtype=torch.bool)
    for b, n in enumerate(ctx):
        lo, P = (0, 100) if b < 5 else (5, 64)
        for j in range(max(n, P) if b == lo else n):
            if j < n or j < P:
                used[c["bt"][lo if j < P else b, j // 16], j % 16] = True
    k[~used], v[~used] = float("nan"), odd
    k[c["bt"][0, 5], 10], v[c["bt"][0, 4], 3] = float("nan"), odd     # tokens 90, 67: not in sequence 2
    v[c["bt"][3, 18], 11, 1, 7] = odd                                 # token 299 of sequence 3, its last
    v[c["bt"][3, 18], 10, 0, 3] = float("nan") if kv == "fp8" else -odd
    k8, v8 = c["k"], c["v"]
    c["k"], c["v"] = k.to(k8.dtype), v.to(v8.dtype)
    out = {"f16": "f16", "bf16": "bf16", "fp8": "f16"}[kv]
    got = check(pa, dev, c, out).reshape(9, S, H, 64)
    assert got[2].isfinite().all() and got[5:].isfinite().all()
    assert not got[3, -1, H // 2:, 7].isfinite().any() and not got[0].isfinite().any()


def test_scales(pa, dev):
    c = case(7, 8, 2, 64, 16, [0, 7], [90], [100, 91, 95, 300, 90, 30, 140], kv="f16", q="f32")
    for scale in (-0.125, 0.0, 3.0):
        check(pa, dev, c, "f32", scale=scale)
    c["q"] = c["q"] * 3e4  # past fp16's range
    check(pa, dev, c, "f32", scale=1e-5)


def test_one_layer_of_a_pool_and_far_offsets(pa, dev):
    """A strided layer of a pool, with page offsets past 2^32 bytes."""
    B, H, HKV, D, BS, starts, prefix, ctx = 5, 8, 2, 64, 16, [0, 5], [50], [60, 51, 100, 50, 20]
    c = case(B, H, HKV, D, BS, starts, prefix, ctx, kv="bf16", q="bf16", extra=0)
    NB = c["k"].shape[0]
    pool = torch.empty((2, 40, 2, 1 << 25), dtype=torch.bfloat16, device=dev)  # 64 MB between pages' planes
    k = pool[1].as_strided((NB, BS, HKV, D), (1 << 26, HKV * D, D, 1), pool[1].storage_offset())
    v = pool[1].as_strided((NB, BS, HKV, D), (1 << 26, HKV * D, D, 1), pool[1].storage_offset() + (1 << 25))
    k.copy_(c["k"].to(dev))
    v.copy_(c["v"].to(dev))
    assert (NB - 1) * (1 << 26) * 2 > 1 << 30
    print("far offsets", NB, flush=True)
    a = [c[n].to(dev) for n in ("bt", "ctx", "starts", "prefix")]
    got = pa.paged_attention_shared_prefix(c["q"].to(dev), k, v, *a, 0.125)
    want = pa.paged_attention_shared_prefix(c["q"].to(dev), c["k"].to(dev), c["v"].to(dev), *a, 0.125)
    assert torch.equal(got, want)


def test_streams_and_graphs(pa, dev):
    """Two calls at once on two streams, and a captured call replayed on other inputs: as eager calls."""
    cs = [case(12, 8, 2, 64, 16, kv="bf16", q="bf16", seed=s, **RAGGED) for s in range(2)]
    ts = [{n: c[n].to(dev) for n in ("q", "k", "v", "bt", "ctx", "starts", "prefix")} for c in cs]

    def call(t):
        return pa.paged_attention_shared_prefix(t["q"], t["k"], t["v"], t["bt"], t["ctx"], t["starts"], t["prefix"], 0.125,
                                                out_dtype=torch.bfloat16)

    want = [call(t) for t in ts]
    torch.cuda.synchronize()
    print("streams", flush=True)
    sides = [torch.cuda.Stream() for _ in ts]
    for _ in range(3):
        got = []
        for s, t in zip(sides, ts):
            with torch.cuda.stream(s):
                got.append(call(t))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    hold = {n: x.clone() for n, x in ts[0].items()}
    graph = torch.cuda.CUDAGraph()
    print("capture", flush=True)
    with torch.cuda.graph(graph):
        out = call(hold)
    other = dict(ts[1], starts=torch.tensor([0, 1, 7, 7, 12], dtype=torch.int32, device=dev),
                 ctx=torch.tensor([200, 71, 70, 20, 129, 128, 1, 0, 130, 128, 100, 17], dtype=torch.int32, device=dev),
                 bt=ts[1]["bt"].clamp(min=0))
    for t in (ts[1], ts[0], other, ts[1]):
        shape_ok = {n: x for n, x in t.items() if hold[n].shape == x.shape}
        if len(shape_ok) < len(hold):
            continue
        for n, x in t.items():
            hold[n].copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = call(hold)
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), eager.view(torch.int16))


def test_python_paths_agree(pa, dev, monkeypatch, tmp_path):
    """Without the operator library, on views and int64 metadata, the results are the same."""
    import sys
    ops = sys.modules[pa.paged_attention.__module__]
    c = case(12, 8, 2, 64, 16, kv="bf16", q="bf16", **RAGGED)
    t = [c[n].to(dev) for n in ("q", "k", "v", "bt", "ctx", "starts", "prefix")]
    want = pa.paged_attention_shared_prefix(*t, 0.125)
    wide = t[:3] + [x.long() for x in t[3:]]
    print("python paths", flush=True)
    assert torch.equal(pa.paged_attention_shared_prefix(*wide, 0.125), want)
    off = torch.empty(t[0].numel() + 1, dtype=t[0].dtype, device=dev)[1:].view(t[0].shape).copy_(t[0])
    out = torch.empty_like(want)
    assert pa.paged_attention_shared_prefix(off, *t[1:], 0.125, out=out) is out and torch.equal(out, want)
    monkeypatch.setattr(ops, "_ops", None)
    monkeypatch.setattr(ops, "_torch_path", lambda: tmp_path / "none.so")
    assert torch.equal(pa.paged_attention_shared_prefix(*wide, 0.125), want)
    assert torch.equal(pa.paged_attention_shared_prefix(off, *t[1:], 0.125), want)


def test_numbers_past_32_bits(pa, dev, monkeypatch, tmp_path):
    """int64 group starts and prefixes that do not fit are out of range."""
    import sys
    ops = sys.modules[pa.paged_attention.__module__]
    c = case(4, 8, 2, 64, 16, [0, 4], [32], [40, 41, 50, 33], kv="bf16", q="bf16")
    t = [c[n].to(dev) for n in ("q", "k", "v", "bt", "ctx")]
    for native in (True, False):
        if not native:
            monkeypatch.setattr(ops, "_ops", None)
            monkeypatch.setattr(ops, "_torch_path", lambda: tmp_path / "none.so")
        print("wide numbers", native, flush=True)
        for starts, prefix in (([2**32, 4], [32]), ([0, 2**32 + 4], [32]), ([0, 4], [2**32 + 32])):
            got = pa.paged_attention_shared_prefix(*t, torch.tensor(starts), torch.tensor(prefix), 0.125)
            assert got.isnan().all()


def test_long_table(pa, dev):
    """A table near the longest that a call takes, on few pages."""
    MB = (1 << 27) - 128
    k, v = (torch.randn((3, 16, 1, 32), device=dev).half() for _ in range(2))
    q = torch.randn((1, 1, 32), device=dev).half()
    bt = torch.ones((1, MB), dtype=torch.int32, device=dev)
    print("long table", flush=True)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    short = pa.paged_attention_shared_prefix(q, k, v, bt[:, :1].clone(), i([16]), i([0, 1]), i([0]), 0.1)
    for n, P in ((16, 0), (MB * 16 + 1, 0)):
        got = pa.paged_attention_shared_prefix(q, k, v, bt, i([n]), i([0, 1]), i([P]), 0.1)
        assert got.isnan().all() if n > MB * 16 else torch.equal(got, short)
    # Every page alike: the mean over a page's keys stays.  The first half goes to wide work-groups, the second
    # to thin ones, an equal cost each: a row's state sums at most 61 k keys of 2^25 (946 tiles of 64), one
    # rounding of 2^-24 a key in the products and half as many in the weights' sum, and the merge adds 2600
    # states.  Together below 2^-7.  64 times as many keys: below 1/2.
    for n, tol in ((1 << 25, 2.0**-7), (MB * 16, 0.5)):
        print("tokens", n, flush=True)
        got = pa.paged_attention_shared_prefix(q, k, v, bt[:, :n // 16].clone(), i([n]), i([0, 1]), i([n // 2]), 0.1)
        assert (got - short).abs().max() <= tol * v.float().abs().max()


@pytest.mark.parametrize("H,HKV,D,S,kv", [(8, 2, 128, 1, "bf16"), (8, 2, 64, 6, "bf16"), (8, 1, 256, 1, "bf16"), (8, 2, 128, 1, "fp8")])
def test_single_precision(pa, dev, H, HKV, D, S, kv):
    """fp32 results from bf16 pieces: the weights keep three of them, half a step of 2^-8 each, 2^-24 together."""
    check(pa, dev, case(12, H, HKV, D, 16, kv=kv, q="bf16", S=S, seed=S + D, **RAGGED), "f32", wr=2.0**-24)
