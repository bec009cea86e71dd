"""What the cache operators refuse before any device work (no GPU needed), through the C-ABI."""
import ctypes as C

import pytest

FAKE = 0x7F0000000000
F32, F16, BF16, F64, I32, I64, FP8 = range(7)


def T(pa, shape, dtype, stride=None, data=FAKE):
    if stride is None:
        stride, s = [], 1
        for n in reversed(shape):
            stride.insert(0, s)
            s *= n
    return pa.PaTensor.make(data, dtype, shape, stride)


def refs(tensors):
    return [None if t is None else C.byref(t) for t in tensors]


def expect(pa, rc, code, msg):
    err = pa.lib().pa_last_error().decode()
    assert rc == code and msg in err, (rc, err)


# --------------------------------------------- norm, rotation and the write --

ROPE = ("q_out", "k_cache", "v_cache", "q", "key", "value", "slots", "table", "pos", "qw", "kw")


def rope_args(pa, T_=5, H=4, HKV=2, D=64, NB=10, BS=16, rot=64, act=BF16, kv=F16, wt=BF16):
    t = lambda *s, dt: T(pa, list(s), dt)  # noqa: E731
    return dict(q_out=t(T_, H, D, dt=act), k_cache=t(NB, BS, HKV, D, dt=kv), v_cache=t(NB, BS, HKV, D, dt=kv),
                q=t(T_, H, D, dt=act), key=t(T_, HKV, D, dt=act), value=t(T_, HKV, D, dt=act), slots=t(T_, dt=I64),
                table=t(100, rot, dt=F32), pos=t(T_, dt=I32), qw=t(D, dt=wt), kw=t(D, dt=wt))


def rope_call(pa, a, eps=1e-6, ks=1.0, vs=1.0):
    return pa.lib().pa_qk_norm_rope_write_kv(*refs(a[n] for n in ROPE), eps, 0, ks, vs, None)


@pytest.mark.parametrize("sizes,change,code,msg", [
    (dict(act=F64), {}, 1, "q must be float32, float16 or bfloat16"),
    ({}, dict(key=([5, 2, 64], F16)), 1, "key and value must have the dtype of q"),
    ({}, dict(value=([5, 3, 64], BF16)), 1, "key and value must be [5, 2, 64]"),
    ({}, dict(key=([4, 2, 64], BF16)), 1, "key and value must be [5, 2, 64]"),
    ({}, dict(q_out=([5, 4, 32], BF16)), 1, "q_out must have the shape of q"),
    ({}, dict(q_out=([5, 4, 64], FP8)), 1, "q_out must be float32, float16 or bfloat16"),
    (dict(kv=F64), {}, 1, "k_cache must be float16, bfloat16, float32 or float8_e4m3fn"),
    ({}, dict(v_cache=([10, 16, 2, 64], BF16)), 1, "v_cache must have the dtype of k_cache"),
    ({}, dict(v_cache=([10, 8, 2, 64], F16)), 1, "v_cache must have the shape of k_cache"),
    ({}, dict(k_cache=([10, 16, 2, 32], F16), v_cache=([10, 16, 2, 32], F16)), 1, "head_dim (32) != q head_dim (64)"),
    (dict(D=72, rot=64), {}, 2, "head_dim must be a multiple of 16 up to 256"),
    (dict(D=272, rot=64), {}, 2, "head_dim must be a multiple of 16 up to 256"),
    (dict(rot=80), {}, 1, "more columns than head_dim"),
    (dict(rot=24), {}, 2, "multiple of 16 columns"),
    ({}, dict(table=([100, 64], F64)), 1, "cos_sin must be float32, float16 or bfloat16"),
    ({}, dict(slots=([4], I64)), 1, "slot_mapping must have 5 entries"),
    ({}, dict(slots=([5], F32)), 1, "slot_mapping must be int32 or int64"),
    ({}, dict(pos=([6], I32)), 1, "positions must have 5 entries"),
    ({}, dict(pos=([5], I32, [2])), 1, "positions must be contiguous"),
    ({}, dict(qw=([32], BF16)), 1, "must have head_dim entries"),
    ({}, dict(kw=([64], F32)), 1, "must share a type"),
    ({}, dict(q=([5, 4, 64], BF16, [256, 64, 2])), 1, "q must have a contiguous last dimension"),
    ({}, dict(q=([5, 4, 64], BF16, [260, 64, 1])), 2, "q strides must be multiples of 16 bytes"),
    ({}, dict(key=([5, 2, 64], BF16, None, FAKE + 8)), 2, "key must be 16-byte aligned"),
    ({}, dict(v_cache=([10, 16, 2, 64], F16, [-2048, 128, 64, 1])), 2, "v_cache strides must be non-negative"),
    (dict(NB=1 << 27), {}, 2, "too large for 32-bit slot indices"),
])
def test_rope_refusals(pa, sizes, change, code, msg):
    a = rope_args(pa, **sizes)
    for n, s in change.items():
        a[n] = T(pa, *s[:2], *s[2:])
    expect(pa, rope_call(pa, a), code, msg)


def test_rope_scalar_refusals(pa):
    a = rope_args(pa)
    for eps in (-1e-6, float("nan"), float("inf"), 1e39):
        expect(pa, rope_call(pa, a, eps=eps), 1, "eps must be finite")
    for s in (0.0, float("nan"), 1e39, 1e-60):
        expect(pa, rope_call(pa, a, ks=s), 1, "finite and nonzero")
        expect(pa, rope_call(pa, a, vs=s), 1, "finite and nonzero")
    for n in ("q", "q_out", "key", "value", "slots", "table", "pos", "k_cache", "v_cache"):
        expect(pa, rope_call(pa, {**a, n: None}), 1, "is NULL")
    assert rope_call(pa, rope_args(pa, T_=0)) == 0


# -------------------------------------------------------------------- pages --

def page_args(pa, L=2, NB=10, BS=16, W=128, dt=F16, R=4, MB=6, N=3):
    t = lambda *s, d=I32: T(pa, list(s), d)  # noqa: E731
    return dict(k=t(L, NB, BS, W, d=dt), v=t(L, NB, BS, W, d=dt), bt=t(R, MB), lens=t(R), refs=t(NB), parents=t(N),
                rows=t(N), out=t(N), src=t(N), dst=t(N), bt_out=T(pa, [R, MB], I32, data=FAKE + (1 << 20)),
                refs_out=T(pa, [NB], I32, data=FAKE + (2 << 20)), map=t(NB), n=t(1))


def copy_call(pa, a):
    return pa.lib().pa_copy_pages(*refs((a["k"], a["v"], a["src"], a["dst"])), None)


def fork_call(pa, a, ws=FAKE, size=1 << 20):
    return pa.lib().pa_fork_sequences(*refs(a[n] for n in ("k", "v", "bt", "lens", "refs", "parents", "rows", "out")),
                                      ws, size, None)


def free_call(pa, a, bs=16):
    return pa.lib().pa_free_sequences(*refs(a[n] for n in ("bt", "lens", "refs", "rows")), bs, None)


def compact_call(pa, a, ws=FAKE, size=1 << 20):
    return pa.lib().pa_compact_pages(*refs(a[n] for n in ("k", "v", "bt", "refs", "bt_out", "refs_out", "map", "n")),
                                     ws, size, None)


POOL = [
    (dict(k=([2, 10, 16], F16)), 1, "k_cache must be [L, NB, BS, row]"),
    (dict(k=([2, 10, 16, 128], 9), v=None), 1, "k_cache has an unknown type"),
    (dict(v=([2, 10, 16, 128], BF16)), 1, "v_cache must have the dtype of k_cache"),
    (dict(v=([2, 9, 16, 128], F16)), 1, "v_cache must have the shape of k_cache"),
    (dict(k=([2, 10, 0, 128], F16), v=None), 1, "block_size must be positive"),
    (dict(k=([2, 10, 16, 4], F16), v=None), 2, "multiple of 16 bytes"),
    (dict(k=([2, 10, 16, 128], F16, [20480, 2048, 256, 2]), v=None), 1, "contiguous last dimension"),
    (dict(k=([2, 10, 16, 128], F16, [20480, 2052, 128, 1]), v=None), 2, "strides must be multiples of 16 bytes"),
    (dict(k=([2, 10, 16, 128], F16, [20480, 0, 128, 1]), v=None), 1, "pages must not overlap"),
    (dict(k=([2, 10, 16, 128], F16, None, FAKE + 4), v=None), 2, "16-byte aligned"),
    (dict(k=([1, 10, 1 << 26, 1024], F16), v=None), 2, "too large"),
]


@pytest.mark.parametrize("change,code,msg", POOL)
@pytest.mark.parametrize("call", [copy_call, fork_call, compact_call])
def test_pool_refusals(pa, call, change, code, msg):
    a = page_args(pa)
    for n, s in change.items():
        a[n] = None if s is None else T(pa, *s)
    expect(pa, call(pa, a), code, msg)


@pytest.mark.parametrize("calls,change,code,msg", [
    ([copy_call], dict(src=([3], I64)), 1, "src must be int32"),
    ([copy_call], dict(dst=([2], I32)), 1, "dst must have 3 entries"),
    ([fork_call, free_call], dict(bt=([4, 6], I64)), 1, "block_tables must be int32"),
    ([fork_call, free_call, compact_call], dict(bt=([4, 6], I32, [5, 1])), 1, "block_tables rows must be contiguous"),
    ([fork_call, free_call, compact_call], dict(bt=([4, 6], I32, [12, 2])), 1, "block_tables rows must be contiguous"),
    ([fork_call, free_call], dict(lens=([5], I32)), 1, "context_lens must have 4 entries"),
    ([fork_call, free_call], dict(rows=([3], I64)), 1, "rows must be int32"),
    ([fork_call, free_call], dict(rows=([65537], I32)), 2, "at most 65536 rows"),
    ([fork_call, free_call], dict(bt=([4, 1 << 28], I32)), 2, "too large for 32-bit token indices"),
    ([fork_call], dict(refs=([9], I32)), 1, "page_refs must have one entry per page"),
    ([fork_call], dict(parents=([2], I32)), 1, "parents must have 3 entries"),
    ([fork_call], dict(out=([2], I32)), 1, "copied must have 3 entries"),
    ([compact_call], dict(refs=([9], I32)), 1, "page_refs must have 10 entries"),
    ([compact_call], dict(refs_out=([9], I32)), 1, "refs_out must have 10 entries"),
    ([compact_call], dict(map=([9], I32)), 1, "page_map must have 10 entries"),
    ([compact_call], dict(n=([2], I32)), 1, "num_live must have 1 entries"),
    ([compact_call], dict(bt_out=([4, 5], I32)), 1, "tables_out must have the shape of block_tables"),
    ([compact_call], dict(bt_out=([4, 6], I32, None, FAKE + 4)), 1, "tables_out must be block_tables or not overlap"),
    ([compact_call], dict(bt_out=([4, 6], I32, [8, 1], FAKE)), 1, "tables_out must be block_tables or not overlap"),
    ([compact_call], dict(refs_out=([10], I32, None, FAKE + 36)), 1, "refs_out must be page_refs or not overlap"),
])
def test_page_refusals(pa, calls, change, code, msg):
    a = page_args(pa)
    for n, s in change.items():
        a[n] = T(pa, *s)
    for call in calls:
        expect(pa, call(pa, a), code, msg)


def test_page_workspaces(pa):
    L, a = pa.lib(), page_args(pa)
    need = L.pa_fork_workspace_size(*refs((a["bt"], a["refs"], a["rows"])))
    assert need == 4 * (3 * 6 + 3 * 3 + 10)
    assert L.pa_compact_workspace_size(*refs((a["refs"],))) == 4 * (1 + 20 + 1)
    assert L.pa_compact_workspace_size(None) == C.c_size_t(-1).value
    for call in (fork_call, compact_call):
        expect(pa, call(pa, a, size=need - 1 if call is fork_call else 80), 3, "workspace too small")
        expect(pa, call(pa, a, ws=None), 3, "workspace too small")
        expect(pa, call(pa, a, ws=FAKE + 16), 3, "workspace must be 256-byte aligned")
    expect(pa, free_call(pa, a, bs=0), 1, "block_size must be positive")


def test_nothing_to_do(pa):
    a = page_args(pa, N=0)
    assert copy_call(pa, a) == 0 and fork_call(pa, a, ws=None, size=0) == 0 and free_call(pa, a) == 0


# ---------------------------------------------------------- shared prefixes --

SHARED = ("out", "q", "k", "v", "bt", "ctx", "starts", "prefix")


def shared_args(pa, B=4, S=None, H=8, HKV=2, D=64, NB=20, BS=16, MB=6, NG=2, kv=F16, qd=F16, od=F32):
    t = lambda *s, d=I32: T(pa, list(s), d)  # noqa: E731
    rows = (B, H, D) if S is None else (B, S, H, D)
    return dict(out=t(*rows, d=od), q=t(*rows, d=qd), k=t(NB, BS, HKV, D, d=kv), v=t(NB, BS, HKV, D, d=kv),
                bt=t(B, MB), ctx=t(B), starts=t(NG + 1), prefix=t(NG))


def shared_call(pa, a, scale=0.1, ks=1.0, vs=1.0, ws=FAKE, size=1 << 40):
    return pa.lib().paged_attention_shared_prefix(*refs(a[n] for n in SHARED), scale, ks, vs, ws, size, None)


@pytest.mark.parametrize("sizes,change,code,msg", [
    ({}, dict(q=([4, 64], F16)), 1, "q must be [B, H, D] or [B, S, H, D]"),
    ({}, dict(out=([4, 1, 8, 64], F32)), 1, "out must be [B, H, D]"),
    (dict(S=3), dict(out=([4, 2, 8, 64], F32)), 1, "out must have the shape of q"),
    (dict(kv=F32), {}, 1, "need an fp16, bf16 or float8_e4m3fn KV cache"),
    (dict(kv=F64), {}, 1, "need an fp16, bf16 or float8_e4m3fn KV cache"),
    (dict(qd=FP8), {}, 1, "q must be float32, float16 or bfloat16"),
    (dict(od=FP8), {}, 1, "out must be float32, float16 or bfloat16"),
    (dict(H=9), {}, 1, "n_head must be divisible by n_kv_head"),
    (dict(D=96), {}, 2, "unsupported head_dim 96"),
    (dict(B=1025), {}, 2, "at most 1024 sequences"),
    (dict(NG=513), {}, 2, "at most 1024 sequences and 512 groups"),
    ({}, dict(starts=([3], I64)), 1, "group_starts must be int32"),
    ({}, dict(starts=([0], I32), prefix=([0], I32)), 1, "group_starts must have at least one entry"),
    ({}, dict(prefix=([3], I32)), 1, "prefix_lens must have 2 entries"),
    ({}, dict(starts=([3], I32, [2])), 1, "group_starts must be contiguous"),
    ({}, dict(bt=([3, 6], I32)), 1, "block_tables must have B rows"),
    ({}, dict(ctx=([5], I32)), 1, "context_lens must have B entries"),
    ({}, dict(q=([4, 8, 64], F16, [1024, 64, 1])), 1, "q must be contiguous"),
    ({}, dict(q=([4, 8, 64], F16, None, FAKE + 2)), 2, "16-byte aligned q"),
    ({}, dict(k=([20, 16, 2, 64], F16, [2052, 128, 64, 1])), 2, "multiples of 16 bytes"),
])
def test_shared_prefix_refusals(pa, sizes, change, code, msg):
    a = shared_args(pa, **sizes)
    for n, s in change.items():
        a[n] = T(pa, *s)
    expect(pa, shared_call(pa, a), code, msg)


def test_shared_prefix_scalars_and_null(pa):
    a = shared_args(pa)
    for bad in (float("nan"), float("inf"), 1e39):
        expect(pa, shared_call(pa, a, ks=bad), 1, "must be finite")
        expect(pa, shared_call(pa, a, vs=bad), 1, "must be finite")
        expect(pa, shared_call(pa, a, scale=bad), 1, "must be finite")
    expect(pa, shared_call(pa, a, scale=1e30, ks=1e10), 1, "scale * k_scale must be finite")
    for n in SHARED:
        rc = shared_call(pa, {**a, n: None})
        assert rc == 1, (n, rc)
    assert shared_call(pa, shared_args(pa, B=0), ws=None, size=0) == 0
    assert shared_call(pa, shared_args(pa, S=0), ws=None, size=0) == 0
    size = pa.lib().paged_attention_shared_prefix_workspace_size
    for sizes in (dict(B=1025), dict(NG=513), dict(H=9), dict(D=512)):
        b = shared_args(pa, **sizes)
        assert size(*refs(b[n] for n in ("q", "k", "bt", "starts"))) == C.c_size_t(-1).value


# ------------------------------------------------------------ limits and overlaps --

@pytest.mark.parametrize("change,msg", [
    (dict(q_out=([5, 4, 64], BF16, [0, 64, 1])), "q_out's rows must not overlap"),
    (dict(q_out=([5, 4, 64], BF16, [256, 0, 1])), "q_out's rows must not overlap"),
    (dict(k_cache=([10, 16, 2, 64], F16, [0, 128, 64, 1])), "k_cache/v_cache rows must not overlap"),
    (dict(v_cache=([10, 16, 2, 64], F16, [2048, 128, 0, 1])), "k_cache/v_cache rows must not overlap"),
])
def test_rope_outputs_that_overlap(pa, change, msg):
    a = rope_args(pa)
    for n, s in change.items():
        a[n] = T(pa, *s)
    expect(pa, rope_call(pa, a), 1, msg)


def test_limits_of_one_call(pa):
    a = page_args(pa, N=65537)
    expect(pa, copy_call(pa, a), 2, "at most 65536 pages")
    # A table that reaches the last 32-bit token: a unit's last tile would pass it.
    for MB in ((1 << 27) - 1, (1 << 27) - 64):
        b = shared_args(pa, B=1, H=1, HKV=1, NG=1, MB=MB)
        expect(pa, shared_call(pa, b), 2, "block tables too long for 32-bit token indices")
        size = pa.lib().paged_attention_shared_prefix_workspace_size(*refs(b[n] for n in ("q", "k", "bt", "starts")))
        assert size == C.c_size_t(-1).value
