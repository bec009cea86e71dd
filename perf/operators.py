"""The measured cases of the operators around a batch that branches from common
prompts: attention whose group of sequences reads a shared prefix once, the
norm and rotation of new queries and keys on their way into the paged cache,
and the forking, compacting and copying of the cache's pages.

With `own` false, run() computes them in plain torch operations (fp32
arithmetic); with `own` true, through the package's entry points.

Ranges.  Heads are GPT-2 style (12 x 64), GQA groups of 4 and 8 at head_dim 128
and 64; pages of 16 tokens mostly, of 8 and 32 now and then.  Shared prefixes of
1 to 16384 tokens (not whole pages in general) under 1 to 128 sequences in 1 to
8 groups, each with up to 1024 tokens of its own and 1 to 64 new query rows;
1 to 8192 new tokens through the norm and rotation; pools of 64 to 2048 pages
and 1 to 12 layers.
"""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}
FP8_SCALE = 1.0 / 16
EPS = 1e-6

MAX_FLOPS = 6.9e10   # the most matrix work of a drawn shared-prefix call (the quantised listed case)
MAX_KEYS = 1.2e9     # the most K elements that a drawn batch's contexts hold together (the 4 x 32 case)
MAX_COPY = 4.0e8     # the most bytes of a drawn pool (the copy of 256 pages)
MAX_ROPE = 8192 * 48 * 128  # the most new elements (the prompts' case)


def listed():
    gpt2 = dict(H=12, HKV=12, D=64, BS=16)
    gqa4 = dict(H=32, HKV=8, D=128, BS=16)
    gqa8 = dict(H=64, HKV=8, D=128, BS=16)
    return [
        # Four samples of one short prompt, a few tokens in: launch latency.
        dict(name="shared_b4_p512", kind="shared", B=4, NG=1, S=1, prefix=512, own=32, kv="f16", q="f32", out="f32",
             **gpt2),
        # A decode batch behind one system prompt, GPT-2 heads.
        dict(name="shared_b64_p2048", kind="shared", B=64, NG=1, S=1, prefix=2048, own=256, kv="f16", q="f16",
             out="f16", **gpt2),
        # Four prompts with 32 samples each, long prefixes, grouped-query heads.
        dict(name="shared_gqa4_4x32_p8192", kind="shared", B=128, NG=4, S=1, prefix=8192, own=1024, kv="bf16",
             q="bf16", out="bf16", **gqa4),
        # Four drafted rows a sequence (verification) behind one long document in a quantised cache.
        dict(name="shared_gqa8_s4_p16384_fp8", kind="shared", B=32, NG=1, S=4, prefix=16384, own=512, kv="fp8",
             q="bf16", out="bf16", **gqa8),
        # One decode step's new queries and keys.
        dict(name="rope_t32", kind="rope", T=32, rot=128, pairs=False, act="bf16", kv="bf16", norm=True, **gqa4),
        # A batch of prompts into a quantised cache.
        dict(name="rope_t8192_fp8", kind="rope", T=8192, rot=128, pairs=False, act="bf16", kv="fp8", norm=True, **gqa4),
        # Eight beams forked from four in one layer's cache: latency.
        dict(name="fork_n8", kind="fork", L=1, NB=128, NP=4, N=8, ctx=250, HKV=12, D=64, BS=16, kv="f16"),
        # 64 samples forked from four prompts, every layer of the pool.
        dict(name="fork_n64_l12", kind="fork", L=12, NB=1024, NP=4, N=64, ctx=2048, HKV=12, D=64, BS=16, kv="f16"),
        # A small cache made dense again.
        dict(name="compact_nb128", kind="compact", L=1, NB=128, R=8, live=0.4, HKV=12, D=64, BS=16, kv="f16"),
        # A pool of every layer with 40 % of its pages in use, made dense.
        dict(name="compact_nb1024_l12", kind="compact", L=12, NB=1024, R=32, live=0.4, HKV=12, D=64, BS=16, kv="f16"),
        # A few pages copied in one layer's cache.
        dict(name="copy_n16", kind="copy", L=1, NB=256, N=16, HKV=8, D=128, BS=16, kv="bf16"),
        # Whole sequences copied in every layer.
        dict(name="copy_n256_l12", kind="copy", L=12, NB=1024, N=256, HKV=8, D=64, BS=16, kv="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["shared"] * 4 + ["rope"] * 3 + ["fork", "fork", "compact", "copy"])
    H, HKV, D = rng.choice([(12, 12, 64), (32, 8, 128), (64, 8, 128), (8, 2, 128), (8, 1, 128), (16, 4, 64),
                            (16, 16, 128)])
    BS = rng.choice([16, 16, 16, 32, 8])
    kv = rng.choice(["f16", "bf16", "bf16", "fp8"])
    act = kv if kv != "fp8" else rng.choice(["f16", "bf16"])
    c = dict(kind=kind, HKV=HKV, D=D, BS=BS, kv=kv)
    if kind == "shared":
        B = _log(rng, 1, 128)
        c.update(H=H, B=B, NG=min(B, rng.choice([1, 1, 2, 4, 8])), S=rng.choice([1, 1, 1, 2, 4, 17, 64]),
                 prefix=_log(rng, 1, 16384), own=_log(rng, 1, 1024), q=act, out=rng.choice([act, "f32"]))
        while _flops(c) > MAX_FLOPS or B * (c["prefix"] + c["own"] + c["S"]) * HKV * D > MAX_KEYS:
            c["B"] = B = max(1, B // 2)
            c["NG"] = min(B, c["NG"])
            c["prefix"] = max(1, c["prefix"] * 2 // 3)
        return c
    if kind == "rope":
        c.update(H=H, T=_log(rng, 1, min(8192, MAX_ROPE // ((H + 2 * HKV) * D))),
                 rot=rng.choice([D, D, D // 2, D // 4]), pairs=rng.random() < 0.4, act=act, norm=rng.random() < 0.7)
        return c
    c.update(L=rng.choice([1, 1, 2, 12]), NB=_log(rng, 64, 2048))
    c["L"] = max(1, min(c["L"], int(MAX_COPY // (2 * c["NB"] * BS * HKV * D * SIZE[kv]))))
    if kind == "fork":
        c.update(NP=rng.choice([1, 2, 4, 7]))
        c["ctx"] = _log(rng, 1, max(1, c["NB"] * BS // (2 * c["NP"])))
        c["N"] = _log(rng, 1, min(96, c["NB"] // 3))
    elif kind == "compact":
        c.update(R=_log(rng, 1, 64), live=round(rng.uniform(0.05, 0.95), 3))
    else:
        c.update(N=_log(rng, 1, c["NB"] // 2))
    return c


# ------------------------------------------------------------------ inputs --

def _lens(c):
    """(group starts, prefix lengths, contexts) of a shared-prefix case: the first prefix and context the
    longest, the others a little shorter (the same for every seed)."""
    r = np.random.default_rng(c["B"] * 131 + c["prefix"])
    B, NG = c["B"], c["NG"]
    starts = [g * B // NG for g in range(NG + 1)]
    prefix = [c["prefix"]] + [int(x) for x in r.integers(max(1, c["prefix"] // 2), c["prefix"] + 1, NG - 1)]
    mine = [c["own"]] + [int(x) for x in r.integers(1, c["own"] + 1, B - 1)]
    group = [g for g in range(NG) for _ in range(starts[g], starts[g + 1])]
    return starts, prefix, [prefix[g] + c["S"] - 1 + m for g, m in zip(group, mine)], group


def _parent_lens(c):
    """Contexts of the parents of a fork: not whole pages where a page holds more than one token."""
    r = np.random.default_rng(c["NP"] * 17 + c["ctx"])
    lens = [c["ctx"]] + [int(x) for x in r.integers(max(1, c["ctx"] // 2), c["ctx"] + 1, c["NP"] - 1)]
    return [n - 1 if n % c["BS"] == 0 and n > 1 else n for n in lens]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 11)
    return g


def _randn(shape, g, dtype, mul=1.0):
    if dtype == "fp8":
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float16) * mul).to(DT["fp8"])
    return torch.randn(shape, generator=g, device="cuda", dtype=DT[dtype])


def _dev(x, dtype=torch.int32):
    return torch.tensor(np.asarray(x), dtype=dtype, device="cuda")


def _pool(c, g):
    return _randn((c["L"], 2, c["NB"], c["BS"], c["HKV"], c["D"]), g, c["kv"], 1 / FP8_SCALE)


def _shared(c, seed, s):
    starts, prefix, ctx, group = _lens(c)
    g, rng, BS = _gen(seed), np.random.default_rng(seed), c["BS"]
    # A group's members hold the same pages up to the last whole page of the prefix, then their own.
    whole = [p // BS for p in prefix]
    pages = [-(-n // BS) for n in ctx]
    nb = sum(whole) + sum(n - whole[k] for n, k in zip(pages, group))
    perm, at = rng.permutation(nb).astype(np.int32), 0
    bt = np.zeros((c["B"], max(pages)), np.int32)
    for k in range(c["NG"]):
        bt[starts[k]:starts[k + 1], :whole[k]] = perm[at:at + whole[k]]
        at += whole[k]
    for b, k in enumerate(group):
        bt[b, whole[k]:pages[b]] = perm[at:at + pages[b] - whole[k]]
        at += pages[b] - whole[k]
    s["k"] = _randn((nb, BS, c["HKV"], c["D"]), g, c["kv"], 1 / FP8_SCALE)
    s["v"] = _randn((nb, BS, c["HKV"], c["D"]), g, c["kv"], 1 / FP8_SCALE)
    shape = (c["B"], c["H"], c["D"]) if c["S"] == 1 else (c["B"], c["S"], c["H"], c["D"])
    s["q"] = _randn(shape, g, c["q"])
    s["bt"], s["ctx"], s["starts"], s["prefix"] = _dev(bt), _dev(ctx), _dev(starts), _dev(prefix)
    s["scale"], s["kvs"] = 1.0 / math.sqrt(c["D"]), FP8_SCALE if c["kv"] == "fp8" else 1.0


def _rope(c, seed, s):
    g, rng = _gen(seed), np.random.default_rng(seed)
    T, H, HKV, D, BS, rot = c["T"], c["H"], c["HKV"], c["D"], c["BS"], c["rot"]
    # The projection's packed output; q, k and v are views of it.
    qkv = _randn((T, H + 2 * HKV, D), g, c["act"])
    s["q"], s["key"], s["value"] = qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:]
    s["qw"] = s["kw"] = None
    if c["norm"]:
        s["qw"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(DT[c["act"]])
        s["kw"] = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(DT[c["act"]])
    limit = 32768
    angle = np.arange(limit)[:, None] * (10000.0 ** (-np.arange(0, rot, 2) / rot))[None, :]
    s["table"] = _dev(np.concatenate([np.cos(angle), np.sin(angle)], 1), torch.float32)
    nb = -(-T // BS) + 3
    s["k"] = _randn((nb, BS, HKV, D), g, c["kv"], 1 / FP8_SCALE)
    s["v"] = _randn((nb, BS, HKV, D), g, c["kv"], 1 / FP8_SCALE)
    perm, t = rng.permutation(nb), np.arange(T)
    slots = perm[t // BS] * BS + t % BS
    if T <= 256:  # a decode step: every token at a position of its own; one in 16 is padding
        pos = rng.integers(0, limit, T)
        slots[15::16] = -1
    else:
        pos = int(rng.integers(0, limit - T)) + t
    s["pos"], s["slots"] = _dev(pos, torch.int64), _dev(slots, torch.int64)
    s["kvs"] = FP8_SCALE if c["kv"] == "fp8" else 1.0


def _fork(c, seed, s):
    g, rng, BS = _gen(seed), np.random.default_rng(seed), c["BS"]
    lens, NP, N = _parent_lens(c), c["NP"], c["N"]
    pages = [-(-n // BS) for n in lens]
    bt = np.full((NP + N, max(pages)), -1, np.int32)
    perm, at, refs = rng.permutation(c["NB"]).astype(np.int32), 0, np.zeros(c["NB"], np.int32)
    for i, n in enumerate(pages):
        bt[i, :n] = perm[at:at + n]
        refs[perm[at:at + n]] = 1
        at += n
    kv = _pool(c, g)
    s["pool"], s["k"], s["v"] = kv, kv[:, 0], kv[:, 1]
    s["bt"], s["ctx"], s["refs"] = _dev(bt), _dev(lens + [0] * N), _dev(refs)
    s["parents"], s["rows"] = _dev([i % NP for i in range(N)]), _dev(NP + rng.permutation(N))


def _compact(c, seed, s):
    g, rng, NB = _gen(seed), np.random.default_rng(seed), c["NB"]
    live = rng.permutation(NB)[:max(1, int(NB * c["live"]))]
    refs = np.zeros(NB, np.int32)
    refs[live] = rng.integers(1, 4, live.size)
    bt = np.full(c["R"] * (-(-live.size // c["R"]) + 2), -1, np.int32)
    bt[:live.size] = live
    kv = _pool(c, g)
    s["pool"], s["k"], s["v"] = kv, kv[:, 0], kv[:, 1]
    s["bt"], s["refs"] = _dev(rng.permutation(bt).reshape(c["R"], -1)), _dev(refs)
    s["bt_out"], s["refs_out"] = torch.empty_like(s["bt"]), torch.empty_like(s["refs"])


def _copy(c, seed, s):
    g, rng = _gen(seed), np.random.default_rng(seed)
    perm = rng.permutation(c["NB"])
    kv = _pool(c, g)
    s["pool"], s["k"], s["v"] = kv, kv[:, 0], kv[:, 1]
    s["src"], s["dst"] = _dev(perm[:c["N"]]), _dev(perm[c["N"]:2 * c["N"]])


_MAKE = {"shared": _shared, "rope": _rope, "fork": _fork, "compact": _compact, "copy": _copy}


def prepare(case, seed):
    s = {"case": case}
    _MAKE[case["kind"]](case, seed, s)
    return s


# ------------------------------------------------------------- plain forms --

def _plain_shared(s):
    c, q, bt, ctx = s["case"], s["q"], s["bt"].long(), s["ctx"].long()
    B, H, HKV, D, S, BS = c["B"], c["H"], c["HKV"], c["D"], c["S"], c["BS"]
    seq = torch.arange(B, device=q.device)
    group = torch.searchsorted(s["starts"], seq.int(), right=True) - 1
    # Token j of sequence b: before the prefix's end in the pages of its group's first sequence.
    tok = torch.arange(bt.shape[1] * BS, device=q.device)
    first = s["starts"].long()[group]
    row = torch.where(tok < s["prefix"].long()[group][:, None], first[:, None], seq[:, None])
    at = bt[row, tok // BS] * BS + tok % BS
    k = s["k"].view(-1, HKV, D)[at].permute(0, 2, 3, 1).float()   # [B, HKV, D, T]
    x = q.view(B, S, HKV, H // HKV, D).permute(0, 2, 1, 3, 4).float().reshape(B, HKV, S * (H // HKV), D)
    w = torch.matmul(x, k.contiguous()) * (s["scale"] * s["kvs"])
    del k
    last = ctx[:, None] - S + torch.arange(S, device=q.device)    # the row's own position
    seen = (tok <= last[:, :, None]).repeat_interleave(H // HKV, 1)[:, None]
    w = w.masked_fill(~seen, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    v = s["v"].view(-1, HKV, D)[at].permute(0, 2, 1, 3).float().contiguous()
    v = v.masked_fill(~(tok < ctx[:, None])[:, None, :, None], 0.0)
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True) * s["kvs"]
    return o.view(B, HKV, S, H // HKV, D).permute(0, 2, 1, 3, 4).reshape(q.shape).to(DT[c["out"]])


def _rotate(x, w, s):
    c = s["case"]
    x, rot = x.float(), c["rot"]
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    t = s["table"][s["pos"]][:, None]
    cos, sin = t[..., :rot // 2], t[..., rot // 2:]
    if c["pairs"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _to_cache(x, s):
    x = x / s["kvs"]
    if s["case"]["kv"] == "fp8":
        return x.clamp(-448.0, 448.0).to(DT["fp8"])
    return x.to(DT[s["case"]["kv"]])


def _plain_rope(s):
    q = _rotate(s["q"], s["qw"], s).to(s["q"].dtype)
    k, v = _to_cache(_rotate(s["key"], s["kw"], s), s), _to_cache(s["value"].float(), s)
    use = s["slots"] >= 0
    at, size = s["slots"][use], s["k"].shape[2:]
    raw = torch.uint8 if s["case"]["kv"] == "fp8" else k.dtype
    s["k"].view(raw).view(-1, *size)[at] = k[use].view(raw)
    s["v"].view(raw).view(-1, *size)[at] = v[use].view(raw)
    return q, s["k"], s["v"]


def _move(s, src, dst):
    raw = s["pool"].view(torch.uint8)
    raw[:, :, dst] = raw[:, :, src]


def _plain_fork(s):
    bt, ctx, refs, BS = s["bt"].long(), s["ctx"].long(), s["refs"].long(), s["case"]["BS"]
    (R, MB), NB, N = bt.shape, refs.numel(), s["rows"].numel()
    rows, parents, page = s["rows"].long(), s["parents"].long(), torch.arange(MB, device=bt.device)
    idx = torch.arange(N, device=bt.device)
    # The rows' old pages are let go.
    held = (page < -(-ctx[rows] // BS)[:, None]) & (bt[rows] >= 0)
    count = torch.cat([refs, refs.new_zeros(1)])
    count.index_add_(0, torch.where(held, bt[rows], NB).flatten(), -held.flatten().long())
    # Whole pages of the parents are shared.
    n, src = ctx[parents], bt[parents]
    share = page < (n // BS)[:, None]
    count.index_add_(0, torch.where(share, src, NB).flatten(), share.flatten().long())
    # The page begun by the parent: taken over where nobody holds it, copied to the lowest free page otherwise.
    part = n % BS != 0
    last = torch.where(part, src.gather(1, (n // BS).clamp(max=MB - 1)[:, None])[:, 0], NB)
    lowest = torch.full((NB + 1,), N, device=bt.device).scatter_reduce(0, last, idx, "amin")
    take = part & (count[last] == 0) & (lowest[last] == idx)
    count.index_add_(0, torch.where(take, last, NB), take.long())
    need = part & ~take
    free = count[:NB] == 0
    order, rank = torch.argsort((~free).int(), stable=True), torch.cumsum(need, 0) - 1
    got = need & (rank < free.sum())
    new = torch.where(got, order[rank.clamp(min=0)], NB)
    count.index_add_(0, new, got.long())
    copies = got.nonzero()[:, 0]
    _move(s, last[copies], new[copies])
    row = torch.where(share, src, -1)
    tail = torch.where(take, last, new)
    row = torch.where((page == (n // BS)[:, None]) & part[:, None], tail[:, None], row)
    s["bt"][rows] = row.int()
    s["ctx"][rows] = n.int()
    s["refs"].copy_(count[:NB])
    return torch.where(got, new, -1).int()


def _plain_compact(s):
    live = s["refs"] > 0
    n = live.sum()
    page = torch.arange(live.numel(), device=live.device)
    src, dst = (live & (page >= n)).nonzero()[:, 0], (~live & (page < n)).nonzero()[:, 0]
    where = torch.where(live, page, -1)
    where[src] = dst
    _move(s, src, dst)
    refs, bt = s["refs"].clone(), s["bt"].long()
    refs[dst] = refs[src]
    refs[src] = 0
    known = bt >= 0
    s["bt_out"].copy_(torch.where(known, where[bt.clamp(min=0)], bt))
    s["refs_out"].copy_(refs)
    return where.int(), n.int().view(1)


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def run(s):
    c = s["case"]
    kind = c["kind"]
    if kind == "shared":
        if own:
            return _package().paged_attention_shared_prefix(s["q"], s["k"], s["v"], s["bt"], s["ctx"], s["starts"],
                                                            s["prefix"], s["scale"], out_dtype=DT[c["out"]],
                                                            k_scale=s["kvs"], v_scale=s["kvs"])
        return _plain_shared(s)
    if kind == "rope":
        if own:
            q = _package().qk_norm_rope_write_kv(s["q"], s["key"], s["value"], s["k"], s["v"], s["slots"], s["table"],
                                                 s["pos"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                                 interleaved=c["pairs"], k_scale=s["kvs"], v_scale=s["kvs"])
            return q, s["k"], s["v"]
        return _plain_rope(s)
    if kind == "fork":
        if own:
            new = _package().fork_sequences(s["k"], s["v"], s["bt"], s["ctx"], s["refs"], s["parents"], s["rows"])
        else:
            new = _plain_fork(s)
        return new, s["bt"], s["ctx"], s["refs"], s["pool"]
    if kind == "compact":
        if own:
            where, n = _package().compact_pages(s["k"], s["v"], s["bt"], s["refs"], tables_out=s["bt_out"],
                                                refs_out=s["refs_out"])
        else:
            where, n = _plain_compact(s)
        return where, n, s["bt_out"], s["refs_out"], s["pool"]
    if own:
        _package().copy_pages(s["k"], s["v"], s["src"], s["dst"])
    else:
        _move(s, s["src"].long(), s["dst"].long())
    return s["pool"]


# ------------------------------------------------------- what it cannot do without --

def _flops(c):
    """Scores and weighted values of the attended keys: 4 D per (row, head, key)."""
    S = c["S"]
    keys = sum(S * n - S * (S - 1) // 2 for n in _lens(c)[2])
    return 4.0 * c["D"] * c["H"] * keys


def work(case):
    c, kind = case, case["kind"]
    kvb = SIZE[c["kv"]]
    if kind == "shared":
        _, prefix, ctx, group = _lens(c)
        mine = sum(n - prefix[g] for n, g in zip(ctx, group))
        kv = 2 * (sum(prefix) + mine) * c["HKV"] * c["D"] * kvb
        return {"bytes": kv + c["B"] * c["S"] * c["H"] * c["D"] * (SIZE[c["q"]] + SIZE[c["out"]]), "flops": _flops(c)}
    if kind == "rope":
        a = SIZE[c["act"]]
        used = c["T"] - (c["T"] // 16 if c["T"] <= 256 else 0)
        each = 2 * c["H"] * a * c["T"] + 2 * c["HKV"] * (a + kvb) * used
        rows = min(c["T"], 32768) * c["rot"] * 4
        return {"bytes": each * c["D"] + rows + 16 * c["T"], "flops": 8.0 * (c["H"] + c["HKV"]) * c["D"] * c["T"]}
    page = 2 * c["L"] * c["BS"] * c["HKV"] * c["D"] * kvb
    if kind == "fork":
        lens = _parent_lens(c)
        of = [lens[i % c["NP"]] for i in range(c["N"])]
        tables = sum(8 * -(-n // c["BS"]) for n in of)
        return {"bytes": 2 * page * sum(n % c["BS"] != 0 for n in of) + tables + 8 * c["NB"], "flops": 0}
    if kind == "compact":
        live = max(1, int(c["NB"] * c["live"]))
        return {"bytes": 2 * page * live * (1 - live / c["NB"]) + 8 * live + 12 * c["NB"], "flops": 0}
    return {"bytes": 2 * page * c["N"] + 8 * c["N"], "flops": 0}


# ---------------------------------------------------------- definitions in 64 bits --

def _exact_shared(s):
    c = s["case"]
    starts, prefix, ctx, group = _lens(c)
    q = s["q"].double().view(c["B"], c["S"], c["H"], c["D"])
    bt, BS, G = s["bt"].long(), c["BS"], c["H"] // c["HKV"]
    out = torch.zeros_like(q)
    for b in range(c["B"]):
        p, n = prefix[group[b]], ctx[b]
        here = torch.arange(n, device=q.device)
        pages = torch.where(here < p, bt[starts[group[b]]][here // BS], bt[b][here // BS])
        k = s["k"][pages, here % BS].double() * s["kvs"]   # [n, HKV, D]
        v = s["v"][pages, here % BS].double() * s["kvs"]
        for r in range(c["S"]):
            m = n - c["S"] + r + 1
            x = q[b, r].view(c["HKV"], G, -1)
            z = torch.matmul(x, k[:m].permute(1, 2, 0).contiguous()) * s["scale"]
            a = torch.softmax(z, -1)
            out[b, r] = torch.matmul(a, v[:m].permute(1, 0, 2).contiguous()).reshape(c["H"], -1)
    return out.view(s["q"].shape)


def _exact_rope(s):
    c, rot = s["case"], s["case"]["rot"]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        t = s["table"].double()[s["pos"]]
        z = torch.complex(t[:, :rot // 2], t[:, rot // 2:])[:, None]
        a = x[..., :rot].unflatten(-1, (rot // 2, 2) if c["pairs"] else (2, rot // 2))
        if not c["pairs"]:
            a = a.transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(a.contiguous()) * z)
        if not c["pairs"]:
            y = y.transpose(-1, -2)
        return torch.cat([y.flatten(-2), x[..., rot:]], -1)

    k, v = s["k"].double().flatten(0, 1), s["v"].double().flatten(0, 1)
    kept = (s["slots"] >= 0).nonzero()[:, 0]
    top = 448.0 if c["kv"] == "fp8" else math.inf
    k[s["slots"][kept]] = (turned(s["key"], s["kw"])[kept] / s["kvs"]).clamp(-top, top)
    v[s["slots"][kept]] = (s["value"].double()[kept] / s["kvs"]).clamp(-top, top)
    return turned(s["q"], s["qw"]), k.view(s["k"].shape), v.view(s["v"].shape)


def _exact_fork(s):
    bt, ctx, refs = (s[n].cpu().numpy().copy() for n in ("bt", "ctx", "refs"))
    rows, parents, BS = s["rows"].tolist(), s["parents"].tolist(), s["case"]["BS"]
    pool, new, was, length = s["pool"].clone(), [], bt.copy(), ctx.copy()
    for r in rows:
        for p in was[r][:-(-length[r] // BS)]:
            refs[p] -= 1
    for p in parents:
        for j in was[p][:length[p] // BS]:
            refs[j] += 1
    taken = set()
    for p in parents:
        end = was[p][length[p] // BS] if length[p] % BS else -1
        take = end >= 0 and refs[end] == 0
        if take:
            taken.add(len(new))
            refs[end] = 1
        new.append(-1)
    for i, (r, p) in enumerate(zip(rows, parents)):
        n, whole = length[p], length[p] // BS
        bt[r] = -1
        bt[r][:whole] = was[p][:whole]
        if n % BS:
            at = was[p][whole]
            if i not in taken:
                to = int(np.flatnonzero(refs == 0)[0])
                refs[to], new[i] = 1, to
                pool.view(torch.uint8)[:, :, to] = pool.view(torch.uint8)[:, :, int(at)]
                at = to
            bt[r][whole] = at
        ctx[r] = n
    return [torch.tensor(x) for x in (np.asarray(new), bt, ctx, refs)] + [pool.double()]


def _exact_compact(s):
    refs, bt = s["refs"].cpu().numpy().copy(), s["bt"].cpu().numpy()
    live = np.flatnonzero(refs > 0)
    where, pool = np.where(refs > 0, np.arange(refs.size), -1), s["pool"].clone()
    holes = [h for h in range(live.size) if where[h] < 0]
    for p, h in zip([x for x in live if x >= live.size], holes):
        where[p], refs[h], refs[p] = h, refs[p], 0
        pool.view(torch.uint8)[:, :, h] = pool.view(torch.uint8)[:, :, int(p)]
    table = np.where(bt >= 0, where[np.maximum(bt, 0)], bt)
    return [torch.tensor(x) for x in (where, np.asarray([live.size]), table, refs)] + [pool.double()]


def _exact_copy(s):
    pool = s["pool"].clone()
    for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
        pool.view(torch.uint8)[:, :, b] = pool.view(torch.uint8)[:, :, a]
    return pool.double()


def exact(case, seed):
    s = {"case": case}
    _MAKE[case["kind"]](case, seed, s)
    return {"shared": _exact_shared, "rope": _exact_rope, "fork": _exact_fork, "compact": _exact_compact,
            "copy": _exact_copy}[case["kind"]](s)
