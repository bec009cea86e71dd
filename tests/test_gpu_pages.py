"""Pages of the cache copied, forked, freed and compacted, against the same steps
taken one at a time on the host.  Everything here is exact: bytes and whole numbers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64,
      "fp8": torch.float8_e4m3fn}


def pool(L, NB, BS, HKV, D, kv, dev, seed=0):
    """[L, 2, NB, BS, HKV, D] of random bytes (NaN and infinities among them)."""
    g = torch.Generator().manual_seed(seed)
    n = L * 2 * NB * BS * HKV * D * DT[kv].itemsize
    return torch.randint(0, 256, (n,), generator=g, dtype=torch.uint8).to(dev).view(DT[kv]).view(L, 2, NB, BS, HKV, D)


def raw(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


# ----------------------------------------------------------------- by hand --

def fork_by_hand(bytes_, bt, ctx, refs, parents, rows, BS):
    """The documented steps, entry by entry.  bytes_ [L, 2, NB, ...]."""
    (R, MB), NB, N = bt.shape, refs.size, len(rows)
    was, length = bt.copy(), ctx.copy()

    def pages(n):
        return -(-n // BS) if 0 < n <= MB * BS else 0

    copied, kind = np.full(N, -1, np.int32), [None] * N
    for i, r in enumerate(rows):
        if not 0 <= r < R or r in list(rows[:i]):
            copied[i], kind[i] = -3, "skip"
            continue
        for p in was[r][:pages(length[r])]:
            if 0 <= p < NB:
                refs[p] -= 1
        par = -1 if parents is None else parents[i]
        kind[i] = "empty"
        if par >= R:
            copied[i] = -3
        elif par >= 0 and length[par] > 0:
            n = pages(length[par])
            if n == 0 or any(not 0 <= p < NB for p in was[par][:n]):
                copied[i] = -3
            else:
                kind[i] = "fork"
    for i in range(N):
        if kind[i] == "fork":
            for p in was[parents[i]][:length[parents[i]] // BS]:
                refs[p] += 1
    begun = {}
    for i in range(N):
        if kind[i] == "fork" and length[parents[i]] % BS:
            begun[i] = was[parents[i]][length[parents[i]] // BS]
    taken = set()
    for i, p in begun.items():
        if refs[p] == 0 and p not in [begun[j] for j in taken]:
            taken.add(i)
    for i in taken:
        refs[begun[i]] = 1
    undo = []
    free = [p for p in range(NB) if refs[p] == 0]
    for i in range(N):
        if kind[i] == "skip":
            continue
        r = rows[i]
        bt[r], ctx[r] = -1, 0
        if kind[i] != "fork":
            continue
        n = length[parents[i]]
        row = [int(p) for p in was[parents[i]][:n // BS]]
        if i in begun:
            if i in taken:
                row.append(begun[i])
            elif free:
                to = free.pop(0)
                bytes_[:, :, to] = bytes_[:, :, begun[i]]
                refs[to], copied[i] = 1, to
                row.append(to)
            else:
                copied[i] = -2
                undo += row
                continue
        bt[r][:len(row)], ctx[r] = row, n
    for p in undo:
        refs[p] -= 1
    return copied


def compact_by_hand(bytes_, bt, refs):
    live = [p for p in range(refs.size) if refs[p] > 0]
    n = len(live)
    where = np.array([p if refs[p] > 0 else -1 for p in range(refs.size)], np.int32)
    for p, h in zip([p for p in live if p >= n], [h for h in range(n) if refs[h] <= 0]):
        where[p], refs[h], refs[p] = h, refs[p], 0
        bytes_[:, :, h] = bytes_[:, :, p]
    for e in np.ndindex(bt.shape):
        if 0 <= bt[e] < refs.size:
            bt[e] = where[bt[e]]
    return where, n


# ------------------------------------------------------------------- state --

def state(R, MB, NB, BS, lens, rng, share=0):
    """Tables of contexts `lens` on distinct pages; the first `share` pages of every row are row 0's."""
    bt, refs = np.full((R, MB), -1, np.int32), np.zeros(NB, np.int32)
    perm, at = rng.permutation(NB), 0
    for r, n in enumerate(lens):
        k = -(-n // BS)
        own = k if r == 0 else max(0, k - share)
        bt[r, :k] = np.concatenate([bt[0, :k - own], perm[at:at + own]])
        at += own
        np.add.at(refs, bt[r, :k], 1)
    return bt, np.asarray(list(lens) + [0] * (R - len(lens)), np.int32), refs


def run_fork(pa, dev, kv, c, bt, ctx, refs, parents, rows):
    L, NB, BS, HKV, D = c
    data = pool(L, NB, BS, HKV, D, kv, dev)
    t = [torch.from_numpy(x.copy()).to(dev) for x in (bt, ctx, refs)]
    print("fork", kv, c, len(rows), flush=True)
    got = pa.fork_sequences(data[:, 0], data[:, 1], *t, torch.tensor(parents), torch.tensor(rows))
    bytes_ = raw(pool(L, NB, BS, HKV, D, kv, dev))
    want = fork_by_hand(bytes_, bt, ctx, refs, parents, rows, BS)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    for x, y in zip(t, (bt, ctx, refs)):
        np.testing.assert_array_equal(x.cpu().numpy(), y)
    np.testing.assert_array_equal(raw(data), bytes_)
    return want


@pytest.mark.parametrize("kv,c", [("f16", (1, 128, 16, 12, 64)), ("bf16", (3, 96, 16, 2, 128)),
                                  ("fp8", (2, 300, 8, 1, 32)), ("f32", (1, 64, 1, 2, 64)), ("f64", (1, 64, 5, 1, 32)),
                                  ("f16", (1, 9000, 16, 1, 32))])
def test_fork_samples(pa, dev, kv, c):
    """New rows forked from a few parents: whole pages shared, begun ones copied to the lowest free pages."""
    rng = np.random.default_rng(1)
    BS = c[2]
    lens = [3 * BS + BS // 2 + 1, 2 * BS, 1, 0, 5 * BS - 1]
    bt, ctx, refs = state(20, 8, c[1], BS, lens, rng, share=2)
    N = 13
    want = run_fork(pa, dev, kv, c, bt, ctx, refs, [i % 5 for i in range(N)], [5 + int(x) for x in rng.permutation(N)])
    assert (want >= 0).sum() > 0 or BS == 1


@pytest.mark.parametrize("seed", range(6))
def test_fork_beams_in_place(pa, dev, seed):
    """Rows that are parents and replaced in the same call, emptied rows, refused entries."""
    rng = np.random.default_rng(seed)
    R, MB, NB, BS = 12, 6, 90, 4
    lens = [int(x) for x in rng.integers(0, MB * BS + 1, R)]
    bt, ctx, refs = state(R, MB, NB, BS, lens, rng, share=seed % 3)
    for _ in range(3):  # (later steps start from shared rows)
        N = int(rng.integers(1, R + 1))
        rows = [int(x) for x in rng.permutation(R)[:N]]
        parents = [int(x) for x in rng.integers(-1, R, N)]
        if seed == 4:
            rows += [rows[0], -1, R]
            parents += [0, 0, 0]
        if seed == 5:
            parents[0] = R
            ctx[int(rng.integers(0, R))] = MB * BS + 1
            bt[int(rng.integers(0, R)), 0] = NB
        run_fork(pa, dev, "f16", (2, NB, BS, 1, 32), bt, ctx, refs, parents, rows)
        assert (refs >= 0).all() or seed == 5


def test_fork_without_pages(pa, dev):
    """More begun pages than free ones: the first entries get them, the others end empty with nothing held."""
    rng = np.random.default_rng(3)
    bt, ctx, refs = state(10, 4, 7, 16, [50, 20], rng)  # 4 + 2 pages of 7
    want = run_fork(pa, dev, "bf16", (1, 7, 16, 2, 64), bt, ctx, refs, [0, 1, 0, 1], [2, 3, 4, 5])
    assert want[0] >= 0 and (want[1:] == -2).all()
    assert refs.max() == 2 and (ctx[3:] == 0).all()


def test_fork_many_entries(pa, dev):
    """More entries than the allocating work-group has threads."""
    rng = np.random.default_rng(5)
    N = 1500
    bt, ctx, refs = state(N + 3, 3, 4000, 2, [5, 3, 6], rng)
    run_fork(pa, dev, "fp8", (1, 4000, 2, 1, 32), bt, ctx, refs, [i % 3 for i in range(N)], list(range(3, N + 3)))


def test_free(pa, dev):
    rng = np.random.default_rng(2)
    bt, ctx, refs = state(8, 6, 64, 16, [90, 33, 16, 0, 96], rng, share=1)
    before = refs.copy()
    t = [torch.from_numpy(x.copy()).to(dev) for x in (bt, ctx, refs)]
    rows = [0, 4, 0, -1, 8, 3]
    print("free", flush=True)
    pa.free_sequences(*t, torch.tensor(rows), 16)
    fork_by_hand(np.zeros((1, 2, 64, 1), np.uint8), bt, ctx, refs, None, rows, 16)
    for x, y in zip(t, (bt, ctx, refs)):
        np.testing.assert_array_equal(x.cpu().numpy(), y)
    assert refs.sum() < before.sum() and refs[bt[1, 0]] == 2


@pytest.mark.parametrize("NB,live", [(1, 1.0), (3, 0.0), (64, 0.4), (64, 1.0), (2047, 0.5), (2048, 0.9), (2049, 0.05),
                                     (8192, 0.4), (8193, 0.6), (9000, 0.3), (20000, 0.5), (4096, 0.5), (8192, 1.0),
                                     (8192, 0.0), (10240, 1.0)])
def test_compact(pa, dev, NB, live):
    rng = np.random.default_rng(NB)
    L, BS, HKV, D = 2, 4, 1, 32
    refs = np.where(rng.random(NB) < live, rng.integers(1, 5, NB), 0).astype(np.int32)
    bt = rng.integers(-1, NB + 1, (5, 77)).astype(np.int32)  # shared, free and outside pages among them
    data = pool(L, NB, BS, HKV, D, "bf16", dev)
    tb, tr = torch.from_numpy(bt.copy()).to(dev), torch.from_numpy(refs.copy()).to(dev)
    out, ro = torch.zeros_like(tb), torch.zeros_like(tr)
    print("compact", NB, live, flush=True)
    where, n = pa.compact_pages(data[:, 0], data[:, 1], tb, tr, tables_out=out, refs_out=ro)
    np.testing.assert_array_equal(tb.cpu().numpy(), bt)  # the inputs are left as they were
    np.testing.assert_array_equal(tr.cpu().numpy(), refs)
    bytes_ = raw(pool(L, NB, BS, HKV, D, "bf16", dev))
    w, m = compact_by_hand(bytes_, bt, refs)
    np.testing.assert_array_equal(where.cpu().numpy(), w)
    assert int(n) == m
    for x, y in ((out, bt), (ro, refs)):
        np.testing.assert_array_equal(x.cpu().numpy(), y)
    np.testing.assert_array_equal(raw(data), bytes_)
    # In place, from the state as it was: the same; and once dense, nothing moves.
    data = pool(L, NB, BS, HKV, D, "bf16", dev)
    pa.compact_pages(data[:, 0], data[:, 1], tb, tr)
    for x, y in ((tb, bt), (tr, refs)):
        np.testing.assert_array_equal(x.cpu().numpy(), y)
    np.testing.assert_array_equal(raw(data), bytes_)
    where, n = pa.compact_pages(data[:, 0], data[:, 1], tb, tr)
    assert int(n) == m and torch.equal(where[:m].cpu(), torch.arange(m, dtype=torch.int32))
    np.testing.assert_array_equal(raw(data), bytes_)


@pytest.mark.parametrize("kv,layers", [("f16", True), ("fp8", True), ("bf16", False), ("f32", True)])
def test_copy(pa, dev, kv, layers):
    rng = np.random.default_rng(4)
    L, NB, BS, HKV, D = 3, 50, 16, 3, 64
    data = pool(L, NB, BS, HKV, D, kv, dev)
    perm = [int(x) for x in rng.permutation(NB)]
    src = perm[:12] + [-1, NB, 3, perm[0], perm[1], perm[30]]
    dst = perm[20:32] + [perm[40], perm[41], -7, perm[21], NB + 5, perm[30]]  # perm[21] twice: the last pair
    a = (data[:, 0], data[:, 1]) if layers else (data[1, 0], data[1, 1])
    print("copy", kv, layers, flush=True)
    pa.copy_pages(*a, torch.tensor(src), torch.tensor(dst))
    bytes_ = raw(pool(L, NB, BS, HKV, D, kv, dev))
    old = bytes_.copy()
    at = slice(None) if layers else slice(1, 2)
    for s, d in zip(src, dst):
        if 0 <= s < NB and 0 <= d < NB:
            bytes_[at, :, d] = old[at, :, s]
    np.testing.assert_array_equal(raw(data), bytes_)


def test_copy_one_cache_and_strides(pa, dev):
    """One cache alone, of padded token rows and a page stride of its own."""
    big = pool(1, 20, 32, 4, 64, "f16", dev)[0, 0]  # [20, 32, 4, 64]
    view = big[:, :16, :3]
    before = big.clone()
    print("copy strided", flush=True)
    pa.copy_pages(view, None, torch.tensor([1, 2], device=dev), torch.tensor([18, 19], device=dev))
    want = before.clone()
    want[18:20, :16, :3] = before[1:3, :16, :3]
    np.testing.assert_array_equal(raw(big), raw(want))


def test_empty_calls(pa, dev):
    data = pool(1, 8, 4, 1, 32, "f16", dev)
    none = torch.empty(0, dtype=torch.int32, device=dev)
    bt, ctx, refs = (torch.zeros(s, dtype=torch.int32, device=dev) for s in ((2, 2), (2,), (8,)))
    print("empty", flush=True)
    pa.copy_pages(data[:, 0], data[:, 1], none, none)
    assert pa.fork_sequences(data[:, 0], data[:, 1], bt, ctx, refs, none, none).numel() == 0
    pa.free_sequences(bt, ctx, refs, none, 4)
    tables = torch.empty((0, 4), dtype=torch.int32, device=dev)
    where, n = pa.compact_pages(data[:, 0], None, tables, refs)
    assert int(n) == 0 and (where == -1).all()


def test_captured(pa, dev):
    """A fork, a copy and a compaction in one graph, replayed on other entries: as eager calls."""
    rng = np.random.default_rng(8)
    NB, BS = 64, 4
    bt, ctx, refs = state(9, 6, NB, BS, [21, 10, 7], rng)
    data = pool(2, NB, BS, 1, 32, "bf16", dev)
    first = data.clone()
    st = [torch.from_numpy(x).to(dev) for x in (bt, ctx, refs)]
    start = [x.clone() for x in st]
    parents, rows = (torch.zeros(5, dtype=torch.int32, device=dev) for _ in range(2))
    src, dst = (torch.zeros(2, dtype=torch.int32, device=dev) for _ in range(2))

    def step():
        new = pa.fork_sequences(data[:, 0], data[:, 1], *st, parents, rows)
        where, n = pa.compact_pages(data[:, 0], data[:, 1], st[0], st[2])
        pa.copy_pages(data[:, 0], data[:, 1], src, dst)
        return new, where, n

    def reset(k):
        data.copy_(first)
        for x, y in zip(st, start):
            x.copy_(y)
        parents.copy_(torch.tensor([0, 1, 2, k % 3, -1]))
        rows.copy_(torch.tensor([3, 4, 5, 6, k % 3]))
        src.copy_(torch.tensor([0, 1]))
        dst.copy_(torch.tensor([60, 61 + k % 3]))

    reset(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    print("capture", flush=True)
    with torch.cuda.graph(graph):
        out = step()
    for k in (1, 2, 0, 2):
        reset(k)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (*out, *st, data)]
        reset(k)
        want = [*step(), *st, data]
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def test_python_paths_agree(pa, dev, monkeypatch, tmp_path):
    """Without the operator library: the same state, results and refusals."""
    import sys
    ops = sys.modules[pa.paged_attention.__module__]

    def calls():
        bt, ctx, refs = state(9, 6, 64, 4, [21, 10, 7], np.random.default_rng(8))
        data = pool(2, 64, 4, 1, 32, "bf16", dev)
        st = [torch.from_numpy(x).to(dev) for x in (bt, ctx, refs)]
        new = pa.fork_sequences(data[:, 0], data[:, 1], *st, torch.tensor([0, 1, 2, 0]), torch.tensor([3, 4, 5, 6]))
        pa.free_sequences(*st, torch.tensor([1, 4], device=dev), 4)
        where, n = pa.compact_pages(data[:, 0], data[:, 1], st[0], st[2])
        pa.copy_pages(data[:, 0], data[:, 1], torch.tensor([0, 1]), torch.tensor([60, 61]))
        pa.copy_pages(data[1, 0], None, torch.tensor([2]), torch.tensor([62]))
        return [new, where, n, *st, data.view(torch.int16)]

    def refusals():
        data = pool(1, 8, 4, 2, 32, "f16", dev)
        st = [torch.zeros(s, dtype=torch.int32, device=dev) for s in ((2, 2), (2,), (8,))]
        one = torch.tensor([0], device=dev)
        with pytest.raises(RuntimeError, match="must be int32 on CUDA"):
            pa.fork_sequences(data[:, 0], data[:, 1], st[0].long(), *st[1:], one, one)
        with pytest.raises(RuntimeError, match="must be int32 on CUDA"):
            pa.compact_pages(data[:, 0], data[:, 1], st[0], st[2].cpu())
        with pytest.raises(RuntimeError, match="contiguous token rows"):
            pa.copy_pages(data[0, 0].transpose(1, 2), None, one, one)
        with pytest.raises(RuntimeError, match=r"\[NB, BS, HKV, D\]"):
            pa.copy_pages(data, None, one, one)
        with pytest.raises(RuntimeError, match="on CUDA"):
            pa.copy_pages(data[:, 0].cpu(), None, one, one)
        with pytest.raises(RuntimeError, match="parents must have 1 entries"):
            pa.fork_sequences(data[:, 0], data[:, 1], *st, one.repeat(2), one)

    print("python paths", flush=True)
    want = calls()
    refusals()
    monkeypatch.setattr(ops, "_ops", None)
    monkeypatch.setattr(ops, "_torch_path", lambda: tmp_path / "none.so")
    assert ops._native() is ops._CAbi
    for x, y in zip(calls(), want):
        assert torch.equal(x, y)
    refusals()


def test_numbers_past_32_bits(pa, dev, monkeypatch, tmp_path):
    """int64 pages and rows that do not fit are outside, not what is left of them in 32 bits."""
    import sys
    ops = sys.modules[pa.paged_attention.__module__]
    for native in (True, False):
        if not native:
            monkeypatch.setattr(ops, "_ops", None)
            monkeypatch.setattr(ops, "_torch_path", lambda: tmp_path / "none.so")
        data = pool(1, 8, 4, 1, 32, "bf16", dev)
        first = data.clone()
        print("wide indices", native, flush=True)
        pa.copy_pages(data[0, 0], data[0, 1], torch.tensor([2**32, 1, 3, -2**32 + 4]), torch.tensor([5, 2**32 + 6, 7, 2]))
        first[:, :, 7] = first[:, :, 3]
        assert torch.equal(data.view(torch.uint8), first.view(torch.uint8))
        bt, ctx, refs = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([[0, 1], [-1, -1], [-1, -1]], [8, 0, 0],
                                                                                  [1, 1, 0, 0, 0, 0, 0, 0]))
        got = pa.fork_sequences(data[:, 0], data[:, 1], bt, ctx, refs, torch.tensor([2**32, 0, -2**32]),
                                torch.tensor([1, 2**32 + 2, 2]))
        assert got.tolist() == [-3, -3, -1] and ctx.tolist() == [8, 0, 0] and refs.tolist() == [1, 1] + [0] * 6
        pa.free_sequences(bt, ctx, refs, torch.tensor([2**32, -2**33]), 4)
        assert ctx.tolist() == [8, 0, 0] and refs.tolist() == [1, 1] + [0] * 6


@pytest.mark.parametrize("R,MB,most", [(9, 100, 9), (40, 150, 40), (700, 3, 700)])
def test_fork_long_and_many_rows(pa, dev, R, MB, most):
    """Tables longer than a wave, and batches that take one launch more: steps in place, with rows emptied,
    shared and begun pages, and at the end more copies than pages."""
    rng = np.random.default_rng(MB)
    BS = 2
    lens = [int(x) for x in rng.integers(0, MB * BS + 1, R)]
    NB = sum(-(-n // BS) for n in lens) + R // 3
    bt, ctx, refs = state(R, MB, NB, BS, lens, rng)
    for _ in range(3):
        N = int(rng.integers(most // 2, most + 1))
        rows = [int(x) for x in rng.permutation(R)[:N]]
        parents = [int(x) for x in rng.integers(-1, R, N)]
        run_fork(pa, dev, "f16", (1, NB, BS, 1, 32), bt, ctx, refs, parents, rows)
        assert (refs >= 0).all()
    free = int((refs == 0).sum())
    odd = [r for r in range(R) if ctx[r] % BS]
    if odd:
        spare = [r for r in range(R) if r != odd[0]][:free + 5]
        run_fork(pa, dev, "f16", (1, NB, BS, 1, 32), bt, ctx, refs, [odd[0]] * len(spare), spare)
