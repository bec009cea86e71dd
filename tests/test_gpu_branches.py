"""Branching sequences as a server runs them: prompts written with their norm and rotation, rows
forked, decode steps over the shared prefixes, rows freed and forked anew, the cache made dense,
and the steps gone on with, eagerly and as a replayed graph.

A second cache gives each row pages of its own and no sharing.  What the paged cache holds must be
its very bytes, and the attention must be that of its contents in 64 bits within the tolerances
that tests/test_gpu_shared_prefix.py derives."""
import numpy as np
import pytest
import torch

from test_gpu_shared_prefix import DT, HALF, exact

pytestmark = pytest.mark.gpu

L, ROWS, BS, MB = 2, 8, 16, 8
FAR = BS * MB


class Run:
    def __init__(self, pa, dev, H, HKV, D, kv, act, NB, seed):
        self.pa, self.dev, self.kv, self.act = pa, dev, kv, act
        self.H, self.HKV, self.D, self.scale = H, HKV, D, D**-0.5
        self.g = torch.Generator().manual_seed(seed)
        new = lambda *s: torch.zeros(s, dtype=torch.float32, device=dev).to(DT[kv])  # noqa: E731
        self.pool, self.plain = new(L, 2, NB, BS, HKV, D), new(L, 2, ROWS * MB, BS, HKV, D)
        i = lambda *s, fill=0: torch.full(s, fill, dtype=torch.int32, device=dev)  # noqa: E731
        self.bt, self.ctx, self.refs = i(ROWS, MB, fill=-1), i(ROWS), i(NB)
        self.own = torch.arange(ROWS * MB, dtype=torch.int32, device=dev).view(ROWS, MB)
        self.kvs = 1 / 16 if kv == "fp8" else 1.0
        a = torch.arange(FAR, dtype=torch.float64)[:, None] * 1000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
        self.table = torch.cat([a.cos(), a.sin()], 1).float().to(dev)
        self.weights = [[(torch.randn(D, generator=self.g) * 0.2 + 1).to(DT[act]).to(dev) for _ in range(2)] for _ in range(L)]

    def packed(self, T):
        """A projection's output, [T, H + 2 HKV, D] a layer."""
        return torch.randn((L, T, self.H + 2 * self.HKV, self.D), generator=self.g).to(DT[self.act]).to(self.dev)

    def write(self, cache, qkv, slots, positions):
        out, H, HKV = [], self.H, self.HKV
        for n in range(L):
            q, k, v = qkv[n][:, :H], qkv[n][:, H:H + HKV], qkv[n][:, H + HKV:]
            out.append(self.pa.qk_norm_rope_write_kv(q, k, v, cache[n, 0], cache[n, 1], slots, self.table, positions,
                                                     q_weight=self.weights[n][0], k_weight=self.weights[n][1],
                                                     k_scale=self.kvs, v_scale=self.kvs))
        return out

    def grow(self, row, tokens):
        """Pages for `tokens` more of a row: the lowest free ones."""
        n = int(self.ctx[row])
        for j in range(-(-n // BS), -(-(n + tokens) // BS)):
            page = int((self.refs == 0).nonzero()[0])
            self.bt[row, j], self.refs[page] = page, 1

    def prompt(self, row, n):
        self.grow(row, n)
        at = torch.arange(n, device=self.dev)
        qkv = self.packed(n)
        self.write(self.pool, qkv, self.bt[row].long()[at // BS] * BS + at % BS, at)
        self.write(self.plain, qkv, row * FAR + at, at)
        self.ctx[row] = n

    def fork(self, parents, rows):
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        got = self.pa.fork_sequences(self.pool[:, 0], self.pool[:, 1], self.bt, self.ctx, self.refs, i(parents), i(rows))
        assert (got >= -1).all()
        v = self.plain.view(torch.uint8).view(L, 2, ROWS, -1)
        v[:, :, rows] = v[:, :, parents].clone()

    def slots(self, table):
        """Where the step's token of each row goes; a row without tokens writes none."""
        at = self.ctx.long()
        slot = table.gather(1, (at // BS)[:, None]).long()[:, 0] * BS + at % BS
        return torch.where(at > 0, slot, -1)

    def step(self, starts, prefix, qkv):
        """One token of every row that has any: (attention per layer, the queries)."""
        q = self.write(self.pool, qkv, self.slots(self.bt), self.ctx)
        n = torch.where(self.ctx > 0, self.ctx + 1, 0).int()
        return [self.pa.paged_attention_shared_prefix(q[i], self.pool[i, 0], self.pool[i, 1], self.bt, n, starts, prefix,
                                                      self.scale, out_dtype=DT[self.act], k_scale=self.kvs, v_scale=self.kvs)
                for i in range(L)], q

    def decode(self, starts, prefix, call=None):
        for r in (self.ctx > 0).nonzero()[:, 0].tolist():
            self.grow(r, 1)
        i = lambda x: torch.tensor(x, dtype=torch.int32, device=self.dev)  # noqa: E731
        qkv = self.packed(ROWS)
        self.write(self.plain, qkv, self.slots(self.own), self.ctx)
        got, q = (call or self.step)(i(starts), i(prefix), qkv)
        self.ctx += (self.ctx > 0).int()
        torch.cuda.synchronize()
        self.same()
        for n in range(L):
            self.near(got[n], n, q[n], starts, prefix)

    def same(self):
        """Every token of every row, under the table and in the rows' own pages."""
        flat = lambda c: c.view(torch.uint8).view(L, 2, -1, self.HKV * self.D * c.element_size())  # noqa: E731
        for r, n in enumerate(self.ctx.tolist()):
            at = torch.arange(n, device=self.dev)
            for t in at.split(64):
                a = flat(self.pool)[:, :, self.bt[r].long()[t // BS] * BS + t % BS]
                assert torch.equal(a, flat(self.plain)[:, :, r * FAR + t]), ("row", r)

    def near(self, got, n, q, starts, prefix):
        # (the queries as the kernel took them: their own rounding is not this check's)
        c = dict(q=q.cpu(), k=self.plain[n, 0].cpu(), v=self.plain[n, 1].cpu(), bt=self.own.cpu(), ctx=self.ctx.cpu(),
                 starts=torch.tensor(starts), prefix=torch.tensor(prefix), S=1, kvs=self.kvs)
        want, A, es, count = exact(c, self.scale)
        got = got.double().cpu().reshape(want.shape)
        tile = self.act if self.kv == "fp8" else self.kv
        e = es * ((self.D + 8) * 2.0**-24 + 2.0**-23)
        tol = A * (2 * e + (2 * count + 64) * 2.0**-24 + HALF[tile])[..., None]
        tol = tol + HALF[self.act] * (want.abs() + tol) + (2.0**-25 if self.act == "f16" else 0)
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("H,HKV,D,kv,act", [(12, 12, 64, "f16", "f16"), (8, 2, 128, "bf16", "bf16"), (8, 1, 128, "fp8", "bf16")])
def test_branches(pa, dev, H, HKV, D, kv, act):
    r = Run(pa, dev, H, HKV, D, kv, act, NB=48, seed=H)
    print("prompts", H, HKV, D, kv, flush=True)
    r.prompt(0, 37)
    r.prompt(4, 64)
    print("forks", flush=True)
    r.fork([0, 0, 0, 4, 4], [1, 2, 3, 5, 6])
    r.same()
    assert int((r.refs > 0).sum()) == 3 + 3 + 4  # shared pages once, a copied one for each fork of row 0
    groups = ([0, 4, 7], [37, 64])
    for _ in range(12):
        r.decode(*groups)
    print("free, fork, compact", flush=True)
    pa.free_sequences(r.bt, r.ctx, r.refs, torch.tensor([2, 5], dtype=torch.int32, device=dev), BS)
    r.decode(*groups)
    r.fork([3], [2])
    free = int((r.refs == 0).sum())
    where, live = pa.compact_pages(r.pool[:, 0], r.pool[:, 1], r.bt, r.refs)
    assert int(live) == 48 - free and (r.refs[:48 - free] > 0).all() and (r.refs[48 - free:] == 0).all()
    r.same()
    print("a beam step in place", flush=True)
    r.fork([3, 1, 1, 0, 6, 6], [1, 2, 3, 0, 6, 5])
    r.same()
    for _ in range(3):
        r.decode(*groups)

    print("captured", flush=True)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    hold = [i(groups[0]), i(groups[1]), r.packed(ROWS)]
    save = [x.clone() for x in (r.pool, r.bt, r.ctx)]
    for j in (0, 1, 2, 3, 4, 6, 5):
        r.grow(j, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r.step(*hold)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = r.step(*hold)
    r.pool.copy_(save[0])

    def replay(starts, prefix, qkv):
        for x, y in zip(hold, (starts, prefix, qkv)):
            x.copy_(y)
        graph.replay()
        return out

    for k in range(9):
        r.decode(*(groups if k < 6 else ([0, 1, 4], [0, 37])), replay)
        if k == 3:  # (other tables under the same graph)
            r.fork([0], [3])
            pa.compact_pages(r.pool[:, 0], r.pool[:, 1], r.bt, r.refs)
