"""The cache's calls, the tree's attention and its verdict in one run, as a decoding
loop makes them; the same step captured and replayed; and the example."""
import random

import pytest
import torch

from examples import tree_decode
from kv_util import attention
from locus_amd import sampler as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("streams,steps,prompt", [(1, 3, 2), (4, 12, 40)])
def test_example(streams, steps, prompt):
    r = tree_decode.run(streams, steps, prompt)
    assert r["ok"]
    assert r["pages_held"] == r["pages_expected"]
    assert r["length"] == [len(t) - 1 for t in r["text"]]
    assert all(len(t) >= prompt + steps for t in r["text"])


class Run:
    """A cache beside what its sequences hold (per slot the rows of keys and values, in order)."""

    def __init__(self, f8):
        self.L, self.kv, self.H, self.D, self.page, self.R = 2, 2, 6, 64, 16, 5
        g = self.g = torch.Generator().manual_seed(int(f8))
        pages, slots, wide = 60, 6, 12
        shape, dt = (self.L, pages, self.kv, self.page, self.D), torch.float8_e4m3fn if f8 else torch.bfloat16
        sc = {n: torch.zeros(shape[:4], device="cuda") for n in ("k_scale", "v_scale")} if f8 else {}
        self.table = torch.full((slots, wide), -1, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.f8, self.sc = f8, sc
        self.k, self.v = torch.zeros(shape, device="cuda").to(dt), torch.zeros(shape, device="cuda").to(dt)
        self.cache = S.KvCache(self.k, self.v, self.table, self.refs, **sc)
        self.s = S.Sampler(device=0, max_rows=64, max_vocab=1024, max_hist=16, max_top=1)
        self.s.kv_reserve(pages)
        self.rows = {}

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def new(self, n):
        return [torch.randn(self.L, n, self.kv, self.D, generator=self.g).bfloat16() for _ in range(2)]

    def done(self, r):
        torch.cuda.synchronize()
        assert (r == 0).all() and self.s.status() == 0

    def grow(self, seq, start, end):
        r = self.ints([9] * len(seq))
        self.s.kv_grow_dev(self.cache, self.ints(seq), self.ints(start), self.ints(end), r)
        self.done(r)

    def stored(self, x):
        """What the cache holds for bf16 rows, as f64."""
        if not self.f8:
            return x.double()
        x = x.float()
        scale = x.abs().amax(-1, keepdim=True) / 448.0
        return (x / scale).to(torch.float8_e4m3fn).double() * scale.double()

    def check(self, seq):
        """Attention of new tokens in every layer over what each slot should hold."""
        n, R = len(seq), self.R
        q = torch.randn(n * R, self.H, self.D, generator=self.g).bfloat16()
        k, v = self.new(n * R)
        lens = [self.rows[i][0].shape[1] for i in seq]
        out = {"o": torch.empty(n * R, self.H, self.D, device="cuda", dtype=torch.bfloat16), "lse": torch.empty(n * R, self.H, device="cuda")}
        see = torch.ones(R, R).tril().bool()
        for layer in range(self.L):
            self.s.tree_attn_dev(q.cuda(), k[layer].cuda(), v[layer].cuda(), self.cache, out, length=self.ints(lens), seq=self.ints(seq),
                                 rows_per_seq=R, layer=layer)
            torch.cuda.synchronize()
            assert self.s.status() == 0
            for i, slot in enumerate(seq):
                m = slice(i * R, (i + 1) * R)
                ck, cv = (self.stored(t[layer]) for t in self.rows[slot])
                o, lse, weigh, most = attention(q[m], k[layer, m], v[layer, m], R, ck, cv, see, self.D ** -0.5)
                # (as in the attention's own tests: two roundings to bf16, scores in f32; a stored scale is good to 2^-24)
                tol = 2.0 ** -8 * (o.abs() + weigh) * (1 + 2.0 ** -7) + 2.0 ** -18 * (1 + most[..., None]) * weigh
                assert ((out["o"][m].double().cpu() - o).abs() <= tol).all()
                assert ((out["lse"][m].double().cpu() - lse).abs() <= 2.0 ** -18 * (1 + most + lse.abs())).all()


@pytest.mark.parametrize("f8", [False, True])
def test_a_run(f8):
    c, rng = Run(f8), random.Random(f8)
    s = c.s
    # prompts
    n0 = [37, 16, 1]
    k, v = c.new(3 * 40)
    c.grow([0, 1, 2], [0, 0, 0], n0)
    s.kv_append_dev(c.cache, k.cuda(), v.cuda(), c.ints([0, 1, 2]), c.ints([0, 0, 0]), c.ints(n0), rows_per_seq=40)
    for i, n in enumerate(n0):
        c.rows[i] = [t[:, i * 40: i * 40 + n] for t in (k, v)]
    c.check([0, 1, 2])
    # a step whose trees are verified: a path of nodes appended
    R, parent = c.R, [-1, 0, 0, 2, 3]
    best = torch.randint(0, 1000, (3, R), generator=c.g)
    tokens = torch.full((3, R), -1)
    for i, right in enumerate(([], [2], [2, 3, 4])):
        for j in right:
            tokens[i, j] = best[i, parent[j]]
    out = {"argmax_ids": best.int().view(-1).cuda(), "path": c.ints([[0] * R] * 3), "n_path": c.ints([0] * 3), "next_id": c.ints([0] * 3),
           "length": c.ints([0] * 3)}
    s.tree_verify_dev(tokens.int().view(-1).cuda(), c.ints(parent * 3), out, rows_per_seq=R, length=c.ints(n0))
    k, v = c.new(3 * R)
    r = c.ints([9] * 3)
    s.kv_grow_dev(c.cache, c.ints([0, 1, 2]), c.ints(n0), out["length"], r)
    s.kv_append_dev(c.cache, k.cuda(), v.cuda(), c.ints([0, 1, 2]), c.ints(n0), out["n_path"], rows_per_seq=R, index=out["path"])
    c.done(r)
    for i, path in enumerate(([0], [0, 2], [0, 2, 3, 4])):
        c.rows[i] = [torch.cat([a, b[:, [i * R + j for j in path]]], 1) for a, b in zip(c.rows[i], (k, v))]
        assert out["length"][i].item() == c.rows[i][0].shape[1] and out["next_id"][i].item() == best[i, path[-1]].item()
    c.check([2, 0, 1])
    # forks that go on by themselves
    lens = [c.rows[i][0].shape[1] for i in range(3)]
    r = c.ints([9, 9])
    s.kv_fork_dev(c.cache, c.ints([0, 0]), c.ints([3, 4]), c.ints([lens[0], 20]), r)
    c.done(r)
    c.rows[3], c.rows[4] = c.rows[0], [t[:, :20] for t in c.rows[0]]
    who, at = [0, 3, 4], [lens[0], lens[0], 20]
    c.grow(who, at, [a + 7 for a in at])
    k, v = c.new(3 * 7)
    s.kv_append_dev(c.cache, k.cuda(), v.cuda(), c.ints(who), c.ints(at), rows_per_seq=7)
    for i, slot in enumerate(who):
        c.rows[slot] = [torch.cat([a, b[:, i * 7:(i + 1) * 7]], 1) for a, b in zip(c.rows[slot], (k, v))]
    c.check([0, 1, 2, 3, 4])
    # part of a shared context dropped, the rest given back
    n = c.rows[3][0].shape[1]
    keep = sorted(rng.sample(range(n), n // 2))
    c.grow([3], [0], [n])
    r = c.ints([9])
    s.kv_compact_dev(c.cache, c.ints([3]), c.ints([len(keep)]), c.ints([keep]), r)
    c.done(r)
    s.kv_free_dev(c.cache, c.ints([3]), c.ints([len(keep)]), r)
    c.done(r)
    c.rows[3] = [t[:, keep] for t in c.rows[3]]
    c.check([3, 0, 4])
    r = c.ints([9] * 5)
    s.kv_free_dev(c.cache, c.ints([0, 1, 2, 3, 4]), None, r)
    c.done(r)
    assert c.refs.sum().item() == 0 and (c.table == -1).all()
    s.close()


def test_step_in_a_graph():
    """Verdict, pages, append and attention captured: replays with eager steps between give what eager steps alone give."""
    a, b = Run(False), Run(False)
    R, n = a.R, 3
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(2, n * R, 2, 64, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(n * R, 6, 64, generator=g).bfloat16().cuda()
    parent, seq = a.ints([-1, 0, 1, 1, 3] * n), a.ints(list(range(n)))
    tokens, best = torch.zeros(n * R, dtype=torch.int32, device="cuda"), torch.zeros(n * R, dtype=torch.int32, device="cuda")

    def state(c):
        ints = lambda *sh: torch.zeros(*sh, dtype=torch.int32, device="cuda")   # noqa: E731
        return {"length": ints(n), "res": ints(n), "o": torch.zeros(n * R, 6, 64, device="cuda", dtype=torch.bfloat16), "path": ints(n, R),
                "n_path": ints(n), "next_id": ints(n), "new": ints(n)}

    def step(c, st):
        c.s.tree_attn_dev(q, k[1], v[1], c.cache, {"o": st["o"]}, length=st["length"], seq=seq, rows_per_seq=R, layer=1)
        c.s.tree_verify_dev(tokens, parent, {"argmax_ids": best, "path": st["path"], "n_path": st["n_path"], "next_id": st["next_id"],
                                             "length": st["new"]}, rows_per_seq=R, length=st["length"])
        c.s.kv_grow_dev(c.cache, seq, st["length"], st["new"], st["res"])
        c.s.kv_append_dev(c.cache, k, v, seq, st["length"], st["n_path"], rows_per_seq=R, index=st["path"])
        st["length"].copy_(st["new"])

    sa, sb = state(a), state(b)
    step(a, sa)          # (a first eager step)
    step(b, sb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, sa)
    for i in range(12):
        tokens.copy_(torch.randint(0, 3, (n * R,), generator=g))
        best.copy_(torch.randint(0, 3, (n * R,), generator=g))
        q.mul_(-1)
        if i % 3 == 2:
            step(a, sa)
        else:
            graph.replay()
        step(b, sb)
        torch.cuda.synchronize()
        for x in sa:
            assert torch.equal(sa[x].view(torch.uint8), sb[x].view(torch.uint8)), (i, x)
        assert torch.equal(a.table, b.table) and torch.equal(a.refs, b.refs)
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8)) and torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))
        assert a.s.status() == 0
    a.s.close()
    b.s.close()
