"""Attention over the cache and a step's new tokens (lcs_tree_attn) against the formula
in 64 bits.

Tolerances, for exact inputs: a weight is rounded to bf16 once (2^-8 of itself at most)
and the result once (2^-8 of itself), so o is within 2^-8 (|o| + sum_j p_j |v_j|), and
their product of the second order. Scores are f32 sums of exact products: 2^-24 (dim +
8) of the largest scale sum_d |q_d k_d|, for the weights and for lse alike (twice for
the weights: a normaliser's too). The weights' sum is an f32 sum of up to n terms, and
the exponential is good to 2^-21.
"""
import math
import random

import pytest
import torch

from kv_util import attention, quantise
from locus_amd import sampler as S

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def s():
    x = S.Sampler(device=0, max_rows=64, max_vocab=4096, max_hist=64, max_top=4)
    x.kv_reserve(64)
    yield x
    x.close()


def words(see):
    """(rows, n) truth values in 32-bit words."""
    rows, n = see.shape
    out = torch.zeros(rows, (n + 31) // 32, dtype=torch.int64)
    for j in range(n):
        out[:, j // 32] |= see[:, j].long() << (j % 32)
    return torch.where(out >= 1 << 31, out - (1 << 32), out).int()


def tree(rows, rng):
    parent = [-1] + [rng.randrange(max(0, j - 4), j) for j in range(1, rows)]
    see = torch.zeros(rows, rows, dtype=torch.bool)
    for j in range(rows):
        a = j
        while a >= 0:
            see[j, a] = True
            a = parent[a]
    return see


class Case:
    def __init__(self, lengths, rows, heads, kv, dim, page, f8=False, layout="head", mask="tree", layers=2, seed=0, spread=1.0, scale=None):
        rng = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        n = self.n = len(lengths)
        self.lengths, self.rows, self.heads, self.kv, self.dim, self.f8 = lengths, rows, heads, kv, dim, f8
        self.scale = dim ** -0.5 if scale is None else scale
        used = [-(-x // page) for x in lengths]
        pages, max_pages = sum(used) + 3, max(1, max(used)) + 1
        self.page, self.layer = page, layers - 1
        rand = lambda *sh: (torch.randn(*sh, generator=g) * spread).bfloat16()   # noqa: E731
        k, v = rand(layers, pages, kv, page, dim), rand(layers, pages, kv, page, dim)
        self.ks = self.vs = None
        if f8:
            (k, self.ks), (v, self.vs) = quantise(k), quantise(v)
        order = rng.sample(range(pages), pages)
        self.slots = rng.sample(range(n + 2), n)
        self.table = torch.full((n + 2, max_pages), -1, dtype=torch.int32)
        held = torch.zeros(pages, page, dtype=torch.bool)
        for i, x in enumerate(lengths):
            for p in range(used[i]):
                at = order.pop()
                self.table[self.slots[i], p] = at
                held[at, : min(page, x - p * page)] = True
        # what nobody's context holds is not part of any result: it is NaN
        wild = ~held[None, :, None, :].expand(k.shape[:4])
        for t in (k, v):
            t.view(torch.uint8 if f8 else torch.int16)[wild] = 0x7f if f8 else 0x7fc0
        for t in (self.ks, self.vs):
            if t is not None:
                t[wild] = NAN
        self.k, self.v, self.layout = k, v, layout
        self.q, self.k_new, self.v_new = rand(n * rows, heads, dim), rand(n * rows, kv, dim), rand(n * rows, kv, dim)
        at = torch.arange(rows)
        self.mask = None
        self.see = [at[None, :] <= at[:, None] for _ in range(n)]
        if mask == "tree":
            self.see = [tree(rows, rng) for _ in range(n)]
        elif mask == "any":
            self.see = [torch.rand(rows, rows, generator=g) < 0.4 for _ in range(n)]
        elif mask == "none":
            self.see = [torch.zeros(rows, rows, dtype=torch.bool) for _ in range(n)]
        if mask != "chain":
            self.mask = torch.cat([words(x) for x in self.see])

    def put(self, t):
        return t.cuda() if self.layout == "head" else t.transpose(2, 3).contiguous().cuda().transpose(2, 3)

    def upload(self, pad=8):
        n, rows, dim = self.n, self.rows, self.dim
        wide = torch.full((n * rows, (self.heads + 2 * self.kv) * dim + pad), NAN).bfloat16()
        cut, off = [], 0
        for t in (self.q, self.k_new, self.v_new):
            m = t.shape[1] * dim
            wide[:, off: off + m] = t.reshape(n * rows, m)
            cut.append((off, m, t.shape[1]))
            off += m
        w = wide.cuda()
        self.dev = [w[:, o: o + m].unflatten(1, (h, dim)) for o, m, h in cut]
        scales = {} if self.ks is None else {"k_scale": self.ks.cuda(), "v_scale": self.vs.cuda()}
        self.cache = S.KvCache(self.put(self.k), self.put(self.v), self.table.cuda(), torch.ones(self.k.shape[1], dtype=torch.int32).cuda(), **scales)
        self.len_dev = torch.tensor(self.lengths, dtype=torch.int32, device="cuda")
        self.seq_dev = torch.tensor(self.slots, dtype=torch.int32, device="cuda")
        self.mask_dev = None if self.mask is None else self.mask.cuda()
        # a guard row behind the last one
        self.o = torch.full((n * rows + 1, self.heads * dim + 16), 3.0).bfloat16().cuda()
        self.lse = torch.full((n * rows + 1, self.heads), 5.0).cuda()
        self.out = {"o": self.o[:-1, : self.heads * dim].unflatten(1, (self.heads, dim)), "lse": self.lse[:-1]}
        return self

    def launch(self, s, stream=None):
        s.tree_attn_dev(*self.dev, self.cache, self.out, length=self.len_dev, seq=self.seq_dev, rows_per_seq=self.rows, mask=self.mask_dev,
                        layer=self.layer, scale=self.scale, stream=stream)

    def run(self, s):
        self.upload()
        s.status()
        self.launch(s)
        torch.cuda.synchronize()
        return self

    def context(self, i):
        out = []
        for t, sc in ((self.k, self.ks), (self.v, self.vs)):
            idx = self.table[self.slots[i], : -(-self.lengths[i] // self.page)].long()
            x = t[self.layer, idx].double() if sc is None else t[self.layer, idx].float().double() * sc[self.layer, idx].double()[..., None]
            out.append(x.transpose(1, 2).reshape(-1, self.kv, self.dim)[: self.lengths[i]])
        return out

    def check(self, only=None):
        assert (self.o[-1].float() == 3.0).all() and (self.o[:, self.heads * self.dim:].float() == 3.0).all() and (self.lse[-1] == 5.0).all()
        o, lse = self.out["o"].double().cpu(), self.out["lse"].double().cpu()
        for i in range(self.n) if only is None else only:
            mine = slice(i * self.rows, (i + 1) * self.rows)
            ck, cv = self.context(i)
            wo, wl, weigh, most = attention(self.q[mine], self.k_new[mine], self.v_new[mine], self.rows, ck, cv, self.see[i], self.scale)
            terms = self.lengths[i] + self.rows
            score = 2.0 ** -24 * (self.dim + 8) * most
            tol_l = score + 2.0 ** -24 * (terms + wl.abs().nan_to_num(0, 0, 0)) + 2.0 ** -21
            u = 2.0 ** -8
            weight = u + 2 * score + 2.0 ** -24 * terms + 2.0 ** -20
            tol_o = (u * (wo.abs() + (1 + u) * weigh) + (weight - u)[..., None] * weigh) * (1 + u) + 2.0 ** -133
            gone = torch.isinf(wl) & (wl < 0)
            got_l, got_o = lse[mine], o[mine]
            assert torch.equal(torch.isnan(got_l), torch.isnan(wl)) and torch.equal(torch.isnan(got_o), torch.isnan(wo)), f"sequence {i}"
            assert (got_l[gone] == -INF).all() and (got_o[gone] == 0).all(), f"sequence {i}"
            fine = torch.isfinite(wl)
            assert ((got_l - wl).abs() <= tol_l)[fine].all(), (i, (got_l - wl).abs()[fine].max())
            ok = torch.isfinite(wo)
            assert ((got_o - wo).abs() <= tol_o)[ok].all(), (i, ((got_o - wo).abs() / tol_o)[ok].max())
        return self


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 240, 256])
@pytest.mark.parametrize("lengths,rows,heads,kv,page,mask,layout", [
    ([1], 1, 1, 1, 16, "chain", "head"),
    ([0, 0], 3, 2, 2, 16, "tree", "head"),
    ([5, 0, 130], 1, 8, 2, 16, "chain", "token"),
    ([31, 32, 33, 127], 16, 4, 1, 16, "tree", "head"),
    ([128, 129, 500, 1], 7, 15, 5, 32, "any", "token"),
    ([300, 17], 33, 6, 2, 64, "tree", "head"),
    ([64, 1000], 5, 7, 1, 16, "none", "token"),
])
def test_shapes(s, lengths, rows, heads, kv, page, mask, layout, dim, f8):
    Case(lengths, rows, heads, kv, dim, page, f8, layout, mask, seed=dim + rows).run(s).check()
    assert s.status() == 0


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,heads,kv", [(64, 8, 1), (256, 4, 2), (100, 24, 2), (48, 16, 16), (2, 64, 1), (1, 48, 3)])
def test_many_rows(s, rows, heads, kv, f8):
    """More rows than any tile holds, and masks of several words."""
    Case([150, 0, 64], rows, heads, kv, 128, 32, f8, seed=rows).run(s).check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("lengths,page", [([9000], 16), ([20000, 3, 700], 128), ([4096, 4095, 4097], 1024)])
def test_long(s, lengths, page, f8):
    """Contexts that many workgroups share, beside short ones."""
    Case(lengths, 4, 4, 2, 128, page, f8, seed=len(lengths)).run(s).check()


@pytest.mark.parametrize("n", [65, 200, 1024])
def test_many_sequences(s, n):
    rng = random.Random(n)
    lengths = [rng.choice([0, 1, 15, 16, 40, 100]) for _ in range(n)]
    Case(lengths, 2, 2, 1, 64, 16, seed=n, layers=1).run(s).check(only=rng.sample(range(n), 40))


@pytest.mark.parametrize("spread,scale", [(8.0, None), (30.0, None), (1.0, 0.0), (2.0, -0.3), (0.01, 1.0)])
@pytest.mark.parametrize("f8", [False, True])
def test_scores(s, spread, scale, f8):
    """Scores that leave one key, rise block by block, are all equal, or change sign."""
    Case([700, 40], 6, 8, 2, 128, 16, f8, spread=spread, scale=scale, seed=3).run(s).check()


def test_rising_scores(s):
    """Every block's largest score lies above the last one's."""
    c = Case([1500], 3, 4, 1, 64, 16, seed=9)
    idx = c.table[c.slots[0], :94].long()
    up = torch.arange(94 * 16).view(94, 1, 16, 1) * 0.05
    c.k[c.layer, idx] = (c.q[0, 0] * 0.1 + up * c.q[0, 0] / c.q[0, 0].float().norm() ** 2 * 8).bfloat16()
    c.k[c.layer, idx[-1], :, 1500 - 93 * 16:] = NAN
    c.run(s).check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,heads,kv", [(5, 4, 2), (40, 4, 1), (70, 2, 1)])
def test_masked_nan_and_inf(s, rows, heads, kv, f8):
    """NaN and infinities in new tokens that some rows see and others do not."""
    c = Case([90, 0, 33], rows, heads, kv, 64, 16, f8, seed=rows)
    for i, (j, what) in enumerate([(2, NAN), (4, INF), (1, -INF)]):
        c.v_new[i * rows + j, :, ::3] = what
    c.k_new[0 * rows + 3, 0] = NAN
    # a last token that nobody sees, all NaN
    for i in range(3):
        c.see[i][:, rows - 1] = False
        c.k_new[i * rows + rows - 1] = NAN
        c.v_new[i * rows + rows - 1] = NAN
    c.mask = torch.cat([words(x) for x in c.see])
    c.run(s).check()


def test_nan_in_the_context(s):
    """A NaN in a value that all see, an infinity in another; other heads and sequences stay clean."""
    c = Case([50, 60], 3, 4, 2, 64, 16, seed=4)
    c.v[c.layer, c.table[c.slots[0], 1], 0, 3, 7] = NAN
    c.v[c.layer, c.table[c.slots[1], 0], 1, 2, 9] = INF
    c.run(s).check()


def test_missing_pages_and_bad_slots(s):
    """A page missing below the length is not seen; bad slots have no context; the status says so."""
    c = Case([100, 40, 200, 64], 3, 4, 2, 128, 16, seed=5).upload()
    t = c.cache._keep[2]
    slot = c.slots[0]
    gone = c.table[slot, 2].item()
    for bad in (-1, 10 ** 6, -7):
        t[slot, 2] = bad
        s.status()
        c.launch(s)
        torch.cuda.synchronize()
        assert s.status() == 8
    t[slot, 2] = gone
    ctx = c.context
    c.context = lambda i: [torch.cat([x[:32], x[48:]]) for x in ctx(0)] if i == 0 else ctx(i)
    c.check()
    c.context = ctx
    c.launch(s)
    torch.cuda.synchronize()
    assert s.status() == 0
    c.check()
    # no context: slot -1 (no error), slots outside the table and a negative length
    whole = c.lengths
    for slots, lens, status in [([-1, -1, -1, -1], whole, 0), ([6, -2, 2 ** 31 - 1, c.slots[3]], whole, 8), (c.slots, [-1, -2 ** 31, 0, 64], 0)]:
        c.seq_dev.copy_(torch.tensor(slots))
        c.len_dev.copy_(torch.tensor(lens))
        c.launch(s)
        torch.cuda.synchronize()
        assert s.status() == status
        c.context = lambda i: [x[:0] if slots[i] not in c.slots or lens[i] <= 0 else x for x in ctx(i)]
        c.lengths = whole
        c.check()
    # a length past the table: what the table holds
    c.context, c.lengths = ctx, whole
    c.seq_dev.copy_(torch.tensor(c.slots))
    c.len_dev.copy_(torch.tensor([100, 40, 2 ** 31 - 1, 64]))
    c.launch(s)
    torch.cuda.synchronize()
    assert s.status() == 8
    c.check(only=[0, 1, 3])


def test_one_slot_twice_and_no_seq(s):
    c = Case([100, 100], 3, 4, 2, 128, 16, seed=6)
    c.slots = [c.slots[0], c.slots[0]]
    c.run(s).check()
    c = Case([30, 70, 5], 3, 4, 2, 128, 16, seed=7)
    c.table = torch.cat([c.table[c.slots], c.table[:1]])
    c.slots = [0, 1, 2]
    c.upload()
    c.seq_dev = None
    c.launch(s)
    torch.cuda.synchronize()
    c.check()


def test_other_stream_and_graph(s):
    """On a side stream, and captured: replays over lengths, queries and pages that changed, with eager calls between."""
    c = Case([300, 20, 77], 4, 8, 2, 128, 16, seed=8).upload()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.launch(s)
    side.synchronize()
    c.check()
    d = Case([3000, 1], 2, 4, 2, 64, 16, seed=18).upload()      # (another case in a graph of its own, the workspace shared)
    graphs = []
    for x in (c, d):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            x.launch(s)
        graphs.append(gr)
    for lens in ([300, 20, 77], [1, 20, 0], [0, 0, 0], [289, 3, 50]):
        c.lengths = lens
        c.len_dev.copy_(torch.tensor(lens))
        c.dev[0].mul_(0.5)
        c.q = c.dev[0].cpu()
        for gr, x in zip(graphs, (c, d)):
            x.o[:-1, : x.heads * x.dim] = 9.0
            gr.replay()
        torch.cuda.synchronize()
        c.check()
        d.check()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = [t.clone() for t in (c.o, c.lse, d.o, d.lse)]
        c.launch(s)
        d.launch(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(want, (c.o, c.lse, d.o, d.lse)))


def test_same_bits_again(s):
    c = Case([3000, 40], 5, 8, 2, 128, 16, seed=11).run(s)
    first = c.o.clone(), c.lse.clone()
    for _ in range(3):
        c.launch(s)
    torch.cuda.synchronize()
    assert torch.equal(first[0].view(torch.int16), c.o.view(torch.int16)) and torch.equal(first[1], c.lse)


def test_far_pages(s):
    """Offsets past 2^32 bytes: a pool of 6 GB a side, its last pages used."""
    pages, kv, page, dim = 24576, 8, 128, 128
    shape = (1, pages, kv, page, dim)
    k = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    v = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    c = Case([500, 200], 2, 16, 8, 128, 128, seed=12, layers=1)
    for t, w in ((k, c.k), (v, c.v)):
        t[:, -c.k.shape[1]:] = w.cuda()
    c.upload()
    table = torch.where(c.table >= 0, c.table + pages - c.k.shape[1], c.table).int().cuda()
    c.cache = S.KvCache(k, v, table, torch.ones(pages, dtype=torch.int32, device="cuda"))
    c.launch(s)
    torch.cuda.synchronize()
    c.check()


def test_binding_refusals(s):
    c = Case([20, 30], 3, 4, 2, 64, 16, seed=1).upload()
    q, k, v = c.dev
    kw = dict(length=c.len_dev, seq=c.seq_dev, rows_per_seq=3, mask=c.mask_dev, layer=1)
    f32 = torch.empty(6, 4, device="cuda")
    for args, more, out in [((q[:5], k, v), {}, c.out), ((q, k[:, :1], v), {}, c.out), ((q, k, v.float()), {}, c.out), ((q.cpu(), k, v), {}, c.out),
                            ((q.transpose(1, 2), k, v), {}, c.out), ((q[:, :3], k, v), {}, c.out), ((q, k, v), {"rows_per_seq": 2}, c.out),
                            ((q, k, v), {"layer": 2}, c.out), ((q, k, v), {"mask": c.mask_dev.float()}, c.out), ((q, k, v), {"mask": c.mask_dev[:5]}, c.out),
                            ((q, k, v), {"seq": c.seq_dev[:1]}, c.out), ((q, k, v), {"length": c.len_dev.float()}, c.out),
                            ((q, k, v), {"scale": float("nan")}, c.out), ((q, k, v), {}, c.out | {"lse": f32[:5]}), ((q, k, v), {}, {"o": c.out["o"].float()}),
                            ((q.contiguous()[..., 1:], k, v), {}, c.out)]:
        with pytest.raises(S.SamplerError):
            s.tree_attn_dev(*args, c.cache, out, **(kw | more))
    with pytest.raises(S.SamplerError):
        s.tree_attn_dev(q, k, v, None, c.out, **kw)
    s.tree_attn_dev(q, k, v, c.cache, {"o": c.out["o"]}, **(kw | {"scale": None}))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dim", [64, 112, 128])
@pytest.mark.parametrize("lengths,rows,heads,kv,page,mask,layout", [
    ([5000, 0, 63, 64, 65], 13, 10, 2, 16, "tree", "head"),       # 65 rows a head
    ([700, 129], 24, 3, 1, 32, "any", "token"),                   # 72
    ([33, 2000], 128, 2, 2, 64, "tree", "head"),                  # 128, new tokens of a whole step
    ([1, 95, 4000], 129, 1, 1, 16, "chain", "head"),              # 129, of more than a step
    ([300, 3001], 97, 4, 2, 16, "tree", "token"),                 # 194
    ([8000], 64, 8, 2, 128, "tree", "head"),                      # 256, one sequence over all workgroups
    ([40, 0], 256, 3, 1, 16, "any", "head"),                      # 768
    ([1500] * 66, 33, 4, 2, 16, "chain", "head"),                 # 66, several sequences a lane
])
def test_shared_tiles(s, lengths, rows, heads, kv, page, mask, layout, dim):
    """Rows a head on both sides of what makes two or four waves share a tile."""
    Case(lengths, rows, heads, kv, dim, page, False, layout, mask, seed=dim + rows).run(s).check()
    assert s.status() == 0


@pytest.mark.parametrize("rows,heads,kv", [(70, 2, 2), (70, 2, 1), (100, 2, 1)])
def test_masked_nan_in_shared_tiles(s, rows, heads, kv):
    """NaN and infinities in new tokens that some rows see and others do not, in every tile; a missing page."""
    c = Case([90, 0, 333], rows, heads, kv, 128, 16, seed=rows)
    for i in range(3):
        for j, what in ((2, NAN), (4, INF), (33, -INF), (40, NAN), (64, INF), (69, -INF)):
            c.v_new[i * rows + j, :, j % 5::3] = what
        c.see[i][:, rows - 1] = False
        c.k_new[i * rows + rows - 1] = NAN
        c.v_new[i * rows + rows - 1] = NAN
    c.mask = torch.cat([words(x) for x in c.see])
    c.run(s).check()


@pytest.mark.parametrize("dim", [48, 64, 128])
@pytest.mark.parametrize("rows,heads,page,mask", [(10, 32, 16, "tree"), (64, 8, 64, "any"), (33, 8, 32, "chain")])
def test_many_pairs_of_uneven_lengths(s, rows, heads, page, mask, dim):
    lengths = [(37 * i * i) % 1500 if i % 5 else i for i in range(17)]
    Case(lengths, rows, heads, 8, dim, page, mask=mask, seed=dim + rows).run(s).check()
    assert s.status() == 0


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("lengths,rows,heads,kv,page,mask,layout", [
    ([3000, 0, 64, 65, 1], 11, 6, 2, 16, "tree", "token"),        # 33 rows a head
    ([500, 33], 129, 2, 2, 64, "tree", "head"),                   # new tokens of more than a step
    ([2000, 700], 65, 4, 1, 32, "any", "head"),                   # 260
    ([31] * 40, 41, 5, 5, 16, "tree", "head"),
])
@pytest.mark.parametrize("dim", [144, 256])
def test_wide_heads(s, lengths, rows, heads, kv, page, mask, layout, dim, f8):
    Case(lengths, rows, heads, kv, dim, page, f8, layout, mask, seed=dim + rows).run(s).check()
    assert s.status() == 0


def test_masked_nan_in_wide_heads(s):
    rows = 70
    c = Case([90, 0, 333], rows, 2, 1, 256, 16, seed=2)
    for i in range(3):
        for j, what in ((2, NAN), (4, INF), (33, -INF), (40, NAN), (64, INF)):
            c.v_new[i * rows + j, :, j % 5::3] = what
        c.see[i][:, rows - 1] = False
        c.k_new[i * rows + rows - 1] = NAN
        c.v_new[i * rows + rows - 1] = NAN
    c.mask = torch.cat([words(x) for x in c.see])
    c.run(s).check()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,heads,kv,dim", [(3, 4, 2, 64), (9, 8, 2, 128), (70, 2, 1, 128), (40, 4, 2, 256)])
def test_nan_and_inf_in_queries(s, rows, heads, kv, dim, f8):
    """A row whose query holds a NaN, or an infinity that makes a score one, is NaN; the others are as they were."""
    c = Case([200, 0, 45], rows, heads, kv, dim, 16, f8, seed=dim)
    c.q[1, 0, 3] = NAN
    c.q[rows, heads - 1, 0] = NAN
    c.q[2 * rows + 1, 1, dim - 1] = INF
    hit = torch.zeros(3 * rows, heads, dtype=torch.bool)
    for r, h in ((1, 0), (rows, heads - 1), (2 * rows + 1, 1)):
        hit[r, h] = True
    c.run(s)
    o, lse = c.out["o"].cpu(), c.out["lse"].cpu()
    assert torch.isnan(o[hit]).all() and torch.isnan(lse[hit]).all()
    # the rest: the formula's (beside those queries' results without the NaN and the infinity)
    c.q[1, 0, 3] = c.q[rows, heads - 1, 0] = c.q[2 * rows + 1, 1, dim - 1] = 0.0
    c.run(s)
    c.out["o"][~hit.cuda()] = o[~hit].cuda()
    c.out["lse"][~hit.cuda()] = lse[~hit].cuda()
    c.check()


@pytest.mark.parametrize("rows,heads,kv,dim", [(3, 4, 2, 64), (9, 8, 2, 128), (9, 8, 2, 256)])
def test_nan_codes_in_an_8_bit_context(s, rows, heads, kv, dim):
    """NaN codes in a key, in a value and in a value's scale: their head's rows, their channel, their head's values."""
    c = Case([200, 60, 45, 45], rows, heads, kv, dim, 16, True, seed=dim)
    at = lambda i, t: (c.layer, int(c.table[c.slots[i], t // 16]))   # noqa: E731
    c.k[at(0, 77)].view(torch.uint8)[1, 77 % 16, 5] = 0xff
    c.v[at(1, 3)].view(torch.uint8)[0, 3, dim - 1] = 0x7f
    c.vs[at(2, 44)][1, 44 % 16] = NAN
    c.run(s).check()
    assert torch.isnan(c.out["o"].float()).any() and not torch.isnan(c.out["o"][3 * rows:].float()).any()


@pytest.mark.parametrize("rows,heads,dim,f8", [(256, 10, 64, True), (256, 9, 256, False), (256, 17, 128, False), (129, 9, 256, True)])
def test_more_row_tiles_than_a_launch(s, rows, heads, dim, f8):
    """Rows of one kv head past the 32 tiles that a launch takes."""
    Case([300, 70], rows, heads, 1, dim, 16, f8, seed=heads, layers=1).run(s).check(only=[0] if dim > 64 else None)
    assert s.status() == 0


@pytest.mark.parametrize("f8", [False, True])
def test_most_pairs(s, f8):
    """1024 sequences of 64 kv heads, the most of a call."""
    rng = random.Random(1)
    lengths = [rng.choice([0, 1, 15, 16, 40]) for _ in range(1024)]
    Case(lengths, 1, 64, 64, 16, 16, f8, seed=3, layers=1).run(s).check(only=[0, 1023, *rng.sample(range(1024), 14)])
    assert s.status() == 0
