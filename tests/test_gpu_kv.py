"""The paged cache's bookkeeping and row moves on the GPU (lcs_kv_*) against the model
of kv_util: tables, counts, results and every row bit by bit."""
import random

import pytest
import torch

from kv_util import Model, quantise
from locus_amd import sampler as S

pytestmark = pytest.mark.gpu
STATUS_PAGES = 8
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def s():
    x = S.Sampler(device=0, max_rows=64, max_vocab=4096, max_hist=64, max_top=4)
    x.kv_reserve(4096)
    yield x
    x.close()


def bits(t):
    return t.contiguous().view(torch.uint8)


class Pair:
    """A cache on the GPU beside the model of it."""

    def __init__(self, s, layers=2, pages=40, heads=3, page=16, dim=64, seqs=6, max_pages=9, f8=False, layout="head", seed=0):
        g = torch.Generator().manual_seed(seed)
        shape = (layers, pages, heads, page, dim)
        k, v = (torch.randn(shape, generator=g).bfloat16() for _ in range(2))
        k[0, 0, 0, 0, 0] = float("nan")
        v[-1, -1, -1, -1, -1] = float("inf")
        scales = {}
        if f8:
            (k, ks), (v, vs) = quantise(k.nan_to_num(1.0)), quantise(v.nan_to_num(1.0, 1.0))
            scales = {"k_scale": ks.contiguous(), "v_scale": vs.contiguous()}
        table = torch.full((seqs, max_pages), -1, dtype=torch.int32)
        refs = torch.zeros(pages, dtype=torch.int32)
        self.model = Model(k.clone(), v.clone(), table.clone(), refs.clone(), **{n: t.clone() for n, t in scales.items()})

        def put(t):
            if layout == "head":
                return t.cuda()
            if layout == "token":
                return t.transpose(2, 3).contiguous().cuda().transpose(2, 3)
            both = torch.zeros(layers, pages, 2, heads, page, dim, dtype=t.dtype)   # k and v of a page together
            return both.cuda()

        if layout == "both":
            buf = torch.stack([k, v], 2).contiguous().cuda()
            self.k, self.v = buf[:, :, 0], buf[:, :, 1]
        else:
            self.k, self.v = put(k), put(v)
        self.scales = {n: t.cuda() for n, t in scales.items()}
        self.table, self.refs = table.cuda(), refs.cuda()
        self.s, self.f8 = s, f8
        self.cache = S.KvCache(self.k, self.v, self.table, self.refs, **self.scales)

    def ints(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def call(self, fn, want, n, *args, **kw):
        r = torch.full((n,), 77, dtype=torch.int32, device="cuda")
        self.s.status()
        fn(self.cache, *args, r, **kw)
        torch.cuda.synchronize()
        assert r.tolist() == want
        assert self.s.status() == (STATUS_PAGES if -1 in want else 0)
        self.same()

    def same(self):
        m = self.model
        assert torch.equal(self.table.cpu(), m.table)
        assert torch.equal(self.refs.cpu(), m.refs)
        for t, w in zip([self.k, self.v, *self.scales.values()], m.rows):
            assert torch.equal(bits(t.cpu()), bits(w))

    def grow(self, seq, start, end, cap=4096):
        self.call(self.s.kv_grow_dev, self.model.grow(seq, start, end, cap), len(seq), self.ints(seq), self.ints(start), self.ints(end))

    def fork(self, src, dst, tokens):
        self.call(self.s.kv_fork_dev, self.model.fork(src, dst, tokens), len(src), self.ints(src), self.ints(dst), self.ints(tokens))

    def free(self, seq, keep=None):
        self.call(self.s.kv_free_dev, self.model.free(seq, keep), len(seq), self.ints(seq), None if keep is None else self.ints(keep))

    def compact(self, seq, count, keep):
        k = torch.tensor(keep, dtype=torch.int32, device="cuda")
        self.call(self.s.kv_compact_dev, self.model.compact(seq, count, keep), len(seq), self.ints(seq), self.ints(count), k)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("layout", ["head", "token", "both"])
@pytest.mark.parametrize("page,dim", [(16, 16), (16, 80), (32, 128), (64, 256)])
def test_grow_fork_free(s, page, dim, layout, f8):
    c = Pair(s, page=page, dim=dim, layout=layout, f8=f8, pages=30)
    c.grow([0, 1, 2], [0, 0, 5], [3 * page, 2 * page + 1, page])
    c.grow([0, 1], [3 * page, 2 * page + 1], [3 * page, 2 * page + 5])        # (nothing to do, and inside a page)
    c.fork([0, 1, 0], [3, 4, 5], [3 * page - 1, 2 * page + 1, page])
    c.grow([3, 4, 0], [3 * page - 1, 2 * page + 1, 0], [3 * page + 2, 3 * page, 2])   # copies: tails, and a first page
    c.free([5, 3], [0, page])
    c.grow([-1, 5], [0, 0], [5, 1])
    c.free([0, 1, 2, 3, 4, 5, -1])
    assert c.refs.sum().item() == 0


def test_both_holders_grow(s):
    """Two holders of a page that ask in one call both get copies, and the page is free again."""
    c = Pair(s)
    c.grow([0], [0], [20])
    c.fork([0], [1], [20])
    c.grow([0, 1], [20, 20], [21, 21])
    assert c.refs.tolist().count(1) == 2 and c.refs.max().item() == 2


def test_out_of_pages(s):
    """From the first request that there are not enough pages for, none is served."""
    c = Pair(s, pages=12)
    c.grow([0, 1, 2, 3], [0, 0, 0, 0], [5 * 16, 5 * 16, 3 * 16, 16])    # 5 + 5 + 3 > 12: slots 2 and 3 refused
    c.grow([3], [0], [2 * 16])
    c.grow([4, 0], [0, 0], [1, 5 * 16])      # none left: refused, and the request after it too, though it asks for none
    c.free([1])
    c.grow([4], [0], [5 * 16])


def test_few_new_pages_reserved():
    """A call gives out no more pages than lcs_kv_reserve made room for."""
    x = S.Sampler(device=0, max_rows=8, max_vocab=4096, max_hist=64, max_top=4)
    x.kv_reserve(3)
    c = Pair(x)
    c.grow([0, 1, 2], [0, 0, 0], [32, 32, 16], cap=3)
    c.grow([1, 2], [0, 0], [32, 16], cap=3)
    x.kv_reserve(4)
    c.grow([3], [0], [64], cap=4)
    x.close()


def test_refused_requests(s):
    c = Pair(s, seqs=6, max_pages=4)
    top = 4 * 16
    c.grow([0, 6, -2, 0, 1, 2, 3], [0, 0, 0, 0, 5, -1, 0], [33, 5, 5, 9, 4, 3, top + 1])
    c.grow([1, 2], [0, 0], [top, 1])
    c.fork([0, 0, 3, 0, 1, 9, 0], [3, 3, 4, 2, 9, 4, 4], [33, 33, 1, 33, 16, 1, 49])   # twice, a dst, held, outside, missing
    c.fork([0, -1, 1], [5, 3, -1], [0, 5, 5])
    c.fork([2], [2], [1])
    c.fork([0], [4], [-1])
    c.free([0, 0, 7, -1, -5], [16, 0, 0, 0, 0])
    c.free([1, 2], [1000, -3])


@pytest.mark.parametrize("n", [1, 2, 17, 64, 200, 1024])
def test_many_requests(s, n):
    """Every number of lanes a request; long ranges; the pages' order over many rounds of the search."""
    c = Pair(s, layers=1, heads=1, page=16, dim=16, pages=n * 5 + 40000, seqs=n + 1, max_pages=8)
    rng = random.Random(n)
    c.refs[rng.randrange(30):37000] = 1     # most of the pool held by somebody
    c.model.refs.copy_(c.refs.cpu())
    seq = rng.sample(range(n + 1), n)
    start = [rng.randrange(0, 64) for _ in seq]
    end = [min(128, a + rng.randrange(0, 80)) for a in start]
    c.grow(seq, start, end)
    c.free(seq[: n // 2], [rng.randrange(0, 100) for _ in seq[: n // 2]])
    c.grow(seq, start, end)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("layout", ["head", "token", "both"])
@pytest.mark.parametrize("page,dim", [(16, 16), (16, 96), (32, 128), (64, 256), (16, 240)])
def test_compact(s, page, dim, layout, f8):
    c = Pair(s, page=page, dim=dim, layout=layout, f8=f8, pages=40, max_pages=20)
    rng = random.Random(page + dim)
    lengths = [20 * page, 7 * page + 3, page + 1, 1]
    c.grow([0, 1, 2, 3], [0] * 4, lengths)
    keep = [sorted(rng.sample(range(n), max(1, n * f // 10))) for n, f in zip(lengths, (6, 5, 10, 10))]
    wide = max(map(len, keep))
    pad = lambda k: k + [-1] * (wide - len(k))   # noqa: E731
    c.compact([0, 1, -1, 2, 3], [len(keep[0]), len(keep[1]), 4, len(keep[2]), 1],
              [pad(keep[0]), pad(keep[1]), pad([]), pad(keep[2]), pad(keep[3])])
    c.compact([0, 1], [0, -5], [pad([]), pad([])])
    c.compact([0], [10 ** 6], [list(range(wide))])


def test_compact_refused(s):
    c = Pair(s, max_pages=4)
    c.grow([0, 1], [0, 0], [64, 40])
    c.fork([0], [2], [64])
    c.compact([0, 1, 1, 6, -3], [2, 2, 2, 2, 2], [[0, 5], [3, 7], [3, 7], [0, 1], [0, 1]])     # shared; fine; twice; outside
    c.compact([1, 2], [2, 2], [[0, 1], [0, 1]])               # (nothing moves: a shared page may stay)
    c.compact([1], [3], [[0, 5, 5]])
    c.compact([1], [3], [[4, 9, 8]])
    c.compact([1], [2], [[-1, 3]])
    c.compact([1], [2], [[0, 64]])
    c.compact([1], [2], [[0, 50]])                            # (past its pages)
    c.grow([2], [0], [64])
    c.compact([2, 0], [2, 2], [[7, 20], [3, 4]])


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("layout", ["head", "token", "both"])
@pytest.mark.parametrize("page,dim,heads", [(16, 16, 3), (16, 80, 1), (32, 128, 8), (64, 256, 2), (128, 240, 5)])
def test_append(s, page, dim, heads, layout, f8):
    c = Pair(s, page=page, dim=dim, heads=heads, layout=layout, f8=f8, layers=3, pages=20, max_pages=3)
    g = torch.Generator().manual_seed(dim)
    seq, pos, rows = [2, -1, 0, 5], [0, 3, page - 3, 2 * page - 1], 37
    count = [rows, 5, 20 if page > 16 else 18, 1]
    pos = [min(p, 3 * page - n) for p, n in zip(pos, count)]
    c.grow([2, 0, 5], [0, 0, 0], [min(3 * page, 37), min(3 * page, page + 40), 2 * page])
    # rows cut out of a wider buffer; widths that bf16 does not hold exactly in 8 bits, a row of zeros, a NaN, an infinity
    buf = torch.randn(2, 4 * rows, 2 * heads * dim + 16, generator=g).bfloat16()
    buf[:, 3] = 0.0
    buf[0, 5, 1] = float("nan")
    buf[1, 6, 2] = float("-inf")
    buf[:, 7] *= 1e-30
    buf[:, 8] *= 1e30
    new = buf.cuda()
    k, v = (new[:, :, 8 + i * heads * dim:][:, :, : heads * dim].unflatten(2, (heads, dim)) for i in (0, 1))
    index = torch.stack([torch.randperm(rows, generator=g) for _ in range(4)]).int()
    for use in (None, index):
        for cnt in (count, None):
            if cnt is None and (page < 64 or use is None):
                continue
            p = pos if cnt else [0, 0, 0, 0]
            m = c.model
            c.s.status()
            c.s.kv_append_dev(c.cache, k, v, c.ints(seq), c.ints(p), None if cnt is None else c.ints(cnt), rows_per_seq=rows,
                              index=None if use is None else use.cuda(), layer=1)
            torch.cuda.synchronize()
            if cnt is None:
                c.model = m
            for i, q in enumerate(seq):
                for j in range((cnt or [rows] * 4)[i] if q >= 0 else 0):
                    r = i * rows + (j if use is None else int(use[i, j]))
                    pg, off = int(m.table[q, (p[i] + j) // page]), (p[i] + j) % page
                    for t, x in ((0, k), (1, v)):
                        x = x[:, r].cpu()
                        if f8:
                            x, sc = quantise(x)
                            m.rows[2 + t][1:3, pg, :, off] = sc
                        m.rows[t][1:3, pg, :, off] = x
            if f8:   # (a NaN is one whatever its bits)
                for t, w in zip((c.k, c.v), m.rows):
                    assert torch.equal(torch.isnan(t.float()).cpu(), torch.isnan(w.float()))
                    assert torch.equal(t.float().cpu().nan_to_num(), w.float().nan_to_num())
                for t, w in zip(c.scales.values(), m.rows[2:]):
                    assert torch.equal(t.cpu(), w)
                assert torch.equal(c.table.cpu(), m.table) and torch.equal(c.refs.cpu(), m.refs)
            else:
                c.same()
            assert c.s.status() == 0


def test_append_where_it_may_not(s):
    """Missing and shared pages, positions and indexes out of range: nothing is written, and the status says so."""
    c = Pair(s, max_pages=4)
    c.grow([0, 1], [0, 0], [40, 16])
    c.fork([1], [2], [16])
    new = torch.randn(2, 7 * 2, 3, 64, device="cuda").bfloat16()
    for seq, pos, count, index in [([1], [0], [2], None), ([2], [3], [1], None), ([0], [48], [2], None), ([0], [-2], [2], None),
                                   ([0], [64], [1], None), ([0], [2 ** 31 - 1], [2], None), ([6], [0], [1], None), ([-2], [0], [1], None),
                                   ([3], [0], [1], None), ([0], [0], [1], [[7, 0, 0, 0, 0, 0, 0]]), ([0], [0], [1], [[-1, 0, 0, 0, 0, 0, 0]])]:
        s.status()
        s.kv_append_dev(c.cache, new[:, :7], new[:, 7:], c.ints(seq), c.ints(pos), c.ints(count), rows_per_seq=7,
                        index=None if index is None else c.ints(index))
        torch.cuda.synchronize()
        assert s.status() == STATUS_PAGES, (seq, pos)
        c.same()
    s.kv_append_dev(c.cache, new[:, :7], new[:, 7:], c.ints([0]), c.ints([5]), c.ints([-4]), rows_per_seq=7)
    torch.cuda.synchronize()
    assert s.status() == 0
    c.same()


def test_no_requests(s):
    c = Pair(s)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    s.kv_grow_dev(c.cache, none, none, none, none)
    s.kv_fork_dev(c.cache, none, none, none, none)
    s.kv_free_dev(c.cache, none, None, none)
    s.kv_append_dev(c.cache, torch.empty(2, 0, 3, 64, device="cuda", dtype=torch.bfloat16),
                    torch.empty(2, 0, 3, 64, device="cuda", dtype=torch.bfloat16), none, none, rows_per_seq=4)
    torch.cuda.synchronize()
    c.same()


def test_without_reserve():
    x = S.Sampler(device=0, max_rows=8, max_vocab=4096, max_hist=64, max_top=4)
    c = Pair(x)
    one = c.ints([0])
    with pytest.raises(S.SamplerError, match="reserve"):
        x.kv_grow_dev(c.cache, one, one, one, one.clone())
    x.close()


@pytest.mark.parametrize("seed", range(4))
def test_random_runs(s, seed):
    """Calls of every kind in a row, good and bad requests mixed."""
    rng = random.Random(seed)
    c = Pair(s, layers=2, pages=rng.choice([20, 60]), heads=2, page=16, dim=32, seqs=7, max_pages=6, f8=seed % 2 == 1, seed=seed)
    for _ in range(25):
        n = rng.randint(1, 7)
        seq = [rng.choice([-1, rng.randrange(7), rng.randrange(7), rng.randrange(8)]) for _ in range(n)]
        kind = rng.choice(["grow", "grow", "fork", "free", "compact"])
        if kind == "grow":
            start = [rng.randrange(0, 90) for _ in seq]
            c.grow(seq, start, [min(96, a + rng.randrange(0, 60)) for a in start])
        elif kind == "fork":
            c.fork([rng.randrange(7) for _ in seq], seq, [rng.randrange(0, 60) for _ in seq])
        elif kind == "free":
            c.free(seq, rng.choice([None, [rng.randrange(0, 90) for _ in seq]]))
        else:
            keep = [sorted(rng.sample(range(rng.choice([30, 60, 96])), 20)) for _ in seq]
            c.compact(seq, [rng.randint(0, 20) for _ in seq], keep)


@pytest.mark.parametrize("f8", [False, True])
def test_far_pages(s, f8):
    """Places past 2^32 bytes: rows appended to the last pages of a large pool, copied on write and compacted there."""
    pages, heads, page, dim = (24576, 8, 128, 128) if not f8 else (36864, 8, 128, 128)
    shape = (1, pages, heads, page, dim)
    k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn if f8 else torch.bfloat16, device="cuda") for _ in range(2))
    assert k.numel() * k.element_size() > 1 << 32
    scales = {n: torch.empty(shape[:4], device="cuda") for n in ("k_scale", "v_scale")} if f8 else {}
    refs = torch.ones(pages, dtype=torch.int32, device="cuda")
    refs[-5:] = 0
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    c = S.KvCache(k, v, table, refs, **scales)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    g = torch.Generator().manual_seed(1)
    new = [torch.randn(1, 200, heads, dim, generator=g).bfloat16() for _ in range(2)]
    r = [ints(9) for _ in range(4)]
    s.status()
    s.kv_grow_dev(c, ints(0), ints(0), ints(200), r[0])
    s.kv_append_dev(c, new[0].cuda(), new[1].cuda(), ints(0), ints(0), rows_per_seq=200)
    s.kv_fork_dev(c, ints(0), ints(1), ints(200), r[1])
    s.kv_grow_dev(c, ints(1), ints(0), ints(200), r[2])
    keep = sorted(random.Random(2).sample(range(200), 150))
    s.kv_compact_dev(c, ints(1), ints(150), torch.tensor([keep], dtype=torch.int32, device="cuda"), r[3])
    torch.cuda.synchronize()
    assert [int(x) for x in r] == [0] * 4 and s.status() == 0
    assert table.tolist() == [[pages - 5, pages - 4, -1], [pages - 3, pages - 2, -1]] and refs[-5:].tolist() == [1, 1, 1, 1, 0]
    for slot, rows in ((0, list(range(200))), (1, keep)):
        at = table[slot, :2].long()
        for t, n, sc in ((k, new[0], "k_scale"), (v, new[1], "v_scale")):
            want, scale = quantise(n[0, rows]) if f8 else (n[0, rows], None)
            held = t[0, at].permute(0, 2, 1, 3).reshape(2 * page, heads, dim)[: len(rows)].cpu()
            assert torch.equal(bits(held), bits(want))
            if f8:
                assert torch.equal(scales[sc][0, at].permute(0, 2, 1).reshape(2 * page, heads)[: len(rows)].cpu(), scale)


def test_side_stream_and_graph(s):
    """Pages and rows on a side stream, and in two graphs of one context that are replayed in turn with eager calls between."""
    pairs = [Pair(s, pages=60, max_pages=6, seed=i) for i in range(4)]
    rows, dim = 9, 64
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(2, 3 * rows, 3, dim, generator=g).bfloat16().cuda() for _ in range(2))
    seq = pairs[0].ints([2, 0, 5])
    state = [{"start": c.ints([0, 3, 40]), "end": c.ints([9, 12, 49]), "res": c.ints([9] * 3)} for c in pairs]

    def step(c, st, stream=None):
        s.kv_grow_dev(c.cache, seq, st["start"], st["end"], st["res"], stream=stream)
        s.kv_append_dev(c.cache, k, v, seq, st["start"], rows_per_seq=rows, stream=stream)

    graphs = []
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for c, st in zip(pairs[:2], state):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(c, st)
        graphs.append(gr)
    for i in range(4):
        for a in (0, 1):
            if i == 2:
                step(pairs[a], state[a], side)
                side.synchronize()
            else:
                graphs[a].replay()
            torch.cuda.synchronize()
            step(pairs[2 + a], state[2 + a])
            torch.cuda.synchronize()
            assert torch.equal(state[a]["res"], state[2 + a]["res"])
            assert torch.equal(pairs[a].table, pairs[2 + a].table) and torch.equal(pairs[a].refs, pairs[2 + a].refs)
            used = pairs[a].table[pairs[a].table >= 0].long()
            for x, y in ((pairs[a].k, pairs[2 + a].k), (pairs[a].v, pairs[2 + a].v)):
                x, y = x[:, used], y[:, used]
                same = x.view(torch.int16) == y.view(torch.int16)
                filled = torch.zeros(x.shape[:4], dtype=torch.bool, device="cuda")
                for j, q in enumerate(seq.tolist()):
                    for p in range(int(state[a]["start"][j]), int(state[a]["end"][j])):
                        page = int(pairs[a].table[q, p // 16])
                        filled[:, (used == page).nonzero()[0, 0], :, p % 16] = True
                assert bool(same[filled].all())
        for st in state:
            st["start"] += 9
            st["end"] += 9
    assert s.status() == 0


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("layers,heads,dim,page,length,most", [(1, 1, 256, 32, 6000, 5000), (2, 3, 80, 16, 1100, 1024), (1, 2, 128, 64, 900, 257), (1, 2, 128, 16, 900, 256)])
def test_compact_long(s, layers, heads, dim, page, length, most, f8):
    """Lists of several rounds of a workgroup's rows, on both sides of what makes it wide, dense and thin."""
    pages = -(-length // page)
    c = Pair(s, layers=layers, pages=2 * pages + 2, heads=heads, page=page, dim=dim, seqs=3, max_pages=pages, f8=f8)
    c.grow([0, 1], [0, 0], [length, length])
    rng = random.Random(most)
    keep = [sorted(rng.sample(range(length), most)), sorted(rng.sample(range(length // 2 + most // 2), most))]
    c.compact([0, 1], [most, most - 3], keep)
    c.compact([0, 1], [most // 2, most], [sorted(rng.sample(range(most), most // 2)) + [0] * (most - most // 2), list(range(most))])


def test_append_finite_beside_a_nan(s):
    """A row that holds a NaN is stored with a scale of 1: what else it holds stays itself up to 448, which bounds the rest."""
    c = Pair(s, layers=1, heads=2, dim=32, f8=True, pages=8)
    c.grow([0], [0], [16])
    row = torch.linspace(-30.0, 30.0, 32)
    row[:12] = torch.tensor([NAN, 447.0, 448.0, 449.0, 480.0, 500.0, 1e4, 3e38, -500.0, -3e38, INF, -INF])
    k = torch.stack([row, torch.linspace(-900.0, 900.0, 32)]).bfloat16()[None, None].expand(1, 3, 2, 32).contiguous()
    k[0, 1, 1, 5] = -NAN                                     # (in one row of the others too)
    s.kv_append_dev(c.cache, k.cuda(), k.cuda(), c.ints([0]), c.ints([2]), rows_per_seq=3)
    torch.cuda.synchronize()
    want, scale = quantise(k[0])
    assert torch.isfinite(want[0, 0].float()).sum() == 31    # (the oracle's own: the NaN alone is one)
    page = int(c.table[0, 0])
    for t, sc in ((c.k, "k_scale"), (c.v, "v_scale")):
        got = t[0, page, :, 2:5].transpose(0, 1).float().cpu()
        assert torch.equal(c.scales[sc][0, page, :, 2:5].t().cpu(), scale)
        assert torch.equal(torch.isnan(got), torch.isnan(want.float()))
        assert torch.equal(got.nan_to_num(), want.float().nan_to_num())


def test_padding_behind_a_shortage(s):
    """Behind a request that there are not enough pages for, every result of lcs_kv_grow is -1, a slot of -1's too; ahead of it
    and in calls without a shortage that slot's is 0."""
    c = Pair(s, pages=8)
    c.grow([-1, 0, -1, 1, -1], [0] * 5, [5, 64, 5, 80, 5])    # 4 + 5 > 8
    r = c.ints([7] * 5)
    c.s.kv_grow_dev(c.cache, c.ints([-1, 1, -1, 2, -1]), c.ints([0] * 5), c.ints([0, 80, 9, 0, 0]), r)
    torch.cuda.synchronize()
    assert r.tolist() == [0, -1, -1, -1, -1] and s.status() == STATUS_PAGES
    c.same()
    c.grow([-1, 1, -1], [0] * 3, [5, 64, 5])


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("layers,heads,page,dim", [(1, 1024, 16, 16), (300, 1, 16, 32), (2, 3, 1024, 48)])
def test_largest_layouts(s, layers, heads, page, dim, f8):
    """Many heads, many layers, the longest pages: rows appended, copied on write and compacted."""
    c = Pair(s, layers=layers, heads=heads, page=page, dim=dim, f8=f8, pages=8, max_pages=3)
    n = page + 7
    c.grow([0], [0], [n])
    k, v = (torch.randn(layers, n, heads, dim, generator=torch.Generator().manual_seed(i)).bfloat16() for i in (1, 2))
    s.kv_append_dev(c.cache, k.cuda(), v.cuda(), c.ints([0]), c.ints([0]), rows_per_seq=n)
    for t, x in ((0, k), (1, v)):
        sc = None
        if f8:
            x, sc = quantise(x)
        for j in range(n):
            pg, off = int(c.model.table[0, j // page]), j % page
            c.model.rows[t][:, pg, :, off] = x[:, j]
            if f8:
                c.model.rows[2 + t][:, pg, :, off] = sc[:, j]
    torch.cuda.synchronize()
    c.same()
    c.fork([0], [1], [n])
    c.grow([1], [0], [n])
    c.compact([1], [n // 2], [list(range(0, n // 2 * 2, 2))])
