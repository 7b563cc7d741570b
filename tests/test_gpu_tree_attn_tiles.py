"""lcs_tree_attn where a wave walks many tiles of cached tokens, every form of the kernel:
contexts several times what the card's workgroups take a step of, against the formula in
64 bits on the GPU.

Values are zero but in the channel that a token's step of 128 and its place name, and
positive there, so that the bound on an output, which is relative to sum_j p_j |v_j|, is
relative to a few tokens' share: a value row that is lost, doubled or misplaced shows. (16
to 64 tokens share a channel, so that one has about a 64th of an output or more, and the
bound is a 128th. In the longest contexts a lost tile shows, a fortieth.)
Tolerances as in test_gpu_tree_attn.py. Where values are normal, the error's norm is
bounded too: two roundings to bf16, of the weights and of the result, are each
uniform within half a step, 2^-8 of the value at most, and independent: 2^-8 / sqrt(3)
of sqrt(o^2 + sum_j p_j^2 v_j^2) a channel; a quarter more for the sample.
"""
import math

import pytest
import torch

from kv_util import quantise
from locus_amd import sampler as S

pytestmark = pytest.mark.gpu
NAN = float("nan")
CLASSES = 16


@pytest.fixture(scope="module")
def s():
    x = S.Sampler(device=0, max_rows=64, max_vocab=4096, max_hist=64, max_top=4)
    x.kv_reserve(64)
    yield x
    x.close()


def form_of(rows, pairs, dim, f8, cus):
    """What a call runs: (padded dim, 16-row tiles of a wave, waves that share a tile, tiles at once)."""
    dp = 64 if dim <= 64 else 128 if dim <= 128 else 256
    if rows <= 16:
        return dp, 1, 1, 4
    if dp != 256 and not f8:
        if rows > (128 if dp == 64 else 64) and (rows - 1) % 128 >= 64:
            return dp, 2, 4, 2
        if rows > 128 or (rows > 32 and pairs * 2 >= cus):
            return dp, 2, 2, 2
    if dp == 256 and not f8 and rows > 32:
        return dp, 1, 4, 2
    return dp, 2, 1, 4


def tiles_of(lengths, new, rows, kv, form, cus):
    """How many tiles of cached tokens a wave walks in a row, of every stretch of one sequence and head."""
    dp, mt, wr, nw = form
    per_cu = (1 if dp == 256 else 2) if nw * wr == 4 else 1
    pieces = min(cus, 256) * per_cu // min(32, -(-rows // (16 * mt * wr))) // 8 * 8 or 8
    steps = [-(-n // 128) + -(-new // 128) for n in lengths]
    share, unit = max(1, -(-sum(steps) * kv // pieces)), 1
    if len(lengths) <= 64 and share > 1:
        for u in range(share, share + 4):
            if sum(-(-t // u) for t in steps) * kv <= pieces:
                unit, share = u, 1
                break
    found, x = set(), 0
    for n, t in zip(lengths, steps):
        units = -(-t // unit)
        for _ in range(kv):
            at = 0
            while at < units:
                end = min(units, at + share - x % share)
                found.add((min(-(-n // 128), end * unit) - at * unit) * (4 // nw))
                x += end - at
                at = end
    return found


class Long:
    def __init__(self, lengths, new, heads, kv, dim, page, f8, rise=0.0, sparse=True, seed=0):
        self.lengths, self.new, self.heads, self.kv, self.dim, self.page, self.f8 = lengths, new, heads, kv, dim, page, f8
        self.sparse = sparse
        n, self.scale = len(lengths), dim ** -0.5
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        used = [-(-x // page) for x in lengths]
        first = [sum(used[:i]) for i in range(n)]
        pages = sum(used) + 3
        tok = torch.full((pages, page), -1, device="cuda")
        for x, p, u in zip(lengths, first, used):
            flat = torch.arange(u * page, device="cuda")
            tok[p: p + u] = torch.where(flat < x, flat, -1).view(u, page)
        k, v = self.rows(tok, rise)
        order = torch.randperm(pages, generator=g, device="cuda")
        at = order.argsort()                       # (logical page l lies at order[l])
        self.k, self.v = k[at].transpose(1, 2).contiguous()[None], v[at].transpose(1, 2).contiguous()[None]
        self.ks = self.vs = None
        if f8:
            (self.k, self.ks), (self.v, self.vs) = quantise(self.k), quantise(self.v)
            self.ks, self.vs = self.ks.contiguous(), self.vs.contiguous()
        gone = (tok[at] < 0)[None, :, None, :].expand(self.k.shape[:4])
        for t in (self.k, self.v):
            t.view(torch.uint8 if f8 else torch.int16)[gone] = 0x7f if f8 else 0x7fc0
        for t in (self.ks, self.vs):
            if t is not None:
                t[gone] = NAN
        self.table = torch.full((n, max(used) + 1), -1, dtype=torch.int32, device="cuda")
        for i in range(n):
            self.table[i, : used[i]] = order[first[i]: first[i] + used[i]].int()
        new_tok = torch.tensor(lengths, device="cuda")[:, None] + torch.arange(new, device="cuda")
        self.k_new, self.v_new = (t.reshape(n * new, kv, dim) for t in self.rows(new_tok, rise))
        self.q = (torch.randn(n * new, heads, dim, generator=g, device="cuda") * 0.5).bfloat16()
        self.q[..., 0] = 4.0
        self.cache = S.KvCache(self.k, self.v, self.table, torch.ones(pages, dtype=torch.int32, device="cuda"),
                               **({"k_scale": self.ks, "v_scale": self.vs} if f8 else {}))
        self.out = {"o": torch.full_like(self.q, 3.0), "lse": torch.full((n * new, heads), 5.0, device="cuda")}

    def rows(self, tok, rise):
        """Keys whose score rises by 2^rise from step to step, and values, of tokens (.., kv, dim)."""
        shape = (*tok.shape, self.kv, self.dim)
        k = torch.randn(shape, generator=self.g, device="cuda") * 0.5
        k[..., 0] = (tok // 128 * rise / (math.log2(math.e) * self.scale * 4.0))[..., None]
        if not self.sparse:
            return k.bfloat16(), torch.randn(shape, generator=self.g, device="cuda").bfloat16()
        d = torch.arange(self.dim, device="cuda")
        here = (d % CLASSES == (tok // 128 % CLASSES)[..., None]) & (d // CLASSES == (tok % (self.dim // CLASSES))[..., None])
        v = here[..., None, :] * (1.0 + torch.rand((*tok.shape, self.kv, 1), generator=self.g, device="cuda"))
        return k.bfloat16(), v.bfloat16()

    def run(self, s):
        s.status()
        s.tree_attn_dev(self.q, self.k_new, self.v_new, self.cache, self.out, length=torch.tensor(self.lengths, dtype=torch.int32, device="cuda"),
                        rows_per_seq=self.new)
        torch.cuda.synchronize()
        assert s.status() == 0
        return self

    def context(self, t, sc, i):
        at = self.table[i, : -(-self.lengths[i] // self.page)].long()
        x = t[0, at].double() if sc is None else t[0, at].float().double() * sc[0, at].double()[..., None]
        return x.transpose(0, 1).reshape(self.kv, at.numel() * self.page, self.dim)[:, : self.lengths[i]]

    def check(self, only):
        group, N, u = self.heads // self.kv, self.new, 2.0 ** -8
        for i in only:
            mine = slice(i * N, (i + 1) * N)
            K = torch.cat([self.context(self.k, self.ks, i), self.k_new[mine].double().transpose(0, 1)], 1)
            V = torch.cat([self.context(self.v, self.vs, i), self.v_new[mine].double().transpose(0, 1)], 1)
            terms = K.shape[1]
            see = torch.ones(N, terms, dtype=torch.bool, device="cuda")
            see[:, terms - N:] = torch.ones(N, N, device="cuda").tril().bool()
            for h in range(self.kv):
                q = self.q[mine, h * group: (h + 1) * group].double().reshape(N * group, self.dim)
                s = (torch.matmul(q, K[h].t().contiguous()) * self.scale).masked_fill(~see.repeat_interleave(group, 0), -math.inf)
                lse = torch.logsumexp(s, 1)
                p = torch.exp(s - lse[:, None])
                o, weigh = torch.matmul(p, V[h]), torch.matmul(p, V[h].abs())
                most = (torch.matmul(q.abs(), K[h].abs().t().contiguous()).amax(1) * self.scale)
                got = self.out["o"][mine, h * group: (h + 1) * group].double().reshape(o.shape)
                got_l = self.out["lse"][mine, h * group: (h + 1) * group].double().reshape(-1)
                score = 2.0 ** -24 * (self.dim + 8) * most
                assert ((got_l - lse).abs() <= score + 2.0 ** -24 * (terms + lse.abs()) + 2.0 ** -21).all(), (i, h)
                weight = 2 * score + 2.0 ** -24 * terms + 2.0 ** -20
                tol = (u * (o.abs() + (1 + u) * weigh) + weight[:, None] * weigh) * (1 + u) + 2.0 ** -133
                bad = (got - o).abs() / tol
                assert (bad <= 1).all(), (i, h, bad.max().item(), (bad > 1).nonzero()[:4].tolist())
                if not self.sparse:
                    norm = (o.square() + torch.matmul(p.square(), V[h].square())).sum().sqrt()
                    assert (got - o).norm() <= 1.25 * u / math.sqrt(3.0) * norm, (i, h, ((got - o).norm() / norm).item())
        return self


def uneven(n, lo, hi):
    return [lo + (hi - lo) * ((7 * i) % n) // max(1, n - 1) + i % 3 for i in range(n)]


# sequences, new tokens, heads, kv heads, dim, e4m3, the form
FORMS = [
    (32, 2, 16, 8, 64, False, (64, 1, 1, 4)), (32, 6, 32, 8, 48, False, (64, 2, 1, 4)), (8, 50, 32, 8, 64, False, (64, 2, 4, 2)),
    (20, 10, 32, 8, 64, False, (64, 2, 2, 2)),
    (32, 2, 16, 8, 128, False, (128, 1, 1, 4)), (32, 6, 32, 8, 80, False, (128, 2, 1, 4)), (16, 25, 32, 8, 128, False, (128, 2, 4, 2)),
    (20, 10, 32, 8, 112, False, (128, 2, 2, 2)),
    (16, 4, 16, 8, 256, False, (256, 1, 1, 4)), (16, 6, 32, 8, 144, False, (256, 2, 1, 4)), (16, 10, 32, 8, 256, False, (256, 1, 4, 2)),
    (32, 4, 16, 8, 64, True, (64, 1, 1, 4)), (32, 8, 32, 8, 64, True, (64, 2, 1, 4)), (32, 1, 8, 8, 96, True, (128, 1, 1, 4)),
    (32, 8, 32, 8, 128, True, (128, 2, 1, 4)), (16, 3, 16, 8, 256, True, (256, 1, 1, 4)), (16, 8, 32, 8, 240, True, (256, 2, 1, 4)),
]


def planned(lengths, new, heads, kv, dim, f8, form, least):
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    rows = new * heads // kv
    assert form_of(rows, len(lengths) * kv, dim, f8, cus) == form
    found = tiles_of(lengths, new, rows, kv, form, cus)
    assert max(found) >= least, found
    return found


@pytest.mark.parametrize("rise", [0.0, 3.0, -3.0])
@pytest.mark.parametrize("n,new,heads,kv,dim,f8,form", FORMS)
def test_many_tiles(s, n, new, heads, kv, dim, f8, form, rise):
    """Scores alike, and rising or falling by 2^3 a step: what lies 2^8 above the running maximum moves it."""
    # (as many tokens as give each workgroup four or five steps)
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    dp, mt, wr, nw = form
    slots = min(cus, 256) * ((1 if dp == 256 else 2) if nw * wr == 4 else 1) // -(-(new * heads // kv) // (16 * mt * wr))
    mean = slots * 9 // 2 * 128 // (n * kv)
    lengths = uneven(n, mean // 2, mean * 3 // 2)
    found = planned(lengths, new, heads, kv, dim, f8, form, 5 if wr == 1 else 6)
    assert len(found) >= 3 and {x // (4 // nw) % 2 for x in found} == {0, 1}, found    # (odd and even numbers of steps)
    Long(lengths, new, heads, kv, dim, 16, f8, rise=rise, seed=dim + new).run(s).check([0, 1, n // 2, n - 1])


@pytest.mark.parametrize("n,new,heads,kv,dim,f8,form", FORMS)
def test_error_norm(s, n, new, heads, kv, dim, f8, form):
    lengths = uneven(n, 500, 1900)
    planned(lengths, new, heads, kv, dim, f8, form, 2)
    Long(lengths, new, heads, kv, dim, 32, f8, sparse=False, seed=dim + new + 1).run(s).check([1, n - 1])


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("n,new,dim,rise", [(70, 1, 128, 0.0), (130, 4, 64, 3.0), (300, 2, 80, -3.0)])
def test_more_sequences_than_lanes(s, n, new, dim, rise, f8):
    """Several sequences a lane of the line of steps: stretches of many tiles that begin and end anywhere."""
    lengths = uneven(n, 0, 2 * 40000 // n)
    found = planned(lengths, new, 16, 8, dim, f8, (64 if dim == 64 else 128, 1, 1, 4), 3)
    assert len(found) >= 3
    Long(lengths, new, 16, 8, dim, 16, f8, rise=rise, seed=n).run(s).check([0, 1, n // 3, n // 2, n - 1])


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("new,dim,rise", [(1, 128, 0.0), (2, 64, 0.5), (8, 256, -0.5)])
def test_one_long_sequence(s, new, dim, rise, f8):
    """Every workgroup has a piece of one context."""
    lengths = [20011 + 128 * new]
    Long(lengths, new, 8, 2, dim, 64, f8, rise=rise, seed=dim).run(s).check([0])
