"""The paged cache's row moves and the tree's verdict past what one dimension of a launch
counts: 2^32 threads. Most of the moves' requests ask for nothing; the first, one in the
middle and the last do."""
import pytest
import torch

from kv_util import Model
from locus_amd import sampler as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def s():
    x = S.Sampler(device=0, max_rows=64, max_vocab=4096, max_hist=64, max_top=4)
    x.kv_reserve(64)
    yield x
    x.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def pool(layers, heads, slots, tokens, seed):
    """A cache of 16-token pages whose slots hold `tokens` tokens each, and its model."""
    g = torch.Generator().manual_seed(seed)
    per = -(-tokens // 16)
    k, v = (torch.randn(layers, slots * per, heads, 16, 16, generator=g).bfloat16() for _ in range(2))
    table = torch.arange(slots * per, dtype=torch.int32).view(slots, per)
    refs = torch.ones(slots * per, dtype=torch.int32)
    dev = [t.cuda() for t in (k, v, table, refs)]
    return S.KvCache(*dev), dev, Model(k, v, table, refs)


def same(dev, model):
    for t, w in zip(dev[:2], model.rows):
        assert torch.equal(t.cpu().view(torch.int16), w.view(torch.int16))


@pytest.mark.parametrize("layers,heads,most,threads", [(17, 128, 257, 1024), (65, 128, 12, 256)])
def test_compact(s, layers, heads, most, threads):
    n = 1024
    assert n * layers * 2 * heads * threads > 1 << 32
    cache, dev, model = pool(layers, heads, 3, 20, layers)
    seq, count = [-1] * n, [0] * n
    keep = torch.zeros(n, most, dtype=torch.int32)
    for i, slot in ((0, 1), (500, 2), (n - 1, 0)):
        seq[i], count[i] = slot, 11
        keep[i, :11] = torch.tensor([0, 2, 3, 5, 8, 9, 13, 15, 16, 17, 19])
    result = ints([9] * n)
    s.kv_compact_dev(cache, ints(seq), ints(count), keep.cuda(), result)
    torch.cuda.synchronize()
    assert result.tolist() == model.compact(seq, count, keep.tolist()) == [0] * n and s.status() == 0
    same(dev, model)


@pytest.mark.parametrize("layers", [1, 3])
def test_append(s, layers):
    n, rows = 1024, 65540
    assert n * (-(-rows // 4)) * 256 > 1 << 32
    cache, dev, model = pool(4, 1, 3, 32, 7)
    g = torch.Generator().manual_seed(8)
    new = [torch.empty(n * rows, 1, 16, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    seq, pos, count = [-1] * n, [0] * n, [0] * n
    index = torch.zeros(n, rows, dtype=torch.int32, device="cuda")
    for i, slot, at, num in ((0, 2, 3, 9), (511, 0, 31, 1), (n - 1, 1, 13, 19)):
        seq[i], pos[i], count[i] = slot, at, num
        index[i, :num] = ints(range(rows - num, rows))
        for t, x in zip(new, model.rows):
            r = torch.randn(num, 1, 16, generator=g).bfloat16()
            t[i * rows + rows - num: (i + 1) * rows] = r.cuda()
            for j in range(num):
                x[1: 1 + layers, int(model.table[slot, (at + j) // 16]), :, (at + j) % 16] = r[j]
    # (a layer's rows are another's too: a stride of 0)
    k, v = (t.expand(layers, *t.shape) for t in new)
    s.kv_append_dev(cache, k, v, ints(seq), ints(pos), ints(count), rows_per_seq=rows, index=index, layer=1)
    torch.cuda.synchronize()
    assert s.status() == 0
    same(dev, model)


@pytest.mark.parametrize("n,rows", [((1 << 24) + 5, 1), (5600003, 3)])
def test_verdict(s, n, rows):
    """A workgroup of 256 threads a row: every row's argmax, every sequence's path."""
    assert n * rows * 256 > 1 << 32
    vocab = 8
    g = torch.Generator(device="cuda").manual_seed(n)
    logits = torch.randn(n * rows, vocab, generator=g, device="cuda").bfloat16()
    logits[:, 5] = -9.0
    best = torch.randint(0, 2, (n, rows), generator=g, device="cuda", dtype=torch.int32) * 5
    logits[torch.arange(n * rows, device="cuda"), best.view(-1).long()] = 30.0
    tokens = torch.randint(0, 2, (n, rows), generator=g, device="cuda", dtype=torch.int32) * 5
    parent = (torch.arange(rows, device="cuda", dtype=torch.int32) - 1).repeat(n, 1)
    hit = (tokens[:, 1:] == best[:, :-1]).int().cumprod(1)       # (a chain: the leading nodes that are right)
    taken = 1 + hit.sum(1, dtype=torch.int32)
    empty = lambda *sh: torch.full(sh, -7, device="cuda", dtype=torch.int32)   # noqa: E731
    out = {"argmax_ids": empty(n * rows), "path": empty(n, rows), "n_path": empty(n), "next_id": empty(n), "length": empty(n),
           "node_lp": torch.full((n * rows,), 7.0, device="cuda")}
    length = torch.arange(n, device="cuda", dtype=torch.int32)
    s.tree_verify_dev(tokens.view(-1), parent.reshape(-1), out, rows_per_seq=rows, logits=logits, length=length)
    torch.cuda.synchronize()
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    assert torch.equal(out["argmax_ids"].view(n, rows), best)
    assert torch.equal(out["n_path"], taken)
    assert torch.equal(out["path"], torch.where(at < taken[:, None], at, -1))
    assert torch.equal(out["next_id"], best.gather(1, (taken - 1)[:, None].long())[:, 0])
    assert torch.equal(out["length"], length + taken)
    # (a log-probability is 0 or -20 and less: which one tells the row; the normaliser is held to 1e-5, as lcs_verify's)
    lp = out["node_lp"].view(n, rows)
    assert (lp[:, 0] == 0).all()
    assert ((lp[:, 1:] > -1.0) == (tokens[:, 1:] == best[:, :-1])).all() and (lp <= 1e-5).all()


def test_verdict_of_argmaxes(s):
    """Without logits, a wave a sequence."""
    n = (1 << 26) + 7
    assert -(-n // 4) * 256 > 1 << 32
    best = torch.arange(n, device="cuda", dtype=torch.int32)
    zero = torch.zeros(n, device="cuda", dtype=torch.int32)
    out = {"argmax_ids": best.clone(), "path": torch.full((n, 1), -7, device="cuda", dtype=torch.int32),
           "n_path": torch.full((n,), -7, device="cuda", dtype=torch.int32), "next_id": torch.full((n,), -7, device="cuda", dtype=torch.int32)}
    s.tree_verify_dev(zero, zero - 1, out, rows_per_seq=1)
    torch.cuda.synchronize()
    assert (out["path"] == 0).all() and (out["n_path"] == 1).all()
    assert torch.equal(out["next_id"], best) and torch.equal(out["argmax_ids"], best)
