"""The greedy verdict on trees of drafts (lcs_tree_verify) against a walk on the CPU."""
import pytest
import torch

from locus_amd import sampler as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def s():
    x = S.Sampler(device=0, max_rows=512, max_vocab=200000, max_hist=64, max_top=4)
    yield x
    x.close()


def walk(best, tokens, parent):
    path, cur = [0], 0
    while True:
        kids = [j for j in range(1, len(tokens)) if 0 <= parent[j] < j and parent[j] == cur and tokens[j] == best[cur]]
        if not kids:
            return path
        cur = kids[0]
        path.append(cur)


def out_of(n, rows, lp=True, length=True):
    i = lambda *sh: torch.full(sh, -77, device="cuda", dtype=torch.int32)   # noqa: E731
    o = {"argmax_ids": i(n * rows), "path": i(n, rows), "n_path": i(n), "next_id": i(n)}
    if lp:
        o["node_lp"] = torch.full((n * rows,), 7.0, device="cuda")
    if length:
        o["length"] = i(n)
    return o


def check(out, logits, tokens, parent, length, rows):
    n = tokens.numel() // rows
    best = logits.double().argmax(1)
    assert torch.equal(out["argmax_ids"].cpu().long(), best)
    z = torch.logsumexp(logits.double(), 1)
    for i in range(n):
        t, p = tokens[i * rows:][:rows].tolist(), parent[i * rows:][:rows].tolist()
        want = walk(best[i * rows:][:rows].tolist(), t, p)
        assert out["path"][i].tolist() == want + [-1] * (rows - len(want))
        assert out["n_path"][i].item() == len(want)
        assert out["next_id"][i].item() == best[i * rows + want[-1]].item()
        if "length" in out:
            assert out["length"][i].item() == length[i].item() + len(want)
        if "node_lp" in out:
            for j in range(rows):
                lp = 0.0
                if j > 0 and 0 <= p[j] < j and 0 <= t[j] < logits.shape[1]:
                    lp = (logits[i * rows + p[j], t[j]].double() - z[i * rows + p[j]]).item()
                # the rows' normaliser is held to 1e-5 as lcs_verify's, the result rounded to f32
                assert abs(out["node_lp"][i * rows + j].item() - lp) <= 1e-5 + abs(lp) * 2.0 ** -24


def case(n, rows, vocab, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(n * rows, vocab, generator=g) * 3
    tokens = torch.randint(0, min(vocab, 6), (n * rows,), generator=g)   # few ids: hits, twins among siblings
    for r in range(n * rows):
        logits[r, tokens[torch.randint(0, n * rows, (1,), generator=g)]] += 20
    logits = logits.to(dtype)
    up = torch.randint(1, 4, (n, rows), generator=g)
    parent = (torch.arange(rows) - up).clamp(min=-1)
    parent[:, 1:2] = 0
    if rows > 6:
        parent[0, 5], parent[0, 6] = 5, 99           # its own parent, and none at all
    tokens[-1] = -1
    if n * rows > 3:
        tokens[2] = vocab
    return logits, tokens.int(), parent.int().view(-1), torch.randint(0, 1000, (n,), generator=g).int()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,rows,vocab", [(1, 1, 7), (1, 2, 100), (3, 5, 1003), (7, 16, 50257), (2, 64, 32000), (3, 65, 4097), (2, 130, 5000),
                                          (1, 256, 1000), (33, 8, 128256), (5, 7, 8)])
def test_trees(s, n, rows, vocab, dtype):
    logits, tokens, parent, length = case(n, rows, vocab, dtype, n * rows + vocab)
    per = 4 if dtype == torch.float32 else 8
    wide = torch.full((n * rows, (vocab + per - 1) // per * per + 16), 1e4).to(dtype)
    wide[:, :vocab] = logits
    out = out_of(n, rows)
    s.tree_verify_dev(tokens.cuda(), parent.cuda(), out, rows_per_seq=rows, logits=wide.cuda()[:, :vocab], length=length.cuda())
    torch.cuda.synchronize()
    check(out, logits, tokens, parent, length, rows)
    # the same verdict from the argmax alone, the length in place
    again = out_of(n, rows, lp=False) | {"argmax_ids": out["argmax_ids"].clone(), "length": length.cuda()}
    s.tree_verify_dev(tokens.cuda(), parent.cuda(), again, rows_per_seq=rows, length=again["length"])
    torch.cuda.synchronize()
    check(again, logits, tokens, parent, length, rows)


def test_a_chain_is_lcs_verify(s):
    """Along a chain the accepted nodes are lcs_verify's accepted drafts, the logprobs its own."""
    n, rows, vocab = 6, 8, 32000
    logits, tokens, _, _ = case(n, rows, vocab, torch.float32, 5)
    tokens = tokens.clamp(0, vocab - 1).view(n, rows)
    best = logits.argmax(1).view(n, rows)
    for i in range(n):
        tokens[i, 1: 1 + i] = best[i, :i]            # sequence i's first i drafts are right
    parent = (torch.arange(rows) - 1).expand(n, rows).contiguous()
    out = out_of(n, rows, length=False)
    lg = logits.cuda()
    s.tree_verify_dev(tokens.view(-1).cuda(), parent.int().view(-1).cuda(), out, rows_per_seq=rows, logits=lg)
    draft = torch.cat([tokens[:, 1:], torch.full((n, 1), -1)], 1).int().contiguous().cuda()
    b = S._VBatch(n, rows, vocab, S.LCS_F32, vocab, lg.data_ptr(), draft.data_ptr())
    am, acc = (torch.empty(m, dtype=torch.int32, device="cuda") for m in (n * rows, n))
    lp = torch.empty(n * rows, device="cuda")
    s._check(S.lib().lcs_verify(s.ctx, b, S._VOut(am.data_ptr(), lp.data_ptr(), acc.data_ptr()), None))
    torch.cuda.synchronize()
    assert torch.equal(out["argmax_ids"], am)
    assert torch.equal(out["n_path"], acc + 1)
    assert torch.equal(out["node_lp"].view(n, rows)[:, 1:], lp.view(n, rows)[:, :-1])


def test_after_the_lm_head(s):
    """The verdict on the lm-head's argmax, no logits written."""
    n, rows, vocab, hidden = 4, 6, 5000, 128
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n * rows, hidden, device="cuda", generator=g).bfloat16()
    w = torch.randn(vocab, hidden, device="cuda", generator=g).bfloat16()
    out = out_of(n, rows, lp=False, length=False)
    s.lmhead_dev(x, w, {"argmax_ids": out["argmax_ids"]})
    torch.cuda.synchronize()
    best = out["argmax_ids"].cpu().view(n, rows)
    parent = torch.tensor([[0, 0, 0, 1, 3, 2]] * n, dtype=torch.int32)
    tokens = torch.full((n, rows), -1, dtype=torch.int32)
    for i in range(1, n):
        for j in ((1,), (1, 3), (1, 3, 4))[i - 1]:
            tokens[i, j] = best[i, parent[i, j]]
    s.tree_verify_dev(tokens.view(-1).cuda(), parent.view(-1).cuda(), out, rows_per_seq=rows)
    torch.cuda.synchronize()
    assert out["n_path"].tolist() == [1, 2, 3, 4]
    assert out["path"].tolist() == [[0, -1, -1, -1, -1, -1], [0, 1, -1, -1, -1, -1], [0, 1, 3, -1, -1, -1], [0, 1, 3, 4, -1, -1]]


def test_binding_refusals(s):
    i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")   # noqa: E731
    out = out_of(2, 3)
    lg = torch.zeros(6, 8, device="cuda")
    good = dict(rows_per_seq=3, logits=lg, length=i(2))
    s.tree_verify_dev(i(6), i(6), out, **good)
    torch.cuda.synchronize()
    for kw, o in [(dict(rows_per_seq=4), out), (dict(rows_per_seq=0), out), (dict(logits=lg[:5]), out), (dict(logits=lg.double()), out),
                  (dict(logits=lg.cpu()), out), (dict(logits=lg[:, ::2]), out), (dict(logits=lg[:, 1:]), out), (dict(length=None), out), (dict(length=i(3)), out),
                  (dict(logits=None), out), ({}, out | {"path": i(5)}), ({}, out | {"n_path": i(3)}), ({}, out | {"argmax_ids": i(6).float()})]:
        with pytest.raises(S.SamplerError):
            s.tree_verify_dev(i(6), i(6), o, **(good | kw))
    with pytest.raises(S.SamplerError):
        s.tree_verify_dev(i(6), i(5), out, **good)
