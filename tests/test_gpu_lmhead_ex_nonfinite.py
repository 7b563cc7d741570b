"""Infinities and NaNs in an adapter's second factor (lcs_lmhead_ex): the logits
have an inf, with its sign, or a NaN exactly where the formula
  logits[i][v] += sum_q low[i][q] b[slot i][v][q]
has one, and the statistics are those of the logits. In 64 bits the formula's
own terms decide: an inf times a state is an inf of the product's sign, times a
state of zero a NaN, and infs of both signs in one sum are a NaN.

Finite logits: on integers equal, bit for bit; on random operands within
(hidden + 2 ranks + 8) 2^-24 of the sums of magnitudes, for the product, and
hidden 2^-24 of a state's, for the adapters (f32 sums, each rounding half a step)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def sampler():
    from locus_amd.sampler import Sampler
    s = Sampler(device=0, max_rows=600, max_vocab=131072, max_hist=64, max_top=4)
    yield s
    s.close()


def ints(torch, gen, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=gen, device="cuda").float()


def spoil(torch, b, ranks):
    """Infs and NaNs at the first ranks and at the last one that counts, in columns over the whole width."""
    n, vocab, _ = b.shape
    for i in range(n):
        last = ranks[i] - 1
        for c0 in range(0, vocab, 61):
            for k, at in enumerate(((0, INF), (last, -INF), (0, -INF), (last, NAN))):
                c = c0 + 5 * k + i
                if c < vocab:
                    b[i, c, at[0]] = at[1]
            if c0 + 23 < vocab and last > 0:   # two in one column
                b[i, c0 + 23, 0], b[i, c0 + 23, last] = INF, INF if i % 2 else -INF


def problem(torch, rows, vocab, hidden, f8, ranks, whole, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.float8_e4m3fn if f8 else torch.bfloat16
    n, wide = len(ranks), (max(ranks) + 7) // 8 * 8
    if whole:   # states whose lower parts are zero, and some that are zero themselves
        x, w = ints(torch, gen, -2, 2, rows, hidden), ints(torch, gen, -3, 3, vocab, hidden)
        a = ints(torch, gen, -1, 1, n, wide, hidden) * (torch.rand(n, wide, hidden, generator=gen, device="cuda") < 0.05)
        b = ints(torch, gen, -2, 2, n, vocab, wide)
    else:       # states of 24 bits, whose parts may have either sign
        x, w = torch.randn(rows, hidden, generator=gen, device="cuda"), torch.randn(vocab, hidden, generator=gen, device="cuda")
        a = torch.randn(n, wide, hidden, generator=gen, device="cuda")
        b = torch.randn(n, vocab, wide, generator=gen, device="cuda")
    x, w, a, b = x.to(t), w.to(t), a.to(torch.bfloat16), b.to(torch.bfloat16)
    spoil(torch, b, ranks)
    scale = torch.tensor([1.0, -2.0, 0.5, 4.0][:n], device="cuda")
    slot = torch.randint(-1, n, (rows,), generator=gen, device="cuda").to(torch.int32)
    kw = {}
    if f8:
        kw = {"x_scale": torch.exp2(ints(torch, gen, -2, 2, rows)), "w_scale": torch.exp2(ints(torch, gen, -2, 2, vocab))}
    return x, w, a, b, scale, slot, kw


def formula(torch, x, w, a, b, scale, slot, kw, ranks):
    """The logits in 64 bits, and the size of what their roundings are relative to."""
    hidden = x.shape[1]
    xd, wd = x.double(), w.double()
    if kw:
        xd, wd = xd * kw["x_scale"].double()[:, None], wd * kw["w_scale"].double()[:, None]
    ref, size = xd @ wd.t(), (xd.abs() @ wd.abs().t()) * (hidden + 2 * max(ranks) + 8) * U
    for i, r in enumerate(ranks):
        m = (slot == i).nonzero()[:, 0]
        low = (xd[m] @ a[i, :r].double().t()) * scale[i].double()
        big = (xd[m].abs() @ a[i, :r].double().abs().t()) * scale[i].double().abs()
        bd = b[i, :, :r].double()
        for q in range(r):   # (term by term: a library product may skip zeros)
            ref[m] += low[:, q : q + 1] * bd[:, q]
            size[m] += (big[:, q : q + 1] * hidden * U + low[:, q : q + 1].abs() * (2 * r + 8) * U) * bd[:, q].abs()
    return ref, size


def statistics(g, draft):
    """The statistics against the written logits: NaNs have no part in the argmax, and
    a row with a NaN or +inf has a NaN for its log z, as lcs_lmhead's rows have."""
    l = g["logits"].astype(np.float64)
    known = np.where(np.isnan(l), -INF, l)
    assert np.array_equal(g["argmax_ids"], known.argmax(1))
    plain = ~np.isnan(l).any(1) & (l.max(1) < INF)
    top = np.where(plain, l.max(1), 0.0)
    with np.errstate(all="ignore"):
        lz = top + np.log(np.exp(l - top[:, None]).sum(1))
        lp = l[np.arange(len(l)), draft] - lz
    half = 0.5 * np.spacing(np.abs(lz[plain]).astype(np.float32))
    assert (np.abs(g["log_z"][plain] - lz[plain]) <= 1e-5 + half).all()
    assert np.isnan(g["log_z"][~plain]).all()
    low = plain & (lp == -INF)
    assert np.array_equal(g["draft_lp"][plain] == -INF, low[plain])
    ok = plain & ~low
    assert (np.abs(g["draft_lp"][ok] - lp[ok]) <= 2e-5 + 0.5 * np.spacing(np.abs(lp[ok]).astype(np.float32))).all()


def run(sampler, rows, vocab, hidden, f8, ranks, whole, seed, only=None):
    from locus_amd.sampler import Adapters
    torch = sampler.torch
    print("nonfinite", rows, vocab, hidden, "e4m3" if f8 else "bf16", ranks, "whole" if whole else "random", flush=True)
    x, w, a, b, scale, slot, kw = problem(torch, rows, vocab, hidden, f8, ranks, whole, seed)
    if only is not None:   # infs of one sign only, and no NaN
        b = torch.where(torch.isfinite(b.float()), b.float(), torch.full_like(b.float(), only)).to(torch.bfloat16)
    ref, size = formula(torch, x, w, a, b, scale, slot, kw, ranks)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    draft = torch.randint(0, vocab, (rows,), generator=gen, device="cuda").to(torch.int32)
    out = sampler.alloc_lmhead_out(rows, vocab, draft=True)
    pool = Adapters(a, b, rank=torch.tensor(ranks, device="cuda", dtype=torch.int32), scale=scale)
    sampler.lmhead_ex_dev(x, w, out, adapters=pool, slot=slot, draft=draft, **kw)
    torch.cuda.synchronize()
    got = out["logits"].double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (int(torch.isnan(got).sum()), int(torch.isnan(ref).sum()))
    for s in (INF, -INF):
        assert torch.equal(got == s, ref == s)
    if rows > 4:   # (fewer may be without an adapter, or with one of one rank)
        assert (ref == INF).any() and (ref == -INF).any() and (torch.isnan(ref).any() or only is not None)
    ok = torch.isfinite(ref)
    if whole:
        assert torch.equal(got[ok], ref[ok].float().double())
    else:
        assert ((got - ref).abs()[ok] <= size[ok]).all()
    statistics({k: v.cpu().numpy() for k, v in out.items()}, draft.cpu().numpy())


# a case of every tile, and ranks past a tile's share of LDS
@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab", [
    (5, 300), (9, 20001), (31, 33001), (64, 20001), (33, 33001), (2, 80001), (64, 80001), (70, 140), (128, 16001), (300, 8001),
    (128, 50257), (192, 50257), (200, 50257), (511, 30000)])
def test_nonfinite_factors(sampler, rows, vocab, f8, whole):
    run(sampler, rows, vocab, 64, f8, (16, 1, 9, 40), whole, rows + vocab)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab,hidden,ranks", [(40, 500, 1088, (8, 24)), (64, 33001, 64, (256, 7)), (300, 1001, 64, (200, 16))])
def test_nonfinite_factors_of_long_ranks(sampler, rows, vocab, hidden, ranks, f8):
    run(sampler, rows, vocab, hidden, f8, ranks, False, rows + vocab)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("sign", [INF, -INF])
def test_infinities_of_one_sign(sampler, sign, f8):
    run(sampler, 48, 2000, 128, f8, (16, 5), False, 7, only=sign)


@pytest.mark.parametrize("f8", [False, True])
def test_a_column_taken_out_by_minus_infinity(sampler, f8):
    """States above zero and factors of -inf: those columns are out, and log z is the others'."""
    from locus_amd.sampler import Adapters
    torch = sampler.torch
    rows, vocab, hidden, rank = 37, 3000, 128, 8
    gen = torch.Generator(device="cuda").manual_seed(3)
    t = torch.float8_e4m3fn if f8 else torch.bfloat16
    x, w = ints(torch, gen, 1, 4, rows, hidden).to(t), ints(torch, gen, -3, 3, vocab, hidden).to(t)
    a = torch.zeros(1, rank, hidden, device="cuda", dtype=torch.bfloat16)
    a[:, 0] = 0.3   # (0.30078125: states past 16 bits)
    b = torch.zeros(1, vocab, rank, device="cuda", dtype=torch.bfloat16)
    out_of = torch.rand(vocab, generator=gen, device="cuda") < 0.5
    b[0, out_of, 0] = -INF
    o = sampler.alloc_lmhead_out(rows, vocab)
    slot = torch.zeros(rows, device="cuda", dtype=torch.int32)
    sampler.lmhead_ex_dev(x, w, o, adapters=Adapters(a, b), slot=slot)
    torch.cuda.synchronize()
    ref = x.double() @ w.double().t()
    ref[:, out_of] = -INF
    assert torch.equal(o["logits"].double(), ref)
    assert torch.equal(o["argmax_ids"].long(), ref.argmax(1))
    lz = torch.logsumexp(ref, 1)
    assert ((o["log_z"].double() - lz).abs() <= 1e-5 + lz.abs() * U).all()
