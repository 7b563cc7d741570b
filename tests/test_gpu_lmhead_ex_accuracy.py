"""How near lcs_lmhead_ex's logits come to the product in 64 bits: closer than
sums of fewer than f32's 24 bits, or low-rank states of fewer than three bf16
parts, can come.

On random operands, of the logits' norm. A sum of k products of random signs has
at most k / 4 roundings one after the other (four in an instruction of 16), each
off by at most 2^-24 of a partial sum, whose square grows in proportion to its
terms: 2^-24 sqrt(k / 8) of the sum. A logit: that for hidden, and the two products of
its scales. An adapter's part: that for hidden (its states), for three times its rank
(their parts), and four more for the join of a state's summands, its two scales and
the addition. Sums of 8 products in 14 bits miss the first bound by ten times, states
of two parts the second by twice: the CPU tests below hold them to it.

On integers whose products differ by 2^16 in one group of 8, and states of 20
bits, every f32 sum is exact: equal, bit for bit."""
import math

import numpy as np
import pytest

U = 2.0 ** -24


def sum_bound(k):
    return U * math.sqrt(k / 8)


def product_bound(hidden):
    return sum_bound(hidden) + 2 * U


def adapter_bound(hidden, rank):
    return sum_bound(hidden) + sum_bound(3 * rank) + 4 * U


@pytest.fixture(scope="module")
def sampler():
    from locus_amd.sampler import Sampler
    s = Sampler(device=0, max_rows=600, max_vocab=131072, max_hist=64, max_top=4)
    yield s
    s.close()


def to_type(torch, v, f8):
    """Rows as operands, and in 8 bits their scales."""
    if not f8:
        return v.to(torch.bfloat16), None
    s = v.abs().amax(1) / 448
    return (v / s[:, None]).to(torch.float8_e4m3fn), s


def off(got, ref):
    return float((got - ref).norm() / ref.norm())


# a case of every tile (rows, vocab)
TILES = [(3, 300), (9, 20001), (31, 33001), (64, 20001), (33, 33001), (64, 80001), (70, 140), (128, 16001), (300, 8001),
         (128, 50257), (192, 50257), (256, 60000)]


@pytest.mark.gpu
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab", TILES)
def test_products(sampler, rows, vocab, f8):
    torch = sampler.torch
    hidden = 1024
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    x, xs = to_type(torch, torch.randn(rows, hidden, generator=gen, device="cuda"), f8)
    w, ws = to_type(torch, torch.randn(vocab, hidden, generator=gen, device="cuda"), f8)
    out = sampler.alloc_lmhead_out(rows, vocab)
    sampler.lmhead_ex_dev(x, w, out, x_scale=xs, w_scale=ws)
    ref = x.double() @ w.double().t()
    if f8:
        ref *= xs.double()[:, None] * ws.double()
    got = off(out["logits"].double(), ref)
    print("product", rows, vocab, "e4m3" if f8 else "bf16", "%.3g of %.3g" % (got, product_bound(hidden)), flush=True)
    assert got <= product_bound(hidden)


@pytest.mark.gpu
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("hidden,rank", [(256, 32), (512, 16), (2112, 64)])
@pytest.mark.parametrize("rows,vocab", TILES)
def test_adapters(sampler, rows, vocab, hidden, rank, f8):
    """Logits that are the adapters' (a weight of zeros)."""
    from locus_amd.sampler import Adapters
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab + hidden)
    x, xs = to_type(torch, torch.randn(rows, hidden, generator=gen, device="cuda"), f8)
    w = torch.zeros(vocab, hidden, device="cuda", dtype=x.dtype)
    a, b = (torch.randn(3, *s, generator=gen, device="cuda").to(torch.bfloat16) for s in ((rank, hidden), (vocab, rank)))
    scale = torch.rand(3, generator=gen, device="cuda") + 0.5
    slot = (torch.arange(rows, device="cuda") % 3).to(torch.int32)
    out = sampler.alloc_lmhead_out(rows, vocab)
    sampler.lmhead_ex_dev(x, w, out, x_scale=xs, adapters=Adapters(a, b, scale=scale), slot=slot)
    ref = torch.empty(rows, vocab, device="cuda", dtype=torch.float64)
    for i in range(3):
        m = slot == i
        low = x[m].double() @ a[i].double().t() * scale[i].double()
        ref[m] = (low * xs[m].double()[:, None] if f8 else low) @ b[i].double().t()
    got = off(out["logits"].double(), ref)
    bound = adapter_bound(hidden, rank)
    print("adapters", rows, vocab, hidden, rank, "e4m3" if f8 else "bf16", "%.3g of %.3g" % (got, bound), flush=True)
    assert got <= bound


def ints(torch, gen, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=gen, device="cuda").float()


@pytest.mark.gpu
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab", TILES)
def test_products_far_apart_in_one_group(sampler, rows, vocab, f8):
    """One product of +-2^16 in each 8 neighbours, the others up to 9: no sum above 2^24."""
    torch = sampler.torch
    hidden = 1024
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    t = torch.float8_e4m3fn if f8 else torch.bfloat16
    x, w = ints(torch, gen, -3, 3, rows, hidden), ints(torch, gen, -3, 3, vocab, hidden)
    big = torch.arange(0, hidden, 8, device="cuda") + torch.randint(0, 8, (hidden // 8,), generator=gen, device="cuda")
    for v in (x, w):
        v[:, big] = 256.0 * (2 * ints(torch, gen, 0, 1, v.shape[0], hidden // 8) - 1)
    out = sampler.alloc_lmhead_out(rows, vocab)
    sampler.lmhead_ex_dev(x.to(t), w.to(t), out)
    assert torch.equal(out["logits"].double(), x.double() @ w.double().t())


@pytest.mark.gpu
@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab", TILES)
def test_states_of_20_bits(sampler, rows, vocab, f8):
    from locus_amd.sampler import Adapters
    torch = sampler.torch
    hidden, rank = 1024, 8
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab)
    t = torch.float8_e4m3fn if f8 else torch.bfloat16
    x, w = ints(torch, gen, 0, 15, rows, hidden), ints(torch, gen, -3, 3, vocab, hidden)
    a, b = ints(torch, gen, 0, 255, 2, rank, hidden), ints(torch, gen, -1, 1, 2, vocab, rank)
    b[:, :, 3:] = 0.0   # (three states at a time: sums below 2^24)
    slot = (torch.arange(rows, device="cuda") % 2).to(torch.int32)
    out = sampler.alloc_lmhead_out(rows, vocab)
    sampler.lmhead_ex_dev(x.to(t), w.to(t), out, adapters=Adapters(a.to(torch.bfloat16), b.to(torch.bfloat16)), slot=slot)
    ref = x.double() @ w.double().t()
    low = torch.einsum("rk,nqk->nrq", x.double(), a.double())
    assert (low >= 2.0 ** 18).all() and (low.abs().amax() * 3 + ref.abs().amax()) < 2.0 ** 24
    for i in range(2):
        m = slot == i
        ref[m] += low[i][m] @ b[i].double().t()
    assert torch.equal(out["logits"].double(), ref)


@pytest.mark.gpu
@pytest.mark.parametrize("max_rows,rows,wide,hidden", [(1, 1, 256, 8256), (5, 5, 256, 4224), (300, 300, 256, 8256), (520, 520, 200, 4224)])
def test_contexts_of_the_calls_own_rows(max_rows, rows, wide, hidden):
    """The states in as many parts of the hidden size as the context's scratch holds, up to its end."""
    from locus_amd.sampler import Adapters, Sampler
    s = Sampler(device=0, max_rows=max_rows, max_vocab=300, max_hist=1, max_top=1)
    torch = s.torch
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x, w = ints(torch, gen, -4, 4, rows, hidden), ints(torch, gen, -3, 3, 300, hidden)
    a, b = ints(torch, gen, -1, 1, 1, wide, hidden), ints(torch, gen, -2, 2, 1, 300, wide)
    out = s.alloc_lmhead_out(rows, 300)
    slot = torch.zeros(rows, device="cuda", dtype=torch.int32)
    for _ in range(2):
        s.lmhead_ex_dev(x.to(torch.bfloat16), w.to(torch.bfloat16), out,
                        adapters=Adapters(a.to(torch.bfloat16), b.to(torch.bfloat16)), slot=slot)
        assert torch.equal(out["logits"].double(), x.double() @ w.double().t() + (x.double() @ a[0].double().t()) @ b[0].double().t())
    s.close()


# ---------------------------------------------- what the bounds have to see --
def test_the_product_bound_sees_sums_of_14_bits():
    """8 neighbouring products cut 13 bits below the largest of them, the groups added in 64 bits."""
    torch = pytest.importorskip("torch")
    hidden, gen = 1024, torch.Generator().manual_seed(1)
    x, w = (to_type(torch, torch.randn(40, hidden, generator=gen), True)[0].double() for _ in range(2))
    p = (x[:, None] * w[None]).view(40, 40, hidden // 8, 8)
    top = p.abs().amax(-1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 13)
    err = off((torch.trunc(p / step) * step).sum((2, 3)), p.sum((2, 3)))
    print("%.3g against %.3g" % (err, product_bound(hidden)))
    assert err > 5 * product_bound(hidden)


def test_the_adapter_bound_sees_states_of_two_parts():
    rng = np.random.default_rng(2)
    for hidden, rank in ((256, 32), (512, 16)):
        low = (rng.standard_normal((60, hidden)) @ rng.standard_normal((hidden, rank))).astype(np.float32)
        b = rng.standard_normal((500, rank))

        def part(v, nearest):
            u = v.astype(np.float32).view(np.uint32)
            u = u + (0x7fff + ((u >> 16) & 1) if nearest else np.uint32(0))
            return (u.astype(np.uint32) & np.uint32(0xffff0000)).view(np.float32)

        for nearest in (False, True):
            one = part(low, nearest)
            two = one + part(low - one, nearest)
            ref = low.astype(np.float64) @ b.T
            err = np.linalg.norm(two.astype(np.float64) @ b.T - ref) / np.linalg.norm(ref)
            print("%.3g against %.3g" % (err, adapter_bound(hidden, rank)))
            assert err > 2 * adapter_bound(hidden, rank)
