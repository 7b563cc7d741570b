"""The lm-head in 8 bits and with the rows' low-rank adapters (lcs_lmhead_ex).

Two gates, as for lcs_lmhead: on small integers (in e4m3, bf16 and the scales,
powers of two, exactly) every product and partial sum is an exact f32 integer
multiple of the scale, low-rank states fit 16 bits of mantissa, and the logits are
bit-exact; on random operands they are within the f32 bound of the float64
product. The statistics are held against the written logits."""
import numpy as np
import pytest

from tests.test_gpu_lmhead import check_epilogue

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# cases of each tile of lcs_lmhead_ex (rows, vocab, the tile's 64-column and row
# counts), full ones and with a row, a column and a row tile more or less;
# tests/test_lmhead_ex_shape.py holds the choice of the tile to this list (256 CUs)
TILES = [
    (3, 300, 1, 64), (64, 16384, 1, 64), (1, 20001, 2, 32), (32, 32768, 2, 32), (31, 33001, 4, 32), (17, 100001, 4, 32),
    (64, 20001, 2, 64), (33, 32768, 2, 64), (64, 33001, 4, 64), (47, 100001, 4, 64), (2, 80001, 5, 64), (64, 80001, 5, 64),
    (65, 140, 1, 64), (300, 1001, 1, 64), (128, 16001, 2, 64), (128, 20001, 2, 128), (300, 8001, 2, 128),
    (128, 50257, 4, 128), (300, 20001, 4, 128), (192, 50257, 4, 192),
    (150, 60000, 4, 192), (570, 21000, 4, 192), (256, 60000, 4, 256), (200, 50257, 4, 256), (511, 30000, 4, 256)]


@pytest.fixture(scope="module")
def sampler():
    from locus_amd.sampler import Sampler
    s = Sampler(device=0, max_rows=1100, max_vocab=262144, max_hist=64, max_top=4)
    yield s
    s.close()


def say(*a):
    print(*a, flush=True)


def ints(torch, gen, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=gen, device="cuda").float()


def powers(torch, gen, n):
    return torch.exp2(ints(torch, gen, -2, 2, n))


def call(sampler, x, w, out, ad=None, **kw):
    from locus_amd.sampler import Adapters
    if ad is not None:
        kw["slot"] = ad["slot"]
        ad = Adapters(ad["a"], ad["b"], rank=ad.get("rank"), scale=ad.get("scale"))
    sampler.lmhead_ex_dev(x, w, out, adapters=ad, **kw)
    sampler.torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in out.items()}


def whole(torch, gen, rows, vocab, hidden, f8, ranks=(), seed=0, per=1):
    """Integer operands, and the exact logits in float64."""
    t = torch.float8_e4m3fn if f8 else torch.bfloat16
    x, w = ints(torch, gen, -4, 4, rows, hidden), ints(torch, gen, -3, 3, vocab, hidden)
    ref = x.double() @ w.double().t()
    kw = {}
    if f8:
        kw["x_scale"], kw["w_scale"] = powers(torch, gen, rows), powers(torch, gen, vocab)
        ref = ref * kw["x_scale"].double()[:, None] * kw["w_scale"].double()
    ad = None
    if ranks:
        n, wide = len(ranks), (max(max(ranks), 1) + 7) // 8 * 8
        a = ints(torch, gen, -1, 1, n, wide, hidden)
        b = ints(torch, gen, -2, 2, n, vocab, wide)
        scale = powers(torch, gen, n)
        slot = torch.randint(-1, n + 1, (rows // per + 1,), generator=gen, device="cuda")   # (n: none, as -1)
        slot = slot.repeat_interleave(per)[:rows].to(torch.int32)
        xs = kw["x_scale"].double() if f8 else torch.ones(rows, device="cuda", dtype=torch.float64)
        for i, r in enumerate(ranks):
            mine = (slot == i).nonzero()[:, 0]
            if mine.numel() and r > 0:
                low = x[mine].double() @ a[i, :r].double().t() * scale[i].double() * xs[mine][:, None]
                ref[mine] += low @ b[i, :, :r].double().t()
            a[i, max(r, 0):], b[i, :, max(r, 0):] = float("nan"), float("nan")   # (never part of a result)
        ad = {"a": a.to(torch.bfloat16), "b": b.to(torch.bfloat16), "scale": scale, "slot": slot,
              "rank": torch.tensor(ranks, device="cuda", dtype=torch.int32)}
    return x.to(t), w.to(t), kw, ad, ref


def exact_case(sampler, rows, vocab, hidden, f8, ranks, seed, per=1):
    torch = sampler.torch
    say("exact", rows, vocab, hidden, "e4m3" if f8 else "bf16", ranks)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x, w, kw, ad, ref = whole(torch, gen, rows, vocab, hidden, f8, ranks, per=per)
    draft = torch.randint(0, vocab, (rows,), generator=gen, device="cuda").to(torch.int32)
    draft[0], draft[rows - 1] = -1, vocab
    out = sampler.alloc_lmhead_out(rows, vocab, draft=True, stats=True)
    g = call(sampler, x, w, out, ad, draft=draft, **kw)
    want = ref.float().cpu().numpy()
    bad = g["logits"] != want
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], g["logits"][bad][:3], want[bad][:3])
    assert np.array_equal(g["argmax_ids"], np.argmax(want, axis=1))
    check_lse(g, want, draft.cpu().numpy())
    # the statistics do not depend on writing the logits, nor on a call's history
    h = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab, logits=False, draft=True), ad, draft=draft, **kw)
    for k in ("argmax_ids", "log_z", "draft_lp"):
        assert np.array_equal(h[k], g[k]), k


def check_lse(g, logits, draft):
    l = logits.astype(np.float64)
    m = l.max(axis=1)
    lz = m + np.log(np.exp(l - m[:, None]).sum(axis=1))
    half = lambda v: 0.5 * np.spacing(np.abs(v).astype(np.float32))  # noqa: E731
    assert (np.abs(g["log_z"] - lz) <= 1e-5 + half(lz)).all()
    inside = (draft >= 0) & (draft < logits.shape[1])
    lp = np.where(inside, l[np.arange(len(l)), np.where(inside, draft, 0)] - lz, 0.0)
    assert (np.abs(g["draft_lp"] - lp) <= 1e-5 + half(lp)).all()
    if "stats" in g:
        s = g["stats"]
        assert (np.abs(s[:, 0] - lz) <= 1e-5).all()


# every tile, with fewer and more stages than its ring and a half stage at the end
@pytest.mark.parametrize("hidden", [64, 128, 192, 704, 1152])
@pytest.mark.parametrize("rows,vocab", [c[:2] for c in TILES])
def test_8_bits_exact(sampler, rows, vocab, hidden):
    exact_case(sampler, rows, vocab, hidden, True, (), rows + vocab + hidden)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab", [c[:2] for c in TILES])
def test_adapters_exact_on_every_tile(sampler, rows, vocab, f8):
    exact_case(sampler, rows, vocab, 448, f8, (8, 3, 16, 24, 70), rows * 3 + vocab)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab,hidden,ranks,per", [
    (1, 1, 64, (1,), 1), (1, 300, 64, (16,), 1), (2, 65, 128, (0, 5), 1), (5, 700, 192, (256,), 1),
    (33, 1000, 256, (128, 40), 1), (64, 513, 128, tuple(range(1, 65)), 1), (64, 200, 64, (8,) * 200, 1),
    (130, 257, 64, (20, 33, 7), 5), (1024, 300, 64, (16,) * 1024, 1), (1100, 500, 128, (12, 4, 30, 64, 100), 3),
    (1027, 40, 1024, (32,), 1), (640, 333, 64, (-3, 9, 50), 64), (7, 90, 4096, (17, 32), 1),
    # more ranks than a tile's LDS holds at a time, on each tile; hidden sizes past one and two rounds of lm_low
    (511, 30000, 128, (128, 40, 201), 1), (190, 50257, 64, (128, 40, 201), 1), (300, 20001, 64, (256, 30), 1), (128, 20001, 64, (256, 8), 1), (64, 80001, 64, (250,), 1),
    (64, 33001, 64, (256, 7), 1), (64, 20001, 64, (200, 16), 1), (32, 33001, 64, (256, 7), 1), (9, 20001, 64, (200, 16), 1), (64, 300, 64, (256, 100), 1),
    (300, 1001, 64, (256, 30), 1), (128, 16001, 64, (200, 16), 1),
    (5, 70, 4160, (16, 9), 1), (17, 100, 8256, (24,), 1),
    # the states' sums in one, two and four parts of the hidden size, a part in one round and in several
    (9, 70, 1600, (16, 9), 1), (70, 90, 2112, (20, 5), 1), (70, 90, 16448, (33,), 1), (150, 40, 4224, (64, 7) * 20, 1)])
def test_adapters_exact(sampler, rows, vocab, hidden, ranks, per, f8):
    exact_case(sampler, rows, vocab, hidden, f8, ranks, rows + vocab + len(ranks), per)


@pytest.mark.parametrize("f8", [False, True])
def test_no_row_and_every_row_adapted(sampler, f8):
    """Slots all outside the pool (also far outside), and all one adapter."""
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(8)
    rows, vocab, hidden = 70, 500, 128
    x, w, kw, ad, _ = whole(torch, gen, rows, vocab, hidden, f8, (16, 9))
    base = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab), None, **kw)
    for s in (-1, 2, 1 << 30, -(1 << 31)):
        ad["slot"] = torch.full((rows,), s, device="cuda", dtype=torch.int32)
        g = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab), ad, **kw)
        for k in base:
            assert np.array_equal(g[k], base[k]), (s, k)
    ad["slot"] = torch.ones(rows, device="cuda", dtype=torch.int32)
    g = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab), ad, **kw)
    low = x.double() @ ad["a"][1, :9].double().t() * ad["scale"][1].double()
    if f8:
        low = low * kw["x_scale"].double()[:, None]
    want = torch.from_numpy(base["logits"]).double() + (low @ ad["b"][1, :, :9].double().t()).cpu()
    assert np.array_equal(g["logits"], want.float().numpy())


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab", [(40, 300), (300, 700)])
def test_one_adapters_inf_and_nan_stay_with_its_rows(sampler, rows, vocab, f8):
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, w, kw, ad, _ = whole(torch, gen, rows, vocab, 128, f8, (16, 8, 24))
    ad["slot"] = (torch.arange(rows, device="cuda") % 4 - 1).to(torch.int32)
    good = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab), ad, **kw)
    for what in ("a", "b"):
        bad = dict(ad, **{what: ad[what].clone()})
        bad[what][1, 3 if what == "a" else slice(None), 2] = float("nan") if what == "a" else float("inf")
        g = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab), bad, **kw)
        mine = (ad["slot"] == 1).cpu().numpy()
        assert np.array_equal(g["logits"][~mine], good["logits"][~mine])
        assert np.array_equal(g["log_z"][~mine], good["log_z"][~mine])
        assert not np.isfinite(g["logits"][mine]).all(axis=1).any()
        assert ((g["argmax_ids"] >= 0) & (g["argmax_ids"] < vocab)).all()
    # an e4m3 or bf16 NaN in one row of x: that row only
    y = x.float()
    y[5, 9] = float("nan")
    g = call(sampler, y.to(x.dtype), w, sampler.alloc_lmhead_out(rows, vocab), ad, **kw)
    others = np.arange(rows) != 5
    assert np.array_equal(g["logits"][others], good["logits"][others]) and np.isnan(g["logits"][5]).all()


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("rows,vocab,hidden", [(3, 4000, 1024), (64, 20000, 2048), (130, 5000, 576), (300, 9000, 512)])
def test_random_operands_within_the_f32_bound(sampler, rows, vocab, hidden, f8):
    """f32 sums of exact products over hidden terms; a low-rank state's two bf16
    parts (2^-16) and its own sum; the scales' products."""
    torch = sampler.torch
    say("random", rows, vocab, hidden, f8)
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, hidden, generator=gen, device="cuda")
    w = torch.randn(vocab, hidden, generator=gen, device="cuda") * 0.05
    kw = {}
    if f8:
        xs, ws = x.abs().amax(1) / 448, w.abs().amax(1) / 448
        x, w = (x / xs[:, None]).to(torch.float8_e4m3fn), (w / ws[:, None]).to(torch.float8_e4m3fn)
        kw = {"x_scale": xs, "w_scale": ws}
    else:
        x, w = x.to(torch.bfloat16), w.to(torch.bfloat16)
    n, wide = 6, 40
    a = (torch.randn(n, wide, hidden, generator=gen, device="cuda") / hidden ** 0.5).to(torch.bfloat16)
    b = (torch.randn(n, vocab, wide, generator=gen, device="cuda") * 0.3).to(torch.bfloat16)
    slot = torch.randint(-1, n, (rows,), generator=gen, device="cuda").to(torch.int32)
    scale = torch.rand(n, generator=gen, device="cuda") * 3
    out = sampler.alloc_lmhead_out(rows, vocab)
    g = call(sampler, x, w, out, {"a": a, "b": b, "slot": slot, "scale": scale}, **kw)
    xd, wd = x.double(), w.double()
    if f8:
        xd, wd = xd * xs.double()[:, None], wd * ws.double()[:, None]
    ref, size = xd @ wd.t(), xd.abs() @ wd.abs().t()
    extra = torch.zeros_like(ref)
    for i in range(n):
        m = (slot == i).nonzero()[:, 0]
        low = xd[m] @ a[i].double().t() * scale[i].double()
        big = xd[m].abs() @ a[i].double().abs().t() * scale[i].double()
        ref[m] += low @ b[i].double().t()
        extra[m] += (big * (hidden * U) + low.abs() * 2.0 ** -16) @ b[i].double().abs().t()
        size[m] += low.abs() @ b[i].double().abs().t()
    bound = (hidden + 2 * wide + 8) * U * size + extra
    got = torch.from_numpy(g["logits"]).cuda().double()
    assert ((got - ref).abs() <= bound).all(), float(((got - ref).abs() / bound).max())
    check_epilogue(g)


@pytest.mark.parametrize("f8", [False, True])
def test_drafts_and_acceptance(sampler, f8):
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(11)
    seqs, per, vocab, hidden = 24, 8, 20000, 256
    rows = seqs * per
    x, w, kw, ad, _ = whole(torch, gen, rows, vocab, hidden, f8, (16, 32, 8), per=per)
    first = call(sampler, x, w, sampler.alloc_lmhead_out(rows, vocab), ad, **kw)
    am = torch.from_numpy(first["argmax_ids"]).view(seqs, per)
    draft = am.clone()
    prefix = [s % (per + 1) for s in range(seqs)]
    for s, p in enumerate(prefix):
        if p < per:
            draft[s, p] = (am[s, p] + 1) % vocab
    d = draft.reshape(-1).cuda()
    out = sampler.alloc_lmhead_out(rows, vocab, draft=True, n_seq=seqs)
    g = call(sampler, x, w, out, ad, draft=d, rows_per_seq=per, **kw)
    assert np.array_equal(g["logits"], first["logits"])
    check_epilogue(g, draft.reshape(-1).numpy(), per)
    assert g["accept_len"].tolist() == prefix


def test_bf16_without_adapters_is_lcs_lmhead(sampler):
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(37, 256, generator=gen, device="cuda").to(torch.bfloat16)
    w = torch.randn(3001, 256, generator=gen, device="cuda").to(torch.bfloat16)
    a, b = sampler.alloc_lmhead_out(37, 3001), sampler.alloc_lmhead_out(37, 3001)
    sampler.lmhead_dev(x, w, a)
    sampler.lmhead_ex_dev(x, w, b)
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("f8", [False, True])
def test_padded_and_unaligned_logits(sampler, f8):
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(13)
    rows, vocab = 20, 701
    x, w, kw, ad, ref = whole(torch, gen, rows, vocab, 128, f8, (16, 5))
    big = torch.full((rows, vocab + 6), -3.0, device="cuda")
    out = dict(sampler.alloc_lmhead_out(rows, vocab, logits=False), logits=big[:, 1:1 + vocab])
    call(sampler, x, w, out, ad, **kw)
    assert torch.equal(big[:, 1:1 + vocab], ref.float())
    assert (big[:, 0] == -3.0).all() and (big[:, 1 + vocab:] == -3.0).all()


def test_captured_into_a_graph(sampler):
    """Norm into 8 bits, the lm-head with adapters: captured once, replayed with new
    inputs and slots between eager calls, every replay as the eager result."""
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(14)
    from locus_amd.sampler import Adapters
    rows, vocab, hidden = 48, 2000, 512
    _, w, kw, ad, _ = whole(torch, gen, rows, vocab, hidden, True, (16, 8, 32))
    pool = Adapters(ad["a"], ad["b"], rank=ad["rank"], scale=ad["scale"])
    h = torch.randn(rows, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    r = torch.randn(rows, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    g = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)

    def buffers():
        n = {"y": torch.empty(rows, hidden, device="cuda", dtype=torch.float8_e4m3fn),
             "y_scale": torch.empty(rows, device="cuda"), "sum": torch.empty_like(h)}
        return n, sampler.alloc_lmhead_out(rows, vocab)

    def step(n, o, stream=None):
        sampler.add_rmsnorm_dev(h, g, n, residual=r, stream=stream)
        sampler.lmhead_ex_dev(n["y"], w, o, x_scale=n["y_scale"], w_scale=kw["w_scale"], adapters=pool, slot=ad["slot"],
                              stream=stream)

    n1, o1 = buffers()
    n2, o2 = buffers()
    step(n1, o1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(n2, o2)
    for i in range(4):
        h.normal_(generator=gen)
        ad["slot"].copy_(torch.randint(-1, 3, (rows,), generator=gen, device="cuda"))
        step(n1, o1)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in ((n1, n2), (o1, o2)):
            for k in a:
                assert torch.equal(a[k].view(torch.uint8), b[k].view(torch.uint8)), (i, k)


@pytest.mark.parametrize("f8", [False, True])
def test_on_a_side_stream_after_its_inputs(sampler, f8):
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(16)
    x, w, kw, ad, ref = whole(torch, gen, 50, 3000, 256, f8, (16, 5, 40))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    out = sampler.alloc_lmhead_out(50, 3000)
    st.wait_stream(torch.cuda.current_stream())
    from locus_amd.sampler import Adapters
    sampler.lmhead_ex_dev(x, w, out, adapters=Adapters(ad["a"], ad["b"], rank=ad["rank"], scale=ad["scale"]), slot=ad["slot"],
                          stream=st, **kw)
    st.synchronize()
    assert torch.equal(out["logits"], ref.float())


@pytest.mark.parametrize("f8", [False, True])
def test_pools_without_rank_and_scale(sampler, f8):
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(17)
    x, w, kw, ad, _ = whole(torch, gen, 20, 600, 128, f8, (24, 24))
    base = call(sampler, x, w, sampler.alloc_lmhead_out(20, 600), dict(ad, scale=torch.ones(2, device="cuda")), **kw)
    g = call(sampler, x, w, sampler.alloc_lmhead_out(20, 600), {"a": ad["a"], "b": ad["b"], "slot": ad["slot"]}, **kw)
    for k in base:
        assert np.array_equal(g[k], base[k]), k


def test_no_rows(sampler):
    torch = sampler.torch
    w = torch.zeros(100, 64, device="cuda", dtype=torch.bfloat16)
    sampler.lmhead_ex_dev(w[:0], w, {"argmax_ids": torch.zeros(0, device="cuda", dtype=torch.int32)})


def test_refusals_of_the_binding(sampler):
    from locus_amd.sampler import Adapters, SamplerError
    torch = sampler.torch
    gen = torch.Generator(device="cuda").manual_seed(15)
    x, w, kw, ad, _ = whole(torch, gen, 4, 100, 64, True, (8, 8))
    pool = Adapters(ad["a"], ad["b"])
    out = sampler.alloc_lmhead_out(4, 100)
    xb, wb = x.to(torch.bfloat16), w.to(torch.bfloat16)
    for args, more, text in [
            ((x, wb, out), {}, "both be"), ((x.float(), w.float(), out), {}, "both be"), ((x, w[:, :32], out), {}, "contiguous"),
            ((x.cpu(), w, out), {}, "device"), ((xb, wb, out), {"x_scale": kw["x_scale"]}, "scales go"),
            ((x, w, out), {"x_scale": kw["x_scale"].double()}, "x_scale"), ((x, w, out), {"w_scale": kw["w_scale"][:5]}, "w_scale"),
            ((x, w, out), {"adapters": pool}, "need slot"), ((x, w, out), {"slot": ad["slot"]}, "slot given"),
            ((x, w, out), {"adapters": pool, "slot": ad["slot"].long()}, "slot"),
            ((x, w[:90], out), {"adapters": pool, "slot": ad["slot"]}, "adapters'"),
            ((x, w, dict(out, argmax_ids=None)), {}, "argmax_ids"),
            ((x, w, dict(out, logits=out["logits"][:, :99])), {}, "logits must"),
            ((x, w, dict(out, log_z=out["log_z"][:2])), {}, "log_z")]:
        with pytest.raises(SamplerError, match=text):
            sampler.lmhead_ex_dev(*args, **more)
    with pytest.raises(SamplerError, match="multiple of 64"):
        sampler.lmhead_ex_dev(x[:, :32].contiguous(), w[:, :32].contiguous(), out)
    with pytest.raises(SamplerError, match="limits"):
        sampler.lmhead_ex_dev(x.repeat(300, 1), w, {"argmax_ids": torch.zeros(1200, device="cuda", dtype=torch.int32)})
