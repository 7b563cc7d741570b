"""The residual's addition and root-mean-square norm (lcs_add_rmsnorm) against
the formula in float64.

Tolerances: the sum of squares has at most 32 terms one after the other and ten
levels of a tree (relative 42 * 2^-24, half of it after the square root), the
division, the root, the reciprocal and two products add five roundings, h one:
64 * 2^-24 of |y| covers them; the rounding to y's type adds half a step (bf16
2^-8, e4m3 2^-4 or half of the smallest step, 2^-10 of the scale). The sum is one
f32 addition, rounded once: equal, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


@pytest.fixture(scope="module")
def sampler():
    from locus_amd.sampler import Sampler
    s = Sampler(device=0, max_rows=16, max_vocab=4096, max_hist=64, max_top=4)
    yield s
    s.close()


def types(torch):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def wide(torch, rows, hidden, pad, dtype, shift=0, fill=0.0):
    """A (rows, hidden) view into a buffer with `pad` elements between rows, starting `shift` elements in."""
    buf = torch.full((rows * (hidden + pad) + shift,), fill, device="cuda").to(dtype)
    return buf, torch.as_strided(buf, (rows, hidden), (hidden + pad, 1), shift)


def check(torch, x, res, w, y, scale, total, eps=EPS):
    h = x.double() if res is None else x.double() + res.double()
    if res is not None:
        assert torch.equal(total, (x.float() + res.float()).to(x.dtype))
    ref = h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    got = y.double()
    tol = 64 * U * ref.abs()
    if y.dtype == torch.bfloat16:
        tol = tol + ref.abs() * 2.0 ** -8
    elif y.dtype == torch.float8_e4m3fn:
        top = ref.abs().amax(1)
        s = torch.where(top > 0, top / 448.0, torch.ones_like(top))
        assert ((scale.double() - s).abs() <= 70 * U * s).all()
        got = got * scale.double()[:, None]
        tol = tol + torch.maximum(ref.abs() * 2.0 ** -4, s[:, None] * 2.0 ** -10) * (1 + 70 * U)
    bad = (got - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), got[bad][:4], ref[bad][:4])


def make(torch, rows, hidden, dtype, out, residual, pad, shift=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = types(torch)

    def rand(scale):
        _, v = wide(torch, rows, hidden, pad, t[dtype], shift)
        v.copy_(torch.randn(rows, hidden, generator=gen, device="cuda") * scale)
        return v

    x, res = rand(1.0), rand(3.0) if residual else None
    w = (1 + 0.2 * torch.randn(hidden, generator=gen, device="cuda")).to(t[dtype])
    buf, y = wide(torch, rows, hidden, pad, t[out], shift, fill=-7.0)
    o = {"y": y}
    sbuf = None
    if residual:
        sbuf, o["sum"] = wide(torch, rows, hidden, pad, t[dtype], shift, fill=-7.0)
    if out == "e4m3":
        o["y_scale"] = torch.full((rows,), -7.0, device="cuda")
    return x, res, w, o, buf, sbuf


@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,hidden,pad,shift", [
    (1, 1, 0, 0), (1, 7, 0, 0), (3, 8, 0, 0), (5, 9, 3, 1), (4, 64, 0, 0), (7, 511, 1, 0), (6, 512, 0, 0), (5, 513, 0, 3),
    (3, 1031, 7, 5), (9, 2048, 8, 0), (2, 2049, 0, 1), (3, 4096, 0, 0), (3, 4100, 1, 1), (2, 8192, 0, 0), (3, 8193, 6, 0),
    (2, 16384, 0, 0), (2, 16391, 1, 7), (1, 32768, 0, 0), (300, 48, 5, 0)])
def test_norm_against_float64(sampler, rows, hidden, pad, shift, dtype, out):
    torch = sampler.torch
    print("norm", rows, hidden, pad, shift, dtype, out, flush=True)
    for residual in (False, True):
        x, res, w, o, buf, sbuf = make(torch, rows, hidden, dtype, out, residual, pad, shift, seed=hidden + rows)
        sampler.add_rmsnorm_dev(x, w, o, residual=res, eps=EPS)
        torch.cuda.synchronize()
        check(torch, x, res, w, o["y"], o.get("y_scale"), o.get("sum"))
        for b in (buf, sbuf):   # what lies between the rows is left alone
            if b is not None:
                gap = torch.ones(b.shape, dtype=torch.bool, device="cuda")
                torch.as_strided(gap, (rows, hidden), (hidden + pad, 1), shift).fill_(False)
                assert (b.float()[gap] == torch.tensor(-7.0, device="cuda").to(b.dtype).float()).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hidden", [40, 2048, 5000])
def test_rows_of_zeros_and_extreme_values(sampler, hidden, dtype):
    torch = sampler.torch
    t = types(torch)[dtype]
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    x = torch.randn(8, hidden, generator=gen, device="cuda")
    x[0] = 0.0
    x[1] = 0.0
    x[1, hidden // 2] = 1e-20     # (eps alone makes the norm)
    x[2] *= 1e15                  # squares of 1e30
    x[3] *= 1e-30                 # squares below f32: y = h / sqrt(eps)
    x[4, 5] = 1e18                # one value far above the rest
    x = x.to(t)
    w = torch.ones(hidden, device="cuda").to(t)
    w[1] = 0.0
    w[3] = -2.0
    for out in ("f32", "e4m3"):
        o = {"y": torch.empty(8, hidden, device="cuda", dtype=types(torch)[out]), "y_scale": torch.empty(8, device="cuda")}
        sampler.add_rmsnorm_dev(x, w, o, eps=EPS)
        torch.cuda.synchronize()
        check(torch, x, None, w, o["y"], o["y_scale"], None)
        assert (o["y"][0].float() == 0).all()
        if out == "e4m3":
            assert o["y_scale"][0] == 1.0


@pytest.mark.parametrize("hidden", [40, 600, 4099])
def test_nan_and_inf_stay_where_the_formula_has_them(sampler, hidden):
    """Rows with a NaN or an inf, between rows without: NaN where h / sqrt(mean) w
    is one, 0 beside an inf; y_scale is 1 for a row whose largest |y| is a NaN."""
    torch = sampler.torch
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(5, hidden, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
        x[1, hidden - 1] = float("nan")
        x[3, 2] = float("-inf")
        x = x.to(dtype)
        w = torch.full((hidden,), 0.5, device="cuda").to(dtype)
        for out in (torch.float32, torch.bfloat16, torch.float8_e4m3fn):
            o = {"y": torch.empty(5, hidden, device="cuda", dtype=out), "y_scale": torch.empty(5, device="cuda")}
            sampler.add_rmsnorm_dev(x, w, o, eps=EPS)
            torch.cuda.synchronize()
            y = o["y"].float()
            assert torch.isnan(y[1]).all()
            assert torch.isnan(y[3, 2]) and (y[3, torch.arange(hidden, device="cuda") != 2] == 0).all()
            keep = [0, 2, 4]
            s = o["y_scale"][keep]
            check(torch, x[keep], None, w, o["y"].view(torch.uint8)[keep].view(out) if out == torch.float8_e4m3fn else o["y"][keep],
                  s, None)
            if out == torch.float8_e4m3fn:
                assert o["y_scale"][1] == 1.0 and o["y_scale"][3] == 1.0
    # a NaN of the weight: that column only
    w = torch.ones(hidden, device="cuda")
    w[7] = float("nan")
    x = torch.randn(3, hidden, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    o = {"y": torch.empty(3, hidden, device="cuda")}
    sampler.add_rmsnorm_dev(x, w, o)
    assert torch.isnan(o["y"][:, 7]).all() and torch.isfinite(o["y"][:, :7]).all() and torch.isfinite(o["y"][:, 8:]).all()


@pytest.mark.parametrize("hidden", [100, 4096, 20000])
def test_sum_in_place(sampler, hidden):
    """The sum over x or over the residual, as a residual stream is kept."""
    torch = sampler.torch
    for which in ("x", "residual"):
        x, res, w, o, _, _ = make(torch, 5, hidden, "bf16", "e4m3", True, 0, seed=3)
        ref = {k: v.clone() for k, v in o.items()}
        sampler.add_rmsnorm_dev(x, w, ref, residual=res)
        o["sum"] = x if which == "x" else res
        sampler.add_rmsnorm_dev(x, w, o, residual=res)
        for k in ref:
            assert torch.equal(o[k].view(torch.uint8), ref[k].view(torch.uint8)), (which, k)


def test_side_stream_and_no_rows(sampler):
    torch = sampler.torch
    x, res, w, o, _, _ = make(torch, 64, 4096, "bf16", "e4m3", True, 0, seed=4)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    sampler.add_rmsnorm_dev(x, w, o, residual=res, stream=st)
    st.synchronize()
    check(torch, x, res, w, o["y"], o["y_scale"], o["sum"])
    e = {"y": torch.empty(0, 4096, device="cuda", dtype=torch.bfloat16)}
    sampler.add_rmsnorm_dev(x[:0], w, e)


def test_refusals_of_the_binding(sampler):
    from locus_amd.sampler import SamplerError
    torch = sampler.torch
    x = torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)
    w = torch.zeros(64, device="cuda", dtype=torch.bfloat16)
    y = torch.zeros_like(x)
    for args, kw, text in [
            ((x.half(), w, {"y": y}), {}, "x must be"), ((x, w.float(), {"y": y}), {}, "weight"),
            ((x, w[:32], {"y": y}), {}, "weight"), ((x, w, {"y": y.half()}), {}, "y must be"),
            ((x, w, {"y": y[:3]}), {}, "y must be"), ((x.cpu(), w, {"y": y}), {}, "device"),
            ((x, w, {"y": y}), {"residual": x.float()}, "residual"), ((x, w, {"y": y}), {"residual": x.t()}, "residual"),
            ((x, w, {"y": y, "sum": y}), {}, "sum given"), ((x, w, {"y": y}), {"eps": 0.0}, "eps"),
            ((x, w, {"y": y.to(torch.float8_e4m3fn)}), {}, "y_scale")]:
        with pytest.raises(SamplerError, match=text):
            sampler.add_rmsnorm_dev(*args, **kw)
