"""lcs_add_rmsnorm at the ends of its range. Tolerances as in test_gpu_norm.py: 64 2^-24 of |y| for the f32 arithmetic,
half a step for the rounding to y's type."""
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def sampler():
    from locus_amd.sampler import Sampler
    s = Sampler(device=0, max_rows=16, max_vocab=4096, max_hist=64, max_top=4)
    yield s
    s.close()


@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_more_rows_than_one_launch_has_threads(sampler, out):
    """2^26 + 5 rows of a wave each: past 2^32 threads."""
    torch = sampler.torch
    rows, hidden = (1 << 26) + 5, 2
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    r = torch.randn(rows, hidden, generator=gen, device="cuda").to(torch.bfloat16)
    w = torch.tensor([1.0, -0.5], device="cuda").to(torch.bfloat16)
    o = {"y": torch.full((rows, hidden), 3.0, device="cuda").to(torch.bfloat16 if out == "bf16" else torch.float8_e4m3fn),
         "sum": torch.full_like(x, 3.0)}
    if out == "e4m3":
        o["y_scale"] = torch.full((rows,), -7.0, device="cuda")
    sampler.add_rmsnorm_dev(x, w, o, residual=r)
    torch.cuda.synchronize()
    for a in range(0, rows, 1 << 23):
        s = slice(a, min(rows, a + (1 << 23)))
        h = x[s].float() + r[s].float()
        assert torch.equal(o["sum"][s], h.to(torch.bfloat16))
        h = h.double()
        ref = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
        got, tol = o["y"][s].to(torch.float64), 64 * U * ref.abs()
        if out == "bf16":
            tol = tol + ref.abs() * 2.0 ** -8
        else:
            top = ref.abs().amax(1)
            step = torch.where(top > 0, top / 448.0, torch.ones_like(top))
            assert ((o["y_scale"][s].double() - step).abs() <= 70 * U * step).all()
            got = got * o["y_scale"][s].double()[:, None]
            tol = tol + torch.maximum(ref.abs() * 2.0 ** -4, step[:, None] * 2.0 ** -10) * (1 + 70 * U)
        assert ((got - ref).abs() <= tol).all(), a


def against_float64(torch, sampler, x, w, eps, out):
    rows, hidden = x.shape
    o = {"y": torch.empty(rows, hidden, device="cuda", dtype=out), "y_scale": torch.empty(rows, device="cuda")}
    sampler.add_rmsnorm_dev(x, w, o, eps=eps)
    torch.cuda.synchronize()
    h = x.double()
    ref = h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
    got, tol = o["y"].to(torch.float64), 64 * U * ref.abs()
    if out == torch.float8_e4m3fn:
        s = ref.abs().amax(1) / 448.0
        assert ((o["y_scale"].double() - s).abs() <= 70 * U * s).all(), (o["y_scale"], s)
        got = got * o["y_scale"].double()[:, None]
        tol = tol + torch.maximum(ref.abs() * 2.0 ** -4, s[:, None] * 2.0 ** -10) * (1 + 70 * U)
    elif out == torch.bfloat16:
        tol = tol + ref.abs() * 2.0 ** -8
    assert ((got - ref).abs() <= tol).all(), (got[0, :4], ref[0, :4])


@pytest.mark.parametrize("out", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hidden", [40, 2049, 9000])
def test_products_with_the_weight_that_leave_f32(sampler, hidden, dtype, out):
    """h w past 3e38 or below 1e-38, while y is well inside: y = (h / sqrt(...)) w."""
    torch = sampler.torch
    types = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    v, g = (torch.randn(*n, generator=gen, device="cuda") for n in ((4, hidden), (hidden,)))
    for size, weight, eps in ((1e16, 1e25, 1e-6), (1e-25, 1e-20, 1e-36), (1e-12, 1e-30, 1e-20)):
        against_float64(torch, sampler, (v * size).to(types[dtype]), (g * weight).to(types[dtype]), eps, types[out])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hidden", [40, 2049, 9000])
def test_scales_stay_normal_numbers(sampler, hidden, dtype):
    """Rows whose largest |y| / 448 is below 2^-126, by the weight and by eps, beside one
    that is above: y_scale is 2^-126, and y within half a step of it."""
    torch = sampler.torch
    t = {"f32": torch.float32, "bf16": torch.bfloat16}[dtype]
    least = 2.0 ** -126
    gen = torch.Generator(device="cuda").manual_seed(hidden)
    v, g = (torch.randn(*n, generator=gen, device="cuda") for n in ((4, hidden), (hidden,)))
    for size, weight, eps in ((1e12, 2e-38, 1e-6), (1e-5, 1e-10, 1e37), (1e-2, 1.0, 1e37)):
        x, w = (v * size).to(t), (g * weight).to(t)
        o = {"y": torch.empty(4, hidden, device="cuda", dtype=torch.float8_e4m3fn), "y_scale": torch.empty(4, device="cuda")}
        sampler.add_rmsnorm_dev(x, w, o, eps=eps)
        torch.cuda.synchronize()
        h = x.double()
        ref = h / (h.square().mean(1, keepdim=True) + eps).sqrt() * w.double()
        s = (ref.abs().amax(1) / 448.0).clamp(min=least)
        assert ((o["y_scale"].double() - s).abs() <= 70 * U * s).all() and (o["y_scale"].double() >= least).all(), (o["y_scale"], s)
        got = o["y"].to(torch.float64) * o["y_scale"].double()[:, None]
        tol = 64 * U * ref.abs() + torch.maximum(ref.abs() * 2.0 ** -4, s[:, None] * 2.0 ** -10) * (1 + 70 * U)
        assert ((got - ref).abs() <= tol).all()
