"""The example's chain (norm into 8 bits, 8-bit lm-head with adapters, sampler)
against float64 and against the same sampling without the lm-head's statistics."""
import numpy as np
import pytest

from locus_amd import workloads as W

pytestmark = pytest.mark.gpu


def test_chain_against_float64():
    import torch

    from examples.adapted_decode import random_head
    rows, vocab, hidden = 24, 5003, 512
    head, gen = random_head(rows, vocab, hidden, ranks=(16, 5, 32), seed=3)
    slot = (torch.arange(rows, device="cuda") % 4 - 1).to(torch.int32)
    x, residual = (torch.randn(rows, hidden, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
    out = head.logits_of(x, residual, slot)
    torch.cuda.synchronize()
    # the norm, from the inputs; the head, from the norm's own 8 bits
    h = x.double() + residual.double()
    y = h / (h.square().mean(1, keepdim=True) + head.eps).sqrt()
    q = head.norm["y"].double() * head.norm["y_scale"].double()[:, None]
    half = torch.maximum(y.abs() * 2.0 ** -4, head.norm["y_scale"].double()[:, None] * 2.0 ** -10)
    assert ((q - y).abs() <= half * (1 + 2.0 ** -16) + y.abs() * 2.0 ** -18).all()
    assert torch.equal(head.norm["sum"], (x.float() + residual.float()).to(torch.bfloat16))
    w = head.w.double() * head.w_scale.double()[:, None]
    ref, size = q @ w.t(), q.abs() @ w.abs().t()
    a, b = head.adapters._keep[0].double(), head.adapters._keep[1].double()
    for i, r in enumerate((16, 5, 32)):
        m = (slot == i).nonzero()[:, 0]
        low, big = q[m] @ a[i, :r].t(), q[m].abs() @ a[i, :r].abs().t()
        ref[m] += low @ b[i, :, :r].t()
        size[m] += big @ b[i, :, :r].abs().t()
    # f32 sums over hidden and over the ranks (twice in a state's product), the scales' roundings
    assert ((out["logits"].double() - ref).abs() <= (hidden + 128) * 2.0 ** -24 * 2 * size).all()
    # the sampler on them, with and without the statistics
    params = np.zeros(rows, W.PARAMS_DTYPE)
    params["temperature"], params["top_p"], params["min_p"], params["repeat_penalty"] = 0.7, 1.0, 0.05, 1.0
    u = np.random.default_rng(1).random(rows)
    with_stats = head.sample(params, u)
    stats = head.head.pop("stats")
    head.head["stats"] = None
    without = head.sample(params, u)
    head.head["stats"] = stats
    assert np.array_equal(with_stats["ids"], without["ids"]) and ((with_stats["ids"] >= 0) & (with_stats["ids"] < vocab)).all()
    assert np.abs(with_stats["chosen_lp"] - without["chosen_lp"]).max() <= 1e-5
    head.s.close()


def test_the_example_runs(capsys):
    from examples.adapted_decode import main
    tokens = main(["--rows", "9", "--vocab", "1000", "--hidden", "128", "--steps", "2"])
    assert len(tokens) == 2 and all(((t >= 0) & (t < 1000)).all() for t in tokens)
    assert "step 1" in capsys.readouterr().out
