"""A decode step's end for a batch whose requests carry their own adapters: the
residual's addition and norm into 8 bits, the 8-bit lm-head with the requests'
low-rank adapters, and the sampler on its logits and statistics.

    python examples/adapted_decode.py [--rows 64] [--vocab 32000] [--hidden 2048] [--steps 4]

Random weights and hidden states; prints each step's tokens. The three calls are
stream-ordered and allocate nothing, so a step can be captured into a HIP graph.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

from locus_amd import sampler as S  # noqa: E402
from locus_amd import workloads as W  # noqa: E402


def to_e4m3(v):
    """Rows in 8 bits and their scales, as a checkpoint's tool makes them."""
    scale = v.float().abs().amax(1).clamp_(min=1e-12) / 448.0
    return (v.float() / scale[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


class AdaptedHead:
    """The weights that a server holds, and one batch's buffers."""

    def __init__(self, norm_weight, out_weight, adapters: S.Adapters, rows: int, eps: float = 1e-6, device: int = 0):
        self.norm_weight, self.adapters, self.eps, self.rows = norm_weight, adapters, eps, rows
        self.w, self.w_scale = to_e4m3(out_weight)
        self.vocab, hidden = out_weight.shape
        self.s = S.Sampler(device=device, max_rows=rows, max_vocab=self.vocab, max_hist=64, max_top=4)
        dev = torch.device("cuda", device)
        self.norm = {"y": torch.empty(rows, hidden, device=dev, dtype=torch.float8_e4m3fn),
                     "y_scale": torch.empty(rows, device=dev), "sum": torch.empty(rows, hidden, device=dev, dtype=norm_weight.dtype)}
        stride = (self.vocab + 3) // 4 * 4   # (lcs_sample's rows)
        self.logits = torch.empty(rows, stride, device=dev)
        self.head = dict(self.s.alloc_lmhead_out(rows, self.vocab, logits=False, stats=True), logits=self.logits[:, :self.vocab])

    def logits_of(self, x, residual, slot):
        """x + residual, normed, through the lm-head: self.head holds the logits, the argmax, log z and statistics."""
        self.s.add_rmsnorm_dev(x, self.norm_weight, self.norm, residual=residual, eps=self.eps)
        self.s.lmhead_ex_dev(self.norm["y"], self.w, self.head, x_scale=self.norm["y_scale"], w_scale=self.w_scale,
                             adapters=self.adapters, slot=slot)
        return self.head

    def sample(self, params, u):
        """One token a row from the last logits, with its logprob (the statistics spare the sampler its own sum)."""
        rows = self.rows
        w = W.Workload("adapted", rows, self.vocab, "f32", None, params, None, u, want_logprobs=True)
        dev = self.logits.device
        d = {"w": w, "logits": self.logits, "stride": self.logits.stride(0), "params_host": params,
             "params": torch.from_numpy(params.view(np.uint8).copy()).to(dev), "u": torch.from_numpy(u).to(dev)}
        out = self.s.alloc_out(rows, 0, True, diag=False)
        self.s.sample_dev(d, out, raw_stats=self.head["stats"])
        torch.cuda.synchronize()
        return self.s.fetch(out, 0)


def random_head(rows, vocab, hidden, ranks=(16, 8, 32), seed=0):
    """A head with random weights and a pool of adapters of the given ranks."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    wide = (max(ranks) + 7) // 8 * 8
    w = (torch.randn(vocab, hidden, generator=gen, device="cuda") * (2.5 / hidden ** 0.5)).to(torch.bfloat16)
    a = (torch.randn(len(ranks), wide, hidden, generator=gen, device="cuda") / hidden ** 0.5).to(torch.bfloat16)
    b = (torch.randn(len(ranks), vocab, wide, generator=gen, device="cuda") * 0.3).to(torch.bfloat16)
    pool = S.Adapters(a, b, rank=torch.tensor(ranks, device="cuda", dtype=torch.int32),
                      scale=torch.ones(len(ranks), device="cuda"))
    g = torch.ones(hidden, device="cuda", dtype=torch.bfloat16)
    return AdaptedHead(g, w, pool, rows), gen


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("rows", 64), ("vocab", 32000), ("hidden", 2048), ("steps", 4)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args(argv)
    head, gen = random_head(a.rows, a.vocab, a.hidden)
    slot = (torch.arange(a.rows, device="cuda") % 4 - 1).to(torch.int32)   # a quarter without an adapter
    params = np.zeros(a.rows, W.PARAMS_DTYPE)
    params["temperature"], params["top_p"], params["min_p"], params["repeat_penalty"] = 0.7, 1.0, 0.05, 1.0
    rng = np.random.default_rng(0)
    tokens = []
    for step in range(a.steps):
        x, residual = (torch.randn(a.rows, a.hidden, generator=gen, device="cuda").to(torch.bfloat16) for _ in range(2))
        head.logits_of(x, residual, slot)
        r = head.sample(params, rng.random(a.rows))
        tokens.append(r["ids"])
        print(f"step {step}: ids {r['ids'][:8].tolist()} logprobs {np.round(r['chosen_lp'][:4], 3).tolist()}", flush=True)
    return tokens


if __name__ == "__main__":
    main()
