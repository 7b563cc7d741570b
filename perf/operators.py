"""The model's last step before sampling, through the framework's public entry points.

Two kinds of case. "norm": the residual's addition and the root-mean-square
norm that gives the lm-head its input, in bf16, f32 or in 8 bits (e4m3) with a
scale per row (lcs_add_rmsnorm). "head": the lm-head product over a bf16 or an
8-bit weight, with the low-rank adapters of many requests beside it, and the
statistics that the sampler takes from it (lcs_lmhead_ex).

listed() holds the cases, draw() further ones of the same ranges; prepare()
builds a case's inputs from a seed, run() makes one pass (the plain form, or
the framework's call where `own` is true), exact() restates it in 64 bits.
"""
import functools
import math

import torch

own = False

EPS = 1e-6
E4M3_MAX = 448.0
MAX_ROWS, MAX_VOCAB = 2048, 262144
_T = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}


def listed():
    return [
        # one chat stream's last norm before an 8-bit lm-head: pure latency
        {"name": "norm_1", "kind": "norm", "rows": 1, "hidden": 4096, "dtype": "bf16", "out": "e4m3",
         "residual": True, "pad": 0},
        # a decode batch's
        {"name": "norm_64", "kind": "norm", "rows": 64, "hidden": 4096, "dtype": "bf16", "out": "e4m3",
         "residual": True, "pad": 0},
        # scoring long prompts: every position is normed
        {"name": "norm_8192", "kind": "norm", "rows": 8192, "hidden": 8192, "dtype": "bf16", "out": "e4m3",
         "residual": True, "pad": 0},
        # an f32 residual stream of an odd width, cut out of a wider buffer, for a bf16 lm-head
        {"name": "norm_odd", "kind": "norm", "rows": 777, "hidden": 2883, "dtype": "f32", "out": "bf16",
         "residual": False, "pad": 6},
        # one stream under its own adapter, small vocabulary: the smallest call
        {"name": "adapt_1", "kind": "head", "rows": 1, "vocab": 32000, "hidden": 4096, "dtype": "bf16",
         "adapters": 8, "ranks": "16", "per_seq": 0, "logits": True},
        # a decode batch whose requests carry 32 adapters of mixed ranks
        {"name": "adapt_64", "kind": "head", "rows": 64, "vocab": 128256, "hidden": 4096, "dtype": "bf16",
         "adapters": 32, "ranks": "8,16,32,64", "per_seq": 0, "logits": True},
        # a few rows, sizes off every tile, ranks that are no multiple of eight
        {"name": "adapt_odd", "kind": "head", "rows": 37, "vocab": 50257, "hidden": 1600, "dtype": "bf16",
         "adapters": 5, "ranks": "4,12,20", "per_seq": 0, "logits": True},
        # speculative decoding of 64 adapted streams, drafts verified, no logits written
        {"name": "adapt_512", "kind": "head", "rows": 512, "vocab": 128256, "hidden": 4096, "dtype": "bf16",
         "adapters": 16, "ranks": "32", "per_seq": 8, "logits": False},
        # speculative decoding of one stream over an 8-bit weight
        {"name": "q8_5", "kind": "head", "rows": 5, "vocab": 32000, "hidden": 2048, "dtype": "e4m3",
         "adapters": 0, "ranks": "", "per_seq": 5, "logits": True},
        # a decode batch over an 8-bit weight
        {"name": "q8_64", "kind": "head", "rows": 64, "vocab": 128256, "hidden": 4096, "dtype": "e4m3",
         "adapters": 0, "ranks": "", "per_seq": 0, "logits": True},
        # a decode batch over an 8-bit weight, every request with its own adapter
        {"name": "q8_adapt_64", "kind": "head", "rows": 64, "vocab": 151936, "hidden": 3584, "dtype": "e4m3",
         "adapters": 64, "ranks": "16", "per_seq": 0, "logits": True},
        # speculative decoding of a large batch over an 8-bit weight
        {"name": "q8_1024", "kind": "head", "rows": 1024, "vocab": 128256, "hidden": 4096, "dtype": "e4m3",
         "adapters": 0, "ranks": "", "per_seq": 8, "logits": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    if rng.random() < 0.35:
        hidden = rng.choice([2048, 4096, 8192, 64 * _log(rng, 1, 256), _log(rng, 48, 16384)])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        most = 8192 * 8192 // hidden // (2 if dtype == "f32" else 1)
        return {"kind": "norm", "rows": _log(rng, 1, min(16384, most)), "hidden": hidden, "dtype": dtype,
                "out": rng.choice(["e4m3", "e4m3", "bf16", "f32"]), "residual": rng.random() < 0.7,
                "pad": rng.choice([0, 0, 8, rng.randint(1, 64)])}
    dtype = rng.choice(["bf16", "e4m3"])
    vocab = rng.choice([32000, 50257, 128256, 151936, _log(rng, 4000, 200000)])
    hidden = 128 * rng.randint(4, 64)
    vocab = min(vocab, 128256 * 4096 // hidden)
    per = rng.choice([0, 0, 0, 2, 5, 8])
    rows = _log(rng, 1, min(1024, (1024 if dtype == "e4m3" else 512) * 128256 * 4096 // (vocab * hidden)))
    rows = max(1, rows // per) * per if per else rows
    ranks = rng.choice(["8", "16", "32", "64", "128", "8,16,32,64", "4,12,20", "%d" % rng.randint(1, 128)])
    mean = sum(_ranks(ranks)) / len(_ranks(ranks))
    n = _log(rng, 1, max(1, min(64, int(2.4e8 / (2 * vocab * mean)))))
    if dtype == "e4m3" and rng.random() < 0.4:
        n, ranks = 0, ""
    return {"kind": "head", "rows": rows, "vocab": vocab, "hidden": hidden, "dtype": dtype, "adapters": n,
            "ranks": ranks, "per_seq": per, "logits": rows <= 256 and rng.random() < 0.7}


def _ranks(text):
    return [int(t) for t in text.split(",")] if text else []


def _seqs(c):
    """Sequences of a head case, and how many of them carry an adapter (seven in eight; a few streams: all)."""
    n = c["rows"] // c["per_seq"] if c["per_seq"] else c["rows"]
    return n, n - n // 8


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _to_e4m3(v):
    """Rows in 8 bits and their scales, as a checkpoint's tool makes them."""
    scale = v.abs().amax(1).float().clamp_(min=1e-12) / E4M3_MAX
    return (v / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _prepare_norm(c, seed):
    gen = _gen(seed)
    rows, hidden, t = c["rows"], c["hidden"], _T[c["dtype"]]

    def rows_of(scale):   # a few channels far larger than the rest, as residual streams have
        v = _randn(gen, rows, hidden + c["pad"]) * scale
        v[:, :: max(1, hidden // 5)] *= 20.0
        return v.to(t)[:, :hidden]

    x = rows_of(1.0)
    residual = rows_of(3.0) if c["residual"] else None
    weight = (1.0 + 0.2 * _randn(gen, hidden)).to(t)
    out = {"y": torch.empty(rows, hidden, device="cuda", dtype=_T[c["out"]])}
    if residual is not None:
        out["sum"] = torch.empty(rows, hidden, device="cuda", dtype=t)
    if c["out"] == "e4m3":
        out["y_scale"] = torch.empty(rows, device="cuda")
    return {"kind": "norm", "x": x, "residual": residual, "weight": weight, "out": out}


def _prepare_head(c, seed):
    gen = _gen(seed)
    rows, vocab, hidden, n = c["rows"], c["vocab"], c["hidden"], c["adapters"]
    w = _randn(gen, vocab, hidden, dtype=torch.bfloat16).mul_(2.5 / math.sqrt(hidden))
    # hidden states that say a token: its logit stands out
    said = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    toward = w[said].float()
    x = _randn(gen, rows, hidden) + 10.0 * toward / toward.norm(dim=1, keepdim=True)
    st = {"kind": "head", "draft": None, "adapters": None, "per_seq": c["per_seq"]}
    if c["dtype"] == "e4m3":
        st["w"], st["w_scale"] = _to_e4m3(w)
        st["x"], st["x_scale"] = _to_e4m3(x)
    else:
        st["w"], st["x"], st["w_scale"], st["x_scale"] = w, x.to(torch.bfloat16), None, None
    out = {"argmax_ids": torch.empty(rows, device="cuda", dtype=torch.int32),
           "log_z": torch.empty(rows, device="cuda")}
    if c["logits"]:
        out["logits"] = torch.empty(rows, vocab, device="cuda")
    if c["per_seq"]:   # drafts, three in four of them what the model says, a sequence's last one at random
        hit = torch.rand(rows, generator=gen, device="cuda") < 0.75
        hit[c["per_seq"] - 1 :: c["per_seq"]] = False
        other = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        st["draft"] = torch.where(hit, said, other).to(torch.int32)
        out["draft_lp"] = torch.empty(rows, device="cuda")
        out["accept_len"] = torch.empty(rows // c["per_seq"], device="cuda", dtype=torch.int32)
    if n:
        ranks = _ranks(c["ranks"])
        ranks = [ranks[i % len(ranks)] for i in range(n)]
        wide = (max(ranks) + 7) // 8 * 8
        live = torch.arange(wide, device="cuda") < torch.tensor(ranks, device="cuda")[:, None]   # (n, wide)
        a = _randn(gen, n, wide, hidden, dtype=torch.bfloat16).mul_(1.0 / math.sqrt(hidden))
        b = _randn(gen, n, vocab, wide, dtype=torch.bfloat16).mul_(0.3)
        seqs, adapted = _seqs(c)
        order = torch.randperm(seqs, generator=gen, device="cuda")
        slot = torch.full((seqs,), -1, device="cuda")
        slot[order[:adapted]] = torch.arange(adapted, device="cuda") % n
        st["adapters"] = {"a": a * live[:, :, None], "b": b * live[:, None, :],
                          "rank": torch.tensor(ranks, device="cuda", dtype=torch.int32),
                          "scale": torch.tensor([16.0 / r if r > 8 else 1.0 for r in ranks], device="cuda")}
        st["slot"] = slot.repeat_interleave(max(1, c["per_seq"])).to(torch.int32)
    st["out"] = out
    return st


def prepare(case, seed):
    return _prepare_norm(case, seed) if case["kind"] == "norm" else _prepare_head(case, seed)


# --------------------------------------------------------- the plain forms --
def _plain_norm(st):
    h = st["x"].float()
    out = {}
    if st["residual"] is not None:
        h = h + st["residual"].float()
        out["sum"] = h.to(st["x"].dtype)
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * st["weight"].float()
    dtype = st["out"]["y"].dtype
    if dtype == torch.float8_e4m3fn:
        top = y.abs().amax(1)
        scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        out["y_scale"] = scale
        y = (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX)
    out["y"] = y.to(dtype)
    return out


def _plain_head(st):
    x, w = st["x"].float(), st["w"].float()
    if st["x_scale"] is not None:
        x, w = x * st["x_scale"][:, None], w * st["w_scale"][:, None]
    logits = x @ w.t()
    ad = st["adapters"]
    if ad is not None:   # every adapter's low-rank states, kept where the row's slot is that adapter's
        n, wide, hidden = ad["a"].shape
        mine = st["slot"][:, None] == torch.arange(n, device="cuda")
        live = torch.arange(wide, device="cuda") < ad["rank"][:, None]
        p = (x @ ad["a"].float().view(n * wide, hidden).t()).view(-1, n, wide) * ad["scale"][:, None]
        p = torch.where(mine[:, :, None] & live, p, torch.zeros_like(p))
        logits = logits + p.view(-1, n * wide) @ ad["b"].float().transpose(1, 2).reshape(n * wide, -1)
    top = logits.amax(1)
    out = {"argmax_ids": logits.argmax(1).to(torch.int32),
           "log_z": top + (logits - top[:, None]).exp().sum(1).log()}
    if "logits" in st["out"]:
        out["logits"] = logits
    if st["draft"] is not None:
        out["draft_lp"] = logits.gather(1, st["draft"].long()[:, None])[:, 0] - out["log_z"]
        hits = (out["argmax_ids"] == st["draft"]).view(-1, st["per_seq"])
        out["accept_len"] = hits.to(torch.int32).cumprod(1).sum(1).to(torch.int32)
    return out


# ----------------------------------------------------- the framework's calls --
@functools.lru_cache(maxsize=None)
def _sampler():
    """The handle that a serving program creates once."""
    from locus_amd import sampler
    return sampler, sampler.Sampler(device=0, max_rows=MAX_ROWS, max_vocab=MAX_VOCAB, max_hist=64, max_top=4)


def _own(st):
    module, s = _sampler()
    if st["kind"] == "norm":
        s.add_rmsnorm_dev(st["x"], st["weight"], st["out"], residual=st["residual"], eps=EPS)
        return st["out"]
    ad = st["adapters"]
    if ad is not None:
        ad = module.Adapters(ad["a"], ad["b"], rank=ad["rank"], scale=ad["scale"])
    s.lmhead_ex_dev(st["x"], st["w"], st["out"], x_scale=st["x_scale"], w_scale=st["w_scale"], adapters=ad,
                    slot=st.get("slot"), draft=st["draft"], rows_per_seq=st["per_seq"])
    return st["out"]


def run(state):
    if own:
        return _own(state)
    return _plain_norm(state) if state["kind"] == "norm" else _plain_head(state)


# -------------------------------------------------------------- what it takes --
def work(case):
    c = case
    if c["kind"] == "norm":
        each = c["rows"] * c["hidden"]
        size = _SIZE[c["dtype"]]
        return {"bytes": each * (size * (3 if c["residual"] else 1) + _SIZE[c["out"]]) + c["hidden"] * size
                + (4 * c["rows"] if c["out"] == "e4m3" else 0), "flops": 8 * each}
    rows, vocab, hidden, size = c["rows"], c["vocab"], c["hidden"], _SIZE[c["dtype"]]
    bytes_ = (vocab + rows) * hidden * size + (4 * (rows + vocab) if c["dtype"] == "e4m3" else 0) + 8 * rows
    bytes_ += 4 * rows * vocab if c["logits"] else 0
    bytes_ += 8 * rows + 4 * rows // c["per_seq"] if c["per_seq"] else 0
    flops = 2 * rows * vocab * hidden
    if c["adapters"]:
        ranks = _ranks(c["ranks"])
        _, adapted = _seqs(c)
        used = [ranks[i % len(ranks)] for i in range(min(c["adapters"], adapted))]   # each read once
        bytes_ += sum(used) * (hidden + vocab) * 2 + 4 * rows
        each = [ranks[i % c["adapters"] % len(ranks)] for i in range(adapted)]
        flops += 2 * sum(each) * max(1, c["per_seq"]) * (hidden + vocab)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------- in 64 bits --
def _exact_norm(c, st):
    res, out = st["residual"], {}
    h = st["x"].double() if res is None else st["x"].double().add_(res)
    if res is not None:
        out["sum"] = h
    y = h / h.square().mean(1, keepdim=True).add(EPS).sqrt() * st["weight"].double()
    if c["out"] == "e4m3":
        top = y.abs().amax(1)
        out["y_scale"] = torch.where(top > 0, top, top.new_tensor(E4M3_MAX)) / E4M3_MAX
        y = y / out["y_scale"][:, None]
    out["y"] = y
    return out


def _exact_head(c, st):
    x = st["x"].double()
    x = x if st["x_scale"] is None else x * st["x_scale"].double()[:, None]
    logits = torch.empty(c["rows"], c["vocab"], device="cuda", dtype=torch.float64)
    for v in range(0, c["vocab"], 16384):
        w = st["w"][v:v + 16384].double()
        w = w if st["w_scale"] is None else w * st["w_scale"][v:v + 16384].double()[:, None]
        logits[:, v:v + 16384] = x @ w.t()
    if c["adapters"]:
        ad = st["adapters"]
        for i, r in enumerate(ad["rank"].tolist()):
            mine = (st["slot"] == i).nonzero()[:, 0]
            if mine.numel():
                low = (x[mine] @ ad["a"][i, :r].double().t()) * ad["scale"][i].double()
                logits[mine] += low @ ad["b"][i, :, :r].double().t()
    out = {"argmax_ids": None, "log_z": torch.logsumexp(logits, 1)}
    if c["logits"]:
        out["logits"] = logits
    if c["per_seq"]:
        out["draft_lp"] = logits.gather(1, st["draft"].long()[:, None])[:, 0] - out["log_z"]
        out["accept_len"] = None
    return out


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_norm(case, st) if case["kind"] == "norm" else _exact_head(case, st)
