"""Speculative decoding over a paged cache, through the framework's public entry points.

Four kinds of case. "attn": attention of each sequence's drafted tokens, a tree
of them, over its cached context and their own ancestors (lcs_tree_attn).
"accept": the tree's verification against the model's logits and the accepted
path's keys and values appended to the cache (lcs_tree_verify, lcs_kv_grow,
lcs_kv_append). "fork": sequences that give up their pages for a shared copy of
another's, and private ones to go on writing (lcs_kv_free, lcs_kv_fork,
lcs_kv_grow). "compact": sequences that keep some of their tokens
(lcs_kv_compact).

listed() holds the cases, draw() further ones of the same ranges; prepare()
builds a case's inputs from a seed, run() makes one pass (the plain form, or
the framework's calls where `own` is true), exact() restates it in 64 bits.
"""
import functools
import math

import torch

own = False

E4M3_MAX = 448.0
MAX_ROWS, MAX_VOCAB, MAX_NEW_PAGES = 2048, 262144, 65536
_T = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
_SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}


def listed():
    return [
        # one chat stream's next token over a short context: pure latency
        {"name": "attn_1", "kind": "attn", "seqs": 1, "rows": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "ctx_lo": 1000, "ctx_hi": 1000, "dtype": "bf16", "layout": "head", "tree": "chain"},
        # a decode batch with small trees of drafts, contexts of every length
        {"name": "attn_tree", "kind": "attn", "seqs": 16, "rows": 16, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "ctx_lo": 300, "ctx_hi": 6000, "dtype": "bf16", "layout": "head", "tree": "tree"},
        # one stream over a very long document: few rows, a long axis to split
        {"name": "attn_long", "kind": "attn", "seqs": 1, "rows": 8, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "ctx_lo": 131000, "ctx_hi": 131000, "dtype": "bf16", "layout": "head", "tree": "chain"},
        # a large batch over an 8-bit cache
        {"name": "attn_64", "kind": "attn", "seqs": 64, "rows": 8, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "ctx_lo": 1500, "ctx_hi": 8000, "dtype": "e4m3", "layout": "head", "tree": "tree"},
        # wide trees of a model with many query heads: 512 rows share each head's keys
        {"name": "attn_wide", "kind": "attn", "seqs": 8, "rows": 64, "heads": 64, "kv_heads": 8, "dim": 128, "page": 64,
         "ctx_lo": 8192, "ctx_hi": 8192, "dtype": "bf16", "layout": "head", "tree": "tree"},
        # sizes off every tile: odd heads and widths, a cache with tokens ahead of heads, trees with
        # padded nodes, a sequence without a context
        {"name": "attn_odd", "kind": "attn", "seqs": 7, "rows": 13, "heads": 15, "kv_heads": 5, "dim": 80, "page": 16,
         "ctx_lo": 0, "ctx_hi": 1777, "dtype": "bf16", "layout": "token", "tree": "ragged"},
        # one stream's step: a small tree's verdict and a few rows for every layer
        {"name": "accept_1", "kind": "accept", "seqs": 1, "rows": 8, "vocab": 32000, "logits": "f32", "layers": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "ctx_lo": 250, "ctx_hi": 250, "dtype": "bf16"},
        # a batch's step over a large vocabulary and an 8-bit cache
        {"name": "accept_64", "kind": "accept", "seqs": 64, "rows": 16, "vocab": 128256, "logits": "bf16", "layers": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "ctx_lo": 60, "ctx_hi": 250, "dtype": "e4m3"},
        # a few samples of one prompt
        {"name": "fork_4", "kind": "fork", "sources": 1, "forks": 4, "layers": 16, "kv_heads": 8, "dim": 128, "page": 16,
         "ctx_lo": 500, "ctx_hi": 500, "add": 1, "dtype": "bf16"},
        # a beam step of many prompts: every beam goes on from a copy of another's last page
        {"name": "fork_64", "kind": "fork", "sources": 8, "forks": 64, "layers": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "ctx_lo": 700, "ctx_hi": 1000, "add": 16, "dtype": "bf16"},
        # a few sequences drop part of a short context: odd sizes, an 8-bit cache
        {"name": "compact_odd", "kind": "compact", "seqs": 3, "layers": 5, "kv_heads": 3, "dim": 96, "page": 16,
         "ctx_lo": 100, "ctx_hi": 777, "keep": 610, "dtype": "e4m3"},
        # long contexts cut to half
        {"name": "compact_16", "kind": "compact", "seqs": 16, "layers": 4, "kv_heads": 8, "dim": 128, "page": 32,
         "ctx_lo": 4000, "ctx_hi": 8192, "keep": 500, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "accept", "fork", "compact"])
    dim, page = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bf16", "bf16", "e4m3"])
    kv = rng.choice([1, 2, 3, 5, 8, 8])
    if kind == "attn":
        group = rng.choice([1, 2, 3, 4, 4, 7, 8])
        seqs, rows = _log(rng, 1, 64), _log(rng, 1, 64)
        # no more products, and no more bytes, than the largest listed ones
        most = min(131072, int(8 * 64 * 64 * 8192 * 128 / (seqs * rows * kv * group * dim)),
                   int(64 * 4750 * 8 * 128 / (seqs * kv * dim)))
        hi = _log(rng, 16, max(64, most))
        return {"kind": kind, "seqs": seqs, "rows": rows, "heads": kv * group, "kv_heads": kv, "dim": dim, "page": page,
                "ctx_lo": rng.choice([0, 1, hi // 4, hi]), "ctx_hi": hi, "dtype": dtype,
                "layout": rng.choice(["head", "token"]), "tree": rng.choice(["chain", "tree", "ragged"])}
    layers = _log(rng, 1, 32)
    if kind == "accept":
        logits = rng.choice(["f32", "bf16"])
        vocab = rng.choice([32000, 50257, 128256, 151936, _log(rng, 4000, 200000)])
        rows = _log(rng, 1, 64)
        seqs = _log(rng, 1, max(1, min(64, 64 * 16 * 128256 * 2 // (rows * vocab * _SIZE[logits]))))
        hi = rng.randint(1, 250)
        return {"kind": kind, "seqs": seqs, "rows": rows, "vocab": vocab, "logits": logits, "layers": layers,
                "kv_heads": kv, "dim": dim, "page": page, "ctx_lo": rng.randint(0, hi), "ctx_hi": hi, "dtype": dtype}
    if kind == "fork":
        sources = _log(rng, 1, 8)
        hi = rng.randint(20, 1000)
        return {"kind": kind, "sources": sources, "forks": _log(rng, 1, 64 * 128 * 8 // max(1024, dim * kv)),
                "layers": layers, "kv_heads": kv, "dim": dim, "page": page, "ctx_lo": rng.randint(1, hi), "ctx_hi": hi,
                "add": rng.randint(1, 2 * page), "dtype": dtype}
    seqs = _log(rng, 1, 16)
    hi = _log(rng, 20, max(64, min(16384, 4 * 16 * 8192 * 8 * 128 // (layers * seqs * kv * dim))))
    return {"kind": kind, "seqs": seqs, "layers": layers, "kv_heads": kv, "dim": dim, "page": page,
            "ctx_lo": rng.randint(0, hi), "ctx_hi": hi, "keep": rng.randint(50, 1000), "dtype": dtype}


def _lengths(lo, hi, n):
    """n context lengths evenly between lo and hi."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _chain(rows):
    """The accepted path's longest: half the tree's nodes lie on one line."""
    return (rows + 1) // 2


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _to_e4m3(v):
    """Rows in 8 bits and their scales."""
    top = v.abs().amax(-1).float()
    scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
    return (v.float() / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _pool(c, gen, layers, pages):
    """Keys and values of a pool of pages, a few channels of the keys far larger than the rest, as caches have them."""
    heads, page, dim = c["kv_heads"], c["page"], c["dim"]
    st = {"k_scale": None, "v_scale": None}
    k, v = (_randn(gen, layers, pages, heads, page, dim) for _ in range(2))
    k[..., :: 16] *= 4.0
    if c["dtype"] == "e4m3":
        k, st["k_scale"] = _to_e4m3(k)
        v, st["v_scale"] = _to_e4m3(v)
    if c.get("layout") == "token":   # a token's heads together
        k, v = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (k, v))
    st["k"], st["v"] = k, v
    return st


def _tables(c, gen, lengths, wide, spare):
    """Each sequence's pages, anywhere in the pool, and how often each page is held."""
    page = c["page"]
    used = [(n + page - 1) // page for n in lengths]
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    at = torch.arange(wide, device="cuda")[None, :]
    first = _ints([sum(used[:i]) for i in range(len(used))])[:, None]
    held = at < _ints(used)[:, None]
    table = torch.where(held, order[torch.where(held, first + at, 0).long()], -1).int().contiguous()
    refs = torch.zeros(pages, device="cuda", dtype=torch.int32)
    refs[order[: sum(used)].long()] = 1
    return table, refs, pages


def _ancestors(parent):
    """Per node and itself the nodes it descends from: (seqs, rows, rows) truth values."""
    rows = parent.shape[1]
    step = (parent[:, :, None] == torch.arange(rows, device="cuda")).double() + torch.eye(rows, device="cuda", dtype=torch.float64)
    return torch.matrix_power(step, rows) > 0


def _words(mask):
    """Truth values in 32-bit words, the lowest bit first."""
    n = mask.shape[-1]
    bits = torch.nn.functional.pad(mask, (0, -n % 32)).view(*mask.shape[:-1], -1, 32).long()
    words = (bits << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).int()


def _prepare_attn(c, seed):
    gen = _gen(seed)
    seqs, rows, heads, kv, dim, page = (c[k] for k in ("seqs", "rows", "heads", "kv_heads", "dim", "page"))
    lengths = _lengths(c["ctx_lo"], c["ctx_hi"], seqs)
    wide = max(1, (c["ctx_hi"] + page - 1) // page)
    table, refs, pages = _tables(c, gen, lengths, wide, 3)
    st = _pool(c, gen, 1, pages)
    st |= {"kind": "attn", "rows": rows, "table": table, "refs": refs, "length": _ints(lengths), "seq": _ints(range(seqs)),
           "scale": 1.0 / math.sqrt(dim), "mask": None}
    # queries, keys and values of a step in one buffer, as a fused projection leaves them
    qkv = _randn(gen, seqs * rows, (heads + 2 * kv) * dim)
    st["q"] = qkv[:, : heads * dim].view(-1, heads, dim)
    st["k_new"] = qkv[:, heads * dim : (heads + kv) * dim].view(-1, kv, dim)
    st["v_new"] = qkv[:, (heads + kv) * dim :].view(-1, kv, dim)
    if c["tree"] != "chain":
        up = torch.randint(1, 5, (seqs, rows), generator=gen, device="cuda")
        at = torch.arange(rows, device="cuda")
        see = _ancestors(torch.where(at > 0, (at - up).clamp(min=0), -1))
        if c["tree"] == "ragged":   # sequence i's last i nodes (of at most half) are padding: they see none
            pad = (torch.arange(seqs, device="cuda") % (rows // 2 + 1))[:, None]
            see = see & (at < rows - pad)[:, :, None]
        st["mask"] = _words(see)
    st["out"] = {"o": torch.empty(seqs * rows, heads, dim, device="cuda", dtype=torch.bfloat16),
                 "lse": torch.empty(seqs * rows, heads, device="cuda")}
    return st


def _prepare_accept(c, seed):
    gen = _gen(seed)
    seqs, rows, vocab, page = c["seqs"], c["rows"], c["vocab"], c["page"]
    lengths = _lengths(c["ctx_lo"], c["ctx_hi"], seqs)
    wide = (c["ctx_hi"] + rows + page - 1) // page
    table, refs, pages = _tables(c, gen, lengths, wide, seqs * ((rows + page - 1) // page + 1))
    st = _pool(c, gen, c["layers"], pages)
    # a tree: a line of half the nodes, the others beside it, by depth
    line = _chain(rows)
    depth = torch.randint(min(1, line - 1), line, (seqs, rows), generator=gen, device="cuda")
    depth[:, :line] = torch.arange(line, device="cuda")
    side = torch.arange(rows, device="cuda") >= line
    depth, order = torch.sort(depth * 2 + side, dim=1, stable=True)
    at = torch.empty_like(order).scatter_(1, order, torch.arange(rows, device="cuda").expand(seqs, rows).contiguous())
    depth, side = depth // 2, depth % 2 > 0
    spine = at[:, :line]                                    # the line's nodes, by depth
    parent = torch.where(depth > 0, spine.gather(1, (depth - 1).clamp(min=0)), torch.where(side, 0, -1))
    start = torch.randint(0, vocab, (seqs, 1), generator=gen, device="cuda")
    tokens = (start + 61 * torch.arange(rows, device="cuda")) % vocab
    # logits whose largest is the line's next token as far as the sequence's drafts are right
    logits = torch.randn(seqs * rows, vocab, generator=gen, device="cuda").mul_(2.5)
    right = (torch.arange(seqs, device="cuda") % line)[:, None]
    other = (start + 61 * rows + 7) % vocab
    says = torch.where(~side & (depth < right), tokens.gather(1, spine.gather(1, (depth + 1).clamp(max=line - 1))), other)
    logits.scatter_add_(1, says.view(-1, 1), torch.full((seqs * rows, 1), 22.0, device="cuda"))
    pad = -vocab % 8
    logits = torch.nn.functional.pad(logits.to(_T[c["logits"]]), (0, pad))[:, :vocab]
    new = _randn(gen, 2, c["layers"], seqs * rows, c["kv_heads"], c["dim"])
    ints = lambda *shape: torch.empty(*shape, device="cuda", dtype=torch.int32)  # noqa: E731
    return st | {"kind": "accept", "rows": rows, "table": table, "refs": refs, "length": _ints(lengths),
                 "seq": _ints(range(seqs)), "logits": logits, "tokens": tokens.int().view(-1),
                 "parent": parent.int().view(-1), "k_new": new[0], "v_new": new[1], "result": ints(seqs),
                 "out": {"argmax_ids": ints(seqs * rows), "node_lp": torch.empty(seqs * rows, device="cuda"),
                         "path": ints(seqs, rows), "n_path": ints(seqs), "next_id": ints(seqs), "length": ints(seqs)}}


def _prepare_fork(c, seed):
    gen = _gen(seed)
    sources, forks, page = c["sources"], c["forks"], c["page"]
    lengths = _lengths(c["ctx_lo"], c["ctx_hi"], sources)
    extra = (c["add"] + page - 1) // page + 1
    wide = (c["ctx_hi"] + c["add"] + page - 1) // page
    table, refs, pages = _tables(c, gen, lengths, wide, forks * extra * 2)
    st = _pool(c, gen, c["layers"], pages)
    src = torch.arange(forks, device="cuda") % sources
    # each fork still holds what an earlier step gave it: another source's whole pages and one of its own
    was = (src + 1) % sources
    whole = (_ints(lengths)[was] // page)[:, None]
    at = torch.arange(wide, device="cuda")[None, :]
    mine = (refs == 0).nonzero()[:forks].int()
    held = torch.where(at < whole, table[was], torch.where(at == whole, mine, -1))
    counts = torch.zeros(pages + 1, device="cuda", dtype=torch.int32)
    counts.index_add_(0, torch.where(held < 0, pages, held).view(-1), torch.ones(forks * wide, device="cuda", dtype=torch.int32))
    tokens = _ints(lengths)[src].contiguous()
    return st | {"kind": "fork", "table": torch.cat([table, held.int()]).contiguous(), "refs": refs + counts[:pages],
                 "src": src.int(), "dst": _ints(range(sources, sources + forks)), "length": tokens,
                 "end": tokens + c["add"], "none": torch.zeros(forks, device="cuda", dtype=torch.int32),
                 "results": torch.empty(3, forks, device="cuda", dtype=torch.int32)}


def _prepare_compact(c, seed):
    gen = _gen(seed)
    seqs, page = c["seqs"], c["page"]
    lengths = _lengths(c["ctx_lo"], c["ctx_hi"], seqs)
    counts = [n * c["keep"] // 1000 for n in lengths]
    table, refs, pages = _tables(c, gen, lengths, (c["ctx_hi"] + page - 1) // page, 2)
    st = _pool(c, gen, c["layers"], pages)
    at = torch.arange(c["ctx_hi"], device="cuda")
    weight = torch.rand(seqs, c["ctx_hi"], generator=gen, device="cuda")
    weight[:, :4] = 2.0   # the first tokens always stay
    weight = weight.masked_fill(at >= _ints(lengths)[:, None], -1.0)
    rank = weight.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
    most = max(1, max(counts))
    keep = torch.where(rank < _ints(counts)[:, None], at, 1 << 30).sort(1).values[:, :most]
    return st | {"kind": "compact", "table": table, "refs": refs, "seq": _ints(range(seqs)), "length": _ints(lengths),
                 "count": _ints(counts), "keep": torch.where(keep < 1 << 30, keep, -1).int().contiguous(),
                 "result": torch.empty(seqs, device="cuda", dtype=torch.int32)}


_PREPARE = {"attn": _prepare_attn, "accept": _prepare_accept, "fork": _prepare_fork, "compact": _prepare_compact}


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, seed)


# --------------------------------------------------------- the plain forms --
def _context(st, pool, scale):
    """Every sequence's cached rows in f32: (seqs, heads, tokens, dim)."""
    idx = st["table"][st["seq"].long()].clamp(min=0).long()
    x = pool[0][idx].float()                                            # (seqs, pages, heads, page, dim)
    if scale is not None:
        x = x * scale[0][idx][..., None]
    seqs, n, heads, page, dim = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(seqs, heads, n * page, dim)


def _seen(st, tokens):
    """(seqs, rows, tokens + rows): which of its context and of its tree each row sees."""
    rows, seqs = st["rows"], st["seq"].numel()
    ctx = (torch.arange(tokens, device="cuda") < st["length"][:, None])[:, None].expand(seqs, rows, tokens)
    at = torch.arange(rows, device="cuda")
    if st["mask"] is None:
        tree = (at <= at[:, None]).expand(seqs, rows, rows)
    else:
        tree = (st["mask"].view(seqs, rows, -1)[:, :, at // 32] >> (at % 32)) & 1 > 0
    return torch.cat([ctx, tree], 2)


def _plain_attn(st):
    rows, seqs = st["rows"], st["seq"].numel()
    heads, dim = st["q"].shape[1:]
    kv = st["k_new"].shape[1]
    group = heads // kv
    k, v = (torch.cat([_context(st, st[p], st[p + "_scale"]),
                       st[p + "_new"].float().view(seqs, rows, kv, dim).transpose(1, 2)], 2) for p in ("k", "v"))
    see = _seen(st, k.shape[2] - rows)
    q = st["q"].float().view(seqs, rows, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, group * rows, dim)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()).view(seqs, kv, group, rows, -1) * st["scale"]
    s = s.masked_fill_(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = s.sub_(top).exp_()
    z = p.sum(-1, keepdim=True)
    v = v * see.any(1)[:, None, :, None]   # what no row sees weighs nothing, whatever it holds
    o = torch.matmul(p.view(seqs, kv, group * rows, -1), v).view(seqs, kv, group, rows, dim)
    o = torch.where(z > 0, o / z, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(seqs * rows, heads, dim)
    lse = (top + z.log())[..., 0].permute(0, 3, 1, 2).reshape(seqs * rows, heads)
    return {"o": o.to(torch.bfloat16), "lse": lse}


def _plain_grow(st, seq, start, end):
    """Pages for the tokens [start, end) of each sequence, shared ones replaced by copies, from the lowest free page on."""
    table, refs = st["table"], st["refs"]
    page, rows = st["k"].shape[3], seq.long()
    have = table[rows]
    at = torch.arange(table.shape[1], device="cuda")
    want = (at >= (start // page)[:, None]) & (at < ((end + page - 1) // page)[:, None])
    shared = want & (have >= 0) & (refs[have.clamp(min=0).long()] > 1)
    need = shared | (want & (have < 0))
    free = (refs == 0).nonzero()[:, 0]
    new = free[(need.view(-1).cumsum(0) - 1).clamp(min=0, max=free.numel() - 1)].view(need.shape)
    table[rows] = torch.where(need, new.int(), have)
    refs[new[need]] = 1
    old = have[shared].long()
    refs.index_add_(0, old, torch.full_like(have[shared], -1))
    for t in (st["k"], st["v"], st["k_scale"], st["v_scale"]):
        if t is not None:
            t[:, new[shared]] = t[:, old]
    return torch.zeros_like(seq)


def _plain_accept(st):
    rows, seqs = st["rows"], st["seq"].numel()
    logits = st["logits"].float()
    tokens, parent = st["tokens"].view(seqs, rows).long(), st["parent"].view(seqs, rows).long()
    top = logits.amax(1)
    best = logits.argmax(1).view(seqs, rows)
    log_z = (top + (logits - top[:, None]).exp().sum(1).log()).view(seqs, rows)
    up = parent.clamp(min=0)
    lp = logits.view(seqs, rows, -1)[torch.arange(seqs, device="cuda")[:, None], up, tokens] - log_z.gather(1, up)
    # a node is accepted where it and all above it are what the model says
    hit = (parent < 0) | (best.gather(1, up) == tokens)
    above = _ancestors(parent)
    taken = (hit[:, None, :] | ~above).all(2)
    n = taken.sum(1)
    at = torch.arange(rows, device="cuda").expand(seqs, rows)
    path = torch.where(taken, at, rows).sort(1).values
    last = path.gather(1, (n - 1)[:, None])
    path = torch.where(path < rows, path, -1).int()
    out = {"argmax_ids": best.int().view(-1), "node_lp": torch.where(parent < 0, torch.zeros_like(lp), lp).view(-1),
           "path": path, "n_path": n.int(), "next_id": best.gather(1, last)[:, 0].int(), "length": st["length"] + n.int()}
    out["result"] = _plain_grow(st, st["seq"], st["length"], out["length"])
    page = st["k"].shape[3]
    pos = st["length"][:, None] + at
    keep = at < n[:, None]
    pg = st["table"][st["seq"].long()].gather(1, torch.where(keep, pos // page, 0).long())[keep].long()
    off, row = (pos % page)[keep].long(), (torch.arange(seqs, device="cuda")[:, None] * rows + path)[keep]
    for p in ("k", "v"):
        x = st[p + "_new"][:, row].transpose(0, 1)                      # (tokens, layers, heads, dim)
        if st[p + "_scale"] is not None:
            top = x.abs().amax(-1).float()
            scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
            x = (x.float() / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
            st[p + "_scale"][:, pg, :, off] = scale
        st[p][:, pg, :, off] = x
    return out | _state(st)


def _plain_fork(st):
    table, refs, page = st["table"], st["refs"], st["k"].shape[3]
    dst = st["dst"].long()
    held = table[dst]
    refs.index_add_(0, held[held >= 0], torch.full_like(held[held >= 0], -1))
    at = torch.arange(table.shape[1], device="cuda")
    table[dst] = torch.where(at < ((st["length"] + page - 1) // page)[:, None], table[st["src"].long()], -1)
    held = table[dst]
    refs.index_add_(0, held[held >= 0], torch.ones_like(held[held >= 0]))
    return {"results": torch.zeros_like(st["results"]), "grown": _plain_grow(st, st["dst"], st["length"], st["end"])} | _state(st)


def _plain_compact(st):
    page, keep = st["k"].shape[3], st["keep"].long()
    held = st["table"][st["seq"].long()].long()
    to = torch.arange(keep.shape[1], device="cuda").expand_as(keep)
    live = to < st["count"][:, None]
    to, keep = torch.where(live, to, 0), torch.where(live, keep, 0)
    a, b = held.gather(1, keep // page)[live], (keep % page)[live]
    x, y = held.gather(1, to // page)[live], (to % page)[live]
    for t in (st["k"], st["v"], st["k_scale"], st["v_scale"]):
        if t is not None:
            t[:, x, :, y] = t[:, a, :, b]
    return {"result": torch.zeros_like(st["result"])} | _state(st)


def _state(st):
    names = ("k", "v", "k_scale", "v_scale", "table", "refs")
    return {"cache_" + n: st[n] for n in names if st[n] is not None}


_PLAIN = {"attn": _plain_attn, "accept": _plain_accept, "fork": _plain_fork, "compact": _plain_compact}


# ----------------------------------------------------- the framework's calls --
@functools.lru_cache(maxsize=None)
def _sampler():
    """The handle that a serving program creates once."""
    from locus_amd import sampler
    s = sampler.Sampler(device=0, max_rows=MAX_ROWS, max_vocab=MAX_VOCAB, max_hist=64, max_top=4)
    s.kv_reserve(MAX_NEW_PAGES)
    return sampler, s


def _own(st):
    module, s = _sampler()
    cache = st.get("cache")
    if cache is None:   # the plan that a program keeps with its cache
        cache = st["cache"] = module.KvCache(st["k"], st["v"], st["table"], st["refs"], k_scale=st["k_scale"],
                                             v_scale=st["v_scale"])
    if st["kind"] == "attn":
        s.tree_attn_dev(st["q"], st["k_new"], st["v_new"], cache, st["out"], seq=st["seq"], length=st["length"],
                        rows_per_seq=st["rows"], mask=st["mask"], scale=st["scale"])
        return st["out"]
    if st["kind"] == "accept":
        out = st["out"]
        s.tree_verify_dev(st["tokens"], st["parent"], out, rows_per_seq=st["rows"], logits=st["logits"], length=st["length"])
        s.kv_grow_dev(cache, st["seq"], st["length"], out["length"], st["result"])
        s.kv_append_dev(cache, st["k_new"], st["v_new"], st["seq"], st["length"], out["n_path"], rows_per_seq=st["rows"],
                        index=out["path"])
        return out | {"result": st["result"]} | _state(st)
    if st["kind"] == "fork":
        res = st["results"]
        s.kv_free_dev(cache, st["dst"], st["none"], res[0])
        s.kv_fork_dev(cache, st["src"], st["dst"], st["length"], res[1])
        s.kv_grow_dev(cache, st["dst"], st["length"], st["end"], res[2])
        return {"results": res, "grown": res[2]} | _state(st)
    s.kv_compact_dev(cache, st["seq"], st["count"], st["keep"], st["result"])
    return {"result": st["result"]} | _state(st)


def run(state):
    return _own(state) if own else _PLAIN[state["kind"]](state)


# -------------------------------------------------------------- what it takes --
def work(case):
    c = case
    token = 2 * c["kv_heads"] * (c["dim"] * _SIZE[c["dtype"]] + (4 if c["dtype"] == "e4m3" else 0))   # of one layer
    page = c["page"]
    if c["kind"] == "attn":
        seqs, rows, heads, kv, dim = (c[k] for k in ("seqs", "rows", "heads", "kv_heads", "dim"))
        tokens = sum(_lengths(c["ctx_lo"], c["ctx_hi"], seqs))
        bytes_ = tokens * token + seqs * rows * (2 * heads + 2 * kv) * dim * 2 + 4 * seqs * rows * heads
        return {"bytes": bytes_ + 4 * tokens // page, "flops": 4 * rows * heads * dim * (tokens + seqs)}
    if c["kind"] == "accept":
        seqs, rows = c["seqs"], c["rows"]
        taken = sum(1 + i % _chain(rows) for i in range(seqs))
        new = 2 * c["kv_heads"] * c["dim"] * 2
        return {"bytes": seqs * rows * (c["vocab"] * _SIZE[c["logits"]] + 16) + taken * c["layers"] * (new + token),
                "flops": 3 * seqs * rows * c["vocab"]}
    if c["kind"] == "fork":
        lengths = _lengths(c["ctx_lo"], c["ctx_hi"], c["sources"])
        last = [int(n % page > 0) for n in lengths]
        copies = sum(last[i % c["sources"]] for i in range(c["forks"]))
        read = sum(last[: c["forks"]])
        return {"bytes": (read + copies) * page * c["layers"] * token + 16 * c["forks"] * (c["ctx_hi"] // page + 1),
                "flops": 0}
    tokens = sum(n * c["keep"] // 1000 for n in _lengths(c["ctx_lo"], c["ctx_hi"], c["seqs"]))
    return {"bytes": tokens * (2 * c["layers"] * token + 4), "flops": 0}


# ---------------------------------------------------------------- in 64 bits --
def _exact_attn(c, st):
    rows, heads, kv, page = c["rows"], c["heads"], c["kv_heads"], c["page"]
    group = heads // kv
    o, lse = [], []
    lengths = st["length"].tolist()
    for i in range(c["seqs"]):
        n, mine = lengths[i], slice(i * rows, (i + 1) * rows)
        pages = st["table"][i, : (n + page - 1) // page].long()

        def rows_of(p):
            x = st[p][0, pages].double()
            if st[p + "_scale"] is not None:
                x = x * st[p + "_scale"][0, pages].double()[..., None]
            x = x.transpose(1, 2).reshape(-1, kv, c["dim"])[:n]
            return torch.cat([x, st[p + "_new"][mine].double()]).repeat_interleave(group, 1).transpose(0, 1).contiguous()

        see = torch.ones(rows, n + rows, device="cuda", dtype=torch.bool)
        for r in range(rows):
            for j in range(rows):
                see[r, n + j] = j <= r if st["mask"] is None else False
        if st["mask"] is not None:
            words = st["mask"][i].cpu().tolist()
            bits = [[(words[r][j // 32] >> (j % 32)) & 1 for j in range(rows)] for r in range(rows)]
            see[:, n:] = torch.tensor(bits, device="cuda") > 0
        k, v, q = rows_of("k"), rows_of("v"), st["q"][mine].double().transpose(0, 1).contiguous()
        s = torch.bmm(q, k.transpose(1, 2).contiguous()) * st["scale"]
        s = s.masked_fill(~see, -math.inf)
        z = torch.logsumexp(s, 2)
        w = torch.nan_to_num(torch.exp(s - z[..., None]), nan=0.0)
        o.append(torch.bmm(w, v).transpose(0, 1))
        lse.append(z.transpose(0, 1))
    return {"o": torch.cat(o), "lse": torch.cat(lse)}


def _exact_accept(c, st):
    rows = c["rows"]
    none = {"argmax_ids": None, "path": None, "n_path": None, "next_id": None, "length": None, "result": None,
            "cache_k": None, "cache_v": None, "cache_table": None, "cache_refs": None}
    if st["k_scale"] is not None:
        none |= {"cache_k_scale": None, "cache_v_scale": None}
    lp = []
    tokens, parent = st["tokens"].tolist(), st["parent"].tolist()
    for i in range(c["seqs"]):
        x = st["logits"][i * rows : (i + 1) * rows].double()
        z = torch.logsumexp(x, 1)
        for j in range(rows):
            p = parent[i * rows + j]
            lp.append(x[p, tokens[i * rows + j]] - z[p] if p >= 0 else z.new_zeros(()))
    return {"node_lp": torch.stack(lp)} | none


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):   # nothing is computed there: rows are moved as they are
        return None
    st = prepare(case, seed)
    return _exact_attn(case, st) if case["kind"] == "attn" else _exact_accept(case, st)
