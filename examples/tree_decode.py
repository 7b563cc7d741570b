"""Speculative decoding with trees of drafts over a paged cache.

Every call of a decoding step on the device: the tree's attention over the cache
(lcs_tree_attn), the residual norm (lcs_add_rmsnorm), the lm-head's argmax
(lcs_lmhead), the verdict (lcs_tree_verify), pages for the accepted tokens
(lcs_kv_grow) and their keys and values (lcs_kv_append). At the end one stream is
forked (lcs_kv_fork) and another cut to part of its context (lcs_kv_compact).

The model is one attention layer of random weights, without positions; drafts are the
two tokens that last followed the same token in the stream, and one at random.

    python examples/tree_decode.py [--streams 8] [--steps 32]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from locus_amd.sampler import KvCache, Sampler  # noqa: E402

HEADS, KV_HEADS, DIM, PAGE, VOCAB = 8, 2, 64, 16, 512
HIDDEN = HEADS * DIM
PARENT = [-1, 0, 0, 0, 1, 1, 4]        # three continuations, two more of the first, one of theirs
ROWS = len(PARENT)


class Model:
    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()   # noqa: E731
        self.embed = rand(VOCAB, HIDDEN)
        self.qkv = rand(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM) * HIDDEN ** -0.5
        self.out = rand(HEADS * DIM, HIDDEN) * HIDDEN ** -0.5
        self.norm = torch.ones(HIDDEN, device="cuda", dtype=torch.bfloat16)
        self.head = rand(VOCAB, HIDDEN) * HIDDEN ** -0.5

    def project(self, tokens):
        x = self.embed[tokens.long()]
        y = x @ self.qkv
        q, k, v = y.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], 1)
        return x, q.view(-1, HEADS, DIM), k.view(-1, KV_HEADS, DIM), v.view(-1, KV_HEADS, DIM)


def ancestors(parent):
    """Each node's own bit and those of the nodes above it."""
    words = []
    for j, p in enumerate(parent):
        words.append((words[p] if p >= 0 else 0) | 1 << j)
    return words


def run(streams=8, steps=32, prompt=40, seed=0):
    """Decodes and returns the streams' tokens and how many drafts were accepted."""
    model, s = Model(seed), Sampler(device=0, max_rows=streams * ROWS, max_vocab=VOCAB, max_hist=16, max_top=1)
    ints = lambda *shape: torch.empty(*shape, device="cuda", dtype=torch.int32)   # noqa: E731
    slots = streams + 1                                   # (one for the fork)
    max_pages = (prompt + steps * ROWS) // PAGE + 2
    pages = slots * max_pages
    shape = (1, pages, KV_HEADS, PAGE, DIM)
    cache = KvCache(torch.zeros(shape, device="cuda", dtype=torch.bfloat16), torch.zeros(shape, device="cuda", dtype=torch.bfloat16),
                    torch.full((slots, max_pages), -1, device="cuda", dtype=torch.int32), torch.zeros(pages, device="cuda", dtype=torch.int32))
    s.kv_reserve(pages)
    seq = torch.arange(streams, device="cuda", dtype=torch.int32)
    length, result = torch.zeros_like(seq), ints(streams)

    # the prompts' keys and values (all but the last token's, which is the first tree's root)
    g = torch.Generator().manual_seed(seed + 1)
    text = [torch.randint(0, VOCAB // 16, (prompt,), generator=g).tolist() for _ in range(streams)]
    _, _, k, v = model.project(torch.tensor([t for line in text for t in line[:-1]], device="cuda"))
    s.kv_grow_dev(cache, seq, length, length + (prompt - 1), result)
    s.kv_append_dev(cache, k, v, seq, length, rows_per_seq=prompt - 1)
    length += prompt - 1

    parent = torch.tensor(PARENT * streams, device="cuda", dtype=torch.int32)
    mask = torch.tensor(ancestors(PARENT) * streams, device="cuda", dtype=torch.int32).view(-1, 1)
    rows = streams * ROWS
    attn = {"o": torch.empty(rows, HEADS, DIM, device="cuda", dtype=torch.bfloat16)}
    said = {"argmax_ids": ints(rows), "path": ints(streams, ROWS), "n_path": ints(streams), "next_id": ints(streams), "length": ints(streams)}
    normed = {"y": torch.empty(rows, HIDDEN, device="cuda", dtype=torch.bfloat16)}
    accepted = 0
    for _ in range(steps):
        # drafts: what last followed a token in its stream
        trees = []
        for line in text:
            after = {a: b for a, b in zip(line, line[1:])}
            two = {a: b for a, b in zip(line[:-8], line[1:-8])}
            draft = lambda t, of=after: of.get(t, (t * 7 + 3) % VOCAB)   # noqa: E731
            root = line[-1]
            one = draft(root)
            trees += [root, one, draft(root, two), (root + 1) % VOCAB, draft(one), draft(one, two), draft(draft(one))]
        tokens = torch.tensor(trees, device="cuda", dtype=torch.int32)
        x, q, k, v = model.project(tokens)
        s.tree_attn_dev(q, k, v, cache, attn, length=length, seq=seq, rows_per_seq=ROWS, mask=mask)
        s.add_rmsnorm_dev(attn["o"].view(rows, -1) @ model.out, model.norm, normed, residual=x)
        s.lmhead_dev(normed["y"], model.head, {"argmax_ids": said["argmax_ids"]})
        s.tree_verify_dev(tokens, parent, said, rows_per_seq=ROWS, length=length)
        s.kv_grow_dev(cache, seq, length, said["length"], result)
        s.kv_append_dev(cache, k, v, seq, length, said["n_path"], rows_per_seq=ROWS, index=said["path"])
        length.copy_(said["length"])
        paths, nexts = said["path"].tolist(), said["next_id"].tolist()
        for i, line in enumerate(text):
            path = [j for j in paths[i] if j > 0]
            line += [trees[i * ROWS + j] for j in path] + [nexts[i]]
            accepted += len(path)
    # the last stream with every other token of its context, and a second continuation of stream 0
    kept = length.tolist()
    last, cut, fork = seq[-1:], ints(1), ints(1)
    n = (length[-1:] + 1) // 2
    keep = torch.arange(0, kept[-1], 2, device="cuda", dtype=torch.int32)[None]
    s.kv_compact_dev(cache, last, n, keep, cut)
    s.kv_free_dev(cache, last, n, ints(1))
    length[-1:] = n
    s.kv_fork_dev(cache, seq[:1], torch.full_like(last, streams), length[:1], fork)
    torch.cuda.synchronize()
    ok = s.status() == 0 and fork.item() == 0 and cut.item() == 0
    held = length.tolist() + [length[0].item()]
    s.close()
    return {"text": text, "accepted": accepted, "length": kept, "ok": ok, "pages_held": cache._keep[3].sum().item(),
            "pages_expected": sum(-(-n // PAGE) for n in held)}


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--streams", type=int, default=8)
    p.add_argument("--steps", type=int, default=32)
    a = p.parse_args()
    r = run(a.streams, a.steps)
    print("%d streams, %d steps: %.2f tokens a step and stream, pages held %d" %
          (a.streams, a.steps, 1 + r["accepted"] / (a.streams * a.steps), r["pages_held"]))
