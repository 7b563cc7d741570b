"""A paged cache's plain forms, on the CPU: a model of its bookkeeping and the attention
over it in 64 bits."""
import math

import torch


class Model:
    """What a cache's calls do to its table, counts and rows, one request at a time."""

    def __init__(self, k, v, table, refs, k_scale=None, v_scale=None):
        self.rows = [t for t in (k, v, k_scale, v_scale) if t is not None]
        self.table, self.refs = table, refs
        self.pages, self.page = k.shape[1], k.shape[3]
        self.seqs, self.max_pages = table.shape

    def ok(self, page):
        return 0 <= page < self.pages

    def grow(self, seq, start, end, cap):
        held, refs0 = self.table.clone(), self.refs.clone()
        free = [p for p in range(self.pages) if refs0[p] == 0][:cap]
        wants, good = [], []
        for i, s in enumerate(seq):
            valid = s == -1 or (0 <= s < self.seqs and s not in seq[:i] and 0 <= start[i] <= end[i] <= self.max_pages * self.page)
            w = []
            if valid and s != -1 and end[i] > start[i]:
                for p in range(start[i] // self.page, -(-end[i] // self.page)):
                    page = int(held[s, p])
                    if not self.ok(page):
                        w.append((p, -1))
                    elif refs0[page] > 1:
                        w.append((p, page))
            wants.append(w)
            good.append(valid)
        at, result, todo = 0, [], []
        for i, w in enumerate(wants):
            served = good[i] and at + len(w) <= len(free)
            if served:
                todo += [(seq[i], p, src, free[at + n]) for n, (p, src) in enumerate(w)]
            at += len(w)
            result.append(0 if served else -1)
        for s, p, src, new in todo:
            self.table[s, p] = new
            self.refs[new] = 1
            if src >= 0:
                self.refs[src] -= 1
                for t in self.rows:
                    t[:, new] = t[:, src].clone()
        return result

    def fork(self, src, dst, tokens):
        result, held = [], self.table.clone()
        for i, (s, d) in enumerate(zip(src, dst)):
            if s == -1 or d == -1:
                result.append(0)
                continue
            ok = 0 <= s < self.seqs and 0 <= d < self.seqs and d not in dst[:i] and s not in dst
            ok = ok and 0 <= tokens[i] <= self.max_pages * self.page
            n = -(-tokens[i] // self.page)
            ok = ok and not any(self.ok(int(p)) for p in held[d]) and all(self.ok(int(p)) for p in held[s, :n])
            if ok:
                for p in range(n):
                    self.table[d, p] = held[s, p]
                    self.refs[held[s, p]] += 1
            result.append(0 if ok else -1)
        return result

    def free(self, seq, keep):
        result = []
        for i, s in enumerate(seq):
            if s != -1 and (not 0 <= s < self.seqs or s in seq[:i]):
                result.append(-1)
                continue
            result.append(0)
            if s == -1:
                continue
            first = -(-max(0, keep[i] if keep else 0) // self.page)
            for p in range(first, self.max_pages):
                page = int(self.table[s, p])
                if self.ok(page):
                    self.refs[page] -= 1
                self.table[s, p] = -1
        return result

    def compact(self, seq, count, keep):
        result = []
        for i, s in enumerate(seq):
            if s == -1:
                result.append(0)
                continue
            n = min(max(count[i], 0), len(keep[i]))
            ok = 0 <= s < self.seqs and s not in seq[:i]
            for j in range(n if ok else 0):
                pos, last = keep[i][j], keep[i][j - 1] if j else -1
                if pos <= last or pos // self.page >= self.max_pages:
                    ok = False
                    break
                a, b = int(self.table[s, pos // self.page]), int(self.table[s, j // self.page])
                ok = ok and self.ok(a) and self.ok(b) and (pos == j or self.refs[b] <= 1)
            result.append(0 if ok else -1)
            if not ok:
                continue
            for j in range(n):
                a, b = int(self.table[s, keep[i][j] // self.page]), int(self.table[s, j // self.page])
                for t in self.rows:
                    t[:, b, :, j % self.page] = t[:, a, :, keep[i][j] % self.page].clone()
        return result


def quantise(x):
    """bf16 rows in e4m3 and their scales, every step rounded as the formula's f32 says."""
    x = x.float()
    top = x.abs().amax(-1)
    scale = torch.where(top > 0, (top / 448.0).clamp(min=2.0 ** -126), torch.ones_like(top))
    return (x / scale[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale


def attention(q, k_new, v_new, rows, ctx_k, ctx_v, see, scale):
    """One sequence's attention in 64 bits: q (rows, heads, dim), k_new and v_new (rows, kv,
    dim), ctx_k and ctx_v (tokens, kv, dim) as f64, see (rows, rows) truth values. Returns
    o, lse, and for the tolerances sum_j p_j |v_j| and the largest scale sum_d |q_d k_d|."""
    heads, kv, n = q.shape[1], k_new.shape[1], ctx_k.shape[0]
    q = q.double()
    k = torch.cat([ctx_k, k_new.double()]).repeat_interleave(heads // kv, 1)
    v = torch.cat([ctx_v, v_new.double()]).repeat_interleave(heads // kv, 1)
    o, lse = torch.zeros_like(q), torch.full((rows, heads), -math.inf, dtype=torch.float64)
    weigh, most = torch.zeros_like(q), torch.zeros(rows, heads, dtype=torch.float64)
    for r in range(rows):
        mine = torch.cat([torch.ones(n, dtype=torch.bool), see[r]]).nonzero()[:, 0]
        if not len(mine):
            continue
        for h in range(heads):
            kk, vv = k[mine, h], v[mine, h]
            s = (kk * q[r, h]).sum(1) * scale
            lse[r, h] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[r, h])
            o[r, h] = (p[:, None] * vv).sum(0)
            weigh[r, h] = (p[:, None] * vv.abs()).sum(0)
            most[r, h] = ((kk * q[r, h]).abs().sum(1) * abs(scale)).max()
    return o, lse, weigh, most
