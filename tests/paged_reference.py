"""Plain restatements, in 64 bits and with loops over sequences, of the operators over a paged KV cache."""
import math

import torch


def angles(positions, frequencies):
    return torch.as_tensor(positions).double()[:, None] * torch.tensor(frequencies, dtype=torch.float64)


def rotated(x, positions, table, interleaved=False, backward=False):
    """x [tokens, heads, D] -> float64."""
    y = x.detach().cpu().double().clone()
    pairs = table.rotary_dim // 2
    a = angles(positions.cpu(), table.frequencies)[:, None, :]
    cos, sin = table.magnitude * a.cos(), table.magnitude * a.sin() * (-1 if backward else 1)
    i = torch.arange(pairs)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    u, w = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = u * cos - w * sin, w * cos + u * sin
    return y


def pair_norms(x, table, interleaved=False):
    """|u| + |w| of every element's pair (0 where elements are copied): what the rounding of sine and cosine scales with."""
    pairs = table.rotary_dim // 2
    i = torch.arange(pairs)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)
    x = x.detach().cpu().double().abs()
    out = torch.zeros_like(x)
    out[..., first] = out[..., second] = x[..., first] + x[..., second]
    return out


def gathered(pages, table_row, length, page_size):
    """[length, heads, D] rows of one sequence, on the cache's device."""
    at = torch.arange(length, device=pages.device)
    return pages[table_row.long().to(pages.device)[at // page_size], at % page_size]


def attention(q, k, v, table, lengths, starts, scale, causal=True, zero_fully_masked=False):
    """(out, lse, bound_out, bound_lse) in float64 on q's device; rows of no sequence are NaN. The bounds are those of f32
    scores and sums with probabilities and results rounded to q's type:
      scores    |ds| <= scale (D + 4) 2^-24 sum_d |q_d k_d|                    (products and sums in f32, one scaling)
      p         relative 2 |ds| + 2^-20 (exponential, its argument, the sums)  and half a step of the type
      out       half a step of the type on top"""
    size, unit = k.shape[1], torch.finfo(q.dtype).eps / 2
    group = q.shape[1] // k.shape[2]
    nan = float("nan")
    out = torch.full(q.shape, nan, dtype=torch.float64, device=q.device)
    bound = torch.full(q.shape, nan, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], nan, dtype=torch.float64, device=q.device)
    bound_lse = torch.full(q.shape[:2], nan, dtype=torch.float64, device=q.device)
    starts, lengths = starts.tolist(), lengths.tolist()
    for s, length in enumerate(lengths):
        first, n = starts[s], starts[s + 1] - starts[s]
        if n <= 0:
            continue
        rows = slice(first, first + n)
        if length == 0:
            out[rows] = 0.0 if zero_fully_masked else nan
            lse[rows], bound[rows], bound_lse[rows] = -math.inf, 0.0, 0.0
            continue
        keys = gathered(k, table[s], length, size).double().repeat_interleave(group, 1)
        values = gathered(v, table[s], length, size).double().repeat_interleave(group, 1)
        qs = q[rows].double()
        scores = torch.einsum("nhd,lhd->hnl", qs, keys) * scale
        slack = torch.einsum("nhd,lhd->hnl", qs.abs(), keys.abs()) * (scale * (q.shape[2] + 4) * 2.0 ** -24)
        if causal:
            last = torch.arange(n, device=q.device) + (length - n)
            hidden = torch.arange(length, device=q.device)[None, :] > last[:, None]
            scores.masked_fill_(hidden, -math.inf)
            slack.masked_fill_(hidden, 0.0)
        top = torch.logsumexp(scores, -1)
        p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top)[..., None])
        error = 2 * slack.amax(-1) + 2.0 ** -20
        o = torch.einsum("hnl,lhd->nhd", p, values)
        empty = (top == -math.inf).T
        out[rows] = torch.where(empty[..., None], torch.full_like(o, 0.0 if zero_fully_masked else nan), o)
        lse[rows] = top.T
        bound[rows] = torch.einsum("hnl,lhd->nhd", p, values.abs()) * (unit + error.T[..., None]) * (1 + unit) + unit * o.abs()
        bound_lse[rows] = error.T + top.T.abs().nan_to_num(posinf=0.0) * 2.0 ** -22
    return out, lse, bound, bound_lse


class Pages:
    """The page arrays as plain Python lists, changed one sequence at a time."""

    def __init__(self, table, lengths, refs, page_size):
        self.table, self.lengths, self.refs, self.size = table.cpu().tolist(), lengths.cpu().tolist(), refs.cpu().tolist(), page_size

    def count(self, s):
        return -(-self.lengths[s] // self.size)

    def _take(self):
        page = self.refs.index(0)
        self.refs[page] = 1
        return page

    def reserve(self, wanted):
        wanted = wanted.tolist()
        need = [-(-max(w, n) // self.size) for w, n in zip(wanted, self.lengths)]
        if any(n > len(self.table[0]) for n in need):
            return -1
        missing = sum(n - self.count(s) for s, n in enumerate(need)) - self.refs.count(0)
        if missing > 0:
            return missing
        for s, n in enumerate(need):
            for j in range(self.count(s), n):
                self.table[s][j] = self._take()
            self.lengths[s] = max(self.lengths[s], wanted[s])
        return 0

    def fork(self, parents, children):
        parents, children = parents.tolist(), children.tolist()
        inside = range(len(self.lengths))
        if any(i not in inside for i in parents + children) or len(set(children)) < len(children) or set(parents) & set(children) or \
                any(self.lengths[c] for c in children):
            return -1, [-1] * len(parents), [-1] * len(parents)
        missing = sum(1 for p in parents if self.lengths[p] % self.size) - self.refs.count(0)
        if missing > 0:
            return missing, [-1] * len(parents), [-1] * len(parents)
        sources, destinations = [-1] * len(parents), [-1] * len(parents)
        for i, (p, c) in enumerate(zip(parents, children)):
            full, width = self.lengths[p] // self.size, len(self.table[0])
            self.table[c] = self.table[p][:full] + [-1] * (width - full)
            for page in self.table[p][:full]:
                self.refs[page] += 1
            if self.lengths[p] % self.size:
                sources[i], destinations[i] = self.table[p][full], self._take()
                self.table[c][full] = destinations[i]
            self.lengths[c] = self.lengths[p]
        return 0, sources, destinations

    def free(self, sequences):
        for s in sequences.tolist():
            if s < 0 or self.lengths[s] == 0:
                continue
            for page in self.table[s][:self.count(s)]:
                self.refs[page] -= 1
            self.table[s], self.lengths[s] = [-1] * len(self.table[s]), 0

    def compact(self):
        live = sum(1 for r in self.refs if r > 0)
        sources = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        destinations = [p for p in range(live) if self.refs[p] == 0]
        place = dict(zip(sources, destinations))
        for s in range(len(self.lengths)):
            for j in range(self.count(s)):
                self.table[s][j] = place.get(self.table[s][j], self.table[s][j])
        for a, b in zip(sources, destinations):
            self.refs[b], self.refs[a] = self.refs[a], 0
        pad = [-1] * (len(self.refs) // 2 - len(sources))
        return sources + pad, destinations + pad
