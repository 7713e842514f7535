"""Plain 64-bit forms of the serving operators, and how far a kernel may be from them."""

from __future__ import annotations

import math

import torch

# half a step of rounding to nearest, relative to the value
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend(q, k, v, scale, seen):
    """q [n, d], k, v [m, d], seen [n, m] -> (out, A, S): the rows' attention, their weighted mean
    of |v| and their largest sum of |q||k| * scale over the seen keys (all double)."""
    q, k, v = q.double(), k.double(), v.double()
    k = torch.where(seen.any(0)[:, None], k, torch.zeros_like(k))
    v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
    scores = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    top = scores.amax(1, keepdim=True) if scores.shape[1] else scores.new_zeros(scores.shape[0], 1)
    w = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = w.sum(1, keepdim=True)
    w = w / torch.where(total == 0, torch.ones_like(total), total)
    size = (q.abs() @ k.abs().T * scale).masked_fill(~seen, 0.0)
    largest = size.amax(1) if size.shape[1] else size.new_zeros(size.shape[0])
    return w @ v, w @ v.abs(), largest


def tolerance(out, a, s, dtype, keys, head_dim, vmax, p_step):
    """Output rounding; 2 A times the relative error of a weight (its rounding to 16 bits p_step, a
    head_dim-term fp32 score, the hardware's exp2 and a few fp32 roundings) and of `keys` fp32
    additions; and fp16's absolute step below 2^-14, at most 2^-25 of the largest weight per key."""
    u = HALF_STEP[dtype]
    weight = p_step + head_dim * 2.0 ** -24 * s[:, None] + 2.0 ** -20 + keys * 2.0 ** -24
    tol = u * out.abs() + 2 * a * weight + 2.0 ** -24
    if dtype == torch.float16:
        tol = tol + keys * 2.0 ** -25 * vmax
    return tol * (1 + u)


# fp16 weights go into the products up to 2^15: a weight's step is absolute below 2^-14, half of it 2^-25.
# paged_attention: relative to the largest weight 2^-25 / 2^15.  window_attention's reference lies 7 below the
# largest score of the tile that set it, which no later weight undercuts: 2^-25 / 2^7 of the largest weight.
SMALLEST = {"paged": 2.0 ** -40, "window": 2.0 ** -32}


def small_weight_tolerance(out, a, s, dtype, keys, head_dim, vmax, p_step, kind):
    """As `tolerance`, with what a key's weight can lose below fp16's normal range."""
    u = HALF_STEP[dtype]
    weight = p_step + head_dim * 2.0 ** -24 * s[:, None] + 2.0 ** -20 + keys * 2.0 ** -24
    tol = u * out.abs() + 2 * a * weight + 2.0 ** -24
    if dtype == torch.float16:
        tol = tol + 2 * keys * SMALLEST[kind] * vmax
    return tol * (1 + u)


def window_seen(sq, sk, window, sinks, valid=None):
    pos = torch.arange(sk - sq, sk)[:, None]
    j = torch.arange(sk)[None, :]
    seen = (j <= pos) & ((j > pos - window) | (j < sinks))
    return seen if valid is None else seen & valid[None, :]


def window_reference(q, k, v, scale, window, sinks, valid=None):
    """[B, H, Sq, d] inputs -> out and tolerance as [B, Sq, H*d]."""
    b, h, sq, d = q.shape
    group, sk = h // k.shape[1], k.shape[2]
    out = torch.zeros(b, sq, h, d, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for n in range(b):
        seen = window_seen(sq, sk, window, sinks, None if valid is None else valid[n])
        for i in range(h):
            o, a, s = attend(q[n, i], k[n, i // group], v[n, i // group], scale, seen)
            out[n, :, i] = o
            used = v[n, i // group][seen.any(0)].double().abs()
            tol[n, :, i] = tolerance(o, a, s, q.dtype, min(sk, window + sinks), d,
                                     float(used.max()) if used.numel() else 0.0, HALF_STEP[q.dtype])
    return out.flatten(2), tol.flatten(2)


def paged_reference(q, k_pages, v_pages, table, lengths, scale, window=0, sinks=0):
    """[B, H, d] queries over [pages, Hkv, page_size, d] -> out and tolerance as [B, H*d]."""
    b, h, d = q.shape
    pages, hkv, ps, _ = k_pages.shape
    out = torch.zeros(b, h, d, dtype=torch.float64)
    tol = torch.full_like(out, 2.0 ** -24)
    for n in range(b):
        length = min(max(int(lengths[n]), 0), table.shape[1] * ps)
        if length == 0:
            continue
        j = torch.arange(length)
        ids = table[n, j // ps].long()
        seen = (ids >= 0) & (ids < pages)
        if window:
            seen &= (j >= length - window) | (j < sinks)
        ids = torch.where(seen, ids, torch.zeros_like(ids))
        for i in range(h):
            k, v = k_pages[ids, i // (h // hkv), j % ps], v_pages[ids, i // (h // hkv), j % ps]
            o, a, s = attend(q[n, i][None], k, v, scale, seen[None])
            vmax = float(v[seen].double().abs().max()) if bool(seen.any()) else 0.0
            # bf16 weights go into the product as the sum of two bf16 numbers
            p_step = 2.0 ** -16 if q.dtype == torch.bfloat16 else HALF_STEP[q.dtype]
            out[n, i] = o[0]
            tol[n, i] = tolerance(o, a, s, q.dtype, int(seen.sum()), d, vmax, p_step)[0]
    return out.flatten(1), tol.flatten(1)


class Book:
    """The bookkeeping of a cache on Python lists: what the device must arrive at."""

    def __init__(self, table, lengths, refs, page_size):
        self.table, self.lengths, self.refs, self.ps = table.tolist(), lengths.tolist(), refs.tolist(), page_size
        self.width = table.shape[1]
        self.copies = []  # (from page, to page, rows) in order

    def held(self, b):
        return -(-self.lengths[b] // self.ps)

    def free_pages(self):
        return [p for p, r in enumerate(self.refs) if r <= 0]

    def reserve(self, new):
        most = self.width * self.ps
        if any(n < 0 or l < 0 or l + n > most for l, n in zip(self.lengths, new)):
            return -1
        need = [-(-(l + n) // self.ps) - -(-l // self.ps) for l, n in zip(self.lengths, new)]
        free = self.free_pages()
        if sum(need) > len(free):
            return sum(need) - len(free)
        for b, n in enumerate(need):
            for e in range(self.held(b), self.held(b) + n):
                self.table[b][e] = free.pop(0)
                self.refs[self.table[b][e]] = 1
            self.lengths[b] += new[b]
        return 0

    def fork(self, parents, children):
        rows = range(len(self.lengths))
        if any(p not in rows or c not in rows for p, c in zip(parents, children)) or \
                len(set(children)) < len(children) or any(self.lengths[c] for c in children):
            return -1
        free = self.free_pages()
        before = list(self.lengths)
        short = sum(before[p] % self.ps > 0 for p in parents) - len(free)
        if short > 0:
            return short
        for p, c in zip(parents, children):
            whole, begun = divmod(before[p], self.ps)
            for e in range(whole):
                self.table[c][e] = self.table[p][e]
                self.refs[self.table[p][e]] += 1
            if begun:
                self.table[c][whole] = free.pop(0)
                self.refs[self.table[c][whole]] = 1
                self.copies.append((self.table[p][whole], self.table[c][whole], begun))
            self.lengths[c] = before[p]
        return 0

    def free(self, rows):
        for b in rows:
            if 0 <= b < len(self.lengths):
                for e in range(self.held(b)):
                    self.refs[self.table[b][e]] -= 1
                    self.table[b][e] = -1
                self.lengths[b] = 0

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if self.refs[p] <= 0]
        movers = [p for p in range(used, len(self.refs)) if self.refs[p] > 0]
        to = dict(zip(movers, holes))
        for page, hole in to.items():
            self.refs[hole], self.refs[page] = self.refs[page], 0
            self.copies.append((page, hole, self.ps))
        for b in range(len(self.lengths)):
            for e in range(self.held(b)):
                self.table[b][e] = to.get(self.table[b][e], self.table[b][e])
        return used
