"""Serving operators of the library as cases that can be timed and checked.

A case is one pass through one of them: attention over a window of keys and a few first
tokens (``window``), attention of one new token over a paged key/value cache (``paged``),
the write of new tokens into that cache (``append``) and its page bookkeeping (``pages``:
fork, free, compact and reserve, as a scheduler calls them between two steps).

``run`` makes the library's calls where ``own`` is true and computes the same from
elementary torch operations in 32 bits otherwise.  ``listed`` holds the cases, ``draw``
gives further ones of the same ranges.
"""

from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

_DEV = "cuda"
_DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}

# Drawn cases stay below the largest listed ones.
_MOST_PAIRS = 4.0e9  # (query head, visible key) pairs x head_dim / 64
_MOST_BYTES = 1.0e9  # of keys and values read, or of rows written
_MOST_CACHE = 6.0e9  # of a cache


# --------------------------------------------------------------------------- #
# Cases
# --------------------------------------------------------------------------- #


def _window(name, batch, heads, kv_heads, queries, keys, head_dim, window, sinks, dtype, padding=0.0):
    case = dict(kind="window", batch=batch, heads=heads, kv_heads=kv_heads, queries=queries, keys=keys,
                head_dim=head_dim, window=window, sinks=sinks, dtype=dtype, padding=padding)
    return dict(name=name, **case) if name else case


def _paged(name, batch, heads, kv_heads, head_dim, page, shortest, longest, window, sinks, dtype):
    case = dict(kind="paged", batch=batch, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                shortest=shortest, longest=longest, window=window, sinks=sinks, dtype=dtype)
    return dict(name=name, **case) if name else case


def _append(name, batch, kv_heads, head_dim, page, new, longest, dtype):
    case = dict(kind="append", batch=batch, kv_heads=kv_heads, head_dim=head_dim, page=page, new=new,
                longest=longest, dtype=dtype)
    return dict(name=name, **case) if name else case


def _pages(name, layers, kv_heads, head_dim, page, live, longest, forks, frees, dtype):
    case = dict(kind="pages", layers=layers, kv_heads=kv_heads, head_dim=head_dim, page=page, live=live,
                longest=longest, forks=forks, frees=frees, dtype=dtype)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # A few short padded prompts of a small model: latency.
        _window("window_short", 3, 4, 4, 77, 77, 32, 16, 2, "bfloat16", padding=0.4),
        # One chunk of a long prompt: its queries see the cached keys before them, shared key heads.
        _window("window_chunk", 1, 16, 4, 1000, 9001, 128, 2048, 4, "float16"),
        # Whole prompts of the longest configuration (C5) with a window in place of full causal attention.
        _window("window_long", 2, 16, 16, 32768, 32768, 64, 4096, 4, "bfloat16"),
        # One request, a short context, every head with keys of its own: latency.
        _paged("paged_single", 1, 16, 16, 64, 16, 77, 77, 0, 0, "float16"),
        # A running batch of a service: ragged contexts, four heads to a key head.
        _paged("paged_batch", 64, 16, 4, 128, 64, 100, 4096, 0, 0, "bfloat16"),
        # One request with a very long context: few rows, one long axis.
        _paged("paged_long", 1, 16, 2, 128, 256, 100000, 100000, 0, 0, "float16"),
        # A large batch with a window and sinks: most of each sequence's pages are not read.
        _paged("paged_window", 200, 16, 16, 64, 32, 50, 4096, 1000, 4, "float16"),
        # The write of one decode step.
        _append("append_step", 64, 4, 128, 64, 1, 4096, "bfloat16"),
        # The write of whole ragged prompts (C4's widths).
        _append("append_prompt", 4, 16, 128, 64, 8192, 8192, "float16"),
        # Between two steps of a small service: two forks, two requests done.
        _pages("pages_step", 2, 4, 64, 16, 12, 500, 2, 2, "float16"),
        # Parallel samples of many prompts over six layers (C3's widths): many begun pages are copied.
        _pages("pages_fork", 6, 16, 64, 64, 64, 1000, 96, 16, "float16"),
        # A cache full of holes after half of its requests ended: thousands of pages move.
        _pages("pages_compact", 2, 4, 128, 64, 300, 2048, 5, 150, "bfloat16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _cache_bytes(tokens, kv_heads, head_dim):
    return 4.0 * tokens * kv_heads * head_dim


def draw(rng):
    kind = rng.choice(["window", "window", "paged", "paged", "paged", "append", "pages"])
    dtype = rng.choice(["float16", "bfloat16"])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "window":
        head_dim = rng.choice([32, 40, 64, 64, 80, 128, 128, 256])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        queries = _log_int(rng, 1, 16384)
        keys = queries if rng.random() < 0.5 else queries + _log_int(rng, 1, 16384)
        window = _log_int(rng, 1, 8192)
        sinks = rng.choice([0, 0, 1, 4, 5, 64, 100])
        padding = 0.5 * rng.random() if queries == keys and rng.random() < 0.4 else 0.0
        most = _MOST_PAIRS * 64 / (head_dim * heads * queries * min(keys, window + sinks))
        batch = _log_int(rng, 1, max(1, min(16, int(most), int(2 ** 27 / (keys * kv_heads * head_dim)))))
        return _window(None, batch, heads, kv_heads, queries, keys, head_dim, window, sinks, dtype, padding)
    if kind == "paged":
        head_dim = rng.choice([32, 64, 64, 80, 128, 128, 256])
        heads = kv_heads * rng.choice([1, 2, 4, 7, 8, 16])
        longest = _log_int(rng, 1, 100000)
        shortest = longest if rng.random() < 0.3 else rng.randint(0, longest)
        window, sinks = (0, 0) if rng.random() < 0.6 else (_log_int(rng, 1, 4096), rng.choice([0, 1, 4, 60]))
        seen = min(longest, window + sinks) if window else longest
        most = min(_MOST_BYTES / _cache_bytes(seen, kv_heads, head_dim),
                   _MOST_CACHE / _cache_bytes(longest, kv_heads, head_dim))
        return _paged(None, _log_int(rng, 1, max(1, min(256, int(most)))), heads, kv_heads, head_dim, page, shortest,
                      longest, window, sinks, dtype)
    head_dim = rng.choice([32, 64, 80, 128, 256])
    if kind == "append":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, 8192)
        longest = new + _log_int(rng, 1, 4096)
        most = min(_MOST_BYTES / 4 / _cache_bytes(new, kv_heads, head_dim),
                   _MOST_CACHE / _cache_bytes(longest, kv_heads, head_dim))
        return _append(None, _log_int(rng, 1, max(1, min(256, int(most)))), kv_heads, head_dim, page, new, longest,
                       dtype)
    layers = rng.randint(1, 8)
    longest = _log_int(rng, 1, 4096)
    most = _MOST_BYTES / 2 / _cache_bytes(longest * layers, kv_heads, head_dim)
    live = _log_int(rng, 2, max(2, min(256, int(most))))
    return _pages(None, layers, kv_heads, head_dim, page, live, longest, rng.randint(1, live), rng.randint(1, live - 1),
                  dtype)


# --------------------------------------------------------------------------- #
# Inputs
# --------------------------------------------------------------------------- #


def _spread(count, low, high):
    """``count`` lengths between low and high, the longest first; the same for every seed."""
    return [high if i == 0 else low + ((i * 2654435761) % 4294967296) * (high - low + 1) // 4294967296
            for i in range(count)]


def _normal(gen, dtype, *shape, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device=_DEV)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        flat[i:i + (1 << 28)].normal_(0.0, scale, generator=gen)
    return out


def _valid_lengths(case):
    s = case["keys"]
    return [s - int(case["padding"] * s * b / max(1, case["batch"] - 1)) for b in range(case["batch"])]


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _scattered_tables(lengths, page, gen):
    """Each sequence's pages, scattered over a cache with a tenth of free ones."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts)
    pages = total + total // 10 + 1
    order = torch.randperm(pages, generator=gen, device=_DEV).to(torch.int32)
    table = torch.full((len(lengths), max(max(counts), 1)), -1, dtype=torch.int32, device=_DEV)
    start = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[start:start + n]
        start += n
    return table, pages


def _prepare_window(case, gen):
    b, hq, hkv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    sq, sk, dtype = case["queries"], case["keys"], _DTYPES[case["dtype"]]
    if sq == sk:  # views of one fused projection's output, as the layer's attention takes them
        fused = _normal(gen, dtype, b, sk, hq + 2 * hkv, d)
        q, k, v = fused[:, :, :hq], fused[:, :, hq:hq + hkv], fused[:, :, hq + hkv:]
    else:
        q = _normal(gen, dtype, b, sq, hq, d)
        k, v = _normal(gen, dtype, b, sk, hkv, d), _normal(gen, dtype, b, sk, hkv, d)
    state = dict(q=q.transpose(1, 2), k=k.transpose(1, 2), v=v.transpose(1, 2), scale=1.5 * d ** -0.5, valid=None)
    if case["padding"] > 0:
        state["valid"] = torch.arange(sk, device=_DEV)[None, :] < _int32(_valid_lengths(case))[:, None]
    return state


def _prepare_paged(case, gen):
    dtype, d = _DTYPES[case["dtype"]], case["head_dim"]
    lengths = _spread(case["batch"], case["shortest"], case["longest"])
    table, pages = _scattered_tables(lengths, case["page"], gen)
    return dict(q=_normal(gen, dtype, case["batch"], case["heads"], d),
                k=_normal(gen, dtype, pages, case["kv_heads"], case["page"], d),
                v=_normal(gen, dtype, pages, case["kv_heads"], case["page"], d),
                table=table, lengths=_int32(lengths), scale=1.5 * d ** -0.5)


def _prepare_append(case, gen):
    dtype, n = _DTYPES[case["dtype"]], case["new"]
    shape = (case["batch"], n, case["kv_heads"], case["head_dim"])
    # one new token each, or prompts of all lengths from one token on, behind what is there already
    new = [1] * case["batch"] if n == 1 else _spread(case["batch"], 1, n)
    before = _spread(case["batch"], 0, case["longest"] - n)
    lengths = [a + b for a, b in zip(new, before)]
    table, pages = _scattered_tables(lengths, case["page"], gen)
    fused = _normal(gen, dtype, shape[0], n, 2, shape[2], shape[3])
    return dict(new_k=fused[:, :, 0], new_v=fused[:, :, 1],
                k=torch.zeros(pages, case["kv_heads"], case["page"], case["head_dim"], dtype=dtype, device=_DEV),
                v=torch.zeros(pages, case["kv_heads"], case["page"], case["head_dim"], dtype=dtype, device=_DEV),
                table=table, lengths=_int32(lengths), new=_int32(new))


def _prepare_pages(case, gen):
    dtype, page, live = _DTYPES[case["dtype"]], case["page"], case["live"]
    lengths = _spread(live, 1, case["longest"])
    width = -(-case["longest"] // page) + 1
    rows = live + case["forks"]
    table = torch.full((rows, width), -1, dtype=torch.int32)
    # every third sequence was forked from the one before it: it shares that one's whole pages
    counts = []
    for i, n in enumerate(lengths):
        shared = min(n, lengths[i - 1]) // page if i % 3 == 2 else 0
        counts.append((shared, -(-n // page)))
    pages = sum(b - a for a, b in counts) + case["forks"] + rows
    pages += pages // 10
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(gen.initial_seed())).to(torch.int32)
    start = 0
    for i, (shared, n) in enumerate(counts):
        table[i, :shared] = table[i - 1, :shared]
        table[i, shared:n] = order[start:start + n - shared]
        start += n - shared
    used = table[table >= 0].long()
    refs = torch.zeros(pages, dtype=torch.int32).index_add_(0, used, torch.ones(used.numel(), dtype=torch.int32))
    lengths = torch.tensor(lengths + [0] * case["forks"], dtype=torch.int32)
    # the sequences that end are the last ones, those that fork are before them (some more than once)
    parents = [i % (live - case["frees"]) for i in range(case["forks"])]
    ints = torch.cat([table.flatten(), lengths, refs]).to(_DEV)
    new = torch.ones(rows, dtype=torch.int32)
    new[live - case["frees"]:live] = 0
    shape = (case["layers"], pages, case["kv_heads"], page, case["head_dim"])
    return dict(saved=ints.clone(), ints=ints, table=ints[:rows * width].view(rows, width),
                lengths=ints[rows * width:rows * width + rows], refs=ints[rows * width + rows:],
                k=_normal(gen, dtype, *shape), v=_normal(gen, dtype, *shape), parents=_int32(parents),
                children=_int32(list(range(live, rows))), done=_int32(list(range(live - case["frees"], live))),
                new=new.to(_DEV))


_PREPARE = {"window": _prepare_window, "paged": _prepare_paged, "append": _prepare_append, "pages": _prepare_pages}


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    return dict(case=case, **_PREPARE[case["kind"]](case, gen))


# --------------------------------------------------------------------------- #
# The library's calls
# --------------------------------------------------------------------------- #


def _ops():
    package = str(pathlib.Path(__file__).resolve().parents[1] / "transformer-kernel_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from tkmi import ops

    return ops


def _own_run(st):
    ops, case = _ops(), st["case"]
    if case["kind"] == "window":
        return ops.window_attention(st["q"], st["k"], st["v"], st["scale"], case["window"], sinks=case["sinks"],
                                    key_valid=st["valid"])
    if case["kind"] == "paged":
        return ops.paged_attention(st["q"], st["k"], st["v"], st["table"], st["lengths"], st["scale"],
                                   window=case["window"], sinks=case["sinks"], max_length=case["longest"])
    if case["kind"] == "append":
        ops.cache_append(st["new_k"], st["new_v"], st["k"], st["v"], st["table"], st["lengths"], new=st["new"])
        return st["k"], st["v"]
    # the tables are put back first: every pass forks, frees and moves the same pages
    st["ints"].copy_(st["saved"])
    table, lengths, refs = st["table"], st["lengths"], st["refs"]
    forked = ops.cache_fork(st["k"], st["v"], table, lengths, refs, st["parents"], st["children"])
    ops.cache_free(table, lengths, refs, st["done"], case["page"])
    used = ops.cache_compact(st["k"], st["v"], table, lengths, refs)
    reserved = ops.cache_reserve(table, lengths, refs, st["new"], case["page"])
    return table, lengths, refs, forked, used, reserved, st["k"], st["v"]


# --------------------------------------------------------------------------- #
# The plain forms
# --------------------------------------------------------------------------- #


def _softmax_rows(scores, seen):
    """exp(s - max) / sum over the seen keys; rows that see none are zeros."""
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_window(st):
    """Blocks of queries against the sinks and the keys that their windows reach."""
    case = st["case"]
    b, hq, hkv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    sq, sk, w, sinks = case["queries"], case["keys"], case["window"], case["sinks"]
    out = torch.empty(b, sq, hq * d, dtype=st["q"].dtype, device=_DEV)
    step = max(64, min(1024, w))
    for i0 in range(0, sq, step):
        i1 = min(i0 + step, sq)
        pos = torch.arange(sk - sq + i0, sk - sq + i1, device=_DEV)
        first = max(0, sk - sq + i0 - w + 1)
        cols = torch.arange(first, sk - sq + i1, device=_DEV)
        if sinks and first:
            cols = torch.cat([torch.arange(min(sinks, first), device=_DEV), cols])
        seen = (cols[None, :] <= pos[:, None]) & ((cols[None, :] > pos[:, None] - w) | (cols[None, :] < sinks))
        seen = seen[None, None, None]
        if st["valid"] is not None:
            seen = seen & st["valid"][:, cols][:, None, None, None, :]
        q = st["q"][:, :, i0:i1].float().view(b, hkv, hq // hkv, i1 - i0, d)
        k = st["k"][:, :, cols].float().transpose(2, 3).contiguous()
        p = _softmax_rows(torch.matmul(q, k[:, :, None]) * st["scale"], seen)
        o = torch.matmul(p, st["v"][:, :, cols].float()[:, :, None])
        out[:, i0:i1] = o.view(b, hq, i1 - i0, d).transpose(1, 2).reshape(b, i1 - i0, hq * d).to(out.dtype)
    return out


def _plain_paged(st):
    """The rows that a sequence's window and sinks hold, gathered from their pages."""
    case = st["case"]
    b, hq, hkv, d, page = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    lengths = st["lengths"].long()[:, None]
    if case["window"] and case["window"] + case["sinks"] < case["longest"]:
        w, sinks = case["window"], case["sinks"]
        slot = torch.arange(sinks + w, device=_DEV)[None, :]
        pos = torch.where(slot < sinks, slot, torch.clamp(lengths - w, min=sinks) + slot - sinks)
    else:
        pos = torch.arange(case["longest"], device=_DEV)[None, :].expand(b, -1)
    seen = pos < lengths
    pos = torch.where(seen, pos, torch.zeros_like(pos))
    ids = torch.gather(st["table"].long(), 1, pos // page).clamp_min(0)
    k = st["k"][ids, :, pos % page].float().permute(0, 2, 3, 1).contiguous()  # [B, Hkv, D, n]
    q = st["q"].float().view(b, hkv, hq // hkv, d)
    p = _softmax_rows(torch.matmul(q, k) * st["scale"], seen[:, None, None, :])
    del k
    v = st["v"][ids, :, pos % page].float().transpose(1, 2).contiguous()
    return torch.matmul(p, v).reshape(b, hq * d).to(st["q"].dtype)


def _plain_append(st):
    case = st["case"]
    row = torch.arange(case["new"], device=_DEV)[None, :].expand(case["batch"], -1)
    new = st["new"].long()[:, None]
    b, i = torch.nonzero(row < new, as_tuple=True)
    pos = (st["lengths"].long()[:, None] - new + row)[b, i]
    ids = st["table"].long()[b, pos // case["page"]]
    st["k"][ids, :, pos % case["page"]] = st["new_k"][b, i]
    st["v"][ids, :, pos % case["page"]] = st["new_v"][b, i]
    return st["k"], st["v"]


def _plain_pages(st):
    case, page = st["case"], st["case"]["page"]
    st["ints"].copy_(st["saved"])
    table, lengths, refs, k, v = st["table"], st["lengths"], st["refs"], st["k"], st["v"]
    entry = torch.arange(table.shape[1], device=_DEV)[None, :]
    done = torch.zeros(1, dtype=torch.int32, device=_DEV)

    def count(ids, by):
        refs.index_add_(0, ids.long(), torch.full((ids.numel(),), by, dtype=torch.int32, device=_DEV))

    # fork: whole pages are shared, the rows of the begun one are copied into the lowest free pages
    parents, children = st["parents"].long(), st["children"].long()
    begun = lengths[parents] % page
    free = torch.nonzero(refs <= 0).flatten()
    i = torch.nonzero(begun > 0).flatten()
    fresh = free[:i.numel()].to(torch.int32)
    whole = entry < (lengths[parents] // page)[:, None]
    table[children] = torch.where(whole, table[parents], table[children])
    count(table[children][whole], 1)
    at = (lengths[parents[i]] // page).long()
    source = table[parents[i], at].long()
    table[children[i], at] = fresh
    refs[fresh.long()] = 1
    used_rows = torch.arange(page, device=_DEV)[None, :] < begun[i][:, None]
    n, row = torch.nonzero(used_rows, as_tuple=True)
    for cache in (k, v):
        cache[:, fresh.long()[n], :, row] = cache[:, source[n], :, row]
    lengths[children] = lengths[parents]
    # free
    rows = st["done"].long()
    held = entry < ((lengths[rows] + page - 1) // page)[:, None]
    count(table[rows][held], -1)
    table[rows] = table[rows].masked_fill(held, -1)
    lengths[rows] = 0
    # compact: the i-th live page past the number of live ones moves into the i-th hole
    live = refs > 0
    used = live.sum()
    ids = torch.arange(refs.numel(), device=_DEV)
    holes, movers = torch.nonzero(~live & (ids < used)).flatten(), torch.nonzero(live & (ids >= used)).flatten()
    for cache in (k, v):
        cache[:, holes] = cache[:, movers]
    to = ids.clone()
    to[movers] = holes
    held = entry < ((lengths + page - 1) // page)[:, None]
    table.copy_(torch.where(held, to[table.long().clamp_min(0)].to(torch.int32), table))
    refs[holes] = refs[movers]
    refs[movers] = 0
    # reserve: the lowest free pages, row by row
    new_lengths = lengths + st["new"]
    wanted = (entry >= ((lengths + page - 1) // page)[:, None]) & (entry < ((new_lengths + page - 1) // page)[:, None])
    r, c = torch.nonzero(wanted, as_tuple=True)
    fresh = torch.nonzero(refs <= 0).flatten()[:r.numel()]
    table[r, c] = fresh.to(torch.int32)
    refs[fresh] = 1
    lengths.copy_(new_lengths)
    return table, lengths, refs, done, used.to(torch.int32).view(1), done.clone(), k, v


_PLAIN = {"window": _plain_window, "paged": _plain_paged, "append": _plain_append, "pages": _plain_pages}


def run(state):
    return _own_run(state) if own else _PLAIN[state["case"]["kind"]](state)


# --------------------------------------------------------------------------- #
# What a pass cannot do without
# --------------------------------------------------------------------------- #


def _ceil(a, b):
    return -(-a // b)


def work(case):
    kind, d = case["kind"], case["head_dim"]
    if kind == "window":
        sq, sk, w, sinks = case["queries"], case["keys"], case["window"], case["sinks"]
        pos = torch.arange(sk - sq, sk, dtype=torch.int64)
        first = torch.clamp(pos - w + 1, min=0)
        pairs = reached = 0
        for n in _valid_lengths(case):
            pairs += int((torch.clamp(pos + 1, max=n) - first).clamp_min(0).sum()
                         + torch.minimum(torch.full_like(first, min(sinks, n)), first).sum())
            low = max(0, sk - sq - w + 1)
            reached += max(0, n - low) + min(sinks, low, n)
        rows = case["batch"] * case["heads"] * sq
        return {"bytes": 2.0 * d * (2 * rows + 2 * reached * case["kv_heads"]),
                "flops": 4.0 * d * case["heads"] * pairs}
    if kind == "paged":
        lengths = _spread(case["batch"], case["shortest"], case["longest"])
        seen = sum(min(n, case["window"] + case["sinks"]) if case["window"] else n for n in lengths)
        rows = 2 * case["batch"] * case["heads"] + 2 * seen * case["kv_heads"]
        return {"bytes": 2.0 * d * rows + 4.0 * sum(_ceil(n, case["page"]) for n in lengths),
                "flops": 4.0 * d * case["heads"] * seen}
    if kind == "append":
        n = case["new"]
        new = [1] * case["batch"] if n == 1 else _spread(case["batch"], 1, n)
        return {"bytes": 2.0 * 2 * 2 * sum(new) * case["kv_heads"] * d, "flops": 0.0}
    lengths = _spread(case["live"], 1, case["longest"])
    page, keep = case["page"], case["live"] - case["frees"]
    begun = sum(lengths[i % keep] % page for i in range(case["forks"]))
    # live pages lie anywhere in the cache: the share of them past their number is that of the free ones
    counts = [_ceil(n, page) - (min(n, lengths[i - 1]) // page if i % 3 == 2 else 0) for i, n in enumerate(lengths)]
    total = sum(counts) + case["forks"] + case["live"] + case["forks"]
    total += total // 10
    live = sum(counts[:keep]) + case["forks"]
    moved = live * (1.0 - min(1.0, live / total))
    ints = 4.0 * (2 * total + 2 * (sum(counts) + 2 * case["live"]))
    row = 2.0 * 2 * 2 * case["layers"] * case["kv_heads"] * d
    return {"bytes": ints + row * (begun + page * moved), "flops": 0.0}


# --------------------------------------------------------------------------- #
# From the definitions, in 64 bits
# --------------------------------------------------------------------------- #


def _exact_window(case, st):
    """Every key against every query of a block, one head at a time."""
    b, hq, hkv, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    sq, sk = case["queries"], case["keys"]
    if float(b) * hq * sq * sk > 1.2e11:
        return None
    out = torch.zeros(b, sq, hq, d, dtype=torch.float64, device=_DEV)
    j = torch.arange(sk, device=_DEV)
    block = max(1, min(sq, (1 << 26) // sk))
    for n in range(b):
        allowed = torch.ones(sk, dtype=torch.bool, device=_DEV) if st["valid"] is None else st["valid"][n]
        for h in range(hq):
            k, v = st["k"][n, h // (hq // hkv)].double(), st["v"][n, h // (hq // hkv)].double()
            for i in range(0, sq, block):
                at = torch.arange(i, min(sq, i + block), device=_DEV)[:, None] + (sk - sq)
                hidden = (j > at) | ((j <= at - case["window"]) & (j >= case["sinks"])) | ~allowed
                e = torch.mm(st["q"][n, h, i:i + block].double(), k.t()).mul_(st["scale"])
                e.masked_fill_(hidden, -1e300)
                e = torch.exp_(e.sub_(e.amax(1, keepdim=True))).masked_fill_(hidden, 0.0)
                total = e.sum(1, keepdim=True)
                out[n, i:i + block, h] = torch.mm(e, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.view(b, sq, hq * d)


def _exact_paged(case, st):
    """One sequence at a time, its keys laid end to end."""
    b, hq, hkv, d, page = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=_DEV)
    for n, length in enumerate(_spread(b, case["shortest"], case["longest"])):
        if length == 0:
            continue
        ids = st["table"][n, :_ceil(length, page)].long()
        k, v = (st[c][ids].transpose(1, 2).reshape(-1, hkv, d)[:length] for c in ("k", "v"))
        if case["window"] and length > case["window"] + case["sinks"]:
            keep = list(range(case["sinks"])) + list(range(length - case["window"], length))
            k, v = k[keep], v[keep]
        q = st["q"][n].double().view(hkv, hq // hkv, 1, d)
        e = (q * k.double().transpose(0, 1)[:, None]).sum(-1) * st["scale"] if k.shape[0] * hq * d < 1 << 27 else \
            torch.matmul(q[:, :, 0], k.double().permute(1, 2, 0).contiguous()) * st["scale"]
        e = torch.exp(e - e.amax(-1, keepdim=True))
        out[n] = (torch.matmul(e, v.double().transpose(0, 1).contiguous()) / e.sum(-1, keepdim=True)).view(hq, d)
    return out.view(b, hq * d)


def exact(case, seed):
    if case["kind"] == "window":
        return _exact_window(case, prepare(case, seed))
    if case["kind"] == "paged":
        return _exact_paged(case, prepare(case, seed))
    return None  # copies and whole numbers
