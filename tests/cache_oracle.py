"""Attention over a paged cache and the rotation of its keys, in 64 bits on the CPU, and how far 32-bit arithmetic may be from them."""
import torch

U = 2.0 ** -24


def rotated(x, positions, frequencies, neighbours):
    """x [rows, heads, head] by angles positions x frequencies."""
    pairs = frequencies.numel()
    x = x.clone()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if neighbours else (slice(0, pairs), slice(pairs, 2 * pairs))
    angle = positions.double()[:, None, None] * frequencies.double()
    c, s, u, v = angle.cos(), angle.sin(), x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = u * c - v * s, u * s + v * c
    return x


def attended(q, keys, values, tables, lengths, starts, scale, window=0, sinks=0, weigh=None):
    """(out, what bounds are made of), rows of no sequence NaN.  All operands float64 on the CPU; ``weigh`` [pages, 1, page, 1]: factors of the
    weights of places.  Infinities and NaN of places that a row does not see do not reach it."""
    pages, kv, page_size, head = keys.shape
    rows, heads, _ = q.shape
    group = heads // kv
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    parts = {name: torch.zeros(rows, heads, head, dtype=torch.float64) for name in ("spread", "plain", "flat")}
    parts["magnitude"], parts["count"] = torch.zeros(rows, heads, 1, dtype=torch.float64), torch.zeros(rows, 1, 1, dtype=torch.float64)
    for s in range(len(lengths)):
        m = starts[s + 1] - starts[s]
        first = lengths[s] - m
        length = min(max(lengths[s], 0), tables.size(1) * page_size)
        j = torch.arange(length)
        page = tables[s].long()[j // page_size]
        there = (page >= 0) & (page < pages)
        page, slot = page.clamp(0, pages - 1), j % page_size
        for i in range(m):
            p, row = first + i, starts[s] + i
            seen = there & (j <= p)
            if window:
                seen &= (j > p - window) | (j < sinks)
            k, v = keys[page[seen], :, slot[seen]].transpose(0, 1), values[page[seen], :, slot[seen]].transpose(0, 1)   # [kv, seen, head]
            x = q[row].view(kv, group, head)
            if not bool(seen.any()):
                out[row] = 0.0
                continue
            scores = (x @ k.transpose(1, 2)) * scale                                                                     # [kv, group, seen]
            most = scores.amax(-1, keepdim=True)
            w = torch.exp(scores - torch.where(most == -float("inf"), torch.zeros(()).double(), most))
            if weigh is not None:
                w = w * weigh[page[seen], 0, slot[seen], 0]
            total = w.sum(-1, keepdim=True)
            mixed = torch.where(total == 0, torch.zeros(()).double(), (w @ v) / total)
            out[row] = mixed.reshape(heads, head)
            plain = (w @ v.abs()) / total
            # error of a score: that of its sum, and the rounding of its distance to the largest
            size = (x.abs() @ k.abs().transpose(1, 2)) * abs(scale)
            parts["magnitude"][row] = (size + scores.abs() + most.abs()).amax(-1).reshape(heads, 1)
            parts["plain"][row] = plain.reshape(heads, head)
            parts["flat"][row] = (v.abs().sum(1)[:, None, :] / total).reshape(heads, head)
            parts["count"][row] = float(seen.sum())
    return out, parts


def bound_of(parts, head, dtype, compute=None):
    """How far the result may be from ``out`` before it is stored: scores off by (head + 6) U of their terms' magnitude (sums in any order, the
    scale, the exponent's argument), exponentials by 4 U (of 16-bit rows by 12 U: weights relative to another score than the largest, or lifted, have exponents of
    up to 16, half a step of which is 2^-21, times log 2), sums over the places by U each -- in both the weighted values and the weights, which
    are divided by -- and weights rounded to ``compute`` before they meet values of that type (half a step of theirs; of halves at least
    2^-25 of the largest weight)."""
    compute = dtype if compute is None else compute
    each = (head + 6) * U * parts["magnitude"] + (4 if compute == torch.float32 else 12) * U + parts["count"] * U
    step = 0.0 if compute == torch.float32 else torch.finfo(compute).eps / 2
    limit = (2 * each + step) * parts["plain"] * (1 + 2 * each + step)
    if compute != torch.float32:
        # the sum of the weights may be that of the rounded ones or of the others
        limit = limit + step * parts["plain"]
    if compute == torch.float16:
        limit = limit + 2.0 ** -25 * parts["flat"]
    return limit
