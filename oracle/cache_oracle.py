"""CPU restatement of the paged episode cache in 64 bits -- test infrastructure only: imported by tests/, never by the
product path. No counterpart in the reference, whose K/V are dense per episode (src/mk_expert.py:486-495)."""
from __future__ import annotations

import math

import torch


def plan_oracle(length, new, table, free, marks, page_rows: int, rows: int):
    """Plain loops over lists of ints: the state after placing new[b] rows behind length[b], and the rows' maps."""
    table = [list(r) for r in table]
    taken, returned = marks[0], marks[1]
    avail = max(0, returned - taken)
    wide = len(table[0])
    start, slot, episode, position, after, lost = [0], [], [], [], [], 0
    used = 0
    for b, (n, m) in enumerate(zip(length, new)):
        n, m = max(n, 0), max(m, 0)
        fit = min(m, rows - start[-1])
        lost += m - fit
        page = -(-n // page_rows)
        while page * page_rows < n + fit and page < wide and used < avail:
            table[b][page] = free[(taken + used) % len(free)]
            used += 1
            page += 1
        held = max(n, min(n + fit, page * page_rows))
        lost += n + fit - held
        for at in range(n, n + fit):
            ok = at < held and at // page_rows < wide and table[b][at // page_rows] >= 0
            slot.append(table[b][at // page_rows] * page_rows + at % page_rows if ok else -1)
            episode.append(b)
            position.append(at)
        after.append(held)
        start.append(start[-1] + fit)
    pad = rows - start[-1]
    return dict(start=start, slot=slot + [-1] * pad, episode=episode + [-1] * pad, position=position + [0] * pad,
                length=after, marks=[taken + used, returned, lost], table=table)


def axis_of(sections, interleaved: bool):
    """The axis of each frequency."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a, n in enumerate(left):
            if n:
                left[a] -= 1
                out.append(a)
    return out


def angles_oracle(positions, sections, base: float = 10000.0, interleaved: bool = False):
    """[rows, sum(sections)] double: the angle of each frequency."""
    axes = axis_of(sections, interleaved)
    rate = torch.tensor([base ** (-i / len(axes)) for i in range(len(axes))], dtype=torch.float64)
    return positions.cpu().double()[axes].t() * rate


def turn_oracle(x, angle):
    """x [rows, heads, dim] turned by angle [rows, half], in double."""
    half = angle.shape[1]
    x = x.cpu().double()
    a, b = x[..., :half], x[..., half:2 * half]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], -1)


def attend_oracle(q, k_pages, v_pages, table, length, start, *, causal=True, window=0, sinks=0, scale=None):
    """(out, weight) in double on the inputs' device, rows behind start[-1] zero: weight = sum_j p_j |v_j|, the scale of
    an output's error from roundings of p."""
    rows, heads, hd = q.shape
    page, kv = k_pages.shape[1], k_pages.shape[2]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out = torch.zeros(rows, heads, hd, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    start, length = start.tolist(), length.tolist()
    for b, n in enumerate(length):
        r0, r1 = start[b], start[b + 1]
        if r1 <= r0 or n == 0:
            continue
        j = torch.arange(n, device=q.device)
        ids = table[b, : -(-n // page)].long()
        p = n - (r1 - r0) + torch.arange(r1 - r0, device=q.device)[:, None]
        seen = torch.ones(r1 - r0, n, dtype=torch.bool, device=q.device)
        if causal:
            seen &= j <= p
            if window:
                seen &= (j > p - window) | (j < sinks)
        some = seen.any(0).nonzero()[:, 0]   # rows that nobody sees are not read: they may hold anything
        seen = seen[:, some]
        k = k_pages[ids[some // page], some % page].double()
        v = v_pages[ids[some // page], some % page].double()
        for h in range(heads):
            s = q[r0:r1, h].double() @ k[:, h * kv // heads].T * scale
            w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            w = torch.where(seen.any(1, keepdim=True), w, 0.0)
            out[r0:r1, h] = w @ v[:, h * kv // heads]
            weight[r0:r1, h] = w @ v[:, h * kv // heads].abs()
    return out, weight
