"""Inputs of the paged-cache tests: pages in random order, NaN wherever no row may look."""
import torch


def pages_for(new, past, heads, kv, hd, *, page=32, dtype=torch.bfloat16, seed=0, device="cuda", spare=3, extra_width=2,
              q_scale=1.5, tail_rows=0, head_major=False):
    """A filled cache and the q rows of one step: dict for ``attend``. Page rows beyond an episode's length, unused
    pages and unused table entries hold NaN / ids that do not exist."""
    g = torch.Generator().manual_seed(seed)
    B = len(new)
    need = [-(-(a + b) // page) for a, b in zip(new, past)]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g).tolist()
    table = torch.full((B, max(need) + extra_width), 1 << 29, dtype=torch.int32)
    shape = (total, kv, page, hd) if head_major else (total, page, kv, hd)
    k, v = torch.full(shape, float("nan")), torch.full(shape, float("nan"))
    if head_major:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    at = 0
    for b in range(B):
        for j in range(need[b]):
            rows = min(page, new[b] + past[b] - j * page)
            table[b, j] = order[at]
            k[order[at], :rows] = torch.randn(rows, kv, hd, generator=g)
            v[order[at], :rows] = torch.randn(rows, kv, hd, generator=g)
            at += 1
    n = sum(new) + tail_rows
    q = torch.randn(n, heads, hd, generator=g) * q_scale
    start = [0]
    for a in new:
        start.append(start[-1] + a)
    i32 = dict(dtype=torch.int32, device=device)
    return dict(q=q.to(dtype).to(device), k_pages=k.to(dtype).to(device), v_pages=v.to(dtype).to(device),
                table=table.to(device), length=torch.tensor([a + b for a, b in zip(new, past)], **i32),
                start=torch.tensor(start, **i32))


def attend_tolerance(ref, weight, dtype, keys):
    """Half a step of the output, half a step on each probability (the second product's operand is 16 bits wide),
    2^-12 for the fp32 scores (|q||k| products summed over up to 128 dims: below 2^-14 of a score of 16) and the
    exponential, and what fp16 drops below its smallest number (2^-25 for each key)."""
    u = torch.finfo(dtype).eps / 2
    return u * ref.abs() + (u + 2.0 ** -12) * weight + (keys + 1) * 2.0 ** -25 * 4
