"""Cases of the paged episode cache: placing new rows (block tables and slot maps), storing them (rotary
positions with several axes, K/V rows into pages) and reading them (attention of new rows over the pages,
with a sliding window and first rows that stay visible).

``run`` computes an operator in elementary torch operations where ``own`` is false, and by
``reki_megakernel_b200.episode_cache`` where it is true.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # every episode of a small batch adds its 10 action rows to its cache: the smallest call, latency counts
        {"name": "plan: 10 rows of 16 episodes", "op": "plan", "episodes": 16, "rows": 160, "split": "even",
         "past": 9001, "page": 32},
        # a large server's step: camera frames and single rows of hundreds of episodes, ragged
        {"name": "plan: 100003 rows of 700", "op": "plan", "episodes": 700, "rows": 100003, "split": "ragged",
         "past": 2500001, "page": 16},
        # one new row of each of 24 episodes, rotated by (time, height, width) and stored
        {"name": "write: 24 rows", "op": "write", "rows": 24, "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "bf16",
         "page": 32, "pages": 500, "sections": "8,12,12", "interleaved": False, "far": 5000},
        # the image rows of 16 camera frames
        {"name": "write: 16 frames of 256 rows", "op": "write", "rows": 4096, "heads": 12, "kv_heads": 12, "dim": 64,
         "dtype": "bf16", "page": 32, "pages": 700, "sections": "8,12,12", "interleaved": False, "far": 70000},
        # a long prompt's rows, shared K/V heads, axes taken in turn, far positions
        {"name": "write: 30011 rows, shared heads", "op": "write", "rows": 30011, "heads": 32, "kv_heads": 8, "dim": 128,
         "dtype": "fp16", "page": 16, "pages": 2100, "sections": "24,20,20", "interleaved": True, "far": 1000000},
        # one new row of each of 8 episodes over a few hundred source rows: the smallest read
        {"name": "attend: 8 single rows", "op": "attend", "episodes": 8, "rows": 8, "split": "even", "past": 3001,
         "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "bf16", "page": 32, "causal": True, "window": 0, "sinks": 0},
        # one new row of each of 96 episodes over long ragged caches with shared K/V heads: bound by reading the cache
        {"name": "attend: 96 single rows, long", "op": "attend", "episodes": 96, "rows": 96, "split": "even",
         "past": 400001, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "causal": True,
         "window": 0, "sinks": 0},
        # one episode alone with a very long cache: the work has to be split along the cache
        {"name": "attend: 1 row after 250007", "op": "attend", "episodes": 1, "rows": 1, "split": "even",
         "past": 250007, "heads": 16, "kv_heads": 2, "dim": 128, "dtype": "fp16", "page": 128, "causal": True,
         "window": 0, "sinks": 0},
        # the 10 action rows of 128 episodes over their source rows, every row seeing all of them
        {"name": "attend: 10 rows of 128, all", "op": "attend", "episodes": 128, "rows": 1280, "split": "even",
         "past": 60007, "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "bf16", "page": 32, "causal": False,
         "window": 0, "sinks": 0},
        # a long prompt in chunks: 2011 new rows after 6007
        {"name": "attend: 2011 rows after 6007", "op": "attend", "episodes": 1, "rows": 2011, "split": "even",
         "past": 6007, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16", "page": 64, "causal": True,
         "window": 0, "sinks": 0},
        # camera frames of 6 episodes: the instruction's rows stay visible, older frames leave the window
        {"name": "attend: frames of 6, window", "op": "attend", "episodes": 6, "rows": 6001, "split": "ragged",
         "past": 24001, "heads": 12, "kv_heads": 12, "dim": 64, "dtype": "bf16", "page": 32, "causal": True,
         "window": 1024, "sinks": 70},
        # single rows of 48 episodes that have run for long: only the window and the first rows are read
        {"name": "attend: 48 single rows, window", "op": "attend", "episodes": 48, "rows": 48, "split": "even",
         "past": 600011, "heads": 24, "kv_heads": 4, "dim": 128, "dtype": "fp16", "page": 16, "causal": True,
         "window": 4000, "sinks": 4},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attend", "attend", "attend"])
    if op == "plan":
        b = _log(rng, 1, 700)
        rows = min(100003, b * _log(rng, 1, 2000))
        return {"op": op, "episodes": b, "rows": rows, "split": rng.choice(["even", "ragged"]),
                "past": rng.randint(0, b * 3500), "page": rng.choice([16, 32, 64, 128])}
    heads, kv_heads, dim = rng.choice([(12, 12, 64), (12, 4, 64), (32, 8, 128), (16, 2, 128), (24, 4, 128), (7, 1, 64),
                                       (5, 5, 128)])
    kind = {"heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": rng.choice(["bf16", "fp16"]),
            "page": rng.choice([16, 32, 64, 128])}
    if op == "write":
        rows = _log(rng, 1, 30011)
        sections = {64: ["32", "16,16", "8,12,12", "12,10,10"], 128: ["64", "16,24,24", "24,20,20", "16,8,8"]}[dim]
        return {"op": op, "rows": rows, **kind, "pages": rows // kind["page"] + rng.randint(1, 200),
                "sections": rng.choice(sections), "interleaved": rng.random() < 0.5, "far": _log(rng, 10, 1000000)}
    shape = rng.choice(["single", "single", "few", "chunk"])
    window = rng.choice([0, 0, _log(rng, 16, 5000)])
    mask = {"causal": True, "window": window, "sinks": rng.randint(0, 130) if window else 0}
    if shape == "single":
        b = _log(rng, 1, 96)
        return {"op": op, "episodes": b, "rows": b, "split": "even", "past": b * _log(rng, 16, 250007 // b if b > 60 else 4000),
                **kind, **mask}
    if shape == "few":
        b = _log(rng, 1, 128)
        if rng.random() < 0.5:
            mask = {"causal": False, "window": 0, "sinks": 0}
        return {"op": op, "episodes": b, "rows": b * rng.randint(2, 16), "split": rng.choice(["even", "ragged"]),
                "past": b * _log(rng, 16, 1000), **kind, **mask}
    b = rng.randint(1, 6)
    return {"op": op, "episodes": b, "rows": _log(rng, 40, 2011), "split": rng.choice(["even", "ragged"]),
            "past": _log(rng, 1, 6007), **kind, **mask}


def _parts(total, n, split, rng):
    """``total`` rows over ``n`` episodes: as evenly as it goes, or cut at random places (some get none)."""
    if split == "even":
        return [total // n + (i < total % n) for i in range(n)]
    cuts = [0] + sorted(rng.randint(0, total) for _ in range(n - 1)) + [total]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _lengths(case):
    """New rows and rows cached before, of each episode: part of the case, alike for every seed."""
    rng = random.Random(case["episodes"] * 1000003 + case["rows"])
    n = case["episodes"]
    new = _parts(case["rows"], n, case["split"], rng)
    weights = [0.25 + rng.random() for _ in range(n)]  # caches differ by up to five times
    past = [int(case["past"] * w / sum(weights)) for w in weights]
    past[0] += case["past"] - sum(past)
    return new, past


def _up(a, b):
    return -(-a // b)


def _visible(case, past, t, end):
    """How many cached rows the new row ``t`` of an episode sees."""
    if not case["causal"]:
        return end
    p = past + t
    if not case["window"]:
        return p + 1
    low = max(0, p - case["window"] + 1)
    return p + 1 - low + min(case["sinks"], low)


def work(case):
    if case["op"] == "write":
        n, d = case["rows"], case["dim"]
        axes = case["sections"].count(",") + 1
        moved = 2 * 2 * n * d * (case["heads"] + 2 * case["kv_heads"])
        half = sum(map(int, case["sections"].split(",")))
        return {"bytes": moved + n * (8 + 4 * axes), "flops": 6 * n * half * (case["heads"] + case["kv_heads"])}
    new, past = _lengths(case)
    if case["op"] == "plan":
        fresh = sum(_up(a + b, case["page"]) - _up(b, case["page"]) for a, b in zip(new, past))
        return {"bytes": 16 * case["rows"] + 8 * fresh + 16 * case["episodes"], "flops": 0}
    pairs = rows = 0
    for a, b in zip(new, past):
        if a:
            pairs += sum(_visible(case, b, t, a + b) for t in range(a))
            if case["window"]:
                low = max(0, b - case["window"] + 1)
                rows += a + b - low + min(case["sinks"], low)
            else:
                rows += a + b
    d = case["dim"]
    return {"bytes": 2 * 2 * d * (rows * case["kv_heads"] + case["rows"] * case["heads"]) + 4 * rows // case["page"],
            "flops": 4 * d * pairs * case["heads"]}


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(DTYPES[case["dtype"]])

    s = dict(case)
    if case["op"] == "write":
        n, h, kv, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
        # the rows come as slices of one projection, as a layer's q/k/v product gives them
        qkv = normal(n, (h + 2 * kv) * d)
        s["q"] = qkv[:, : h * d].view(n, h, d)
        s["k"] = qkv[:, h * d: (h + kv) * d].view(n, kv, d)
        s["v"] = qkv[:, (h + kv) * d:].view(n, kv, d)
        s["slot"] = torch.randperm(case["pages"] * case["page"], generator=g, device="cuda")[:n].contiguous()
        s["sizes"] = tuple(map(int, case["sections"].split(",")))
        s["positions"] = torch.randint(0, case["far"], (len(s["sizes"]), n), generator=g, device="cuda", dtype=torch.int32)
        for name in ("k_pages", "v_pages"):
            s[name] = torch.zeros(case["pages"], case["page"], kv, d, device="cuda", dtype=DTYPES[case["dtype"]])
        return s
    new, past = _lengths(case)
    page = case["page"]
    had = [_up(b, page) for b in past]
    need = [_up(a + b, page) for a, b in zip(new, past)]
    wide = max(1, max(need))
    spare = 7
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    if case["op"] == "plan":
        # the tables that the episodes have, the pages that are free, in a ring that has been used before
        column = torch.arange(wide, device="cuda")[None, :]
        count = _ints(had)[:, None]
        before = (torch.cumsum(count, 0) - count).long()
        s["table"] = torch.where(column < count, order[(before + column).clamp(max=pages - 1)], -1).to(torch.int32)
        used = sum(had)
        s["free"] = torch.roll(order, -used - 3).contiguous()  # ring place (taken + i) % pages holds order[used + i]
        s["marks"] = _ints([pages - 3, 2 * pages - 3 - used, 0], torch.int64)
        s["length"], s["new"] = _ints(past), _ints(new)
        return s
    n, h, kv, d = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    column = torch.arange(wide, device="cuda")[None, :]
    count = _ints(need)[:, None]
    before = (torch.cumsum(count, 0) - count).long()
    s["table"] = torch.where(column < count, order[(before + column).clamp(max=pages - 1)], -1).to(torch.int32)
    s["length"] = _ints([a + b for a, b in zip(new, past)])
    s["start"] = torch.cat([_ints([0]), torch.cumsum(_ints(new), 0)]).to(torch.int32)
    s["most"] = max(new)
    s["longest"] = max(a + b for a, b in zip(new, past))
    s["q"] = normal(n, h, d, scale=1.5)
    s["k_pages"] = normal(pages, page, kv, d)
    s["v_pages"] = normal(pages, page, kv, d)
    return s


def _plain_plan(s):
    page, n = s["page"], s["rows"]
    length, new, ring = s["length"].long(), s["new"].long(), s["free"].numel()
    wide = s["table"].shape[1]
    end = torch.cumsum(new, 0)
    start = torch.cat([end.new_zeros(1), end])
    first = (length + page - 1) // page
    need = torch.minimum((length + new + page - 1) // page, first.clamp(min=wide)) - first
    offset = torch.cumsum(need, 0) - need
    free = s["marks"][1] - s["marks"][0]
    granted = torch.minimum((free - offset).clamp(min=0), need)
    column = torch.arange(wide, device="cuda")[None, :] - first[:, None]
    fresh = s["free"][(s["marks"][0] + offset[:, None] + column) % ring]
    table = torch.where((column >= 0) & (column < granted[:, None]), fresh, s["table"])
    row = torch.arange(n, device="cuda")
    episode = torch.searchsorted(end, row, right=True)
    position = length[episode] + row - start[episode]
    at = table[episode, (position // page).clamp(max=wide - 1)].long()
    slot = torch.where((at >= 0) & (position // page < wide), at * page + position % page, -1)
    held = torch.maximum(torch.minimum(length + new, (first + granted) * page), length)
    marks = torch.stack([s["marks"][0] + granted.sum(), s["marks"][1], (length + new - held).sum()])
    return {"start": start.int(), "slot": slot, "episode": episode.int(), "position": position.int(), "table": table,
            "length": held.int(), "marks": marks}


def _axis(sizes, interleaved):
    """Which axis turns each frequency: one run per axis, or the axes in turn while each has some left."""
    if not interleaved:
        return [a for a, n in enumerate(sizes) for _ in range(n)]
    left, axes = list(sizes), []
    while any(left):
        for a in range(len(sizes)):
            if left[a]:
                left[a] -= 1
                axes.append(a)
    return axes


def _turned(x, cos, sin):
    half = cos.shape[-1]
    a, b = x[..., :half].float(), x[..., half: 2 * half].float()
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:].float()], -1).to(x.dtype)


def _plain_write(s):
    axes = torch.tensor(_axis(s["sizes"], s["interleaved"]), device="cuda")
    half = axes.numel()
    rate = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angle = s["positions"].double().t()[:, axes] * rate  # 64 bits: positions are far, angles are not small
    cos, sin = angle.cos().float(), angle.sin().float()
    s["k_pages"].view(-1, *s["k"].shape[1:])[s["slot"]] = _turned(s["k"], cos, sin)
    s["v_pages"].view(-1, *s["v"].shape[1:])[s["slot"]] = s["v"]
    return {"q": _turned(s["q"], cos, sin), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attend(s):
    b, page, h, kv, d = s["episodes"], s["page"], s["heads"], s["kv_heads"], s["dim"]
    t, g = s["most"], s["heads"] // s["kv_heads"]
    start, length = s["start"].long(), s["length"].long()
    new = start[1:] - start[:-1]
    row = torch.arange(s["rows"], device="cuda")
    episode = torch.searchsorted(start[1:], row, right=True)
    place = row - start[episode]
    q = torch.zeros(b, t, h, d, device="cuda")
    q[episode, place] = s["q"].float()
    q = q.view(b, t, kv, g, d).permute(0, 2, 3, 1, 4).reshape(b, kv, g * t, d)
    at = s["table"].long().clamp(min=0)
    keys = at.shape[1] * page
    k = s["k_pages"][at].float().view(b, keys, kv, d)
    v = s["v_pages"][at].float().view(b, keys, kv, d)
    j = torch.arange(keys, device="cuda")
    held = j[None, :] < length[:, None]
    v = torch.where(held[:, :, None, None], v, 0.0)
    p = (length - new)[:, None] + torch.arange(t, device="cuda")[None, :]
    seen = held[:, None, :].expand(b, t, keys)
    if s["causal"]:
        seen = seen & (j[None, None, :] <= p[:, :, None])
        if s["window"]:
            seen = seen & ((j[None, None, :] > p[:, :, None] - s["window"]) | (j < s["sinks"]))
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d)).view(b, kv, g, t, keys)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(b, kv, g * t, keys), v.transpose(1, 2)).view(b, kv, g, t, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, t, h, d)
    return o[episode, place].to(s["q"].dtype)


def run(s):
    if own:
        from reki_megakernel_b200 import episode_cache as ec
        if s["op"] == "plan":
            r = ec.plan_rows(s["length"], s["new"], s["table"], s["free"], s["marks"], page_rows=s["page"], rows=s["rows"])
            return {"start": r.start, "slot": r.slot, "episode": r.episode, "position": r.position, "table": s["table"],
                    "length": r.length, "marks": r.marks}
        if s["op"] == "write":
            q = ec.write_rows(s["k"], s["v"], s["slot"], s["k_pages"], s["v_pages"], q=s["q"], positions=s["positions"],
                              sections=s["sizes"], interleaved=s["interleaved"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        return ec.attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["start"], max_rows=s["most"],
                         causal=s["causal"], window=s["window"], sinks=s["sinks"])
    return {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend}[s["op"]](s)


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "write":
        n, kv, d = case["rows"], case["kv_heads"], case["dim"]
        angle = torch.zeros(n, 0, dtype=torch.float64, device="cuda")
        order = _axis(s["sizes"], case["interleaved"])
        for i, axis in enumerate(order):
            turn = s["positions"][axis].double() * math.pow(10000.0, -i / len(order))
            angle = torch.cat([angle, turn[:, None]], 1)
        unit = torch.polar(torch.ones_like(angle), angle)[:, None, :]

        def turned(x):
            x = x.double()
            w = unit.shape[-1]
            z = torch.complex(x[..., :w].contiguous(), x[..., w: 2 * w].contiguous()) * unit
            return torch.cat([z.real, z.imag, x[..., 2 * w:]], -1)

        out = {"q": turned(s["q"])}
        for name, rows in (("k_pages", turned(s["k"])), ("v_pages", s["v"].double())):
            pages = torch.zeros(case["pages"] * case["page"], kv, d, dtype=torch.float64, device="cuda")
            pages.index_copy_(0, s["slot"], rows)
            out[name] = pages.view(case["pages"], case["page"], kv, d)
        return out
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    new, past = _lengths(case)
    if work(case)["flops"] > 4e12:
        return None
    out = torch.zeros(case["rows"], h, d, dtype=torch.float64, device="cuda")
    first = 0
    for e, (a, b) in enumerate(zip(new, past)):
        if not a:
            continue
        pages = s["table"][e, : _up(a + b, case["page"])].long()
        k = s["k_pages"][pages].flatten(0, 1)[: a + b].double()
        v = s["v_pages"][pages].flatten(0, 1)[: a + b].double()
        j = torch.arange(a + b, device="cuda")
        p = (torch.arange(a, device="cuda") + b)[:, None]
        hidden = torch.zeros(a, a + b, dtype=torch.bool, device="cuda")
        if case["causal"]:
            hidden |= j > p
            if case["window"]:
                hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
        for head in range(h):
            q = s["q"][first: first + a, head].double()
            score = q @ k[:, head * kv // h].T / math.sqrt(d)
            score[hidden] = -math.inf
            out[first: first + a, head] = torch.softmax(score, -1) @ v[:, head * kv // h]
        first += a
    return out
