"""The paged episode cache against its restatement in 64 bits (``oracle/cache_oracle.py``)."""
import pytest
import torch

from _cache_cases import attend_tolerance, pages_for
from oracle.cache_oracle import angles_oracle, attend_oracle, plan_oracle, turn_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16


def ec():
    from reki_megakernel_b200 import episode_cache
    return episode_cache


@pytest.mark.parametrize("name", ["plan", "write", "attend"])
def test_refusals(name):
    """What the checks refuse is refused by the calls themselves, before anything is launched; the good arguments run."""
    import test_episode_cache_host as host
    E = ec()
    f = {"plan": E.plan_rows, "write": E.write_rows, "attend": E.attend}[name]
    good, bad = getattr(host, f"{name}_args")(DEV)
    if name != "plan":
        wide = torch.zeros(7, 6, 72, dtype=BF, device=DEV)
        bad += [dict(q=wide[:, :, 4:68]), dict(q=torch.zeros(7, 6, 65, dtype=BF, device=DEV)[:, :, :64]),
                dict(q=torch.zeros(7, 64, 6, dtype=BF, device=DEV).transpose(1, 2)), dict(out=wide[:, :, 1:65])]
    for kw in bad:
        with pytest.raises(ValueError):
            f(**{**good, **kw})
    f(**good)
    if name == "plan":
        ticket = torch.zeros(1, dtype=torch.int32, device=DEV)
        with pytest.raises(ValueError):
            f(**good, ticket=ticket.long())
        assert f(**good, ticket=ticket).length is good["length"] and int(ticket) == 0
    if name == "write":
        for kw in (dict(sections=(20, 20)), dict(sections=(8, 8, 8)), dict(base=-1.0), dict(positions=torch.zeros(2, 7, dtype=torch.int32, device=DEV)),
                   dict(positions=torch.zeros(1, 7, dtype=torch.int64, device=DEV)), dict(positions=torch.zeros(7, 2, dtype=torch.int32, device=DEV).t(), sections=(16, 16))):
            with pytest.raises(ValueError):
                f(**{**good, **kw})
    torch.cuda.synchronize()


# ---- placing -------------------------------------------------------------------------------------------

def _plan_case(B, page, wide, pages, seed, rows=None, slack=0, most=70):
    g = torch.Generator().manual_seed(seed)
    length = torch.randint(0, max(1, min(wide * page - most, 5 * page)) + 1, (B,), generator=g).tolist()
    new = [int(x) if x % 3 else 0 for x in torch.randint(0, most + 1, (B,), generator=g)]
    had = [-(-n // page) for n in length]
    assert sum(had) <= pages
    free = torch.randperm(pages, generator=g).tolist()
    used, at = sum(had), 0
    taken = used + 3 * pages        # the ring has been round three times
    ring = [0] * pages
    for i, f in enumerate(free):
        ring[(3 * pages + i) % pages] = f
    table = [[-1] * wide for _ in range(B)]
    for b in range(B):
        for j in range(had[b]):
            table[b][j] = ring[at % pages]
            at += 1
    rows = sum(new) + slack if rows is None else rows
    return length, new, table, ring, [taken, 4 * pages, 0], rows


def _tensors(length, new, table, ring, marks):
    i = dict(dtype=torch.int32, device=DEV)
    return (torch.tensor(length, **i), torch.tensor(new, **i), torch.tensor(table, **i), torch.tensor(ring, **i),
            torch.tensor(marks, dtype=torch.int64, device=DEV))


def _same_plan(r, table, ref):
    for name in ("start", "slot", "episode", "position", "length", "marks"):
        assert getattr(r, name).tolist() == ref[name], name
    assert table.tolist() == ref["table"]


@pytest.mark.parametrize("B,page,wide,pages,slack", [
    (1, 16, 8, 40, 0), (3, 16, 10, 60, 5), (17, 32, 8, 300, 0), (300, 16, 12, 4000, 3), (1000, 64, 7, 8000, 0),
    (4096, 128, 6, 30000, 1)])
def test_plan_matches(B, page, wide, pages, slack):
    args = _plan_case(B, page, wide, pages, seed=B, slack=slack)
    ref = plan_oracle(*args[:5], page, args[5])
    assert ref["marks"][2] == 0
    t = _tensors(*args[:5])
    r = ec().plan_rows(*t, page_rows=page, rows=args[5])
    _same_plan(r, t[2], ref)
    assert t[0].tolist() == args[0] and t[4].tolist() == args[4]   # the old state is untouched


@pytest.mark.parametrize("kind", ["pages", "width", "rows", "none free"])
def test_plan_runs_out(kind):
    """Rows that get no slot are counted, the others placed, and the state stays whole."""
    length, new, table, ring, marks, rows = _plan_case(24, 16, 14, 400, seed=5, most=120)
    if kind == "pages":
        marks[1] = marks[0] + 9
    elif kind == "none free":
        marks[1] = marks[0]
    elif kind == "width":
        table = [r[:7] for r in table]
    else:
        rows -= 131
    ref = plan_oracle(length, new, table, ring, marks, 16, rows)
    assert ref["marks"][2] > 0
    t = _tensors(length, new, table, ring, marks)
    r = ec().plan_rows(*t, page_rows=16, rows=rows)
    _same_plan(r, t[2], ref)


def test_plan_of_an_impossible_state():
    """Lengths and marks that no plan leaves behind: rows without a slot, and nothing outside of the arrays."""
    most = 2 ** 31 - 1
    for marks, length in (([-5, 3, 0], [0, 0]), ([2 ** 40 + 1, 2 ** 50, 0], [5, 0]), ([0, 4, 0], [most, -3]),
                          ([9, 2, 0], [most, most]), ([-2 ** 62, 2 ** 62, 0], [17, most])):
        table = torch.full((2, 3), -1, dtype=torch.int32, device=DEV)
        ring = torch.arange(4, dtype=torch.int32, device=DEV)
        as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        plan = ec().plan_rows(as_int(length), as_int([40, 60]), table, ring,
                              torch.tensor(marks, dtype=torch.int64, device=DEV), page_rows=16, rows=100)
        assert int(plan.slot.min()) >= -1 and int(plan.slot.max()) < 4 * 16
        got = plan.slot[plan.slot >= 0]
        assert got.unique().numel() == got.numel()
        assert plan.start.tolist() == [0, 40, 100] and plan.episode.tolist() == [0] * 40 + [1] * 60
        assert int(plan.length.min()) >= 0 and int(table.min()) >= -1 and int(table.max()) < 4


def test_plan_nothing_new():
    length, new, table, ring, marks, _ = _plan_case(5, 32, 8, 90, seed=1)
    t = _tensors(length, [0] * 5, table, ring, marks)
    r = ec().plan_rows(*t, page_rows=32, rows=0)
    assert r.start.tolist() == [0] * 6 and r.length.tolist() == length and r.marks.tolist() == marks
    r = ec().plan_rows(*t, page_rows=32, rows=9)
    assert r.slot.tolist() == [-1] * 9 and r.episode.tolist() == [-1] * 9 and r.position.tolist() == [0] * 9
    assert t[2].tolist() == table


def test_cache_steps_and_releases():
    """Forty steps of a cache with episodes that end: tables, lengths and the ring against a book kept by hand; no page
    belongs to two episodes, none is lost."""
    E = ec()
    pages, B, page = 150, 9, 16
    c = E.EpisodeCache(layers=1, pages=pages, episodes=B, page_rows=page, kv_heads=1, head_dim=64, pages_per_episode=30,
                       device=DEV)
    g = torch.Generator().manual_seed(3)
    state = dict(length=[0] * B, table=c.table.tolist(), marks=[0, pages, 0])
    ring = list(range(pages))
    for step in range(40):
        new = torch.randint(0, 41, (B,), generator=g).tolist()
        r = c.plan(torch.tensor(new, dtype=torch.int32, device=DEV), sum(new) + 2)
        ref = plan_oracle(state["length"], new, state["table"], ring, state["marks"], page, sum(new) + 2)
        _same_plan(r, c.table, ref)
        assert c.length.tolist() == ref["length"] and c.marks.tolist() == ref["marks"]
        ended = (torch.rand(B, generator=g) < 0.25).tolist()
        returned = ref["marks"][1]
        for b in range(B):
            if ended[b]:
                for j in range(-(-ref["length"][b] // page)):
                    ring[returned % pages] = ref["table"][b][j]
                    returned += 1
                ref["table"][b] = [-1] * 30
                ref["length"][b] = 0
        c.release(torch.tensor(ended, device=DEV))
        state = dict(length=ref["length"], table=ref["table"], marks=[ref["marks"][0], returned, ref["marks"][2]])
        assert c.table.tolist() == state["table"] and c.length.tolist() == state["length"]
        assert c.marks.tolist() == state["marks"] and c.free.tolist() == ring
        held = [p for row in state["table"] for p in row if p >= 0]
        free = [ring[i % pages] for i in range(state["marks"][0], state["marks"][1])]
        assert sorted(held + free) == list(range(pages))


# ---- rotary positions and storing ----------------------------------------------------------------------

@pytest.mark.parametrize("hd,sections,interleaved,far", [
    (64, None, False, 4096), (64, (8, 12, 12), False, 70000), (64, (12, 10, 10), True, 10 ** 6),
    (128, (24, 20, 20), True, 10 ** 7), (128, (16, 8, 8), False, 1000), (80, (4, 4), True, 100), (256, (128,), False, 2 ** 31 - 1),
    (64, (0, 16, 16, 0), True, 500)])
def test_rope_tables(hd, sections, interleaved, far):
    """Angles are formed in turns with an exact remainder: four fp32 roundings of values below 1 turn (2^-25 turns each,
    2^-24 * 2 pi = 4e-7 rad apiece at most) and the rate's two floats (2^-48 of the angle: 1e-6 rad at 2^31 / 2 pi turns)."""
    n = 77
    sec = sections or (hd // 2,)
    g = torch.Generator().manual_seed(hd)
    pos = torch.randint(-far if far < 10 ** 6 else 0, far, (len(sec), n), generator=g, dtype=torch.int64).to(torch.int32)
    cos, sin = ec().rope_tables(pos.to(DEV), hd, sections=sections, interleaved=interleaved)
    ang = angles_oracle(pos, sec, interleaved=interleaved)
    half = ang.shape[1]
    rest = torch.zeros(n, hd - 2 * half, dtype=torch.float64)
    tol = 2e-6 + far * 2.0 ** -48
    assert (cos.cpu().double() - torch.cat([ang.cos(), ang.cos(), rest + 1], 1)).abs().max() <= tol
    assert (sin.cpu().double() - torch.cat([ang.sin(), ang.sin(), rest], 1)).abs().max() <= tol


def test_tables_are_the_expert_ones():
    """One axis, all frequencies: the tables of ``synthetic.rope_cos_sin``."""
    from reki_megakernel_b200.synthetic import rope_cos_sin
    pos = torch.arange(300, dtype=torch.int32)
    got = ec().rope_tables(pos.to(DEV), 64)
    for a, b in zip(got, rope_cos_sin(pos, 64)):
        assert (a.cpu() - b).abs().max() <= 2e-6


def _check_turned(got, x, ang):
    ref = turn_oracle(x, ang)
    half = ang.shape[1]
    size = torch.cat([x.cpu().double()[..., :half].abs() + x.cpu().double()[..., half:2 * half].abs()] * 2
                     + [torch.zeros_like(ref[..., 2 * half:])], -1)
    u = torch.finfo(x.dtype).eps / 2
    tol = u * ref.abs() + size * 4e-6 + 2.0 ** -25   # half a step, and the angle's 2e-6 on both terms
    err = (got.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("rows,heads,kv,hd,page,dtype,sections,interleaved", [
    (1, 12, 12, 64, 32, BF, (8, 12, 12), False), (24, 12, 4, 64, 16, FP, None, False), (257, 32, 8, 128, 64, BF, (24, 20, 20), True),
    (1003, 7, 1, 128, 256, FP, (16, 8, 8), False), (33, 5, 5, 80, 16, BF, (4, 4), True), (40, 3, 2, 256, 128, FP, (64, 64), True)])
def test_write_rows(rows, heads, kv, hd, page, dtype, sections, interleaved):
    """q rotated, K and V rows at their slots, everything else in the pages as it was; rows with a slot outside of the
    pages are dropped."""
    g = torch.Generator().manual_seed(rows)
    pages = rows // page + 3
    qkv = torch.randn(rows, (heads + 2 * kv) * hd, generator=g).to(dtype).to(DEV)
    q = qkv[:, :heads * hd].view(rows, heads, hd)
    k = qkv[:, heads * hd:(heads + kv) * hd].view(rows, kv, hd)
    v = qkv[:, (heads + kv) * hd:].view(rows, kv, hd)
    slot = torch.randperm(pages * page, generator=g)[:rows]
    if rows > 20:
        slot[3], slot[7], slot[11] = -1, pages * page, 1 << 40
    sec = sections or (hd // 2,)
    pos = torch.randint(0, 100000, (len(sec), rows), generator=g).to(torch.int32)
    kp = torch.full((pages, page, kv, hd), 3.0, dtype=dtype, device=DEV)
    vp = torch.full((pages, page, kv, hd), -5.0, dtype=dtype, device=DEV)
    out = ec().write_rows(k, v, slot.to(DEV), kp, vp, q=q, positions=pos.to(DEV), sections=sections, interleaved=interleaved)
    ang = angles_oracle(pos, sec, interleaved=interleaved)
    _check_turned(out, q, ang)
    ok = (slot >= 0) & (slot < pages * page)
    flat = kp.view(-1, kv, hd)
    _check_turned(flat[slot[ok].to(DEV)], k[ok.to(DEV)], ang[ok])
    assert torch.equal(vp.view(-1, kv, hd)[slot[ok].to(DEV)], v[ok.to(DEV)])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[slot[ok]] = False
    assert (flat[rest.to(DEV)] == 3.0).all() and (vp.view(-1, kv, hd)[rest.to(DEV)] == -5.0).all()


def test_write_rotates_k_alone():
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(37, 2, 128, generator=g).to(FP).to(DEV) for _ in range(2))
    slot, pos = torch.randperm(64, generator=g)[:37].to(DEV), torch.randint(0, 900, (2, 37), generator=g).to(torch.int32)
    kp, vp = (torch.zeros(4, 16, 2, 128, dtype=FP, device=DEV) for _ in range(2))
    assert ec().write_rows(k, v, slot, kp, vp, positions=pos.to(DEV), sections=(40, 24), base=500.0) is None
    _check_turned(kp.view(64, 2, 128)[slot], k, angles_oracle(pos, (40, 24), base=500.0))
    assert torch.equal(vp.view(64, 2, 128)[slot], v)


def test_write_without_positions_and_in_place():
    """K as it is where there are no positions; q may be rotated in place; pages may be laid out head by head."""
    g = torch.Generator().manual_seed(0)
    k, v, q = (torch.randn(50, 4, 64, generator=g).to(BF).to(DEV) for _ in range(3))
    slot = torch.randperm(96, generator=g)[:50].to(DEV)
    kp = torch.zeros(3, 4, 32, 64, dtype=BF, device=DEV).transpose(1, 2)
    vp = torch.zeros(3, 4, 32, 64, dtype=BF, device=DEV).transpose(1, 2)
    assert ec().write_rows(k, v, slot, kp, vp) is None
    assert torch.equal(kp[slot // 32, slot % 32], k) and torch.equal(vp[slot // 32, slot % 32], v)
    pos = torch.arange(50, dtype=torch.int32, device=DEV)
    want = ec().write_rows(k, v, slot, kp, vp, q=q, positions=pos)
    x = q.clone()
    got = ec().write_rows(k, v, slot, kp, vp, q=x, positions=pos, out=x)
    assert got is x and torch.equal(x, want)
    empty = torch.empty(0, 4, 64, dtype=BF, device=DEV)
    assert ec().write_rows(empty, empty, slot[:0], kp, vp, q=empty, positions=pos[:0]).shape == (0, 4, 64)


# ---- attention -----------------------------------------------------------------------------------------

def _check_attend(c, max_rows=None, tail=0, out=None, **kw):
    E = ec()
    got = E.attend(**c, max_rows=max_rows, out=out, **kw)
    torch.cuda.synchronize()
    E.check_device_error(DEV)
    ref, weight = attend_oracle(**c, **kw)
    n = got.shape[0] - tail
    tol = attend_tolerance(ref, weight, c["q"].dtype, int(c["length"].max()))
    err = (got.double() - ref).abs()[:n]
    assert torch.isfinite(got[:n].float()).all()
    assert bool((err <= tol[:n]).all()), float((err / tol[:n]).max())
    return got


# Beyond 16 rows of a K/V head the kernel goes by what the tables can hold (how long the caches are is not known when a
# call is launched): a tight table brings these small caches to the kernel of 16-row tiles, a wide one to that of chunks.
WIDTHS = pytest.mark.parametrize("extra_width", [2, 300000])

SHAPES = [(12, 12, 64), (32, 8, 128), (7, 1, 64), (16, 2, 128), (40, 2, 64), (5, 5, 128)]
LENGTHS = [  # new, past
    ([1], [0]), ([1, 1, 1], [0, 16, 700]), ([10] * 5, [31, 0, 64, 1000, 129]), ([0, 3, 0, 17, 1], [40, 0, 0, 260, 513]),
    ([130], [0]), ([77, 200, 5], [500, 1, 33]), ([2, 300], [1500, 90])]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("new,past", LENGTHS)
@WIDTHS
def test_attend_causal(heads, kv, hd, new, past, extra_width):
    dtype, page = (BF, 32) if (heads + len(new)) % 2 else (FP, 16)
    c = pages_for(new, past, heads, kv, hd, page=page, dtype=dtype, seed=heads + sum(new), extra_width=extra_width)
    _check_attend(c, max_rows=max(new))


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("new,past", LENGTHS[1:5])
@WIDTHS
def test_attend_all(heads, kv, hd, new, past, extra_width):
    c = pages_for(new, past, heads, kv, hd, page=64, dtype=FP if heads % 2 else BF, seed=sum(past), extra_width=extra_width)
    _check_attend(c, causal=False)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 130), (64, 4), (100, 0), (128, 64), (333, 70), (5000, 9)])
@pytest.mark.parametrize("new,past,heads,kv,hd,page", [
    ([1, 1], [900, 3], 12, 12, 64, 32), ([9, 1, 0, 40], [400, 0, 12, 1000], 16, 4, 128, 16),
    ([260, 35], [700, 0], 6, 2, 64, 128), ([150], [2000], 4, 1, 128, 256)])
@WIDTHS
def test_attend_window(window, sinks, new, past, heads, kv, hd, page, extra_width):
    """Pages that no row sees any more hold NaN: they may have gone to somebody else."""
    c = pages_for(new, past, heads, kv, hd, page=page, seed=window, extra_width=extra_width)
    for b in range(len(new)):
        for j in range(-(-(new[b] + past[b]) // page)):
            if new[b] and (j + 1) * page <= past[b] - window + 1 and j * page >= sinks:
                c["k_pages"][c["table"][b, j]] = float("nan")
                c["v_pages"][c["table"][b, j]] = float("nan")
                if j % 2:
                    c["table"][b, j] = -1
    _check_attend(c, max_rows=max(new), window=window, sinks=sinks)


@pytest.mark.parametrize("most", [1, 5, 40])
@WIDTHS
def test_attend_many_episodes(most, extra_width):
    """More episodes than a block has threads, many without new rows or without any."""
    g = torch.Generator().manual_seed(most)
    new = [int(x) for x in torch.randint(0, most + 1, (700,), generator=g)]
    past = [int(x) if x % 3 else 0 for x in torch.randint(0, 200, (700,), generator=g)]
    c = pages_for(new, past, 4, 2, 64, page=16, seed=most, extra_width=min(extra_width, 20000))
    _check_attend(c, max_rows=most)
    _check_attend(c, max_rows=most, window=30, sinks=2)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 200])
@WIDTHS
def test_attend_page_sizes(page, hd, new, extra_width):
    for n in (page - 1, page, page + 1, 3 * page + 5):
        c = pages_for([new, new], [n, 2 * n], 4, 2, hd, page=page, seed=n, extra_width=extra_width)
        _check_attend(c)


@WIDTHS
def test_attend_rows_that_see_nothing(extra_width):
    """An episode without any row (length 0) and new rows that were never stored (length below the new rows)."""
    c = pages_for([4, 6, 2], [0, 20, 50], 4, 2, 64, extra_width=extra_width)
    c["length"][0] = 0
    got = _check_attend(c)
    assert (got[:4] == 0).all()
    c = pages_for([4, 150, 2], [0, 20, 50], 4, 2, 64, extra_width=extra_width)
    c["length"][1] = 60      # 90 rows lie before position 0
    got = ec().attend(**c)
    assert (got[4:94] == 0).all() and torch.isfinite(got.float()).all()
    got = ec().attend(**c, causal=False)
    assert torch.isfinite(got.float()).all() and not (got[4:94] == 0).any()


@pytest.mark.parametrize("new", [[3, 1], [150, 40]])
@WIDTHS
def test_attend_leaves_rows_behind_the_last(new, extra_width):
    c = pages_for(new, [70, 9], 4, 4, 64, tail_rows=13, extra_width=extra_width)
    out = torch.full_like(c["q"], 7.0)
    got = _check_attend(c, tail=13, out=out)
    assert got is out and (out[sum(new):] == 7.0).all()
    # rows beyond max_rows stay as well, and the others keep their positions
    out2 = torch.full_like(c["q"], 7.0)
    ec().attend(**c, max_rows=2, out=out2)
    ref, weight = attend_oracle(**c)
    tol = attend_tolerance(ref, weight, BF, int(c["length"].max()))
    assert bool(((out2.double() - ref).abs()[:2] <= tol[:2]).all())
    assert (out2[2:new[0]] == 7.0).all()


@pytest.mark.parametrize("new", [[2, 1, 9], [140, 300]])
@WIDTHS
def test_attend_strides(new, extra_width):
    """q and out as slices of wider rows, pages laid out head by head and as a slice of a pool of layers."""
    past = [300] * len(new)
    c = pages_for(new, past, 6, 2, 64, head_major=True, seed=4, extra_width=extra_width)
    n = sum(new)
    wide = torch.zeros(n, 10 * 64, dtype=BF, device=DEV)
    wide[:, 128:512] = c["q"].reshape(n, -1)
    c["q"] = wide[:, 128:512].view(n, 6, 64)
    pool = torch.full((c["k_pages"].shape[0], 2, 32, 4, 64), float("nan"), dtype=BF, device=DEV)
    pool[:, 1, :, 2:] = c["k_pages"]
    c["k_pages"] = pool[:, 1, :, 2:]
    assert not c["v_pages"].is_contiguous()
    out = torch.zeros(n, 6, 128, dtype=BF, device=DEV)[:, :, 64:]
    _check_attend(c, out=out)


@WIDTHS
def test_attend_scale_and_large_scores(extra_width):
    """Scores of thousands: one key takes all; a scale of zero: the mean."""
    c = pages_for([3, 200], [90, 50], 4, 2, 64, q_scale=400.0, seed=8, extra_width=extra_width)
    ref, _ = attend_oracle(**c)
    got = ec().attend(**c)
    # scores up to 2^13 have fp32 error 2^-10: a tie within that may go either way, elsewhere the row is a copy
    near = (got.double() - ref).abs() <= 2.0 ** -7 * ref.abs() + 2.0 ** -6
    assert near.double().mean() >= 0.995 and torch.isfinite(got.float()).all()
    c = pages_for([3, 200], [90, 50], 4, 2, 64, seed=8, extra_width=extra_width)
    _check_attend(c, scale=0.0)
    _check_attend(c, scale=-0.2)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("drop", [8, 13, 18])
def test_attend_many_small_weights(drop, new, dtype):
    """One key far above all others: weights of e^-drop (e^-18 < 2^-25, half the smallest fp16), which count together.
    Half a step of the output and of each weight, 2^-12 for scores and exponentials, and 2^-32 of |v| < 6 for each key:
    weights enter 2^7 times as large or more, so that fp16's 2^-25 is 2^-32 of the largest."""
    c = pages_for([new], [20000], 4, 1, 64, page=64, dtype=dtype, seed=3)
    here = c["table"][0][:-(-(20000 + new) // 64)].long()
    k, v = (c[name][here].flatten(0, 1) for name in ("k_pages", "v_pages"))
    k[:20000 + new] = 0.0
    k[0, :, 0] = 1.0
    v[:20000 + new] = v[:20000 + new].abs() + 0.5
    v[0] = 0.0
    c["k_pages"][here], c["v_pages"][here] = k.view(-1, 64, 1, 64), v.view(-1, 64, 1, 64)
    c["q"].zero_()
    c["q"][..., 0] = float(drop)
    # 400 such episodes on the same pages: more tiles than blocks, so that stretches of keys stay long
    ref, weight = (x.repeat(400, 1, 1) for x in attend_oracle(**c, scale=1.0))
    c["q"], c["table"], c["length"] = c["q"].repeat(400, 1, 1), c["table"].repeat(400, 1), c["length"].repeat(400)
    c["start"] = torch.arange(401, dtype=torch.int32, device=DEV) * new
    got = ec().attend(**c, max_rows=new, scale=1.0)
    u = torch.finfo(dtype).eps / 2
    tol = u * ref.abs() + (u + 2.0 ** -12) * weight + 20041 * 2.0 ** -32 * 6
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@WIDTHS
def test_attend_into_its_queries(extra_width):
    c = pages_for([40, 3, 150], [700, 2000, 90], 8, 2, 128, page=32, seed=21, extra_width=min(extra_width, 100000))
    apart = ec().attend(**c, max_rows=150, window=500, sinks=3)
    q = c.pop("q").clone()
    assert ec().attend(q, **c, max_rows=150, window=500, sinks=3, out=q) is q
    assert torch.equal(q, apart)


def test_attend_long_cache_and_far_pages():
    """A pool of more than 2^31 elements whose pages lie at both ends; one episode split over many blocks."""
    pages, page, kv, hd = 9000, 256, 8, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.empty(pages, page, kv, hd, dtype=BF, device=DEV).normal_(generator=g)
    v = torch.empty(pages, page, kv, hd, dtype=BF, device=DEV).normal_(generator=g)
    assert k.numel() > 2 ** 31
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.randperm(pages, generator=g, device=DEV)[:150].to(torch.int32).view(1, 150)
    for new in (1, 40):
        c = dict(q=torch.randn(new, 16, hd, generator=g, device=DEV).to(BF), k_pages=k, v_pages=v, table=table,
                 length=torch.tensor([38001], **i32), start=torch.tensor([0, new], **i32))
        _check_attend(c)


def test_attend_is_deterministic_and_captured_twice():
    """Split tiles are joined in the order of their parts; two graphs may run at once."""
    E = ec()
    c = pages_for([1, 1], [9000, 5000], 8, 2, 128, page=64, seed=2)
    d = pages_for([200], [6000], 8, 2, 128, page=64, seed=3)
    want = [E.attend(**x) for x in (c, d)]
    for _ in range(5):
        for x, w in zip((c, d), want):
            assert torch.equal(E.attend(**x), w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for x in (c, c, d):
            E.attend(**x)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(E.attend(**x))
            graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, t in zip(graphs, streams):
            with torch.cuda.stream(t):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[0]) and torch.equal(outs[2], want[1])
    E.check_device_error(DEV)


def test_attend_on_two_streams_at_once():
    E = ec()
    cases = [pages_for([1, 1], [9000, 5000], 8, 2, 128, page=64, seed=2), pages_for([180], [6000], 8, 2, 64, page=64, seed=3)]
    want = [E.attend(**c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(E.attend(**c))
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for i, w in enumerate(want) for g in got[i])


def test_a_step_of_serving_captured():
    """place -> store -> read, captured once and replayed over steps, against the oracle on the rows kept by hand."""
    E = ec()
    B, heads, kv, hd, T = 5, 6, 2, 64, 3
    c = E.EpisodeCache(layers=2, pages=60, episodes=B, page_rows=16, kv_heads=kv, head_dim=hd, pages_per_episode=12, device=DEV)
    new = torch.zeros(B, dtype=torch.int32, device=DEV)
    rows = B * T
    x = {n: torch.zeros(rows, h, hd, dtype=BF, device=DEV) for n, h in (("q", heads), ("k", kv), ("v", kv))}
    pos = torch.zeros(3, rows, dtype=torch.int32, device=DEV)

    def step():
        plan = c.plan(new, rows)
        outs = []
        for layer in range(2):
            q = c.write(layer, x["k"], x["v"], plan, q=x["q"], positions=pos, sections=(8, 12, 12))
            outs.append(c.attend(layer, q, plan, max_rows=T, window=20, sinks=3))
        return plan, outs

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()          # nothing new: the state stays
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        plan, outs = step()
    gen = torch.Generator().manual_seed(0)
    kept_k = [torch.zeros(0, kv, hd, dtype=BF) for _ in range(B)]
    kept_v = [torch.zeros(0, kv, hd, dtype=BF) for _ in range(B)]
    for it in range(12):
        counts = torch.randint(0, T + 1, (B,), generator=gen)
        new.copy_(counts)
        for t in x.values():
            t.copy_(torch.randn(t.shape, generator=gen))
        pos.copy_(torch.randint(0, 5000, pos.shape, generator=gen))
        if it == 7:
            c.release(torch.tensor([True, False, False, True, False], device=DEV))
            for b in (0, 3):
                kept_k[b], kept_v[b] = kept_k[b][:0], kept_v[b][:0]
        g.replay()
        torch.cuda.synchronize()
        assert int(c.marks[2]) == 0
        ang = angles_oracle(pos, (8, 12, 12))
        turned = [turn_oracle(x[n], ang) for n in ("q", "k")]
        at = 0
        for b in range(B):
            n = int(counts[b])
            kept_k[b] = torch.cat([kept_k[b], turned[1][at:at + n].to(BF)])
            kept_v[b] = torch.cat([kept_v[b], x["v"][at:at + n].cpu()])
            at += n
        assert c.length.tolist() == [len(k) for k in kept_k]
        top = max(16, -(-max(len(k) for k in kept_k) // 16) * 16)
        pk, pv = torch.zeros(B, top // 16, 16, kv, hd, dtype=BF), torch.zeros(B, top // 16, 16, kv, hd, dtype=BF)
        for b in range(B):
            pk[b].view(-1, kv, hd)[:len(kept_k[b])] = kept_k[b]
            pv[b].view(-1, kv, hd)[:len(kept_v[b])] = kept_v[b]
        table = torch.arange(B * (top // 16)).view(B, -1)
        ref, weight = attend_oracle(turned[0].to(BF), pk.flatten(0, 1), pv.flatten(0, 1), table,
                                    torch.tensor([len(k) for k in kept_k]), plan.start.cpu(), window=20, sinks=3)
        # q and k may differ by a step from the oracle's rounding of them: 2^-7 of each score's size on top
        tol = attend_tolerance(ref, weight, BF, top) + 2.0 ** -5 * weight
        for o in outs:
            assert bool(((o.cpu().double() - ref).abs()[:at] <= tol[:at]).all())
    c.check_device_error()


def test_prepare_takes_positions():
    """``RegisterPrepare.run`` with source positions of three axes equals the run with their tables."""
    from reki_megakernel_b200.prepare import RegisterPrepare
    from reki_megakernel_b200.synthetic import ExpertDims, make_prepare_weights, make_source
    d = ExpertDims(L=2)
    rp = RegisterPrepare(make_prepare_weights(d, seed=0).to(DEV))
    src = make_source(70, d.src_dim, seed=1).to(DEV)
    pos = torch.stack([torch.arange(70) // 35, torch.arange(70) % 35 // 7, torch.arange(70) % 7]).to(torch.int32).to(DEV)
    k, v = rp.run(src, positions=pos, sections=(8, 12, 12))
    cos, sin = ec().rope_tables(pos, d.HD, sections=(8, 12, 12))
    k2, v2 = rp.run(src, cos, sin)
    k3, _ = rp.run(src)
    torch.cuda.synchronize()
    rp.check_device_error()
    assert torch.equal(k, k2) and torch.equal(v, v2) and not torch.equal(k, k3)
    with pytest.raises(ValueError):
        rp.run(src, cos, sin, positions=pos)
    rp.close()
