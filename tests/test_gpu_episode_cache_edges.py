"""Calls of the paged episode cache at its edges: queries that are not finite, parts of split tiles one by one, geometries and
arguments that are refused, several threads. Oracles as in ``test_gpu_episode_cache.py``."""
import ctypes as C
import threading

import pytest
import torch

from _cache_cases import attend_tolerance, pages_for
from oracle.cache_oracle import angles_oracle, attend_oracle, turn_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, FP = torch.bfloat16, torch.float16
WIDTHS = pytest.mark.parametrize("extra_width", [2, 300000])  # the kernel of 16-row tiles, that of chunks


def ec():
    from reki_megakernel_b200 import episode_cache
    return episode_cache


# ---- queries that are not finite -----------------------------------------------------------------------

@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (2, 0), (2, 3), (40, 1)])
@pytest.mark.parametrize("hd", [64, 128])
@WIDTHS
def test_attend_queries_not_finite(value, window, sinks, hd, extra_width):
    """NaN in a query makes its scores NaN, infinity makes them infinite (or NaN): softmax has no value there, and the row of
    that head is NaN, in whichever columns its keys lie. All other rows are what they are without, and a row that sees nothing
    is zero whatever its query holds."""
    new, past = [150, 40, 30], [0, 70, 0]
    c = pages_for(new, past, 4, 2, hd, page=16, dtype=BF if hd == 64 else FP, seed=window, extra_width=extra_width)
    c["length"][2] = 20                       # ten new rows lie before position 0
    ref, weight = attend_oracle(**c, window=window, sinks=sinks)
    tol = attend_tolerance(ref, weight, c["q"].dtype, int(c["length"].max()))
    g = torch.Generator().manual_seed(1)
    spoilt = torch.rand(sum(new), 4, generator=g) < 0.3
    dim = torch.randint(0, hd, (sum(new), 4), generator=g)
    q = c["q"].clone()
    for r, h in spoilt.nonzero().tolist():
        q[r, h, dim[r, h]] = value
    c["q"] = q
    got = ec().attend(**c, max_rows=150, window=window, sinks=sinks).double()
    ec().check_device_error(DEV)
    spoilt = spoilt.to(DEV)
    blind = torch.zeros_like(spoilt)
    blind[190:200] = True
    assert (got[blind] == 0).all()
    assert torch.isnan(got[spoilt & ~blind]).all()
    assert bool(((got - ref).abs() <= tol)[~spoilt].all())


# ---- scores of any size --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,bits", [(FP, b) for b in (0, 12, 20, 24, 25, 26, 27, 28, 30, 31)] + [(BF, b) for b in (0, 24, 28, 31, 36, 60, 100)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("hd", [64, 128])
@WIDTHS
def test_attend_scores_of_any_size(dtype, bits, sign, hd, extra_width):
    """Finite queries and keys have a finite output, however large their scores: here sign * 2^bits * c of whole numbers c
    up to 40, exact in fp32 (a factor of 2^6 of the sum over 64 dims, the others zero), so that equal scores stay equal and all
    others are units apart. From 2^24 on a unit in the last place of a score is more than what the kernels shift it by. The rounding of
    score x scale to fp32 is off by 2^-24 of it: 2^-18 at scores of 40, more where one key takes all."""
    new, past = [40, 3, 150], [700, 0, 90]
    c = pages_for(new, past, 4, 2, hd, page=32, dtype=dtype, seed=bits, extra_width=extra_width)
    g = torch.Generator().manual_seed(bits)
    n = c["k_pages"].shape[0]
    k = torch.zeros(n, 32, 2, hd)
    of_k = (bits - 6) // 2 if dtype == BF else min((bits - 6) // 2, 10)     # 40 * 2^10 and 2^15 are below 65504
    k[..., :64] = sign * torch.randint(1, 41, (n, 32, 2, 1), generator=g).float() * 2.0 ** of_k
    held = ~torch.isnan(c["k_pages"])
    c["k_pages"] = torch.where(held, k.to(dtype).to(DEV), c["k_pages"])
    c["q"] = torch.zeros_like(c["q"])
    c["q"][..., :64] = 2.0 ** (bits - 6 - of_k)
    assert torch.isfinite(c["q"]).all() and torch.isfinite(c["k_pages"][held]).all()
    got = _attended(c, scale=1.0)
    ref, weight = attend_oracle(**c, scale=1.0)
    tol = attend_tolerance(ref, weight, dtype, 0)
    assert bool(((got.double() - ref).abs() <= tol).all()), float(((got.double() - ref).abs() / tol).max())


def _attended(c, **kw):
    got = ec().attend(**c, **kw)
    ec().check_device_error(DEV)
    assert torch.isfinite(got.float()).all()
    return got


# ---- parts of split tiles ------------------------------------------------------------------------------

def _stripes(c, page):
    """V in head_dim stretches of an episode's keys, each 1 in a dim of its own: every output dim is the weight of one
    stretch, so that a part of a tile that is lost, or counted twice, shows in it."""
    hd = c["q"].shape[2]
    for b, n in enumerate(c["length"].tolist()):
        j = torch.arange(n, device=DEV)
        v = torch.nn.functional.one_hot(j * hd // n, hd).to(c["v_pages"].dtype)
        c["v_pages"][c["table"][b, :-(-n // page)].long()[j // page], j % page] = v[:, None].expand(n, c["v_pages"].shape[2], hd)
    return c


def _check_stripes(got, c, **kw):
    """Half a step of the output and of each weight, 2^-12 for scores and exponentials as everywhere; what fp16 drops of a
    key is below 2^-32 of the largest weight (lifted by 2^7 or more). No term grows with the keys in bf16."""
    ref, weight = attend_oracle(**c, **kw)
    u = torch.finfo(c["q"].dtype).eps / 2
    lost = int(c["length"].max()) * 2.0 ** -32 if c["q"].dtype == FP else 2.0 ** -133
    tol = u * ref.abs() + (u + 2.0 ** -12) * weight + lost
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


# 16-row tiles in up to 26 parts, in more; chunks in a few parts, in more than 12 (joined in two levels); those of the
# tests of determinism and of two streams
SPLIT = pytest.mark.parametrize("heads,kv,hd,page,new,past", [
    (12, 12, 64, 32, [1], [20000]), (16, 2, 128, 128, [1], [60000]), (16, 8, 128, 64, [1, 1, 3], [38000, 17, 9000]),
    (4, 1, 64, 256, [1], [70000]), (16, 8, 128, 256, [40], [38000]), (8, 1, 64, 128, [100], [50000]),
    (32, 8, 128, 64, [300], [9000]), (12, 4, 64, 32, [500, 33, 200], [7000, 3000, 0]),
    (8, 2, 128, 64, [1, 1], [8999, 4999]), (8, 2, 128, 64, [200], [5800]), (8, 2, 64, 64, [180], [5820])])


@SPLIT
@pytest.mark.parametrize("dtype", [BF, FP])
def test_attend_counts_every_part_once(heads, kv, hd, page, new, past, dtype):
    c = _stripes(pages_for(new, past, heads, kv, hd, page=page, dtype=dtype, seed=5, q_scale=0.7, extra_width=1), page)
    for kw in (dict(), dict(causal=False), dict(window=max(past) // 2, sinks=300)):
        want = ec().attend(**c, max_rows=max(new), **kw)
        ec().check_device_error(DEV)
        _check_stripes(want, c, **kw)
        for _ in range(3):      # whichever block comes last
            assert torch.equal(ec().attend(**c, max_rows=max(new), **kw), want)


def test_stripes_show_a_lost_part():
    """The check above with one stretch of 1024 of 38,001 keys left out, or counted twice, on the oracle's side."""
    c = _stripes(pages_for([1], [38000], 4, 2, 128, page=256, seed=5, q_scale=0.7), 256)
    got = ec().attend(**c)
    _check_stripes(got, c)
    for factor in (0.0, 2.0):
        ids = c["table"][0, 40:44].long()
        spoilt = dict(c, v_pages=c["v_pages"].clone())
        spoilt["v_pages"][ids] *= factor
        with pytest.raises(AssertionError):
            _check_stripes(got, spoilt)


# ---- rotary geometries ---------------------------------------------------------------------------------

def test_prepare_turns_k_by_its_positions():
    """K of ``RegisterPrepare.run`` with positions is K without turned by the formula's angles; sections that leave dims out
    are refused. K without is rounded to bf16 (half a step of each of two terms), K with once more, and the tables are
    off by 2e-6."""
    from reki_megakernel_b200.prepare import RegisterPrepare
    from reki_megakernel_b200.synthetic import ExpertDims, make_prepare_weights, make_source
    d = ExpertDims(L=1)
    rp = RegisterPrepare(make_prepare_weights(d, seed=0).to(DEV))
    src = make_source(70, d.src_dim, seed=1).to(DEV)
    pos = torch.stack([torch.arange(70) // 35, torch.arange(70) % 35 // 7, torch.arange(70) % 7]).to(torch.int32)
    plain, v0 = rp.run(src, positions=torch.zeros_like(pos).to(DEV), sections=(8, 12, 12))
    u = torch.finfo(BF).eps / 2
    for n, sections, interleaved in ((3, (8, 12, 12), False), (2, (20, 12), True), (1, None, False)):
        k, v = rp.run(src, positions=pos[:n].to(DEV), sections=sections, interleaved=interleaved)
        ang = angles_oracle(pos[:n], sections or (32,), interleaved=interleaved)
        ref = turn_oracle(plain[0], ang)
        x = plain[0].cpu().double().abs()
        c, s = ang.cos().abs()[:, None], ang.sin().abs()[:, None]
        a, b = x[..., :32], x[..., 32:]
        size = torch.cat([a * c + b * s, b * c + a * s], -1)
        err = (k[0].cpu().double() - ref).abs()
        assert bool((err <= u * ref.abs() + (u * (1 + u) + 4e-6) * size).all()), float((err / (u * ref.abs() + u * size)).max())
        assert torch.equal(v, v0)
    with pytest.raises(ValueError):
        rp.run(src, positions=pos[:2].to(DEV), sections=(8, 8))
    with pytest.raises(ValueError):
        rp.run(src, sections=(16, 16))
    torch.cuda.synchronize()
    rp.check_device_error()
    rp.close()


@pytest.mark.parametrize("base", [1.0, 0.3, 1e-4, 1e-6])
def test_rope_tables_of_a_base_up_to_one(base):
    """Frequencies of many turns a position. 2e-6 as for any base; the rates in 64 bits, here and in the oracle, are off by
    two units of 2^-53 of the angle each (a power, a quotient)."""
    g = torch.Generator().manual_seed(0)
    pos = torch.randint(10 ** 6 - 5000, 10 ** 6, (1, 77), generator=g).to(torch.int32)
    cos, sin = ec().rope_tables(pos.to(DEV), 64, base=base)
    ang = angles_oracle(pos, (32,), base=base)
    tol = 2e-6 + 4 * 2.0 ** -53 * float(ang.abs().max())
    assert (cos.cpu().double() - torch.cat([ang.cos()] * 2, 1)).abs().max() <= tol
    assert (sin.cpu().double() - torch.cat([ang.sin()] * 2, 1)).abs().max() <= tol


# ---- several threads -----------------------------------------------------------------------------------

def test_plans_of_two_threads():
    """The C ABI from two threads at once (ctypes lets go of Python's lock), both with more episodes than the default shared
    memory holds, and not as many: no launch fails, and both plans are right."""
    from reki_megakernel_b200 import _lib
    lib = _lib.load()
    failed, starts = [], {}

    def plans(B, times):
        i32 = dict(dtype=torch.int32, device=DEV)
        length, new, ring = torch.zeros(B, **i32), torch.ones(B, **i32), torch.arange(B, **i32)
        table, marks = torch.full((B, 2), -1, **i32), torch.tensor([0, B, 0], dtype=torch.int64, device=DEV)
        start, slot = torch.zeros(B + 1, **i32), torch.zeros(B, dtype=torch.int64, device=DEV)
        episode, position, after, marks_after = torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros_like(marks)
        a = _lib.PlanInputs(*(t.data_ptr() for t in (length, new, table, ring, marks, start, slot, episode, position, after, marks_after)),
                            None, B, 2, B, 16, B)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        for _ in range(times):
            if lib.mkx_cache_plan(C.byref(a), 0, stream.cuda_stream):
                failed.append(B)
        torch.cuda.synchronize()
        starts[B] = (start.tolist(), slot.tolist(), marks_after.tolist())

    threads = [threading.Thread(target=plans, args=(B, 4000)) for B in (4096, 2100)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for B in (4096, 2100):
        assert starts[B] == (list(range(B + 1)), [16 * b for b in range(B)], [B, B, 0])


# ---- autograd ------------------------------------------------------------------------------------------

def test_gradients_are_not_dropped_in_silence():
    """A tensor that requires grad is refused by the calls while gradients are recorded, and taken under no_grad."""
    import test_episode_cache_host as host
    from test_episode_cache_edges_host import grad_cases
    for name, good, floats in grad_cases(host, DEV):
        f = {"write": ec().write_rows, "attend": ec().attend}[name]
        for arg in floats:
            kw = {**good, arg: good[arg].clone().requires_grad_(True)}
            with pytest.raises(ValueError, match=f"{arg} requires grad"):
                f(**kw)
            with torch.no_grad():
                assert not f(**kw).requires_grad
    torch.cuda.synchronize()


def test_writes_in_place_are_seen_by_autograd():
    """What a call writes in place has a new version, so that a backward pass that saved it refuses; inference tensors,
    which have none, are taken as well."""
    E = ec()

    def changed(f, *tensors):
        before = [t._version for t in tensors]
        f()
        return [t._version > b for t, b in zip(tensors, before)]

    c = E.EpisodeCache(layers=2, pages=8, episodes=2, page_rows=16, kv_heads=2, pages_per_episode=4, device=DEV)
    new = torch.ones(2, dtype=torch.int32, device=DEV)
    x = torch.ones(2, 2, 64, dtype=BF, device=DEV)
    plans = []
    assert all(changed(lambda: plans.append(c.plan(new, 2)), c.table, c.length, c.marks))
    pos = torch.arange(2, dtype=torch.int32, device=DEV)
    q = x.clone()
    assert all(changed(lambda: c.write(1, x, x, plans[0], q=q, positions=pos, out=q), c.k, c.v, q))
    assert all(changed(lambda: c.attend(1, x, plans[0], out=q), q)) and changed(lambda: c.attend(1, x, plans[0]), c.k, c.v, x) == [False] * 3
    w = torch.ones((), device=DEV, requires_grad=True)
    loss = (c.k[1].float() * w * c.k[1].float()).sum() + (c.k[1] * w).sum()
    c.write(1, x, x, plans[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    assert all(changed(lambda: c.release(torch.ones(2, dtype=torch.bool, device=DEV)), c.table, c.length, c.marks, c.free))
    with torch.inference_mode():
        i = E.EpisodeCache(layers=1, pages=8, episodes=2, page_rows=16, kv_heads=2, pages_per_episode=4, device=DEV)
    plan = i.plan(new, 2)
    i.write(0, x, x, plan)
    i.attend(0, x, plan)
    i.release(torch.ones(2, dtype=torch.bool, device=DEV))
    torch.cuda.synchronize()


# ---- outputs that overlap ------------------------------------------------------------------------------

def test_outputs_that_share_a_place_are_refused():
    """An expanded tensor may be read (one row for all heads), but not written to, nor be the pages of attend."""
    import test_episode_cache_host as host
    good = host.write_args(DEV)[0]
    one = torch.ones(7, 1, 64, dtype=BF, device=DEV)
    pool = torch.zeros(1, 32, 2, 64, dtype=BF, device=DEV)
    wide = ec().write_rows(**{**good, "q": one.expand(7, 6, 64), "k": one.expand(7, 2, 64)})
    assert wide.shape == (7, 6, 64) and (wide[:, 0] == wide[:, 5]).all()
    for kw in (dict(out=one.clone().expand(7, 6, 64)), dict(k_pages=pool.expand(4, 32, 2, 64)), dict(v_pages=pool.expand(4, 32, 2, 64))):
        with pytest.raises(ValueError, match="share a place"):
            ec().write_rows(**{**good, **kw})
    good = host.attend_args(DEV)[0]
    for kw in (dict(out=one.clone().expand(7, 6, 64)), dict(k_pages=pool.expand(4, 32, 2, 64)), dict(v_pages=pool[:, :, :1].expand(1, 32, 2, 64))):
        kw = {**good, **kw}
        if kw["v_pages"].shape[0] == 1:
            kw["k_pages"] = pool
        with pytest.raises(ValueError, match="share a place"):
            ec().attend(**kw)
    torch.cuda.synchronize()
