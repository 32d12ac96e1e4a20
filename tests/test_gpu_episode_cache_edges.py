"""Calls of the paged episode cache at its edges: queries that are not finite, parts of split tiles one by one, geometries and
arguments that are refused, several threads. Oracles as in ``test_gpu_episode_cache.py``."""
import pytest
import torch

from _cache_cases import attend_tolerance, pages_for
from oracle.cache_oracle import attend_oracle

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
