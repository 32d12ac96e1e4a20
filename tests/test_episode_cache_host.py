"""The paged episode cache without a GPU: struct layouts, argument checks of the C entry points and of the Python
wrappers (``meta`` tensors stand for the device's), and the restatement the GPU tests compare with."""
import ctypes as C
import re
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT
from oracle.cache_oracle import attend_oracle, axis_of, plan_oracle

META = torch.device("meta")
BF, I32, I64 = torch.bfloat16, torch.int32, torch.int64


def _t(shape, dtype=BF, device=META):
    return torch.empty(shape, dtype=dtype, device=device)


@pytest.mark.parametrize("struct,cls", [("mkx_rotary", "Rotary"), ("mkx_plan_inputs", "PlanInputs"),
                                        ("mkx_release_inputs", "ReleaseInputs"), ("mkx_store_inputs", "StoreInputs"),
                                        ("mkx_attend_inputs", "AttendInputs")])
def test_struct_layout_matches_c(struct, cls, tmp_path):
    from reki_megakernel_b200 import _lib
    gcc = shutil.which("gcc")
    if not gcc:
        pytest.skip("gcc missing")
    ct = getattr(_lib, cls)
    fields = [f[0] for f in ct._fields_]
    body = "".join(f'printf("{f} %zu\\n", offsetof({struct}, {f}));' for f in fields)
    (tmp_path / "l.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "mkx_cache.h"\n'
                                  f'int main(void){{{body} printf("sizeof %zu\\n", sizeof({struct})); return 0;}}\n')
    subprocess.run([gcc, "-I", str(ROOT / "include"), "-I", "/usr/local/cuda/include", str(tmp_path / "l.c"), "-o",
                    str(tmp_path / "l")], check=True)
    c = dict(line.split() for line in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True).stdout.splitlines())
    assert {f: getattr(ct, f).offset for f in fields} == {f: int(c[f]) for f in fields}
    assert C.sizeof(ct) == int(c["sizeof"])


def test_constants_match_the_header():
    from reki_megakernel_b200 import _lib
    from reki_megakernel_b200 import episode_cache as E
    text = (ROOT / "include" / "mkx_cache.h").read_text()
    assert E.MAX_EPISODES == int(re.search(r"MKX_MAX_EPISODES (\d+)", text)[1])
    want = _lib.Rotary(1e6, 3, (C.c_int * 4)(8, 12, 16, 0), 1)
    assert _lib.pack_rotary(1e6, 3, 8, 12, 16, 0, 1) == bytes(want)


def test_torch_binding_refuses_what_it_does_not_know():
    """It answers None (the wrappers then say what is wrong), whatever it is given."""
    from reki_megakernel_b200 import _lib
    m = _lib.load_torch()
    x = torch.zeros(3)
    for f in (m.plan, m.store, m.attend):
        assert f() is None and f(1, 2, 3) is None
        for n in (8, 9, 12):
            assert f(*[x] * n) is None and f(*[None] * n) is None and f(*["a"] * n) is None


def test_null_arguments_are_rejected_without_a_device():
    from reki_megakernel_b200 import _lib
    lib, bad = _lib.load(), _lib.MKX_ERR_INVALID_ARG
    assert lib.mkx_cache_plan(None, 0, None) == bad
    assert lib.mkx_cache_plan(C.byref(_lib.PlanInputs()), 0, None) == bad
    assert lib.mkx_cache_release(None, 0, None) == bad
    assert lib.mkx_cache_release(C.byref(_lib.ReleaseInputs()), 0, None) == bad
    assert lib.mkx_rope_tables(None, None, 0, 4, 64, None, None, 0, None) == bad
    assert lib.mkx_cache_store(None, 0, None) == bad
    assert lib.mkx_cache_store(C.byref(_lib.StoreInputs()), 0, None) == bad
    assert lib.mkx_cache_attend(None, 0, 0, None) == bad
    assert lib.mkx_attend_workspace(None, 0) == 0


def _plan_inputs(**kw):
    from reki_megakernel_b200 import _lib
    a = dict(length=64, new_rows=64, table=64, ring=64, marks=64, start=64, slot=64, episode=64, position=64,
             length_out=128, marks_out=128, ticket=None, B=2, table_width=4, ring_pages=8, page_rows=16, rows=4)
    return _lib.PlanInputs(**{**a, **kw})


@pytest.mark.parametrize("kw", [dict(B=0), dict(B=4097), dict(page_rows=24), dict(page_rows=8), dict(page_rows=512), dict(rows=-1),
                                dict(table_width=0), dict(ring_pages=0), dict(slot=72), dict(position=68), dict(table=None),
                                dict(length_out=64), dict(marks_out=64), dict(slot=None)])
def test_c_plan_refuses(kw):
    from reki_megakernel_b200 import _lib
    assert _lib.load().mkx_cache_plan(C.byref(_plan_inputs(**kw)), 0, None) == _lib.MKX_ERR_INVALID_ARG


def _store_inputs(**kw):
    from reki_megakernel_b200 import _lib
    rot = _lib.Rotary(10000.0, 3, (C.c_int * 4)(8, 12, 12, 0), 0)
    a = dict(q=64, k=64, v=64, q_out=64, k_pages=64, v_pages=64, slot=64, positions=64, pos_stride=4, q_row=128, q_head=64,
             k_row=128, k_head=64, v_row=128, v_head=64, qo_row=128, qo_head=64, kp_page=2048, kp_row=128, kp_head=64,
             vp_page=2048, vp_row=128, vp_head=64, rows=4, heads=2, kv_heads=2, head_dim=64, dtype=0, pages=3, page_rows=16, rot=rot)
    return _lib.StoreInputs(**{**a, **kw})


@pytest.mark.parametrize("kw", [dict(rows=-1), dict(kv_heads=0), dict(pages=0), dict(page_rows=17), dict(k=72), dict(q_out=None),
                                dict(k_row=100), dict(vp_head=4), dict(kp_page=-8), dict(positions=None), dict(slot=None),
                                dict(head_dim=72), dict(head_dim=272), dict(head_dim=48), dict(dtype=2), dict(heads=0)])
def test_c_store_refuses(kw):
    from reki_megakernel_b200 import _lib
    st = _lib.load().mkx_cache_store(C.byref(_store_inputs(**kw)), 0, None)
    assert st in (_lib.MKX_ERR_INVALID_ARG, _lib.MKX_ERR_UNSUPPORTED)
    assert _lib.load().mkx_cache_store(C.byref(_store_inputs(rows=0)), 0, None) == _lib.MKX_OK   # nothing to store


@pytest.mark.parametrize("base,sections", [(0.0, (32,)), (float("nan"), (32,)), (1e4, (33,)), (1e4, (20, 8, 8)), (1e4, (4,)), (1e4, (-8, 32)),
                                           (1e4, (8, 12)), (1e4, (8, 8, 8, 8, 0))])
def test_rotary_refuses(base, sections):
    from reki_megakernel_b200 import episode_cache as E
    with pytest.raises(ValueError):
        E._rotary(64, sections, base, False)


def _attend_inputs(**kw):
    from reki_megakernel_b200 import _lib
    a = dict(q=64, k_pages=64, v_pages=64, out=64, table=64, length=64, start=64, workspace=64, error=64, q_row=128, q_head=64,
             o_row=128, o_head=64, kp_page=2048, kp_row=128, kp_head=64, vp_page=2048, vp_row=128, vp_head=64, rows=4, B=2, heads=2,
             kv_heads=2, head_dim=64, dtype=0, pages=3, page_rows=16, table_width=4, max_rows=4, causal=1, window=0, sinks=0, scale=0.1)
    return _lib.AttendInputs(**{**a, **kw})


@pytest.mark.parametrize("kw", [dict(head_dim=80), dict(dtype=3), dict(window=-1), dict(sinks=-1), dict(sinks=3),
                                dict(window=4, causal=0), dict(scale=float("inf")), dict(q=72), dict(workspace=8), dict(error=None),
                                dict(q_row=4), dict(kp_page=12), dict(table=None)])
def test_c_attend_refuses(kw):
    from reki_megakernel_b200 import _lib
    st = _lib.load().mkx_cache_attend(C.byref(_attend_inputs(**kw)), 1 << 30, 0, None)
    assert st in (_lib.MKX_ERR_INVALID_ARG, _lib.MKX_ERR_UNSUPPORTED)


# ---- the wrappers ---------------------------------------------------------------------------------------

def plan_args(dev=META):
    t = lambda shape, dtype, d=dev: torch.zeros(shape, dtype=dtype, device=d)  # noqa: E731
    good = dict(length=t(3, I32), new=t(3, I32), table=t((3, 5), I32), free=t(9, I32), marks=t(3, I64), page_rows=16, rows=7)
    bad = [dict(length=t(0, I32)), dict(length=t(5000, I32)), dict(new=t(4, I32)), dict(new=t(3, I64)), dict(table=t((2, 5), I32)),
           dict(table=t((3, 0), I32)), dict(table=t((5, 3), I32).t()), dict(table=t((3, 5), I64)), dict(free=t(0, I32)), dict(free=t((3, 3), I32)),
           dict(marks=t(2, I64)), dict(marks=t(3, I32)), dict(page_rows=48), dict(rows=-1), dict(rows=1 << 31), dict(new=t(3, I32, "cpu")),
           dict(table=t((1, 1), I32).expand(3, (1 << 26) + 1)), dict(length=t((3, 1), I32)), dict(new=t(6, I32)[::2])]
    return good, bad


def write_args(dev=META):
    t = lambda shape, dtype=BF, d=dev: torch.zeros(shape, dtype=dtype, device=d)  # noqa: E731
    good = dict(k=t((7, 2, 64)), v=t((7, 2, 64)), slot=t(7, I64), k_pages=t((4, 32, 2, 64)), v_pages=t((4, 32, 2, 64)), q=t((7, 6, 64)),
                positions=t((1, 7), I32), out=None)
    bad = [dict(v=t((7, 1, 64))), dict(k=t((7, 2, 72)), v=t((7, 2, 72))), dict(k=t((7, 2, 64), torch.float32)), dict(slot=t(6, I64)),
           dict(slot=t(7, I32)), dict(k_pages=t((4, 20, 2, 64)), v_pages=t((4, 20, 2, 64))), dict(v_pages=t((4, 32, 3, 64))),
           dict(k_pages=t((4, 32, 2, 64), torch.float16)), dict(k_pages=t((4, 32, 2, 64), BF, "cpu")), dict(q=t((6, 6, 64))),
           dict(q=t((7, 6, 32))), dict(q=t((7, 6, 64), torch.float16)), dict(positions=None), dict(out=t((7, 6, 32))),
           dict(q=None, out=t((7, 6, 64))), dict(k=t((7, 128))), dict(out=t((7, 6, 64), BF, "cpu"))]
    return good, bad


def attend_args(dev=META):
    t = lambda shape, dtype=BF, d=dev: torch.zeros(shape, dtype=dtype, device=d)  # noqa: E731
    good = dict(q=t((7, 6, 64)), k_pages=t((4, 32, 2, 64)), v_pages=t((4, 32, 2, 64)), table=t((3, 5), I32), length=t(3, I32), start=t(4, I32),
                max_rows=None, causal=True, window=8, sinks=2, scale=None, out=None)
    bad = [dict(q=t((7, 6, 80))), dict(q=t((7, 6, 64), torch.float32)), dict(q=t((7, 5, 64))), dict(k_pages=t((4, 32, 2, 128))),
           dict(v_pages=t((4, 16, 2, 64))), dict(v_pages=t((4, 32, 2, 64), torch.float16)), dict(table=t((2, 5), I32)),
           dict(table=t((3, 5), I64)), dict(length=t(3, I64)), dict(start=t(3, I32)), dict(max_rows=-1), dict(max_rows=-2), dict(causal=False),
           dict(window=-1), dict(window=0), dict(sinks=-2), dict(scale=float("nan")), dict(out=t((7, 6, 128))), dict(out=t((7, 6, 64), BF, "cpu")),
           dict(k_pages=t((4, 24, 2, 64)), v_pages=t((4, 24, 2, 64))), dict(length=t(0, I32), start=t(1, I32), table=t((0, 5), I32))]
    return good, bad


@pytest.mark.parametrize("name", ["plan", "write", "attend"])
def test_arguments(name):
    from reki_megakernel_b200 import episode_cache as E
    check = getattr(E, f"check_{name}_args")
    good, bad = globals()[f"{name}_args"]()
    check(**good)
    if name == "write":
        check(**{**good, "q": None, "positions": None})
    for kw in bad:
        with pytest.raises(ValueError):
            check(**{**good, **kw})


def test_wrappers_refuse_the_cpu_and_odd_strides():
    from reki_megakernel_b200 import episode_cache as E
    for name, f in (("plan", E.plan_rows), ("write", E.write_rows), ("attend", E.attend)):
        with pytest.raises(ValueError, match="CUDA"):
            f(**globals()[f"{name}_args"]("cpu")[0])
    with pytest.raises(ValueError):
        E.rope_tables(torch.zeros(4, dtype=I32), 64)
    for good in (torch.zeros(4, 2, 64, dtype=BF), torch.zeros(8, 2, 72, dtype=BF)[::2, :1, :64], torch.zeros(2, 3, 4, 64, dtype=BF).transpose(1, 2)):
        E._check_strides(good, "x")
    for bad in (torch.zeros(4, 2, 65, dtype=BF)[:, :, :64], torch.zeros(4, 2, 72, dtype=BF)[:, :, 1:65], torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)):
        with pytest.raises(ValueError):
            E._check_strides(bad, "x")


# ---- the restatement ------------------------------------------------------------------------------------

def test_axes_in_turn():
    assert axis_of((3, 1, 2), False) == [0, 0, 0, 1, 2, 2]
    assert axis_of((3, 1, 2), True) == [0, 1, 2, 0, 2, 0]


def test_plan_by_hand():
    r = plan_oracle([17, 0, 3], [16, 2, 0], [[4, 5, -1], [-1, -1, -1], [7, -1, -1]], [9, 8, 6], [1, 3, 0], 16, 19)
    assert r["table"] == [[4, 5, 8], [6, -1, -1], [7, -1, -1]]
    assert r["slot"] == [81 + i for i in range(15)] + [128, 96, 97, -1] and r["marks"] == [3, 3, 0] and r["length"] == [33, 2, 3]


def test_attention_by_hand():
    """Two keys with scores 0 and log 3: weights 1/4 and 3/4; a window of one row sees itself."""
    k = torch.zeros(1, 16, 1, 64)
    v = torch.zeros(1, 16, 1, 64)
    k[0, 1, 0, 0] = torch.log(torch.tensor(3.0))
    v[0, 0], v[0, 1] = 4.0, 8.0
    q = torch.zeros(1, 1, 64)
    q[..., 0] = 1.0
    a = (q, k, v, torch.tensor([[0]]), torch.tensor([2]), torch.tensor([0, 1]))
    assert torch.allclose(attend_oracle(*a, scale=1.0)[0], torch.tensor(7.0, dtype=torch.float64))
    assert torch.allclose(attend_oracle(*a, scale=1.0, window=1)[0], torch.tensor(8.0, dtype=torch.float64))
    assert torch.allclose(attend_oracle(*a, scale=1.0, window=1, sinks=1)[0], torch.tensor(7.0, dtype=torch.float64))
