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


def test_packed_structs_match_ctypes():
    from reki_megakernel_b200 import _lib
    for cls in (_lib.Rotary, _lib.PlanInputs, _lib.StoreInputs, _lib.AttendInputs):
        flat, want = [], cls()
        n = 1

        def fill(obj, n):
            for name, kind in obj._fields_:
                if issubclass(kind, C.Structure):
                    n = fill(getattr(obj, name), n)
                elif kind is C.c_int * 4:
                    for i in range(4):
                        getattr(obj, name)[i] = n
                        flat.append(n)
                        n += 1
                else:
                    setattr(obj, name, n)
                    flat.append(n)
                    n += 1
            return n

        fill(want, n)
        assert _lib.packer(cls)(*flat) == bytes(want), cls


def test_ticket_bytes_match_the_header():
    from reki_megakernel_b200 import episode_cache as E
    text = (ROOT / "include" / "mkx_cache.h").read_text()
    assert E._TICKET_BYTES == 4 * int(re.search(r"MKX_ATTEND_TICKETS (\d+)", text)[1])
    assert E.MAX_EPISODES == int(re.search(r"MKX_MAX_EPISODES (\d+)", text)[1])


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

def _plan_args():
    return dict(length=_t(3, I32), new=_t(3, I32), table=_t((3, 5), I32), free=_t(9, I32), marks=_t(3, I64), page_rows=16, rows=7)


def test_plan_args():
    from reki_megakernel_b200.episode_cache import check_plan_args
    check_plan_args(**_plan_args())
    bad = [dict(length=_t(0, I32)), dict(length=_t(5000, I32)), dict(new=_t(4, I32)), dict(new=_t(3, I64)), dict(table=_t((2, 5), I32)),
           dict(table=_t((3, 0), I32)), dict(table=_t((5, 3), I32).t()), dict(table=_t((3, 5), I64)), dict(free=_t(0, I32)), dict(free=_t((3, 3), I32)),
           dict(marks=_t(2, I64)), dict(marks=_t(3, I32)), dict(page_rows=48), dict(rows=-1), dict(rows=1 << 31),
           dict(new=_t(3, I32, "cpu")), dict(table=_t((3, (1 << 26) + 1), I32))]
    for kw in bad:
        with pytest.raises(ValueError):
            check_plan_args(**{**_plan_args(), **kw})


def _write_args():
    return dict(k=_t((7, 2, 64)), v=_t((7, 2, 64)), slot=_t(7, I64), k_pages=_t((4, 32, 2, 64)), v_pages=_t((4, 32, 2, 64)),
                q=_t((7, 6, 64)), positions=_t((1, 7), I32), out=None)


def test_write_args():
    from reki_megakernel_b200.episode_cache import check_write_args
    check_write_args(**_write_args())
    check_write_args(**{**_write_args(), "q": None, "positions": None})
    bad = [dict(v=_t((7, 1, 64))), dict(k=_t((7, 2, 72)), v=_t((7, 2, 72))), dict(k=_t((7, 2, 64), torch.float32)), dict(slot=_t(6, I64)),
           dict(slot=_t(7, I32)), dict(k_pages=_t((4, 20, 2, 64)), v_pages=_t((4, 20, 2, 64))), dict(v_pages=_t((4, 32, 3, 64))),
           dict(k_pages=_t((4, 32, 2, 64), torch.float16)), dict(k_pages=_t((4, 32, 2, 64), BF, "cpu")), dict(q=_t((6, 6, 64))),
           dict(q=_t((7, 6, 32))), dict(q=_t((7, 6, 64), torch.float16)), dict(positions=None), dict(out=_t((7, 6, 32))),
           dict(q=None, out=_t((7, 6, 64)))]
    for kw in bad:
        with pytest.raises(ValueError):
            check_write_args(**{**_write_args(), **kw})


def _attend_args():
    return dict(q=_t((7, 6, 64)), k_pages=_t((4, 32, 2, 64)), v_pages=_t((4, 32, 2, 64)), table=_t((3, 5), I32), length=_t(3, I32),
                start=_t(4, I32), max_rows=None, causal=True, window=8, sinks=2, scale=None, out=None)


def test_attend_args():
    from reki_megakernel_b200.episode_cache import check_attend_args
    check_attend_args(**_attend_args())
    bad = [dict(q=_t((7, 6, 80))), dict(q=_t((7, 6, 64), torch.float32)), dict(q=_t((7, 5, 64))), dict(k_pages=_t((4, 32, 2, 128))),
           dict(v_pages=_t((4, 16, 2, 64))), dict(v_pages=_t((4, 32, 2, 64), torch.float16)), dict(table=_t((2, 5), I32)),
           dict(table=_t((3, 5), I64)), dict(length=_t(3, I64)), dict(start=_t(3, I32)), dict(max_rows=-1), dict(causal=False),
           dict(window=-1), dict(window=0), dict(sinks=-2), dict(scale=float("nan")), dict(out=_t((7, 6, 128))), dict(out=_t((7, 6, 64), BF, "cpu"))]
    for kw in bad:
        with pytest.raises(ValueError):
            check_attend_args(**{**_attend_args(), **kw})


def test_wrappers_refuse_the_cpu_and_odd_strides():
    from reki_megakernel_b200 import episode_cache as E
    a = {k: (torch.zeros(v.shape, dtype=v.dtype) if isinstance(v, torch.Tensor) else v) for k, v in _attend_args().items()}
    with pytest.raises(ValueError):
        E.attend(**a)
    with pytest.raises(ValueError):
        E.rope_tables(torch.zeros(4, dtype=I32), 64)
    x = torch.zeros(4, 2, 64, dtype=BF)
    assert E._strides(x, "x") == (x.data_ptr(), [128, 64])
    assert E._strides(x[:, 1:], "x")[1] == [128, 64]
    assert E._strides(torch.zeros(8, 2, 72, dtype=BF)[::2, :1, :64], "x")[1] == [288, 64]
    assert E._strides(torch.zeros(2, 3, 4, 64, dtype=BF).transpose(1, 2), "x")[1] == [768, 64, 256]
    for bad in (torch.zeros(4, 2, 65, dtype=BF)[:, :, :64], torch.zeros(4, 2, 72, dtype=BF)[:, :, 1:65], torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)):
        with pytest.raises(ValueError):
            E._strides(bad, "x")


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
