"""Arguments at the edges of the paged episode cache, without a GPU."""
import pytest
import torch


def test_prepare_refuses_sections_that_leave_dims_out():
    """K's dims d and d + HD / 2 turn together; tables of fewer frequencies pair others. Sections without positions, and
    positions beside tables, have no meaning."""
    from reki_megakernel_b200.prepare import check_position_args
    from reki_megakernel_b200.synthetic import ExpertDims
    d = ExpertDims(L=1)
    assert d.HD == 64
    pos, table = torch.zeros(2, 5, dtype=torch.int32), torch.zeros(5, 64)
    for sections in (None, (16, 16), (0, 32), (8, 12, 12)):
        check_position_args(d, pos, None, None, sections, False)
    check_position_args(d, None, table, table, None, False)
    check_position_args(d, None, None, None, None, False)
    for args in ((pos, None, None, (8, 8), False), (pos, None, None, (40,), False), (pos, table, None, None, False),
                 (pos, None, table, (32,), False), (None, None, None, (8, 8), False), (None, table, table, None, True)):
        with pytest.raises(ValueError):
            check_position_args(d, *args)


def test_no_binding_but_that_of_these_sources(monkeypatch):
    """Another torch, Python or source has a binding of its own, and where that one cannot be built, none is loaded."""
    import importlib.metadata
    import shutil
    from reki_megakernel_b200 import _lib, build
    _lib.load_torch()
    here = build.torch_lib()
    assert here.exists() and here.suffix == ".so"
    monkeypatch.setattr(_lib, "_TORCH", None)
    monkeypatch.setattr(shutil, "which", lambda name: None)
    assert _lib.load_torch() is not None            # it is there: nothing to build
    monkeypatch.setattr(_lib, "_TORCH", None)
    for change in ("torch", "source"):
        with monkeypatch.context() as m:
            if change == "torch":
                m.setattr(importlib.metadata, "version", lambda name: "0.0.1")
            else:
                m.setattr(build, "TORCH_SOURCES", build.TORCH_SOURCES[1:])
            assert build.torch_lib() != here
            with pytest.raises(RuntimeError):
                _lib.load_torch()
            assert _lib._TORCH is None and here.exists()


def test_binding_refuses_a_library_of_another_header():
    from reki_megakernel_b200 import _lib, build
    m, lib = _lib.load_torch(), _lib.load()
    key = lib.mkx_cache_key()
    assert key == build.cache_key() != 0
    assert m.bind(key + 1, 8, 8, 8, 8) is None and m.bind(key, 8, 8, 8) is None and m.bind(0, 8, 8, 8, 8) is None
    assert m.plan(*[torch.zeros(3)] * 8) is None    # and what was bound still is


def grad_cases(host, dev):
    """(name, good arguments, names of the tensors that must not require grad)."""
    return [("write", host.write_args(dev)[0], ("k", "v", "q", "k_pages", "v_pages")), ("attend", host.attend_args(dev)[0], ("q", "k_pages", "v_pages"))]


def test_gradients_are_not_dropped_in_silence():
    import test_episode_cache_host as host
    from reki_megakernel_b200 import episode_cache as E
    for name, good, floats in grad_cases(host, host.META):
        check = getattr(E, f"check_{name}_args")
        for arg in floats + ("out",):
            t = torch.empty(7, 6, 64, dtype=host.BF, device=host.META) if arg == "out" else good[arg].clone()
            kw = {**good, arg: t.requires_grad_(True)}
            with pytest.raises(ValueError, match=f"{arg} requires grad"):
                check(**kw)
            with torch.no_grad():
                check(**kw)


def test_binding_answers_none_to_a_flag_without_a_truth_value():
    """It returned with Python's error set, which the interpreter makes a SystemError of."""
    from reki_megakernel_b200 import _lib
    x = torch.zeros(3)
    assert _lib.load_torch().attend(x, x, x, x, x, x, 1, x, 0, 0, None, None) is None


def test_c_attend_refuses_pages_without_a_stride():
    import ctypes as C
    import test_episode_cache_host as host
    from reki_megakernel_b200 import _lib
    for name in ("kp_page", "vp_page", "kp_row", "vp_row", "kp_head", "vp_head"):
        a = host._attend_inputs(**{name: 0})
        assert _lib.load().mkx_cache_attend(C.byref(a), 1 << 30, 0, None) == _lib.MKX_ERR_INVALID_ARG


def test_what_is_written_to_is_not_expanded():
    from reki_megakernel_b200 import episode_cache as E
    t = torch.zeros(7, 1, 64, dtype=torch.bfloat16).expand(7, 6, 64)
    E._check_strides(t, "q")
    E._check_strides(torch.zeros(7, 6, 64, dtype=torch.bfloat16)[:, :1].expand(7, 1, 64), "out", apart=True)
    with pytest.raises(ValueError, match="share a place"):
        E._check_strides(t, "out", apart=True)


def test_rotary_refuses_a_base_without_an_inverse():
    from reki_megakernel_b200 import episode_cache as E
    E._rotary(64, (32,), 1e-300, False)
    with pytest.raises(ValueError):
        E._rotary(64, (32,), 1e-310, False)
