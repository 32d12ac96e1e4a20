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
