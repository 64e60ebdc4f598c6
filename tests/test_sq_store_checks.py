"""Scalar-quantised rows: groups near and beyond the range of an int, as the C ABI
and the Python binding check them (no GPU).  The addresses are never read: every
call here is refused, or has no rows."""
import pytest

import insitu_b200 as ib

P = 1 << 20
OK, EINVAL = 0, -1
LARGEST = (1 << 31) - 16         # the largest group that an int holds


def write(**change):
    L = ib.load_library(require_device=False)
    args = dict(x=None, x_type=0, n=0, d=32, ldx=32, slots=P, bits=8, group=0, codes=P, ldc=32, scales=P, lds=1,
                capacity=16, claim=None, stream=None)
    return L.ivf_sq_write(*{**args, **change}.values())


def read(**change):
    L = ib.load_library(require_device=False)
    args = dict(codes=P, ldc=32, scales=P, lds=1, capacity=16, bits=8, group=0, slots=P, n=0, d=32, out=None,
                out_type=0, ldo=32, stream=None)
    return L.ivf_sq_read(*{**args, **change}.values())


@pytest.mark.parametrize("call", [write, read])
@pytest.mark.parametrize("group", [0, 16, 32, 48, 1 << 20, 1 << 30, LARGEST - 16, LARGEST])
@pytest.mark.parametrize("d", [17, 32, 1 << 20])
def test_rows_have_room_for_their_scales(call, group, d):
    """the distance between rows of scales is at least the number of groups, whatever the group"""
    least = -(-d // group) if group else 1
    rows = dict(d=d, ldx=d) if call is write else dict(d=d, ldo=d)
    for lds, rc in ((least, OK), (least + 5, OK), (least - 1, EINVAL), (0, EINVAL), (-1, EINVAL)):
        assert call(group=group, lds=lds, ldc=d, **rows) == rc, lds


@pytest.mark.parametrize("group", [1 << 31, (1 << 32) + 16, 1 << 40])
def test_binding_refuses_groups_that_no_int_holds(group):
    """(ctypes would pass their last 32 bits on: a group of 16, with more scales than the store has room for)"""
    import torch

    rows = ib.SQRows.__new__(ib.SQRows)
    with pytest.raises(ValueError, match="group"):
        rows._adopt(torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 8)[:, :1], 20, 8, group)
