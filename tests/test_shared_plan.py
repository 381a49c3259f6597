"""Into how many parts a plan of rows with shared prefixes cuts the rows' own keys.  (A plan for the CPU
has all but the addresses of its buffers.)"""
import pytest

from orinfer_b200.ops import functional as F, native


def plan(groups, rows, max_kv_len, qh=32, kvh=8, d=128, **kw):
    if not native.loaded():
        pytest.skip("the kernel library is not built")
    return F.SharedPrefix(groups, rows, qh=qh, kvh=kvh, head_dim=d, max_kv_len=max_kv_len, device="cpu",
                          **{"force": True, **kw})


@pytest.mark.parametrize("qh,kvh,d", [(32, 8, 128), (32, 4, 128), (16, 2, 256), (16, 8, 64)])
@pytest.mark.parametrize("rows", [8, 16, 64])
def test_a_long_row_beside_a_group_is_cut(qh, kvh, d, rows):
    """In no group, behind a shorter prefix, or in a group by itself; where the plan knows every row's
    length, and where it knows one for all."""
    for groups in ([(0, rows, 16384)], [(0, rows, 16384), (rows, 1, 128)]):
        exact = plan(groups, rows + 1, [16500] * (rows + 1), qh, kvh, d)
        assert exact.own_keys >= 16372 and exact.splits >= 4
        assert plan(groups, rows + 1, 16500, qh, kvh, d).splits >= 2


def test_rows_that_are_short_behind_unlike_prefixes_are_not():
    groups = [(0, 16, 4096), (16, 16, 512)]
    p = plan(groups, 32, [4296] * 16 + [712] * 16)
    assert (p.own_keys, p.splits) == (200, 1) and p.scratch is None


def test_parts_follow_rows_and_keys():
    """More rows want fewer parts, more keys want more."""
    for qh, kvh, d in ((32, 8, 128), (32, 4, 128), (16, 2, 256), (16, 8, 64)):
        for groups, rows in (([], (1, 2, 3, 8, 21, 64, 128)), (True, (2, 3, 8, 21, 64, 128))):
            last = None
            for n in rows:
                at = [plan([(0, n, 8192)] if groups else [], n, (8192 if groups else 0) + own, qh, kvh,
                           d).splits for own in (1, 40, 130, 380, 390, 420, 600, 1000, 2000, 5000)]
                assert at == sorted(at) and at[0] == 1
                assert last is None or all(a <= b for a, b in zip(at, last))
                last = at
    assert plan([], 8, 384).splits == plan([], 8, 420).splits


def test_bounds_of_rows():
    from orinfer_b200.ops.native import KernelError
    for rows, bounds in ((3, [10, 10]), (2, [10, -1]), (2, [100, 100])):
        with pytest.raises(KernelError):
            plan([(0, 2, 128)], rows, bounds)
    assert plan([(0, 2, 128)], 3, (128, 130, 5)).own_keys == 5       # a row may end inside its prefix
    assert plan([], 0, []).splits == 1
