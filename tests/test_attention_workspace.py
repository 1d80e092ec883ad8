"""The workspaces that the head asks for: what its passes write there, and no more (no GPU needed)."""
import pytest

from flashlog_b200 import _lib as L

SIZE = {L.FL_F32: 4, L.FL_F16: 2, L.FL_BF16: 2}


def line(n):
    return (n + 63) // 64 * 64


@pytest.mark.parametrize("dtype", [L.FL_F32, L.FL_F16, L.FL_BF16])
@pytest.mark.parametrize("act", [L.FL_ACT_NONE, L.FL_ACT_GELU])
@pytest.mark.parametrize("rows,n,k", [(4608, 29649, 1024), (4608, 1645, 1024), (20000, 1645, 500)])
def test_backward_workspace(rows, n, k, dtype, act):
    sums = 4 * (-(-rows // 128)) * n
    if dtype == L.FL_F32:
        # two planes of 16 bits: dz scaled by rows and by columns, the weight and x; dz itself of an activation
        need = 2 * 4 * rows * line(n) + 4 * (n + rows) * line(k) + 8 * (rows + n + 2 * k)
        need += 4 * rows * line(n) if act != L.FL_ACT_NONE else 0
    else:
        # dz in 16 bits, two planes of an activation's; copies of the weight and x where their rows start anywhere
        need = 2 * rows * line(n) * (1 if act == L.FL_ACT_NONE else 2) + 2 * (n + rows) * line(k)
    got = L.lib().fl_linear_backward_workspace(rows, n, k, dtype, act)
    assert got <= need + sums + 64 * 1024, (got, need + sums)
