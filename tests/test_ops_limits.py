"""The operators' C ABI without a GPU, continued: workspaces and refusals."""

from f16acc_amd import _ops


def test_column_sums_checks():
    need = _ops.column_sums_workspace(4096, 100)
    assert need >= 2 * 100 * 4 and _ops.column_sums_workspace(256, 100) == 0 == _ops.column_sums_workspace(0, 100)

    def call(rows=4096, cols=100, x=256, t=0, out=256, ws=256, n=need):
        return _ops.column_sums(x, t, rows, cols, cols, 1, out, ws, n, None)

    assert call(ws=None) == call(ws=128) == call(n=need - 1) == _ops.E_WORKSPACE
    assert call(rows=-1) == call(cols=-1) == call(x=None) == call(t=3) == call(out=None) == _ops.E_ARG
    assert call(cols=1 << 30) == call(rows=1 << 41) == _ops.E_UNSUPPORTED
    assert call(cols=0) == 0
