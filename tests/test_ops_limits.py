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


def test_an_experts_workspace_holds_fewer_tokens_too():
    """A batch comes in parts, or a program allocates for its largest: no smaller T needs more."""
    for k, E, D, I in ((8, 64, 2048, 1024), (1, 1, 16, 16), (16, 16, 16, 4096), (3, 20, 1040, 720), (16, 1000, 128, 4096),
                       (2, 3, 8, 20000), (17, 40, 64, 64)):
        most, at = 0, 0
        for T in [*range(1, 1500), *range(1500, 40000, 97)]:
            need = _ops.experts_workspace(T, k, E, D, I)
            assert need >= most, (k, E, D, I, T, at)
            most, at = need, T
