"""CPU: the training operators at the edges of their arguments, without a device: room in workspaces, refusals."""
import ctypes as C


def test_head_workspace_has_a_row_of_column_sums_for_every_workgroup():
    """A head of at most 64 classes: the gradient runs over the tokens padded to 64, 16 of them a workgroup up to 8192 and 64 beyond, and each
    workgroup writes one fp32 value per class behind the padded operands and d.  Everything but these sums depends on the padded number only."""
    from sgpo_amd import _lib as L
    lib = L.load()
    up = lambda n, a: (n + a - 1) // a * a               # noqa: E731
    H = 512
    a = L.LinearCeArgs(hidden=1 << 30, weight=1 << 31, targets=4096, H=H, ld_hidden=H, ld_weight=H, reduction=1)
    ref = C.byref(a)
    need = lib.sgpo_linear_ce_workspace_bytes
    for dtype, planes in ((0, 3), (1, 1)):
        a.dtype = dtype
        for V in range(1, 65):
            a.V = V
            weights = up(V * H * planes * 2, 256) if planes == 3 else 0     # bf16 rows of whole K steps are read as they are
            for N in [*range(1, 8193), 8255, 8256, 8257, 20011]:
                a.N = N
                rows = up(N, 64)
                parts = up(rows * H * planes * 2, 256) + weights + up(rows * 64 * planes * 2, 256) + rows // (16 if N <= 8192 else 64) * V * 4
                got = need(ref, 1)
                assert got >= parts, (dtype, V, N)
                a.N = rows
                assert got >= need(ref, 1), (dtype, V, N)
