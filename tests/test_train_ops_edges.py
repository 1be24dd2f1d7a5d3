"""CPU: the training operators at the edges of their arguments, without a device: room in workspaces, refusals."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fw


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


def test_tangents_are_refused_where_nothing_carries_them_on():
    """Forward-mode inputs: without this, the result would have no tangent, i.e. a derivative of 0."""
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    t = torch.zeros(3, dtype=torch.int64)
    f = torch.zeros(4, dtype=torch.float64)
    q = torch.zeros(1, 2, 2, 8)
    with fw.dual_level():
        def dual(x):
            return fw.make_dual(x, torch.ones_like(x))

        h, w, b = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5)
        for call in (lambda: T.rotary_positions(q, q, dual(f)), lambda: T.rotary_positions_(dual(q), None, f), lambda: T.rotary_positions_(q, dual(q), f),
                     lambda: T.linear_cross_entropy(dual(h), w, t), lambda: T.linear_cross_entropy(h, dual(w), t), lambda: T.linear_cross_entropy(h, w, t, dual(b)),
                     lambda: T.newton_schulz(dual(w)), lambda: T.muon_step(dual(w), w, w, 0.1), lambda: T.muon_step(w, dual(w), w, 0.1), lambda: T.muon_step(w, w, dual(w), 0.1)):
            with pytest.raises(L.SgpoError, match='derivative'):
                call()


def test_lazily_negated_views_are_refused():
    """Their memory holds the values with the other sign."""
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    neg = torch._neg_view
    t = torch.zeros(3, dtype=torch.int64)
    f = torch.zeros(4, dtype=torch.float64)
    q, h, w, b = torch.zeros(1, 2, 2, 8), torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(5)
    for call in (lambda: T.rotary_positions(neg(q), q, f), lambda: T.rotary_positions(q, neg(q), f), lambda: T.rotary_positions(q, None, neg(f)), lambda: T.rotary_positions_(neg(q), None, f),
                 lambda: T.rotary_positions_(q, neg(q), f), lambda: T.linear_cross_entropy(neg(h), w, t), lambda: T.linear_cross_entropy(h, neg(w), t),
                 lambda: T.linear_cross_entropy(h, w, t, neg(b)), lambda: T.newton_schulz(neg(w)), lambda: T.muon_step(neg(w), w, w, 0.1), lambda: T.muon_step(w, neg(w), w, 0.1),
                 lambda: T.muon_step(w, w, neg(w), 0.1)):
        with pytest.raises(L.SgpoError, match='negated'):
            call()


def test_transformed_and_traced_tensors_are_refused():
    """A torch.func transform's tensor, a sparse one and a lazy zero have no memory to read; a trace would keep the call's result as a constant."""
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    w, q, f = torch.ones(3, 5, 8), torch.ones(1, 2, 2, 8), torch.zeros(4, dtype=torch.float64)
    t = torch.zeros(5, dtype=torch.int64)
    one = torch.ones(5, 8)
    for call in (lambda: torch.func.vmap(T.newton_schulz)(w), lambda: torch.func.vmap(lambda x: T.linear_cross_entropy(one, x, t))(w),
                 lambda: torch.func.grad(lambda x: T.linear_cross_entropy(x, one, t))(one), lambda: torch.func.grad(lambda x: T.rotary_positions(x, None, f)[0].sum())(q),
                 lambda: torch.func.vmap(lambda x: T.muon_step(x, one, one, 0.1))(w), lambda: T.newton_schulz(one.to_sparse()),
                 lambda: T.rotary_positions(q, torch._efficientzerotensor(q.shape), f), lambda: T.newton_schulz(torch._efficientzerotensor((5, 8)))):
        with pytest.raises(L.SgpoError, match='memory of its own'):
            call()
    for call, args in ((lambda x: T.newton_schulz(x), (one,)), (lambda x: T.rotary_positions(x, None, f)[0], (q,)), (lambda x: T.linear_cross_entropy(x, one, t), (one,))):
        with pytest.raises(L.SgpoError, match='trace'):
            torch.jit.trace(call, args)


def test_loss_gradients_that_overlap_are_refused():
    """No output of the backward pass may lie over an input or another output; the places are numbers that no call gets to read."""
    from sgpo_amd import _lib as L
    lib = L.load()
    N, H, V = 4, 8, 5
    sizes = dict(hidden=N * H * 4, weight=V * H * 4, targets=N * 8, bias=V * 4, lse=N * 4, g=N * 4, inv=4, dh=N * H * 4, dw=V * H * 4, db=V * 4)
    base = {k: (i + 1) << 20 for i, k in enumerate(sizes)}

    def call(reduction, **moved):
        p = dict(base, **moved)
        a = L.LinearCeArgs(hidden=p['hidden'], weight=p['weight'], bias=p['bias'], targets=p['targets'], N=N, H=H, V=V, ld_hidden=H, ld_weight=H, reduction=reduction)
        # the workspace is too small, which is found last
        rc = lib.sgpo_linear_ce_backward(C.byref(a), p['lse'], p['g'], p['inv'], p['dh'], p['dw'], p['db'], 1 << 30, 16, None)
        assert rc < 0
        return lib.sgpo_last_error().decode()

    for reduction in (L.REDUCE_NONE, L.REDUCE_SUM):
        assert 'workspace' in call(reduction)
        for out in ('dh', 'dw', 'db'):
            assert 'workspace' in call(reduction, **{out: None})
            for other in sizes:
                if other == out or (reduction == L.REDUCE_NONE and other == 'inv'):
                    continue
                size = 4 if other == 'g' and reduction == L.REDUCE_SUM else sizes[other]
                for at in (base[other], base[other] + size - 4, base[other] - sizes[out] + 4):
                    assert 'overlaps' in call(reduction, **{out: at}), (reduction, out, other)
                for at in (base[other] + size, base[other] - sizes[out]):
                    assert 'workspace' in call(reduction, **{out: at}), (reduction, out, other)


def test_rotation_refuses_more_heads_than_it_can_count():
    from sgpo_amd import _lib as L
    lib = L.load()
    n = 1 << 30
    a = L.RotaryArgs(B=1, L=1, heads_q=n, heads_k=n, head_dim=1, rot=0, q=1 << 40, q_out=1 << 41, k=1 << 42, k_out=1 << 43)
    for field in ('q', 'q_out', 'k', 'k_out'):
        setattr(a, field + '_stride', (C.c_int64 * 3)(n, n, 1))
    assert lib.sgpo_rotary(C.byref(a), None) < 0 and 'heads in one call' in lib.sgpo_last_error().decode()


def test_stretched_frequencies_ramp_in_turns():
    """The pairs between beta_slow and beta_fast turns: the share that is kept is linear in the turns, not in the pair's index."""
    from sgpo_amd import train_ops as T
    rot, factor, length = 64, 8.0, 4096
    f, _ = T.rotary_frequencies(rot, device='cpu')
    got, _ = T.rotary_frequencies(rot, scaling='yarn', factor=factor, original_length=length, device='cpu')
    turns = length * f / (2 * torch.pi)
    keep = (got / f - 1 / factor) / (1 - 1 / factor)
    between = (turns > 1) & (turns < 32)
    assert int(between.sum()) >= 10 and bool((keep[turns >= 32] > 1 - 1e-12).all()) and bool((keep[turns <= 1].abs() < 1e-12).all())
    torch.testing.assert_close(keep[between], (turns[between] - 1) / 31, rtol=1e-12, atol=1e-12)
