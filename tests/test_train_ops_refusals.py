"""CPU: what the training operators refuse, before anything reaches a device."""
import ctypes as C
import random

import pytest
import torch


def test_host_tensors_are_refused():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    q = torch.zeros(1, 2, 2, 8)
    f = torch.zeros(4, dtype=torch.float64)
    h, w, t = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: T.rotary_positions(q, q, f), lambda: T.rotary_positions_(q, None, f), lambda: T.linear_cross_entropy(h, w, t),
                 lambda: T.newton_schulz(w), lambda: T.muon_step(w, w, w, 0.1)):
        with pytest.raises(L.SgpoError, match='host tensor'):
            call()


def test_what_has_no_gradient_is_refused():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    w = torch.zeros(5, 8, requires_grad=True)
    f = torch.zeros(4, dtype=torch.float64, requires_grad=True)
    q, b = torch.zeros(1, 2, 2, 8), torch.zeros(5, 8)
    for call, text in ((lambda: T.rotary_positions(q, q, f), 'frequencies'), (lambda: T.rotary_positions_(q, None, f), 'frequencies'),
                       (lambda: T.newton_schulz(w), 'no gradient'), (lambda: T.muon_step(w * 2, b, b, 0.1), 'graph'),
                       (lambda: T.muon_step(b, b, w * 2, 0.1), 'graph'), (lambda: T.newton_schulz(b, coefficients=()), 'triples'),
                       (lambda: T.newton_schulz(b, steps=0), 'triples'), (lambda: T.muon_step(b, b, b, 0.1, coefficients=[(1.0, 2.0)] * 5), 'triples')):
        with pytest.raises(L.SgpoError, match=text):
            call()


def test_frequencies():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    f, s = T.rotary_frequencies(64, device='cpu')
    assert s == 1.0 and f.dtype == torch.float64
    torch.testing.assert_close(f, 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64), rtol=1e-15, atol=0)
    lin, _ = T.rotary_frequencies(64, scaling='linear', factor=4.0, device='cpu')
    torch.testing.assert_close(lin, f / 4, rtol=1e-15, atol=0)
    ntk, _ = T.rotary_frequencies(64, scaling='ntk', factor=4.0, device='cpu')
    assert float(ntk[0]) == 1.0 and abs(float(ntk[-1] / f[-1]) - 0.25) < 1e-12
    yarn, s = T.rotary_frequencies(64, scaling='yarn', factor=4.0, device='cpu')
    assert float(yarn[0]) == 1.0 and abs(float(yarn[-1] / f[-1]) - 0.25) < 1e-12 and abs(s - (1 + 0.1 * 1.3862943611198906)) < 1e-12
    assert bool((yarn <= f).all()) and bool((yarn >= f / 4 * (1 - 1e-12)).all())
    assert T.rotary_frequencies(0, device='cpu')[0].numel() == 0
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, factor=0.5), dict(rotary_dim=8, scaling='cubic'), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, scaling='yarn', beta_fast=1.0, beta_slow=2.0)):
        with pytest.raises(L.SgpoError):
            T.rotary_frequencies(device='cpu', **bad)


def test_library_refuses_bad_arguments_without_a_device():
    from sgpo_amd import _lib as L
    lib = L.load()

    def refused(rc, text):
        assert rc < 0 and text in lib.sgpo_last_error().decode()

    refused(lib.sgpo_rotary(None, None), 'null')
    a = L.RotaryArgs(B=1, L=2, heads_q=1, head_dim=8, rot=10)
    refused(lib.sgpo_rotary(C.byref(a), None), 'rot=10')
    a = L.RotaryArgs(B=1, L=2, heads_q=1, head_dim=8, rot=3)
    refused(lib.sgpo_rotary(C.byref(a), None), 'rot=3')
    a = L.RotaryArgs(B=1, L=2, heads_q=1, head_dim=8, rot=8, dtype=7)
    refused(lib.sgpo_rotary(C.byref(a), None), 'dtype')
    a = L.RotaryArgs(B=1, L=2, heads_q=1, head_dim=8, rot=8, q=4096, q_out=8192, q_stride=(16, 8, 8), q_out_stride=(16, 8, 8))
    refused(lib.sgpo_rotary(C.byref(a), None), 'frequencies')
    a = L.RotaryArgs(B=1 << 16, L=1 << 16, heads_q=1, head_dim=8, rot=0)
    refused(lib.sgpo_rotary(C.byref(a), None), 'tokens')
    a = L.RotaryArgs(B=1, L=2, heads_q=1, head_dim=8, rot=0)
    refused(lib.sgpo_rotary(C.byref(a), None), 'null')
    a = L.RotaryArgs(B=0, L=2, heads_q=1, head_dim=8, rot=8)
    assert lib.sgpo_rotary(C.byref(a), None) == 0                # nothing to do

    def loss(**kw):
        v = dict(N=4, H=8, V=5, ld_hidden=8, ld_weight=8, reduction=1)
        v.update(kw)
        return C.byref(L.LinearCeArgs(**v))

    for kw, text in ((dict(H=0), 'sizes'), (dict(V=0), 'sizes'), (dict(N=-1), 'sizes'), (dict(dtype=3), 'dtype'), (dict(reduction=4), 'reduction'),
                     (dict(ld_hidden=7), 'pitch'), (dict(ld_weight=1 << 22), 'pitch')):
        refused(lib.sgpo_linear_ce_forward(loss(**kw), None, None, None, None, None, 0, None), text)
        refused(lib.sgpo_linear_ce_backward(loss(**kw), None, None, None, None, None, None, None, 0, None), text)
        assert lib.sgpo_linear_ce_workspace_bytes(loss(**kw), 1) == 0
    refused(lib.sgpo_linear_ce_forward(loss(), None, None, None, None, None, 0, None), 'null')
    one = C.c_void_p(4096)                                       # never read: the workspace is refused first
    refused(lib.sgpo_linear_ce_forward(C.byref(L.LinearCeArgs(hidden=4096, weight=4096, targets=4096, N=4, H=8, V=500, ld_hidden=8, ld_weight=8)),
                                       one, one, one, one, one, 16, None), 'workspace')
    odd = C.c_void_p(4096 + 128)
    big = L.LinearCeArgs(hidden=1 << 30, weight=1 << 31, targets=4096, N=4, H=8, V=500, ld_hidden=8, ld_weight=8)
    refused(lib.sgpo_linear_ce_forward(C.byref(big), one, one, one, one, odd, 1 << 40, None), 'aligned')
    refused(lib.sgpo_linear_ce_backward(C.byref(big), one, one, one, None, None, one, odd, 1 << 40, None), 'aligned')
    coef = (C.c_float * 3)(1, 0, 0)
    refused(lib.sgpo_newton_schulz(one, 0, 1, 400, 4, 1600, 4, coef, 1, 1e-7, one, odd, 1 << 30, None), 'aligned')
    refused(lib.sgpo_muon_step(one, 0, one, 0, one, 1, 400, 4, 0.1, 0.9, 1, 0.0, coef, 1, 1e-7, odd, 1 << 30, None), 'aligned')
    refused(lib.sgpo_newton_schulz(one, 0, 1, 4, 4, 16, 4, coef, 0, 1e-7, one, one, 1 << 30, None), 'triples')
    refused(lib.sgpo_newton_schulz(one, 5, 1, 4, 4, 16, 4, coef, 1, 1e-7, one, one, 1 << 30, None), 'dtype')
    refused(lib.sgpo_newton_schulz(one, 0, 1, 4, 4, 16, 3, coef, 1, 1e-7, one, one, 1 << 30, None), 'pitch')
    refused(lib.sgpo_newton_schulz(one, 0, 1, 400, 4, 1600, 4, coef, 1, 1e-7, one, one, 16, None), 'workspace')
    refused(lib.sgpo_newton_schulz(one, 0, 1, -4, 4, 16, 4, coef, 1, 1e-7, one, one, 16, None), 'negative')
    refused(lib.sgpo_muon_step(one, 0, one, 9, one, 1, 4, 4, 0.1, 0.9, 1, 0.0, coef, 1, 1e-7, one, 1 << 30, None), 'dtype')
    refused(lib.sgpo_muon_step(one, 0, None, 0, one, 1, 4, 4, 0.1, 0.9, 1, 0.0, coef, 1, 1e-7, one, 1 << 30, None), 'null')
    refused(lib.sgpo_newton_schulz(one, 0, 1, 4, (1 << 22) + 1, 1 << 24, 1 << 23, coef, 1, 1e-7, one, one, 1 << 60, None), 'at most')
    refused(lib.sgpo_newton_schulz(one, 0, 1, (1 << 22) + 1, 4, 1 << 26, 4, coef, 1, 1e-7, one, one, 1 << 60, None), 'at most')

    def at(n):
        return C.c_void_p(4096 + n)

    # what a call writes overlaps what it reads: 2 matrices of 4 x 6, fp32 (192 bytes) or bf16 (96)
    for out in (-95, 0, 191 + 64 * 4):
        refused(lib.sgpo_newton_schulz(at(0), 0, 2, 4, 6, 88, 6, coef, 1, 1e-7, at(out), one, 1 << 30, None), 'overlaps')
    for w, g, b in ((0, 191, 1000), (0, 1000, 191), (1000, 0, 95), (95, 0, 1000), (0, 0, 0)):
        refused(lib.sgpo_muon_step(at(w), 0, at(g), 1, at(b), 2, 4, 6, 0.1, 0.9, 1, 0.0, coef, 1, 1e-7, one, 1 << 30, None), 'overlap')
    ce = C.byref(L.LinearCeArgs(hidden=1 << 20, weight=1 << 21, targets=4096, N=4, H=8, V=5, ld_hidden=8, ld_weight=10))
    for dh, dw in ((1 << 20, None), (None, 1 << 20), ((1 << 20) + 127, None), ((1 << 21) - 127, None), (None, (1 << 21) + 191), (4096, 4096 + 127)):
        refused(lib.sgpo_linear_ce_backward(ce, one, one, one, dh, dw, None, one, 1 << 40, None), 'overlaps')
    assert lib.sgpo_newton_schulz(None, 0, 0, 4, 4, 16, 4, coef, 1, 1e-7, None, None, 0, None) == 0


def test_workspace_covers_every_split():
    """Sizes that grow with the problem: positive, and never above a few copies of the operands and one piece of the vocabulary."""
    from sgpo_amd import _lib as L
    lib = L.load()
    for dtype in (0, 1):
        for N, H, V in ((1, 1, 1), (7, 517, 31), (1003, 517, 50021), (8192, 2048, 131072), (200000, 512, 31)):
            a = L.LinearCeArgs(N=N, H=H, V=V, ld_hidden=H, ld_weight=H, dtype=dtype, reduction=1)
            for backward in (0, 1):
                got = lib.sgpo_linear_ce_workspace_bytes(C.byref(a), backward)
                pad = lambda n: n + 64                           # noqa: E731
                operands = 6 * (pad(N) + V) * pad(H)
                assert (0 if V <= 64 and not backward else 1) <= got <= operands + (6 * max(1 << 27, pad(N) * 1088) + 4 * 64 * (pad(N) + 1024) * pad(H) + (1 << 28)), (dtype, N, H, V, backward, got)


def test_rotation_refuses_outputs_that_overlap():
    """Views of one buffer, against the sets of places that they cover.  No call gets as far as a launch: the frequencies are missing, and
    what passes the check of the memory is refused for that."""
    from sgpo_amd import _lib as L
    lib = L.load()
    base = 1 << 40
    rng = random.Random(5)

    def places(v, B, n, H, D):
        return [v[0] + b * v[1] + i * v[2] + h * v[3] + d for b in range(B) for i in range(n) for h in range(H) for d in range(D)]

    def call(B, n, D, views, dtype=0):
        a = L.RotaryArgs(B=B, L=n, head_dim=D, rot=2, dtype=dtype)
        for name, (heads, src, dst) in zip('qk', views):
            setattr(a, 'heads_' + name, heads)
            for field, v in ((name, src), (name + '_out', dst)):
                setattr(a, field, base + v[0] * (2 if dtype else 4))
                setattr(a, field + '_stride', (C.c_int64 * 3)(*v[1:]))
        assert lib.sgpo_rotary(C.byref(a), None) < 0
        text = lib.sgpo_last_error().decode()
        assert 'overlap' in text or 'frequencies' in text, text
        return 'overlap' in text

    # a packed projection in place: (batch, token, 3, heads, 8), q and k beside each other, with as many heads or fewer
    q, k = (0, 5 * 96, 96, 8), (32, 5 * 96, 96, 8)
    assert not call(2, 5, 8, [(4, q, q), (4, k, k)])
    assert not call(2, 5, 8, [(4, q, q), (1, k, k)])
    assert not call(2, 5, 8, [(4, q, q), (1, (32, 5 * 96, 96, 12345), (32, 5 * 96, 96, 12345))])    # one head has no stride
    assert call(2, 5, 8, [(4, q, q), (4, q, q)])                                                    # twice the same heads
    assert call(2, 5, 8, [(4, q, q), (4, (31, 5 * 96, 96, 8), (31, 5 * 96, 96, 8))])
    assert call(2, 5, 8, [(4, q, (1, 5 * 96, 96, 8))])                                              # shifted by one
    assert call(2, 5, 8, [(4, (0, 0, 96, 8), (0, 0, 96, 8))])                                       # one batch for all
    assert not call(2, 5, 8, [(4, (0, 0, 96, 8), (10000, 5 * 96, 96, 8))])                          # read only: may be broadcast
    assert call(2, 5, 8, [(4, q, (10000, 5 * 96, 96, 8)), (4, k, (10032, 5 * 96, 96, 7))])
    seen = [0, 0]
    for _ in range(3000):
        B, n, D, heads = rng.randint(1, 3), rng.randint(1, 4), rng.choice([2, 3, 4]), [rng.randint(1, 3), rng.randint(0, 3)]
        steps = [rng.choice([0, D, 2 * D, 3 * D, 4 * D]) for _ in range(3)] if rng.random() < 0.3 else [n * (3 * D + 2) + rng.randint(0, 9), 3 * D + rng.randint(0, 9), D]
        if rng.random() < 0.3:
            rng.shuffle(steps)
        views = []
        for h in heads:
            src = (rng.randint(0, 60), *steps)
            views.append((h, src, src if rng.random() < 0.7 else (rng.randint(0, 400), *steps)))
        live = [(h, places(s, B, n, h, D), places(d, B, n, h, D), s == d) for h, s, d in views if h]
        shared = any(len(set(d)) < len(d) for _, _, d, _ in live)
        for i, (_, _, d, _) in enumerate(live):
            for j, (_, s2, d2, same) in enumerate(live):
                shared |= i != j and bool(set(d) & (set(d2) | set(s2)))
                shared |= i == j and not same and bool(set(d) & set(s2))
        got = call(B, n, D, views, rng.randint(0, 1))
        assert got or not shared, (B, n, D, views)
        # strides that reach over each other without a shared place are refused too: only ordinary ones are told apart exactly
        order = sorted((st, c) for st, c in ((steps[0], B), (steps[1], n), (steps[2], max(heads))) if c > 1)
        nested, span = True, D
        for st, c in order:
            nested &= st >= span
            span += (c - 1) * st
        if nested:
            assert got == shared, (B, n, D, views)
        seen[got] += 1
    assert min(seen) > 300
