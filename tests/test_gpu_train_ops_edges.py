"""GPU: the training operators at the edges of their arguments: workspaces of exactly the size asked for, tensors that are more than plain memory."""
import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
GUARD = 1 << 16


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _lib():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    T.newton_schulz(torch.zeros(1, 1, device='cuda'))         # the first call binds the process to its GPU
    return L, L.load()


class Guarded:
    """`need` bytes, 256-byte aligned, with a filled region behind them."""
    def __init__(self, need):
        self.need = need
        self.buf = torch.full((need + GUARD + 256,), 0xA5, dtype=torch.uint8, device='cuda')
        self.skip = -self.buf.data_ptr() % 256
        self.ptr = C.c_void_p(self.buf.data_ptr() + self.skip)

    def whole(self):
        return bool((self.buf[:self.skip] == 0xA5).all()) and bool((self.buf[self.skip + self.need:] == 0xA5).all())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


# heads of every number of padded workgroups, the largest that share tokens among waves; then the tiles, cut and not, in one piece and in several
SIZES = [(N, 64, V) for N in (1, 16, 17, 33, 48, 49, 64, 513, 1537, 8145, 8192, 8193) for V in (1, 31, 64)] + [
    (1, 512, 31), (17, 512, 64), (300, 517, 31), (257, 517, 1003), (130, 72, 257), (3, 2048, 20011), (2100, 33, 70), (40000, 64, 8000)]


@pytest.mark.parametrize('dtype', [F32, BF])
def test_loss_leaves_what_lies_behind_its_workspace(dtype):
    L, lib = _lib()
    g = _gen(1)
    for N, H, V in SIZES:
        h, w = torch.randn(N, H, generator=g, device='cuda').to(dtype), torch.randn(V, H, generator=g, device='cuda').to(dtype)
        b, t = torch.randn(V, generator=g, device='cuda'), torch.randint(0, V, (N,), generator=g, device='cuda')
        a = L.LinearCeArgs(hidden=h.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), targets=t.data_ptr(), ld_hidden=H, ld_weight=H, ignore_index=-100, N=N, H=H, V=V,
                           dtype=int(dtype == BF), reduction=L.REDUCE_MEAN)
        out = {k: Guarded(n * 4) for k, n in (('nll', N), ('lse', N), ('loss', 1), ('inv', 1), ('db', V))}
        out.update(dh=Guarded(N * H * h.element_size()), dw=Guarded(V * H * h.element_size()))
        up = torch.ones(1, device='cuda')
        for backward in (0, 1):
            need = lib.sgpo_linear_ce_workspace_bytes(C.byref(a), backward)
            ws = Guarded(need)
            if backward:
                rc = lib.sgpo_linear_ce_backward(C.byref(a), out['lse'].ptr, C.c_void_p(up.data_ptr()), out['inv'].ptr, out['dh'].ptr, out['dw'].ptr, out['db'].ptr, ws.ptr, need, _stream())
            else:
                rc = lib.sgpo_linear_ce_forward(C.byref(a), out['nll'].ptr, out['lse'].ptr, out['loss'].ptr, out['inv'].ptr, ws.ptr, need, _stream())
            assert rc == 0, lib.sgpo_last_error()
            torch.cuda.synchronize()
            assert ws.whole(), (N, H, V, backward)
        assert all(o.whole() for o in out.values()), (N, H, V)


@pytest.mark.parametrize('dtype', [F32, BF])
def test_updates_leave_what_lies_behind_their_workspace(dtype):
    L, lib = _lib()
    g = _gen(2)
    coef = (C.c_float * 15)(*([3.4445, -4.7750, 2.0315] * 5))
    for batch, m, n in [(1, 1, 1), (3, 64, 64), (2, 128, 100), (1, 31, 512), (3, 64, 4000), (2, 1003, 17), (1, 100, 900), (2, 150, 9000), (1, 513, 129), (3, 400, 1000),
                        (1, 1000, 1001), (1, 40000, 3), (8, 70, 5000)]:
        grad = torch.randn(batch, m, n, generator=g, device='cuda').to(dtype)
        need = lib.sgpo_newton_schulz_workspace_bytes(batch, m, n)
        x, weight, buf = Guarded(batch * m * n * 2), Guarded(batch * m * n * 4), Guarded(batch * m * n * 4)
        for o in (weight, buf):
            o.buf[o.skip:o.skip + o.need] = 0
        for step in (0, 1):
            ws = Guarded(need)
            if step:
                rc = lib.sgpo_muon_step(weight.ptr, 0, C.c_void_p(grad.data_ptr()), int(dtype == BF), buf.ptr, batch, m, n, 0.02, 0.9, 1, 0.0, coef, 5, 1e-7, ws.ptr, need, _stream())
            else:
                rc = lib.sgpo_newton_schulz(C.c_void_p(grad.data_ptr()), int(dtype == BF), batch, m, n, m * n, n, coef, 5, 1e-7, x.ptr, ws.ptr, need, _stream())
            assert rc == 0, lib.sgpo_last_error()
            torch.cuda.synchronize()
            assert ws.whole() and x.whole() and weight.whole() and buf.whole(), (batch, m, n, step)


@pytest.mark.parametrize('dtype,interleaved', [(F32, False), (BF, True)])
def test_rotation_in_forward_mode(dtype, interleaved):
    """The rotation is linear: the tangent is the rotated tangent, alone, for q and k together, over a reverse pass and under one."""
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    g = _gen(3)
    q, dq, u = (torch.randn(2, 7, 3, 16, generator=g, device='cuda').to(dtype) for _ in range(3))
    k, dk = (torch.randn(2, 7, 1, 16, generator=g, device='cuda').to(dtype) for _ in range(2))
    freq, _ = T.rotary_frequencies(8)
    pos = torch.randint(0, 100, (2, 7), generator=g, device='cuda')

    def turn(a, b, **kw):
        return T.rotary_positions(a, b, freq, pos, interleaved=interleaved, **kw)

    want, dwant = turn(q, k), turn(dq, dk)
    with fw.dual_level():
        for a, b in ((1, 1), (1, 0), (0, 1)):
            out = turn(fw.make_dual(q, dq) if a else q, fw.make_dual(k, dk) if b else k)
            for x, y, dy, has in zip(out, want, dwant, (a, b)):
                p, t = fw.unpack_dual(x)
                assert torch.equal(p, y) and (torch.equal(t, dy) if has else t is None)
        p, t = fw.unpack_dual(turn(fw.make_dual(q, dq), None)[0])
        assert torch.equal(p, want[0]) and torch.equal(t, dwant[0])
        # a tangent that is a lazy zero
        p, t = fw.unpack_dual(turn(fw.make_dual(q, torch._efficientzerotensor(q.shape, dtype=dtype, device='cuda')), None)[0])
        assert torch.equal(p, want[0]) and float(t.abs().max()) == 0.0
        # the gradient's tangent: R^T of the upstream gradient's
        leaf = q.clone().requires_grad_()
        back, = torch.autograd.grad(turn(leaf, None)[0], leaf, fw.make_dual(u, dq))
        p, t = fw.unpack_dual(back)
        leaf2 = q.clone().requires_grad_()
        y = turn(leaf2, None)[0]
        assert torch.equal(p, torch.autograd.grad(y, leaf2, u, retain_graph=True)[0]) and torch.equal(t, torch.autograd.grad(y, leaf2, dq)[0])
        # the tangent's gradient
        leaf = dq.clone().requires_grad_()
        t = fw.unpack_dual(turn(fw.make_dual(q, leaf), None)[0]).tangent
        got, = torch.autograd.grad(t, leaf, u)
        assert torch.equal(got, p)
        # a leaf of both modes
        leaf = q.clone().requires_grad_()
        x, t = fw.unpack_dual(turn(fw.make_dual(leaf, dq), None)[0])
        assert torch.equal(t, dwant[0]) and torch.equal(torch.autograd.grad(x, leaf, u)[0], p)
        # the loss's gradient has none
        h, w = torch.randn(4, 8, generator=g, device='cuda', requires_grad=True), torch.randn(9, 8, generator=g, device='cuda')
        loss = T.linear_cross_entropy(h, w, torch.zeros(4, dtype=torch.int64, device='cuda'))
        with pytest.raises((L.SgpoError, RuntimeError), match='forward-mode'):
            torch.autograd.grad(loss, h, fw.make_dual(torch.ones((), device='cuda'), torch.ones((), device='cuda')))


def test_lazily_negated_views():
    """Refused as inputs; gradients that autograd hands over so are read with their sign."""
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    g = _gen(4)
    neg = torch._neg_view
    q, u = (torch.randn(2, 5, 3, 16, generator=g, device='cuda') for _ in range(2))
    freq, _ = T.rotary_frequencies(8)
    h, w, b = (torch.randn(s, generator=g, device='cuda') for s in ((6, 16), (9, 16), (9,)))
    t = torch.randint(0, 9, (6,), generator=g, device='cuda')
    for call in (lambda: T.rotary_positions(q, neg(q), freq), lambda: T.rotary_positions(q, None, neg(freq)), lambda: T.rotary_positions_(q, neg(q), freq),
                 lambda: T.linear_cross_entropy(neg(h), w, t), lambda: T.linear_cross_entropy(h, neg(w), t), lambda: T.linear_cross_entropy(h, w, t, neg(b)),
                 lambda: T.newton_schulz(neg(w)), lambda: T.muon_step(neg(w), w, w.clone(), 0.1), lambda: T.muon_step(w, neg(h), w.clone(), 0.1),
                 lambda: T.muon_step(w, h, neg(w), 0.1)):
        with pytest.raises(L.SgpoError, match='negated'):
            call()
    leaf = q.clone().requires_grad_()
    y, k = T.rotary_positions(leaf, leaf, freq)
    assert torch.equal(torch.autograd.grad((y, k), leaf, (neg(u), u), retain_graph=True)[0], torch.autograd.grad((y, k), leaf, (-u, u))[0])
    for red, up in (('none', torch.rand(6, generator=g, device='cuda')), ('mean', torch.rand((), generator=g, device='cuda'))):
        leaves = [x.clone().requires_grad_() for x in (h, w, b)]
        loss = T.linear_cross_entropy(*leaves[:2], t, leaves[2], reduction=red)
        got, want = (torch.autograd.grad(loss, leaves, x, retain_graph=True) for x in (neg(up), -up))
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize('dtype', [F32, BF])
@pytest.mark.parametrize('N,H,V', [(100, 64, 31), (9000, 40, 31), (130, 72, 257), (1000, 96, 3000)])
def test_an_infinite_upstream_gradient_does_not_reach_ignored_tokens(N, H, V, dtype):
    """As a loss scale that overflowed hands over: an ignored token's gradient is 0 all the same, and every gradient is if no token has a loss."""
    from sgpo_amd import train_ops as T
    g = _gen(5)
    h, w = torch.randn(N, H, generator=g, device='cuda').to(dtype).requires_grad_(), torch.randn(V, H, generator=g, device='cuda').to(dtype).requires_grad_()
    b = torch.zeros(V, device='cuda', requires_grad=True)
    t = torch.randint(0, V, (N,), generator=g, device='cuda')
    drop = torch.rand(N, generator=g, device='cuda') < 0.3
    t[drop] = -100
    for up in (math.inf, math.nan):
        for red in ('mean', 'sum', 'none'):
            out = T.linear_cross_entropy(h, w, t, b, reduction=red)
            dh, dw, db = torch.autograd.grad(out, (h, w, b), torch.full_like(out, up))
            assert bool((dh[drop] == 0).all()), (up, red)
            assert not bool(dh[~drop].isfinite().any()) and not bool(dw.isfinite().any()) and not bool(db.isfinite().any()), (up, red)
            out = T.linear_cross_entropy(h, w, torch.full_like(t, -100), b, reduction=red)
            assert all(bool((x == 0).all()) for x in torch.autograd.grad(out, (h, w, b), torch.full_like(out, up))), (up, red)


@pytest.mark.parametrize('V', [31, 300])
def test_head_whose_bias_has_the_weights_type(V):
    """A linear layer in bf16 as it is: the bias is read as it stands (bf16 values are fp32 values), and its gradient rounded once."""
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    g = _gen(6)
    head = torch.nn.Linear(64, V, dtype=BF, device='cuda')
    h, t = torch.randn(50, 64, generator=g, device='cuda').to(BF), torch.randint(0, V - 1, (50,), generator=g, device='cuda')
    with torch.no_grad():
        head.bias[V - 1] = -math.inf
    T.linear_cross_entropy(h, head.weight, t, head.bias).backward()
    w, b = head.weight.detach().requires_grad_(), head.bias.detach().float().requires_grad_()
    want = torch.autograd.grad(T.linear_cross_entropy(h, w, t, b), (w, b))
    assert torch.equal(head.weight.grad, want[0]) and head.bias.grad.dtype == BF and torch.equal(head.bias.grad, want[1].to(BF))
    for bad in (head.bias.detach().half(), head.bias.detach().double()):
        with pytest.raises(L.SgpoError, match='bias'):
            T.linear_cross_entropy(h, head.weight, t, bad)
    with pytest.raises(L.SgpoError, match='bias'):
        T.linear_cross_entropy(h.float(), head.weight.float(), t, head.bias)


@pytest.mark.parametrize('shape', [(31, 128), (64, 300), (20, 90), (500, 48)])
def test_low_rank_updates_of_few_rows_or_columns_stay_in_32_bits(shape):
    """Updates of five directions whose iteration runs on d x d matrices, seen through an fp32 weight that takes them unrounded.  X_0 has norm 1 and is rounded by
    2^-24; a product adds d terms, each sum rounded by 2^-24 / sqrt(3) with a random sign; what the five triples leave outside of the five directions
    grows by 3.4445^5 = 485 at most: 5 x 485 x 2^-24 sqrt(d / 3), 3.7e-4 to 6.7e-4 of a result of norm 2.  (With Q mirrored from one triangle, instead of
    multiplied whole, the same arithmetic on the CPU is off by 6e-4 to 3e-3; whole, by 2e-5 to 9e-5.)"""
    from sgpo_amd import train_ops as T
    g = _gen(7)
    m, n = shape
    u = torch.randn(m, 5, generator=g, device='cuda') @ torch.randn(5, n, generator=g, device='cuda')
    u[::7] = 0
    for x in (u, u * torch.logspace(0, -3, m, device='cuda')[:, None], u.to(BF)):
        want = x.double() / (x.double().norm() + 1e-7)
        for _ in range(5):
            a, b, c = T.NS_COEFFICIENTS
            gram = want @ want.T if m < n else want.T @ want
            p = b * gram + c * gram @ gram
            want = a * want + (p @ want if m < n else want @ p)
        w = torch.zeros(shape, device='cuda')
        T.muon_step(w, x, torch.zeros(shape, device='cuda'), lr=1 / math.sqrt(max(1, m / n)), momentum=0.0, nesterov=False)
        assert float((w.double() + want).norm()) <= 5 * 485 * 2.0 ** -24 * math.sqrt(min(m, n) / 3) + 4 * 2.0 ** -24 * float(want.norm())


def _pi(bits):
    """pi 2^bits as a whole number, by Machin's formula."""
    def inverse_arctan(n):
        total, term, k = 0, (1 << bits + 32) // n, 0
        while term:
            total += -(term // (2 * k + 1)) if k & 1 else term // (2 * k + 1)
            term //= n * n
            k += 1
        return total
    return 4 * (4 * inverse_arctan(5) - inverse_arctan(239)) >> 32


def test_rotation_angles_against_whole_number_arithmetic():
    """Angles whose product is not rounded: a frequency is a whole number of 2^-e, the angle's rest after whole turns is formed in whole numbers.  The kernel's
    is off by the product's rounding, 2^-53 of the angle, besides 10 units of fp32 (angle rounded within half a turn, sin, cos, products and sum)."""
    from fractions import Fraction
    from sgpo_amd import train_ops as T
    g = _gen(8)
    rot, places = 16, 1 << 160
    freq, _ = T.rotary_frequencies(rot)
    pos = [0, 1, 4095, (1 << 22) + 1, (1 << 29) - 1, (1 << 31) + 7, 123456789012, (1 << 40) - 3, (1 << 50) - 1, -(1 << 30) - 1]
    q = torch.randn(1, len(pos), 2, rot, generator=g, device='cuda')
    got = T.rotary_positions(q, None, freq, torch.tensor(pos, device='cuda'))[0].double().cpu()
    q = q.double().cpu()
    turn = Fraction(2 * _pi(160), places)
    for i, p in enumerate(pos):
        for j, f in enumerate(freq.tolist()):
            angle = p * Fraction(f)
            rest = angle - round(angle / turn) * turn
            c, s = math.cos(rest), math.sin(rest)
            a, b = q[0, i, :, j], q[0, i, :, j + rot // 2]
            tol = (10 * 2.0 ** -24 + abs(float(angle)) * 2.0 ** -53) * (a.abs() + b.abs())
            assert bool(((got[0, i, :, j] - (a * c - b * s)).abs() <= tol).all()) and bool(((got[0, i, :, j + rot // 2] - (a * s + b * c)).abs() <= tol).all()), (p, j)


def test_hooks_and_checkpoints():
    """What autograd lets a program do around a call: tensors saved on the host between the passes (where they lose their strides), gradients changed by hooks,
    the forward pass run again in the backward pass."""
    from torch.utils.checkpoint import checkpoint
    from sgpo_amd import train_ops as T
    g = _gen(9)
    wide = torch.randn(300, 72, generator=g, device='cuda').to(BF)
    h, w = wide[:200, :64], wide[200:, 8:]
    b, t = torch.randn(100, generator=g, device='cuda'), torch.randint(0, 100, (200,), generator=g, device='cuda')
    qkv = torch.randn(2, 9, 3, 4, 16, generator=g, device='cuda')
    freq, _ = T.rotary_frequencies(16)

    def loss(hh, ww, bb):
        return T.linear_cross_entropy(hh, ww, t, bb)

    def turned(x):
        q, k = T.rotary_positions(x[:, :, 0], x[:, :, 1], freq)
        return (q * k).sum()

    for call, args in ((loss, (h, w, b)), (turned, (qkv,))):
        leaves = [x.detach().requires_grad_() for x in args]
        want = torch.autograd.grad(call(*leaves), leaves)
        with torch.autograd.graph.save_on_cpu():
            out = call(*leaves)
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(out, leaves), want))
        assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(checkpoint(call, *leaves, use_reentrant=False), leaves), want))
        out = call(*leaves)
        seen = []
        leaves[0].register_hook(lambda x: seen.append(x) or -x)
        out.register_hook(lambda x: x * 2)
        got = torch.autograd.grad(out, leaves)
        assert len(seen) == 1 and bool((got[0] == -seen[0]).all())
        for x, y in zip(got, want):             # twice the gradient, exactly: a factor of 2 rounds nothing
            assert torch.equal(x.abs(), (2 * y).abs())
