"""GPU: the training operators against their definitions in 64 bits, gradients also against differences, through the public calls.

Tolerances are worst cases by arithmetic, written beside each: a rounding is off by at most half a step (fp32 2^-24, bf16 2^-8 of the value), a
sum of n products in fp32 by n 2^-24 of the sum of their sizes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32, UBF = 2.0 ** -24, 2.0 ** -8
STEP = {torch.float32: U32, torch.bfloat16: UBF}
BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), f'{what}: {float((got - want).abs().max()):.3g} off, {int((off > 0).sum())} of {off.numel()} values over tolerance'


# ---------------------------------------------------------------------------------------------------------------- rotation

def _turn64(x, pos, freq, scale, interleaved, inverse=False):
    rot = 2 * freq.numel()
    ang = pos.double()[..., None] * freq
    cos, sin = ang.cos()[:, :, None] * scale, ang.sin()[:, :, None] * scale * (-1 if inverse else 1)
    y = x.double().clone()
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    y[..., a], y[..., b] = x[..., a].double() * cos - x[..., b].double() * sin, x[..., a].double() * sin + x[..., b].double() * cos
    return y


def _turn_tol(x, want, freq, scale, interleaved):
    # angle: rounded to fp32 within half a turn, pi 2^-24 (rounded up to 4 u); sin and cos 2 u each; their product with scale u; two products and a sum
    # 2 u: under 10 u (|a| + |b|) scale, and the output's own rounding
    rot = 2 * freq.numel()
    s = torch.zeros_like(want)
    i = torch.arange(rot // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    both = x[..., a].double().abs() + x[..., b].double().abs()
    s[..., a], s[..., b] = both, both
    return 10 * U32 * scale * s + (STEP[x.dtype] * want.abs() if x.dtype == BF else 0)


ROTARY = [
    # B, L, Hq, Hk, D, rot, dtype, interleaved, layout, positions
    (1, 1, 1, 1, 2, 2, F32, False, 'plain', None),
    (3, 1, 8, 8, 64, 64, BF, False, 'plain', 'far'),
    (2, 119, 8, 8, 64, 64, BF, False, 'packed', None),
    (2, 119, 8, 8, 64, 64, BF, True, 'packed', 'ragged'),
    (2, 37, 6, 2, 80, 40, F32, False, 'plain', 'ragged'),
    (2, 37, 6, 2, 80, 40, BF, False, 'heads_first', 'row'),
    (1, 515, 4, 1, 128, 64, BF, True, 'heads_first', None),
    (2, 33, 3, 3, 66, 62, BF, False, 'plain', 'one'),
    (2, 33, 3, 3, 66, 62, F32, True, 'odd', 'ragged'),
    (2, 33, 3, 1, 15, 6, BF, True, 'odd', 'ragged'),
    (2, 33, 3, 1, 15, 6, F32, False, 'odd', 'negative'),
    (5, 2000, 2, 2, 256, 256, F32, False, 'plain', 'huge'),
    (2, 9, 2, 2, 64, 0, BF, False, 'plain', None),
    (2, 9, 5, 0, 64, 16, BF, False, 'plain', None),
    # the last run of a part shorter than the others: 31 pairs and 2 copied, 3 and 60, 13 and 7, odd heads
    (2, 37, 3, 1, 64, 62, BF, False, 'plain', 'ragged'),
    (2, 37, 3, 1, 66, 6, F32, False, 'heads_first', None),
    (3, 50, 2, 2, 33, 26, BF, True, 'plain', 'ragged'),
    (3, 50, 2, 2, 33, 26, F32, False, 'plain', 'row'),
    (2, 119, 8, 8, 64, 62, BF, False, 'packed', None),
]


@pytest.mark.parametrize('B,L,Hq,Hk,D,rot,dtype,interleaved,layout,positions', ROTARY)
def test_rotation_and_its_gradient(B, L, Hq, Hk, D, rot, dtype, interleaved, layout, positions):
    from sgpo_amd import train_ops as T
    g = _gen(B * 1000 + L)
    freq, scale = T.rotary_frequencies(rot, scaling='yarn' if interleaved else None, factor=8.0 if interleaved else 1.0)

    def make(H):
        if layout == 'packed':
            return torch.randn(B, L, 3, H, D, generator=g, device='cuda').to(dtype)
        if layout == 'heads_first':
            return torch.randn(B, H, L, D, generator=g, device='cuda').to(dtype).transpose(1, 2)
        if layout == 'odd':         # a view at an odd offset with an odd pitch
            return torch.randn(B, L, H, D + 3, generator=g, device='cuda').to(dtype)[..., 1:D + 1]
        return torch.randn(B, L, H, D, generator=g, device='cuda').to(dtype)

    if layout == 'packed':
        qkv = make(Hq)
        q, k = qkv[:, :, 0], qkv[:, :, 1]
    else:
        q, k = make(Hq), make(Hk) if Hk else None
    steps = torch.arange(L, device='cuda')
    pos = {None: None, 'row': steps + 7, 'one': (steps * 3)[None], 'ragged': torch.randint(0, 5000, (B, 1), generator=g, device='cuda') + steps,
           'far': torch.randint(0, 1 << 22, (B, L), generator=g, device='cuda'), 'negative': (steps - 1000).expand(B, L),
           'huge': torch.randint(1 << 31, 1 << 40, (B, L), generator=g, device='cuda')}[positions]
    pos64 = (steps if pos is None else pos).expand(B, L)
    was = [x.clone() if x is not None else None for x in (q, k)]
    leaves = [x.detach().requires_grad_() if x is not None else None for x in (q, k)]
    out = T.rotary_positions(*leaves, freq, pos, interleaved=interleaved, scale=scale)
    for name, x, y in (('q', q, out[0]), ('k', k, out[1])):
        if x is None:
            assert y is None
            continue
        want = _turn64(x, pos64, freq, scale, interleaved)
        _within(y.detach(), want, _turn_tol(x, want, freq, scale, interleaved), name)
        assert y.dtype == dtype and torch.equal(y[..., rot:], x[..., rot:])
    live = [(x, y) for x, y in zip(leaves, out) if x is not None]
    ups = [torch.randn(y.shape, generator=g, device='cuda').to(dtype) for _, y in live]
    grads = torch.autograd.grad([y for _, y in live], [x for x, _ in live], ups)
    for u, dx in zip(ups, grads):
        want = _turn64(u, pos64, freq, scale, interleaved, inverse=True)
        _within(dx, want, _turn_tol(u, want, freq, scale, interleaved), 'gradient')
    assert torch.equal(q, was[0]) and (k is None or torch.equal(k, was[1]))      # inputs are left as they were


def test_rotation_in_place_touches_nothing_else():
    from sgpo_amd import train_ops as T
    qkv = torch.randn(3, 50, 3, 4, 64, generator=_gen(5), device='cuda').to(BF)
    was = qkv.clone()
    freq, _ = T.rotary_frequencies(32)
    want = T.rotary_positions(qkv[:, :, 0], qkv[:, :, 1], freq)
    T.rotary_positions_(qkv[:, :, 0], qkv[:, :, 1], freq)
    assert torch.equal(qkv[:, :, 0], want[0]) and torch.equal(qkv[:, :, 1], want[1]) and torch.equal(qkv[:, :, 2], was[:, :, 2])


def test_rotation_offsets_beyond_32_bits():
    from sgpo_amd import train_ops as T
    x = torch.zeros(1, 70000, 1, 32768, dtype=BF, device='cuda').view(1, 70000, 256, 128)      # 2.3e9 elements
    x[0, -1, -1] = 1.0
    freq, _ = T.rotary_frequencies(128)
    T.rotary_positions_(x[:, 69000:], None, freq, torch.arange(69000, 70000, device='cuda'))
    one = torch.ones(1, 1, 1, 128, dtype=BF, device='cuda')
    assert torch.equal(x[0, -1, -1], T.rotary_positions(one, None, freq, torch.tensor([69999], device='cuda'))[0][0, 0, 0])
    T.rotary_positions_(x, None, freq)
    assert float(x[0, -1, -1].float().norm()) > 10.0 and float(x[0, :-1].abs().max()) == 0.0
    del x
    torch.cuda.empty_cache()


def test_rotation_of_nothing_and_refusals():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    freq, _ = T.rotary_frequencies(8)
    for shape in ((0, 5, 2, 8), (3, 0, 2, 8), (3, 5, 0, 8)):
        x = torch.zeros(shape, device='cuda', requires_grad=True)
        y, none = T.rotary_positions(x, None, freq)
        assert y.shape == x.shape and none is None
    q = torch.zeros(2, 5, 2, 8, device='cuda')
    for bad in (lambda: T.rotary_positions(q.half(), None, freq), lambda: T.rotary_positions(q, q.to(BF), freq), lambda: T.rotary_positions(q[0], None, freq),
                lambda: T.rotary_positions(q, None, freq.float()), lambda: T.rotary_positions(q, None, freq, torch.zeros(4, dtype=torch.int64, device='cuda')),
                lambda: T.rotary_positions(q, None, freq, torch.zeros(5, dtype=torch.int32, device='cuda')),
                lambda: T.rotary_positions(q[..., :4], None, freq), lambda: T.rotary_positions(q, q[:1], freq),
                lambda: T.rotary_positions(q, None, freq, torch.zeros(5, dtype=torch.int64)),
                lambda: T.rotary_positions_(q[..., ::2], None, freq[:2]), lambda: T.rotary_positions_(q[:1].expand(2, 5, 2, 8), None, freq),
                lambda: T.rotary_positions_(q.clone().requires_grad_(), None, freq), lambda: T.rotary_positions_(q, q, freq),
                lambda: T.rotary_positions_(q[:, :4], q[:, 1:], freq), lambda: T.rotary_positions(torch._neg_view(q), None, freq)):
        with pytest.raises(L.SgpoError):
            bad()


# -------------------------------------------------------------------------------------------------------------------- loss

def _loss64(h, w, t, b, ignore, g):
    """(nll, lse, p - onehot scaled by g, |z| sizes) in 64 bits; g (N,) the factor on each token's loss."""
    h, w = h.double(), w.double()
    keep = t != ignore
    h = torch.where(keep[:, None], h, 0.0)
    z = h @ w.T + (0 if b is None else b.double())
    lse = torch.logsumexp(z, 1)
    tt = t.clamp(0, w.shape[0] - 1)
    nll = torch.where(keep, lse - z.gather(1, tt[:, None])[:, 0], 0.0)
    p = torch.softmax(z, 1)
    d = p.clone()
    d[torch.arange(len(t), device=t.device), tt] -= 1.0
    d = torch.where(keep[:, None], d * g[:, None], 0.0)
    p = torch.where(keep[:, None], p * g[:, None].abs(), 0.0)
    size = h.abs() @ w.abs().T
    return nll, lse, z, d, p, size, h, w


def _check_loss(N, H, V, dtype, bias, closed, ignored, reduction, seed, strided=False, scale=1.0):
    from sgpo_amd import train_ops as T
    g = _gen(seed)
    pitch = H + 8 if strided else H
    h = (torch.randn(N, pitch, generator=g, device='cuda') * scale).to(dtype)[:, :H]
    w = (torch.randn(V, pitch, generator=g, device='cuda') * H ** -0.5).to(dtype)[:, :H]
    b = torch.randn(V, generator=g, device='cuda') * 0.5 if bias else None
    t = torch.randint(0, V - 1 if closed else V, (N,), generator=g, device='cuda')
    if closed:
        b[V - 1] = -math.inf
    drop = torch.rand(N, generator=g, device='cuda') < ignored
    t = torch.where(drop, -100, t)
    if ignored:                                     # what an ignored token holds does not matter
        h[drop] = float('nan')
    hl, wl = h.detach().requires_grad_(), w.detach().requires_grad_()
    bl = None if b is None else b.detach().requires_grad_()
    out = T.linear_cross_entropy(hl, wl, t, bl, reduction=reduction)
    kept = int((t != -100).sum())
    up = torch.rand(N, generator=g, device='cuda') if reduction == 'none' else torch.tensor(1.5, device='cuda')
    f = up.double() if reduction == 'none' else torch.full((N,), 1.5 / (max(kept, 1) if reduction == 'mean' else 1), dtype=torch.float64, device='cuda')
    nll, lse, z, d, p, size, h64, w64 = _loss64(h, w, t, b, -100, f)
    # a logit: H products summed in fp32 (three planes: 3 more units of 2^-24 per product), the bias added
    zt = (H + 4) * U32 * size + U32 * torch.where(z.isfinite(), z.abs(), 0.0)
    zmax = zt.max(1).values
    # lse: the worst logit's error, V exponentials summed pairwise in tiles and joined in a chain (under 40 + V / 64 additions), exp2's own 2 u and its
    # argument's 3 u |z - max| (counted with 32, beyond which a term is below 2^-46), log and the last addition 2 u |lse|
    rel = (40 + V / 64 + 2 + 3 * 32) * U32
    nt = torch.where(t != -100, 2 * zmax + rel + 4 * U32 * (lse.abs() + 1), 0.0)
    leaves = [x for x in (hl, wl, bl) if x is not None]
    if reduction == 'none':
        _within(out.detach(), nll, nt, 'nll')
    else:
        div = max(kept, 1) if reduction == 'mean' else 1
        _within(out.detach(), nll.sum() / div, nt.sum() / div + U32 * (nll.sum() / div).abs(), 'loss')
    grads = torch.autograd.grad(out, leaves, up)
    # d: p's relative error is twice the logits' plus rel; factor and product 3 u; the rounding to the operands' planes (2^-8, or 2^-26 and counted
    # as 2^-24); differences p - 1 are rounded once more
    own = UBF if dtype == BF else U32
    # a single p is off by exp2's argument too, 3 u |z - lse| of it, and below 2^-126 it may be 0
    pt = p * ((2 * zmax + rel)[:, None] + 3 * U32 * torch.where(z.isfinite(), (z - lse[:, None]).abs(), 0.0)) + 2.0 ** -126
    dt = pt + (own + 4 * U32) * d.abs()
    ht = dt @ w64.abs() + (V + 4) * U32 * (d.abs() @ w64.abs()) + STEP[dtype] * (d @ w64).abs()
    wt = dt.T @ h64.abs() + (N + 4) * U32 * (d.abs().T @ h64.abs()) + STEP[dtype] * (d.T @ h64).abs()
    _within(grads[0], d @ w64, ht * (1 + STEP[dtype]), 'dhidden')
    _within(grads[1], d.T @ h64, wt * (1 + STEP[dtype]), 'dweight')
    if b is not None:
        bt = pt.sum(0) + (N + 8) * U32 * d.abs().sum(0)
        _within(grads[2], d.sum(0), bt, 'dbias')
    assert bool((grads[0][drop] == 0).all())
    # no_grad gives the same bits, and again the same
    with torch.no_grad():
        assert torch.equal(T.linear_cross_entropy(h, w, t, b, reduction=reduction), out)
    again = torch.autograd.grad(T.linear_cross_entropy(hl, wl, t, bl, reduction=reduction), leaves, up)
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


LOSS = [
    # N, H, V, bias, closed, ignored, reduction
    (1, 1, 1, False, False, 0.0, 'mean'),
    (1, 512, 31, True, True, 0.0, 'none'),
    (119, 512, 31, True, True, 0.0, 'none'),
    (300, 512, 31, True, True, 0.6, 'mean'),
    (65, 64, 26, True, False, 0.2, 'sum'),
    (257, 517, 1003, False, False, 0.1, 'mean'),
    (130, 72, 257, True, True, 0.3, 'none'),
    (1000, 128, 5000, True, False, 0.15, 'mean'),
    (3, 2048, 20011, False, False, 0.0, 'mean'),
    (2100, 33, 70, True, True, 0.5, 'sum'),
    (300, 517, 31, True, True, 0.2, 'none'),
    (9001, 75, 31, True, False, 0.3, 'mean'),
    (70, 7, 64, False, False, 0.0, 'sum'),
]


@pytest.mark.parametrize('dtype', [F32, BF])
@pytest.mark.parametrize('N,H,V,bias,closed,ignored,reduction', LOSS)
def test_loss_and_gradients(N, H, V, bias, closed, ignored, reduction, dtype):
    _check_loss(N, H, V, dtype, bias, closed, ignored, reduction, seed=N + V)


@pytest.mark.parametrize('dtype', [F32, BF])
def test_loss_of_strided_rows_and_large_logits(dtype):
    _check_loss(200, 128, 300, dtype, True, True, 0.2, 'mean', seed=3, strided=True)
    _check_loss(100, 100, 300, dtype, True, False, 0.2, 'none', seed=4, strided=True, scale=60.0)


def test_loss_in_several_pieces_and_tile_sizes():
    # 40000 tokens: pieces of 3355 -> 3328 classes, so 3 of 8000; the largest tiles
    _check_loss(40000, 64, 8000, BF, True, True, 0.4, 'mean', seed=9)
    _check_loss(9000, 96, 20000, F32, True, False, 0.4, 'mean', seed=10)


def test_loss_of_more_tokens_than_a_tile_of_transposed_features_reaches():
    # 256 rows of 8421600 bf16 tokens are over 2^32 bytes.  All but a few tokens are ignored, so that the sums stay short; those few are everywhere.
    from sgpo_amd import train_ops as T
    g = _gen(13)
    N, H, V = 8421600, 64, 70
    h = torch.randn(N, H, generator=g, device='cuda').to(BF).requires_grad_()
    w = (torch.randn(V, H, generator=g, device='cuda') * H ** -0.5).to(BF).requires_grad_()
    at = torch.cat([torch.randint(0, N, (500,), generator=g, device='cuda'), torch.tensor([0, N - 1], device='cuda')]).unique()
    t = torch.full((N,), -100, device='cuda')
    t[at] = torch.randint(0, V, (len(at),), generator=g, device='cuda')
    out = T.linear_cross_entropy(h, w, t)
    dh, dw = torch.autograd.grad(out, (h, w))
    few = h.detach()[at].requires_grad_()
    want = T.linear_cross_entropy(few, w, t[at])              # checked above against 64 bits
    fh, fw = torch.autograd.grad(want, (few, w))
    _within(out.detach(), want.detach(), 2 * U32 * want.detach().double(), 'loss')      # the same losses, summed in 64 bits
    # the same d; its products' sums in another order, and each side's own rounding to bf16
    z = few.detach().double() @ w.detach().double().T
    d = (torch.softmax(z, 1) + torch.nn.functional.one_hot(t[at], V)) / len(at) * (1 + 2 ** -6)
    _within(dh[at], fh, 2 * V * U32 * (d @ w.detach().double().abs()) + 2.01 * UBF * fh.double().abs(), 'dhidden')
    _within(dw, fw, 2 * (len(at) + 70) * U32 * (d.T @ few.detach().double().abs()) + 2.01 * UBF * fw.double().abs(), 'dweight')
    dh[at] = 0
    assert int(dh.count_nonzero()) == 0
    del h, dh
    torch.cuda.empty_cache()


def test_loss_of_rows_far_apart():
    from sgpo_amd import train_ops as T
    g = _gen(14)
    far = torch.randn(3, 1 << 22, generator=g, device='cuda')
    h, w = far[:, 5:69], torch.randn(40, 64, generator=g, device='cuda')
    t = torch.tensor([1, 2, 39], device='cuda')
    assert torch.equal(T.linear_cross_entropy(h, w, t), T.linear_cross_entropy(h.clone(), w, t))


def test_loss_gradient_against_differences():
    from sgpo_amd import train_ops as T
    g = _gen(11)
    N, H, V = 40, 24, 50
    h, w = torch.randn(N, H, generator=g, device='cuda'), torch.randn(V, H, generator=g, device='cuda') * 0.3
    b = torch.randn(V, generator=g, device='cuda')
    t = torch.randint(0, V, (N,), generator=g, device='cuda')
    leaves = [x.requires_grad_() for x in (h, w, b)]
    grads = torch.autograd.grad(T.linear_cross_entropy(h, w, t, b, reduction='sum'), leaves)
    for i, x in enumerate(leaves):
        e = torch.randn(x.shape, generator=g, device='cuda')
        step = 2.0 ** -7
        with torch.no_grad():
            args = [[y + s * e if j == i else y for j, y in enumerate((h, w, b))] for s in (step, -step)]
            hi, lo = (T.linear_cross_entropy(a[0], a[1], t, a[2], reduction='none').double().sum() for a in args)
        # third-order term of the difference: step^2 / 6 times a third derivative of at most N max|dz|^3; each loss is off by some 2^-20 at most
        slope = float((hi - lo) / (2 * step))
        dz = float((e.abs().max() * max(1.0, float(h.detach().abs().sum(1).max()), float(w.detach().abs().sum(1).max()))))
        want = float((grads[i].double() * e.double()).sum())
        z2 = [(e @ w.detach().T if i == 0 else h.detach() @ e.T if i == 1 else e.expand(N, V))][0]
        assert abs(slope - want) <= step ** 2 / 6 * float((2 * z2.abs().max(1).values.double() ** 3).sum()) + 2 * N * 2.0 ** -18 / (2 * step) and dz > 0


def test_loss_edges():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    g = _gen(12)
    h, w = torch.randn(6, 16, generator=g, device='cuda', requires_grad=True), torch.randn(9, 16, generator=g, device='cuda', requires_grad=True)
    none = torch.full((6,), -100, device='cuda')
    for red in ('mean', 'sum', 'none'):          # no token has a loss
        out = T.linear_cross_entropy(h, w, none, reduction=red)
        assert float(out.detach().abs().sum()) == 0.0
        assert all(float(x.abs().sum()) == 0.0 for x in torch.autograd.grad(out.sum(), (h, w)))
    for red in ('mean', 'sum', 'none'):          # no token
        for dt in (F32, BF):
            e = torch.zeros(0, 15, device='cuda', dtype=dt, requires_grad=True)
            wd = torch.ones(3, 15, device='cuda', dtype=dt, requires_grad=True)
            bb = torch.ones(3, device='cuda', requires_grad=True)
            out = T.linear_cross_entropy(e, wd, torch.zeros(0, dtype=torch.int64, device='cuda'), bb, reduction=red)
            assert out.shape == ((0,) if red == 'none' else ()) and float(out.detach().sum()) == 0.0
            got = torch.autograd.grad(out.sum(), (e, wd, bb))
            assert got[0].shape == e.shape and float(got[1].abs().sum()) == 0.0 and float(got[2].abs().sum()) == 0.0
    t = torch.tensor([0, 8, 9, -1, 1 << 40, -(1 << 40)], device='cuda')      # classes 0 and 8; the others are none
    out = T.linear_cross_entropy(h, w, t, reduction='none')
    assert out.isnan().tolist() == [False, False, True, True, True, True]
    dh = torch.autograd.grad(out.sum(), h)[0]
    assert dh.isnan().any(1).tolist() == [False, False, True, True, True, True]
    lead = T.linear_cross_entropy(h.view(2, 3, 16), w, torch.zeros(2, 3, dtype=torch.int64, device='cuda'), reduction='none')
    assert lead.shape == (2, 3)
    # a target in a closed class has an infinite loss; the others do not see the class
    b = torch.zeros(9, device='cuda')
    b[4] = -math.inf
    out = T.linear_cross_entropy(h, w, torch.tensor([4, 0, 1, 2, 3, 5], device='cuda'), b, reduction='none')
    assert out.isinf().tolist() == [True] + [False] * 5
    # a NaN feature stays in its row
    hn = h.detach().clone()
    hn[2, 3] = float('nan')
    assert T.linear_cross_entropy(hn, w, torch.zeros(6, dtype=torch.int64, device='cuda'), reduction='none').isnan().tolist() == [False, False, True, False, False, False]
    ok = torch.zeros(6, dtype=torch.int64, device='cuda')
    for bad in (lambda: T.linear_cross_entropy(h, w.to(BF), ok), lambda: T.linear_cross_entropy(h, w[:, :8], ok), lambda: T.linear_cross_entropy(h, w, ok[:5]),
                lambda: T.linear_cross_entropy(h, w, ok.int()), lambda: T.linear_cross_entropy(h, w, ok, torch.zeros(8, device='cuda')),
                lambda: T.linear_cross_entropy(h, w, ok, torch.zeros(9, device='cuda', dtype=BF)), lambda: T.linear_cross_entropy(h, w, ok, reduction='max'),
                lambda: T.linear_cross_entropy(h.half(), w.half(), ok), lambda: T.linear_cross_entropy(h, w[:0], ok), lambda: T.linear_cross_entropy(h, w, ok.cpu())):
        with pytest.raises(L.SgpoError):
            bad()


# ----------------------------------------------------------------------------------------------------------------- updates

def _schulz64(u, coefficients, eps):
    """The result in 64 bits and a bound on what iterates of two planes can be off by (Frobenius norm, first order)."""
    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.norm() + eps)
    fro, two = (lambda y: float(y.norm())), (lambda y: float(torch.linalg.matrix_norm(y, 2)))
    err = 2.0 ** -17 * fro(x)
    for a, b, c in coefficients:
        gram = x @ x.T
        p = b * gram + c * gram @ gram
        # a product of two-plane operands: pairs left out 2^-16, stored again 2^-17, sums K 2^-24 -- of the product of the norms
        unit = 2.0 ** -16 + 2.0 ** -17 + x.shape[1] * U32
        dg = unit * fro(x) ** 2
        dp = abs(b) * dg + abs(c) * (2 * dg * two(gram) + unit * fro(gram) ** 2) + 2.0 ** -16 * fro(p)
        fresh = 2.0 ** -16 * abs(a) * fro(x) + dp * two(x) + unit * fro(p) * fro(x)
        # what was off before is carried by the derivative, at most max|f'| and max|f(s) / s| over the spectrum
        s = torch.linspace(0, max(1.0, two(x)), 1000, dtype=torch.float64)
        slope = max(float((a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()), float((a + b * s ** 2 + c * s ** 4).abs().max()))
        x = a * x + p @ x
        err = err * slope + fresh
    return (x.T if tall else x), err


ORTHO = [((8, 8), F32), ((1, 1), F32), ((1, 40), BF), ((40, 1), F32), ((64, 64), F32), ((33, 65), BF), ((100, 70), F32), ((200, 130), BF), ((130, 517), F32),
         ((513, 129), BF), ((512, 2048), BF), ((1536, 512), F32), ((3, 64, 48), F32), ((2, 2, 150, 40), BF), ((3, 64, 4000), F32), ((5000, 70), BF), ((2, 150, 9000), BF),
         ((31, 512), F32), ((512, 31), BF), ((7, 200), F32), ((1, 129), BF), ((20, 65), BF), ((128, 32), F32), ((33, 128), F32), ((1003, 17), F32), ((3, 64, 129), BF), ((2, 33, 4100), F32), ((30000, 64), BF), ((3, 40000), F32)]


@pytest.mark.parametrize('shape,dtype', ORTHO)
def test_newton_schulz(shape, dtype):
    from sgpo_amd import train_ops as T
    u = (torch.randn(shape, generator=_gen(sum(shape)), device='cuda') * 1e-3).to(dtype)
    got = T.newton_schulz(u)
    assert got.dtype == BF and got.shape == u.shape
    for x, y in zip(u.reshape(-1, *shape[-2:]), got.reshape(-1, *shape[-2:])):
        want, err = _schulz64(x, [T.NS_COEFFICIENTS] * 5, 1e-7)
        off = float((y.double() - want).norm())
        assert off <= err + UBF * float(want.norm()), (off, err, float(want.norm()))
        # away from the bound, as sharp as the output's type: iterates are 2^-16 wide and random in sign
        assert off <= (UBF + 2.0 ** -9) * float(want.norm()), (off, float(want.norm()))
    assert torch.equal(got, T.newton_schulz(u))


@pytest.mark.parametrize('shape', [(40, 60), (64, 300), (700, 20), (100, 900)])
def test_newton_schulz_of_uneven_spectra_and_other_tables(shape):
    # nearly one direction; singular values over six orders; and one to nine triples, whose products grow small ones by up to 5^2 each
    from sgpo_amd import train_ops as T
    g = _gen(23)
    m, n = shape
    d = min(shape)
    noise = torch.randn(shape, generator=g, device='cuda')
    a, b = torch.randn(m, 1, generator=g, device='cuda'), torch.randn(1, n, generator=g, device='cuda')
    left, right = torch.linalg.qr(torch.randn(m, d, generator=g, device='cuda').double())[0], torch.linalg.qr(torch.randn(n, d, generator=g, device='cuda').double())[0]
    spread = (left * torch.logspace(0, -6, d, dtype=torch.float64, device='cuda')) @ right.T
    for u in (a @ b + 1e-3 * noise, spread.float()):
        for table in ([T.NS_COEFFICIENTS], [T.NS_COEFFICIENTS] * 5, [(5.0, -9.0, 4.5)] * 4, [(15 / 8, -10 / 8, 3 / 8)] * 9):
            want, err = _schulz64(u, table, 1e-7)
            off = float((T.newton_schulz(u, steps=len(table), coefficients=table).double() - want).norm())
            assert off <= err + UBF * float(want.norm()), (off, err, float(want.norm()))


@pytest.mark.parametrize('shape', [(31, 128), (64, 300), (20, 90), (500, 48), (150, 400), (60, 60)])
def test_newton_schulz_of_low_rank_updates(shape):
    # five directions, and rows of zeros: what rounding leaves in the other directions is multiplied by a^5 = 485.  X_0 of norm 1 is rounded by 2^-17, and
    # X_k, whose norm is at most a^k, again before the remaining factors a^(5 - k): 5 x 485 x 2^-17 at most, and the output's own rounding
    from sgpo_amd import train_ops as T
    g = _gen(24)
    m, n = shape
    u = torch.randn(m, 5, generator=g, device='cuda') @ torch.randn(5, n, generator=g, device='cuda')
    u[::7] = 0
    for x in (u, u * torch.logspace(0, -3, m, device='cuda')[:, None], u.to(BF)):
        want, _ = _schulz64(x, [T.NS_COEFFICIENTS] * 5, 1e-7)
        off = float((T.newton_schulz(x).double() - want).norm())
        assert off <= 5 * 485 * 2.0 ** -17 + UBF * float(want.norm()), (off, float(want.norm()))


@pytest.mark.parametrize('tall', [False, True])
def test_newton_schulz_of_the_longest_updates(tall):
    # 200 x 2^22, zero but for some columns everywhere: the others' updates are those of the small matrix that is left
    from sgpo_amd import train_ops as T
    g = _gen(22)
    n = 1 << 22
    at = torch.cat([torch.randint(0, n, (300,), generator=g, device='cuda'), torch.tensor([0, n - 1], device='cuda')]).unique()
    few = torch.randn(200, len(at), generator=g, device='cuda').to(BF)
    u = torch.zeros((n, 200) if tall else (200, n), dtype=BF, device='cuda')
    if tall:
        u[at] = few.T
    else:
        u[:, at] = few
    got = T.newton_schulz(u)
    got = got.T if tall else got
    want, err = _schulz64(few, [T.NS_COEFFICIENTS] * 5, 1e-7)
    off = float((got[:, at].double() - want).norm())
    assert off <= err + UBF * float(want.norm()) and off <= (UBF + 2.0 ** -9) * float(want.norm())
    assert int(got.count_nonzero()) == int(got[:, at].count_nonzero())
    del u, got
    torch.cuda.empty_cache()


def test_newton_schulz_properties():
    from sgpo_amd import _lib as L
    from sgpo_amd import train_ops as T
    g = _gen(21)
    u = torch.randn(96, 160, generator=g, device='cuda')
    s = torch.linalg.svdvals(T.newton_schulz(u).float())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3           # the polynomial's own range over this spectrum
    # independent of scale, where eps does not count; nothing over- or underflows
    base = T.newton_schulz(u, eps=0.0)
    for scale in (2.0 ** -60, 2.0 ** 60):
        assert torch.equal(T.newton_schulz(u * scale, eps=0.0), base)
    assert float(T.newton_schulz(torch.zeros(40, 50, device='cuda')).abs().max()) == 0.0
    assert bool(T.newton_schulz(torch.full((4, 4), float('nan'), device='cuda')).isnan().all())
    # views: transposed, a slice of a larger matrix
    big = torch.randn(200, 300, generator=g, device='cuda').to(BF)
    assert torch.equal(T.newton_schulz(big[3:67, 5:105]), T.newton_schulz(big[3:67, 5:105].contiguous()))
    assert torch.equal(T.newton_schulz(big.T), T.newton_schulz(big.T.contiguous()))
    assert torch.equal(T.newton_schulz(big[None].expand(3, 200, 300))[2], T.newton_schulz(big))
    # coefficients of its own for every step
    table = [(3.0, -3.2, 1.2), (2.0, -1.5, 0.5), (15 / 8, -10 / 8, 3 / 8)]
    want, err = _schulz64(u, table, 1e-7)
    assert float((T.newton_schulz(u, steps=3, coefficients=table).double() - want).norm()) <= err + UBF * float(want.norm())
    for shape in ((0, 4), (4, 0), (0, 3, 4)):
        assert T.newton_schulz(torch.zeros(shape, device='cuda')).shape == shape
    for bad in (lambda: T.newton_schulz(u[0]), lambda: T.newton_schulz(u.half()), lambda: T.newton_schulz(u, steps=0), lambda: T.newton_schulz(u, steps=2, coefficients=table),
                lambda: T.muon_step(u, u[:5], u, 0.1), lambda: T.muon_step(u, u, u.to(BF), 0.1), lambda: T.muon_step(u.T, u.T, u.T, 0.1)):
        with pytest.raises(L.SgpoError):
            bad()


@pytest.mark.parametrize('wdt,gdt,shape,nesterov', [(F32, F32, (96, 64), True), (F32, BF, (64, 200), False), (BF, BF, (2, 130, 70), True), (BF, F32, (512, 512), True),
                                                      (F32, F32, (31, 512), True), (BF, F32, (3, 400, 24), False), (F32, BF, (50, 333), True)])
def test_muon_step(wdt, gdt, shape, nesterov):
    from sgpo_amd import train_ops as T
    g = _gen(31)
    w = (torch.randn(shape, generator=g, device='cuda') * 0.05).to(wdt)
    buf = torch.randn(shape, generator=g, device='cuda') * 1e-2
    lr, mu, wd = 0.02, 0.9, 0.1
    rate = lr * max(1.0, shape[-2] / shape[-1]) ** 0.5
    for _ in range(3):
        grad = (torch.randn(shape, generator=g, device='cuda') * 1e-3).to(gdt)
        w0, b0 = w.clone(), buf.clone()
        assert T.muon_step(w, grad, buf, lr, momentum=mu, nesterov=nesterov, weight_decay=wd) is w
        want_b = mu * b0.double() + grad.double()
        _within(buf, want_b, 2 * U32 * (b0.abs().double() + grad.abs().double()), 'buffer')   # mu itself is rounded, and the sum
        u = grad.double() + mu * want_b if nesterov else want_b
        for i, (ui, wi, w0i) in enumerate(zip(u.reshape(-1, *shape[-2:]), w.reshape(-1, *shape[-2:]), w0.reshape(-1, *shape[-2:]))):
            x, err = _schulz64(ui, [T.NS_COEFFICIENTS] * 5, 1e-7)
            want = (1 - lr * wd) * w0i.double() - rate * x
            # the update is 2^-10 of its norm off at most (two planes, random signs), constants and sums 4 u, the weight's rounding
            tol = min(rate * err, rate * 2.0 ** -10 * float(x.norm())) + float((4 * U32 * (w0i.double().abs() + rate * x.abs()) + (STEP[wdt] * want.abs() if wdt == BF else 0)).norm())
            assert float((wi.double() - want).norm()) <= tol, i


# ---------------------------------------------------------------------------------------------- streams, graphs, together

def test_another_stream_and_device_memory_reuse():
    from sgpo_amd import train_ops as T
    g = _gen(41)
    h, w = torch.randn(700, 200, generator=g, device='cuda').to(BF), torch.randn(3000, 200, generator=g, device='cuda').to(BF)
    t = torch.randint(0, 3000, (700,), generator=g, device='cuda')
    freq, _ = T.rotary_frequencies(64)
    q = torch.randn(4, 100, 5, 64, generator=g, device='cuda')

    def both():
        hl, wl = h.detach().requires_grad_(), w.detach().requires_grad_()
        loss = T.linear_cross_entropy(hl, wl, t)
        return [loss.detach(), *torch.autograd.grad(loss, (hl, wl)), T.newton_schulz(w), T.rotary_positions(q, None, freq)[0]]

    want = both()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in side:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(both())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_captured_graphs_replay_with_new_inputs():
    from sgpo_amd import train_ops as T
    g = _gen(42)
    h = torch.randn(300, 160, generator=g, device='cuda').to(BF).requires_grad_()
    w = torch.randn(2000, 160, generator=g, device='cuda').to(BF).requires_grad_()
    b = torch.zeros(2000, device='cuda', requires_grad=True)
    t = torch.randint(0, 2000, (300,), generator=g, device='cuda')
    buf = torch.zeros(2000, 160, device='cuda')
    q = torch.randn(2, 60, 4, 64, generator=g, device='cuda')
    freq, _ = T.rotary_frequencies(64)

    def step():
        loss = T.linear_cross_entropy(h, w, t, b)
        dh, dw, db = torch.autograd.grad(loss, (h, w, b))
        with torch.no_grad():
            weight = w.detach().clone()
            state = buf.clone()
            T.muon_step(weight, dw, state, 0.02)
        return loss.detach(), dh, dw, db, weight, state, T.rotary_positions(q, None, freq)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                      # two graphs, each with scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for r in range(4):
        with torch.no_grad():
            h.copy_(torch.randn(300, 160, generator=g, device='cuda'))
            buf.normal_(generator=g)
            q.normal_(generator=g)
            t.copy_(torch.randint(-1, 2000, (300,), generator=g, device='cuda').where(torch.arange(300, device='cuda') % 3 > 0, -100).clamp(min=-100))
            t[t == -1] = -100
        want = step()
        torch.cuda.synchronize()
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want)), r


@pytest.mark.parametrize('V,shape', [(31, (31, 512)), (26, (3, 700, 40)), (100, (48, 48)), (70, (2, 96, 3000))])
def test_captured_graphs_of_heads_many_tokens_and_narrow_updates(V, shape):
    from sgpo_amd import train_ops as T
    g = _gen(43)
    N = 20011                               # the losses' total in parts
    h = torch.randn(N, 64, generator=g, device='cuda').to(BF).requires_grad_()
    w = torch.randn(V, 64, generator=g, device='cuda').to(BF).requires_grad_()
    t = torch.randint(0, V, (N,), generator=g, device='cuda')
    u = torch.randn(shape, generator=g, device='cuda')

    def step():
        loss = T.linear_cross_entropy(h, w, t)
        return [loss.detach(), *torch.autograd.grad(loss, (h, w)), T.newton_schulz(u)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        with torch.no_grad():
            h.normal_(generator=g)
            u.normal_(generator=g)
            t.random_(0, V, generator=g)
            t[::5] = -100
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want))


def test_calls_of_two_threads_at_once():
    import threading
    from sgpo_amd import train_ops as T
    g = _gen(44)
    h, w = torch.randn(500, 96, generator=g, device='cuda'), torch.randn(700, 96, generator=g, device='cuda')
    t = torch.randint(0, 700, (500,), generator=g, device='cuda')
    freq, _ = T.rotary_frequencies(32)
    q = torch.randn(2, 30, 4, 32, generator=g, device='cuda')

    def calls():
        hl = h.detach().requires_grad_()
        loss = T.linear_cross_entropy(hl, w, t)
        return [loss.detach(), torch.autograd.grad(loss, hl)[0], T.newton_schulz(w), T.newton_schulz(w[:64]), T.newton_schulz(w[:50, :60]), T.rotary_positions(q, None, freq)[0]]

    want = calls()
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got[i].append(calls())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    for out in got[0] + got[1]:
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    assert len(got[0]) == len(got[1]) == 10


def test_a_training_step_of_a_small_denoiser():
    """The operators together, as one training step uses them: rotated heads, attention, the head's loss with the mask class closed, gradients
    through all of it, orthogonalised updates of the matrices; against the same step in 64 bits."""
    from sgpo_amd import train_ops as T
    g = _gen(51)
    B, L, H, D, V = 4, 50, 4, 32, 31
    E = H * D
    par = {'embed': torch.randn(V, E, generator=g, device='cuda'), 'qkv': torch.randn(3 * E, E, generator=g, device='cuda') * E ** -0.5,
           'out': torch.randn(E, E, generator=g, device='cuda') * E ** -0.5, 'head': torch.randn(V, E, generator=g, device='cuda') * E ** -0.5}
    bias = torch.zeros(V, device='cuda')
    bias[28] = -math.inf
    x0 = torch.randint(0, 20, (B, L), generator=g, device='cuda')
    masked = torch.rand(B, L, generator=g, device='cuda') < 0.5
    xt = torch.where(masked, 28, x0)
    target = torch.where(masked, x0, -100)
    freq, _ = T.rotary_frequencies(D)

    def body(p, rotate, loss):
        x = p['embed'][xt]
        qkv = (x @ p['qkv'].T).view(B, L, 3, H, D)
        q, k = rotate(qkv[:, :, 0], qkv[:, :, 1])
        a = torch.softmax((q.transpose(1, 2) @ k.permute(0, 2, 3, 1).contiguous()) * D ** -0.5, -1) @ qkv[:, :, 2].transpose(1, 2).contiguous()
        return loss(x + a.transpose(1, 2).reshape(B, L, E) @ p['out'].T, p['head'])

    leaves = {k: v.clone().requires_grad_() for k, v in par.items()}
    loss = body(leaves, lambda q, k: T.rotary_positions(q, k, freq), lambda h, w: T.linear_cross_entropy(h, w, target, bias))
    loss.backward()
    p64 = {k: v.double().cpu().requires_grad_() for k, v in par.items()}
    xt, tc, fc = xt.cpu(), target.cpu(), freq.cpu()

    def rot64(*heads):
        ang = torch.arange(L, dtype=torch.float64)[:, None] * fc
        c, s = ang.cos()[None, :, None], ang.sin()[None, :, None]
        return [torch.cat((x[..., :D // 2] * c - x[..., D // 2:] * s, x[..., :D // 2] * s + x[..., D // 2:] * c), -1) for x in heads]

    want = body(p64, rot64, lambda h, w: torch.nn.functional.cross_entropy((h @ w.T + bias.double().cpu()).view(-1, V), tc.view(-1), ignore_index=-100))
    want.backward()
    # a chain of five fp32 products of up to 128 terms forward and as many back: 2 * 5 * 128 u = 2^-13.7 of a gradient's norm
    assert abs(float(loss.detach()) - float(want.detach())) <= 2.0 ** -14 * float(want.detach())
    for k, v in leaves.items():
        d = v.grad.double().cpu() - p64[k].grad
        assert float(d.norm()) <= 2.0 ** -13 * float(p64[k].grad.norm()), k
        buf = torch.zeros_like(par[k])
        new = T.muon_step(par[k].clone(), v.grad, buf, 0.02)
        x, _ = _schulz64(v.grad * 1.95, [T.NS_COEFFICIENTS] * 5, 1e-7)
        rate = 0.02 * max(1.0, v.shape[0] / v.shape[1]) ** 0.5
        assert float((new.double() - (par[k].double() - rate * x)).norm()) <= rate * 2.0 ** -9 * float(x.norm()) + 4 * U32 * float(par[k].norm())


def test_second_derivatives():
    """The rotation is linear: its gradient can be differentiated again.  The loss's cannot, and says so only where it is used."""
    from sgpo_amd import train_ops as T
    g = _gen(61)
    q, k = (torch.randn(2, 5, 3, 16, generator=g, device='cuda', requires_grad=True) for _ in range(2))
    u = torch.randn(2, 5, 3, 16, generator=g, device='cuda', requires_grad=True)
    freq, _ = T.rotary_frequencies(8)
    out, _ = T.rotary_positions(q, k, freq)
    dq, = torch.autograd.grad(out, q, u, create_graph=True)
    ddu, = torch.autograd.grad((dq * q.detach()).sum(), u)
    # d/du <R^T u, q> = R q
    assert torch.equal(ddu, out.detach())
    h = torch.randn(6, 16, generator=g, device='cuda', requires_grad=True)
    w = torch.randn(9, 16, generator=g, device='cuda', requires_grad=True)
    t = torch.arange(6, device='cuda')
    first = torch.autograd.grad(T.linear_cross_entropy(h, w, t), (h, w))
    again = torch.autograd.grad(T.linear_cross_entropy(h, w, t), (h, w), create_graph=True)
    assert all(torch.equal(a, b.detach()) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match='differentiated once'):
        torch.autograd.grad(again[0].sum(), h)
    # only what is asked for is computed, and in any combination
    for needs in ((True, False), (False, True)):
        hh, ww = h.detach().requires_grad_(needs[0]), w.detach().requires_grad_(needs[1])
        got, = torch.autograd.grad(T.linear_cross_entropy(hh, ww, t), [x for x, n in zip((hh, ww), needs) if n])
        assert torch.equal(got, first[0] if needs[0] else first[1])
    bias = torch.zeros(9, device='cuda', requires_grad=True)
    got, = torch.autograd.grad(T.linear_cross_entropy(h.detach(), w.detach(), t, bias), bias)
    assert got.shape == (9,) and float(got.sum().abs()) <= 20 * U32


def test_versions_tell_autograd_of_writes_in_place():
    from sgpo_amd import train_ops as T
    freq, _ = T.rotary_frequencies(8)
    w = torch.randn(8, 8, device='cuda')
    x = torch.randn(8, 8, device='cuda', requires_grad=True)
    y = x @ w
    T.muon_step(w, torch.randn(8, 8, device='cuda'), torch.zeros(8, 8, device='cuda'), 0.1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()
    q = torch.randn(1, 4, 2, 8, device='cuda')
    y = (x[:1, :4].reshape(1, 4, 1, 1) * q).sum()
    T.rotary_positions_(q, None, freq)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    with torch.inference_mode():
        q = torch.randn(1, 4, 2, 8, device='cuda')
        T.rotary_positions_(q, None, freq)
        T.muon_step(torch.zeros(8, 8, device='cuda'), q.new_ones(8, 8), torch.zeros(8, 8, device='cuda'), 0.1)
