"""The training operators of a denoiser, as workloads: position rotation of query and key heads, the cross entropy of a linear
vocabulary head without its logits, and updates orthogonalised by Newton-Schulz products.

`own` False: the plain form, elementary torch operations in 32 bits.  `own` True: the calls of sgpo_amd.train_ops.
"""
import math

import torch

own = False

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
IGNORE = -100
DTYPES = {'bf16': torch.bfloat16, 'fp32': torch.float32}


# ------------------------------------------------------------------------------------------------------------------ cases

def _rotary(name, B, L, Hq, Hk, D, rot, dtype, **kw):
    c = dict(op='rotary', B=B, L=L, Hq=Hq, Hk=Hk, D=D, rot=rot, dtype=dtype, interleaved=False, packed=False,
             scaling='none', factor=1.0, positions='range', step=False)
    c.update(kw)
    return dict(c, name=name) if name else c


def _loss(name, N, H, V, dtype, **kw):
    c = dict(op='loss', N=N, H=H, V=V, dtype=dtype, bias=True, closed=True, ignored=0.0, step=True)
    c.update(kw)
    return dict(c, name=name) if name else c


def _ortho(name, batch, m, n, dtype, **kw):
    c = dict(op='ortho', batch=batch, m=m, n=n, dtype=dtype, update=False, nesterov=True)
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of each of 64 sequences, at positions all over a long context: a sampler's smallest call
        _rotary('rotary_token', 64, 1, 8, 8, 64, 64, 'bf16', positions='far'),
        # the DiT's heads (8 of 64) on 256 sequences of 119 residues, read in place from the packed projection; training step
        _rotary('rotary_denoiser', 256, 119, 8, 8, 64, 64, 'bf16', packed=True, step=True),
        # 389 residues, odd batch, shared key heads, part of the head, positions of its own per sequence, stretched by 4
        _rotary('rotary_ragged', 37, 389, 6, 2, 80, 40, 'fp32', scaling='linear', factor=4.0, positions='ragged', step=True),
        # one long context of 131072 positions, interleaved pairs, half the head, frequency-dependent stretch; training step
        _rotary('rotary_long', 1, 131072, 32, 8, 128, 64, 'bf16', interleaved=True, scaling='yarn', factor=16.0, step=True),
        # scoring one sequence of 119 residues with the denoiser's own head (31 classes, the mask class closed)
        _loss('loss_score', 119, 512, 31, 'fp32', step=False),
        # a training step on 64 sequences with the denoiser's own head; unmasked tokens carry no loss
        _loss('loss_denoiser', 64 * 119, 512, 31, 'bf16', ignored=0.6),
        # a 32-bit head of odd sizes everywhere: 1003 tokens, 517 features, 50021 classes
        _loss('loss_odd', 1003, 517, 50021, 'fp32', closed=False, ignored=0.1),
        # a large vocabulary: 8192 tokens, 2048 features, 131072 classes; training step
        _loss('loss_large', 8192, 2048, 131072, 'bf16', bias=False, closed=False),
        # the 64 x 64 layers of an ensemble of ten value functions in one call
        _ortho('ortho_ensemble', 10, 64, 64, 'fp32'),
        # the QKV projection of one DiT block (1536 x 512): the whole update of an fp32 weight
        _ortho('ortho_projection', 1, 1536, 512, 'fp32', update=True),
        # the MLP weights of the eight DiT blocks (512 x 2048) in one call
        _ortho('ortho_blocks', 8, 512, 2048, 'bf16'),
        # one large bf16 weight, whole update
        _ortho('ortho_large', 1, 4096, 4096, 'bf16', update=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['rotary', 'loss', 'ortho'])
    if op == 'rotary':
        D = rng.choice([16, 32, 48, 64, 80, 96, 128, 256])
        Hk = rng.choice([1, 2, 3, 4, 8, 16])
        Hq = Hk * rng.choice([1, 1, 2, 4, 8])
        per_token = (Hq + Hk) * D
        L = _log_int(rng, 1, min(131072, 300_000_000 // per_token))
        B = max(1, min(_log_int(rng, 1, 512), 300_000_000 // (L * per_token)))
        scaling = rng.choice(['none', 'linear', 'ntk', 'yarn'])
        return _rotary(None, B, L, Hq, Hk, D, rng.choice([D, D, D // 2, max(2, D // 4), D - 2]), rng.choice(['bf16', 'bf16', 'fp32']),
                       interleaved=rng.random() < 0.5, packed=Hq == Hk and rng.random() < 0.5, scaling=scaling,
                       factor=1.0 if scaling == 'none' else float(rng.choice([2, 4, 8, 16, 32])),
                       positions=rng.choice(['range', 'ragged', 'far']), step=rng.random() < 0.6)
    if op == 'loss':
        dtype = rng.choice(['bf16', 'bf16', 'fp32'])
        H, V = _log_int(rng, 16, 2048), rng.choice([31, 26, _log_int(rng, 2, 131072), _log_int(rng, 2, 131072)])
        most = 8192 * 2048 * 131072 // (16 if dtype == 'fp32' else 1)
        N = max(1, min(_log_int(rng, 1, 8192 if V > 1024 else 65536), most // (H * V)))
        return _loss(None, N, H, V, dtype, bias=rng.random() < 0.6, closed=rng.random() < 0.5,
                     ignored=rng.choice([0.0, 0.0, 0.15, 0.6]), step=rng.random() < 0.7)
    m, n = _log_int(rng, 8, 4096), _log_int(rng, 8, 4096)
    batch = max(1, min(rng.randint(1, 16), 4096 ** 3 // (min(m, n) ** 2 * max(m, n))))
    return _ortho(None, batch, m, n, rng.choice(['bf16', 'fp32']), update=batch == 1 and rng.random() < 0.7,
                  nesterov=rng.random() < 0.8)


# ----------------------------------------------------------------------------------------------------------------- inputs

def _frequencies(rot, scaling, factor, base=10000.0, original=4096):
    """Angles per position of the rot / 2 pairs, in 64 bits, and the factor on the rotated part."""
    j = torch.arange(0, rot, 2, dtype=torch.float64, device='cuda') / rot
    if scaling == 'linear':
        return base ** -j / factor, 1.0
    if scaling == 'ntk':
        return (base * factor ** (rot / max(rot - 2, 1))) ** -j, 1.0
    f = base ** -j
    if scaling == 'yarn':
        turns = original * f / (2 * math.pi)            # whole turns of a pair within the original context
        lo, hi = 1.0, 32.0
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(int(seed) * 7919 + 13)
    dt = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)

    if case['op'] == 'rotary':
        B, L, Hq, Hk, D = (case[k] for k in ('B', 'L', 'Hq', 'Hk', 'D'))
        if case['packed']:
            qkv = normal(B, L, 3, Hq, D)
            q, k = qkv[:, :, 0], qkv[:, :, 1]
        else:
            q, k = normal(B, L, Hq, D), normal(B, L, Hk, D)
        if case['positions'] == 'range':
            pos = None
        else:
            top = 4096 if case['positions'] == 'ragged' else 4_000_000
            pos = torch.randint(0, top, (B, 1), generator=g, device='cuda') + torch.arange(L, device='cuda')
        freq, scale = _frequencies(case['rot'], case['scaling'], case['factor'])
        s = dict(case=case, q=q, k=k, positions=pos, frequencies=freq, scale=scale)
        if case['step']:
            s['q'], s['k'] = q.detach().requires_grad_(), k.detach().requires_grad_()
            s['dq'], s['dk'] = normal(B, L, Hq, D), normal(B, L, Hk, D)
        return s
    if case['op'] == 'loss':
        N, H, V = case['N'], case['H'], case['V']
        weight = normal(V, H, scale=H ** -0.5)
        targets = torch.randint(0, V - 1 if case['closed'] else V, (N,), generator=g, device='cuda')
        # normalised features that lean towards their class, as a partly trained model's do
        hidden = torch.randn(N, H, generator=g, device='cuda') + 2.0 * weight[targets].float()
        hidden = hidden.to(dt)
        bias = normal(V, scale=0.1, dtype=torch.float32) if case['bias'] or case['closed'] else None
        if case['closed']:
            bias[V - 1] = -math.inf                     # a class that is never predicted, as an absorbing state's mask
        if case['ignored']:
            targets = torch.where(torch.rand(N, generator=g, device='cuda') < case['ignored'], IGNORE, targets)
        s = dict(case=case, hidden=hidden, weight=weight, bias=bias, targets=targets)
        if case['step']:
            for k in ('hidden', 'weight', 'bias'):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    shape = (case['batch'], case['m'], case['n'])
    # gradients: a few strong directions over noise
    r = max(1, min(shape[1:]) // 8)
    grad = torch.randn(*shape, generator=g, device='cuda')
    for_b = torch.randn(shape[0], shape[1], r, generator=g, device='cuda') @ torch.randn(shape[0], r, shape[2], generator=g, device='cuda')
    grad = ((grad + for_b * (2.0 / r ** 0.5)) * 1e-3).to(dt)
    if not case['update']:
        return dict(case=case, grad=grad)
    buf = torch.randn(*shape[1:], generator=g, device='cuda') * 5e-3
    return dict(case=case, grad=grad[0], weight=normal(*shape[1:], scale=0.04), buffer=buf)


# ------------------------------------------------------------------------------------------------------------ plain forms

def _rotate_plain(x, cos, sin, rot, interleaved):
    x = x.float()
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :rot // 2], r[..., rot // 2:])
    lo, hi = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((lo, hi), -1).flatten(-2) if interleaved else torch.cat((lo, hi), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _rotary_plain(s):
    c, q, k = s['case'], s['q'].detach(), s['k'].detach()
    pos = s['positions'] if s['positions'] is not None else torch.arange(c['L'], device=q.device)[None]
    ang = pos[..., None].double() * s['frequencies']
    cos, sin = ((f * s['scale']).float()[:, :, None] for f in (ang.cos(), ang.sin()))
    out = [_rotate_plain(x, cos, sin, c['rot'], c['interleaved']).to(x.dtype) for x in (q, k)]
    if c['step']:       # the transposed rotation
        out += [_rotate_plain(x, cos, -sin, c['rot'], c['interleaved']).to(x.dtype) for x in (s['dq'], s['dk'])]
    return out


def _loss_plain(s):
    h, w = s['hidden'].detach().float(), s['weight'].detach().float()
    t, keep = s['targets'].clamp(min=0), s['targets'] != IGNORE
    z = h @ w.t()
    if s['bias'] is not None:
        z += s['bias'].detach()
    top = z.max(1, keepdim=True).values
    at = z.gather(1, t[:, None])
    p = z.sub_(top).exp_()
    total = p.sum(1, keepdim=True)
    nll = torch.where(keep, (total.log() + top - at)[:, 0], 0.0)
    if not s['case']['step']:
        return [nll]
    count = keep.sum().clamp(min=1)
    loss = (nll.double().sum() / count).float()
    d = p.div_(total)
    d.scatter_add_(1, t[:, None], torch.full_like(total, -1.0))
    d *= keep[:, None] / count.float()
    out = [loss, (d @ w).to(s['hidden'].dtype), (d.t() @ h).to(s['weight'].dtype)]
    return out + ([d.sum(0)] if s['bias'] is not None else [])


def _orthogonal_plain(u):
    a, b, c = NS_COEFFICIENTS
    x = u.float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (x.double().square().sum((-2, -1), keepdim=True).sqrt().float() + 1e-7)
    x = _five(x, a, b, c)
    return x.transpose(-2, -1).contiguous() if tall else x


def _five(x, a, b, c, left=5):
    g = x @ x.transpose(-2, -1).contiguous()
    x = a * x + (b * g + c * (g @ g)) @ x
    return x if left == 1 else _five(x, a, b, c, left - 1)


def _ortho_plain(s):
    c = s['case']
    if not c['update']:
        return [_orthogonal_plain(s['grad']).to(torch.bfloat16)]
    w, buf, g = s['weight'], s['buffer'], s['grad'].float()
    buf.mul_(0.95).add_(g)
    u = g + 0.95 * buf if c['nesterov'] else buf
    w.copy_(w.float() * (1 - 0.02 * 0.01) - 0.02 * max(1.0, c['m'] / c['n']) ** 0.5 * _orthogonal_plain(u))
    return [w, buf]


def run(state):
    c = state['case']
    if not own:
        return {'rotary': _rotary_plain, 'loss': _loss_plain, 'ortho': _ortho_plain}[c['op']](state)
    from sgpo_amd import train_ops
    s = state
    if c['op'] == 'rotary':
        q, k = train_ops.rotary_positions(s['q'], s['k'], s['frequencies'], s['positions'], interleaved=c['interleaved'], scale=s['scale'])
        if not c['step']:
            return [q, k]
        return [q, k, *torch.autograd.grad((q, k), (s['q'], s['k']), (s['dq'], s['dk']))]
    if c['op'] == 'loss':
        if not c['step']:
            return [train_ops.linear_cross_entropy(s['hidden'], s['weight'], s['targets'], s['bias'], ignore_index=IGNORE, reduction='none')]
        loss = train_ops.linear_cross_entropy(s['hidden'], s['weight'], s['targets'], s['bias'], ignore_index=IGNORE, reduction='mean')
        leaves = [s[k] for k in ('hidden', 'weight', 'bias') if s[k] is not None]
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    if not c['update']:
        return [train_ops.newton_schulz(s['grad'])]
    train_ops.muon_step(s['weight'], s['grad'], s['buffer'], lr=0.02, momentum=0.95, nesterov=c['nesterov'], weight_decay=0.01)
    return [s['weight'], s['buffer']]


# -------------------------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    size = 2 if case['dtype'] == 'bf16' else 4
    if case['op'] == 'rotary':
        n = case['B'] * case['L'] * (case['Hq'] + case['Hk']) * case['D']
        passes = 2 if case['step'] else 1
        turned = n * case['rot'] // case['D']
        return dict(bytes=passes * 2 * n * size + (0 if case['positions'] == 'range' else 8 * case['B'] * case['L']), flops=passes * 3 * turned)
    if case['op'] == 'loss':
        N, H, V = case['N'], case['H'], case['V']
        io = (N * H + V * H) * size + 8 * N + (4 * V if case['bias'] or case['closed'] else 0)
        return dict(bytes=2 * io if case['step'] else io + 4 * N, flops=(6 if case['step'] else 2) * N * H * V)
    b, m, n = case['batch'], min(case['m'], case['n']), max(case['m'], case['n'])
    # per step: both symmetric products at half, one full product
    flops = b * 5 * (m * m * n + m ** 3 + 2 * m * m * n)
    elems = b * m * n
    return dict(bytes=elems * (3 * size + 8) if case['update'] else elems * (size + 2), flops=flops)


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'rotary':
        rot, D = case['rot'], case['D']
        pos = s['positions'] if s['positions'] is not None else torch.arange(case['L'], device='cuda').expand(case['B'], -1)
        turn = torch.polar(torch.full((), s['scale'], dtype=torch.float64, device='cuda'), pos.double()[..., None] * s['frequencies'])[:, :, None]
        first = torch.arange(rot // 2, device='cuda') * (2 if case['interleaved'] else 1)
        second = first + (1 if case['interleaved'] else rot // 2)

        def turned(x, t):
            y = x.detach().double()
            z = torch.complex(y[..., first], y[..., second]) * t
            y[..., first], y[..., second] = z.real, z.imag
            return y

        out = [turned(s['q'], turn), turned(s['k'], turn)]
        return out + ([turned(s['dq'], turn.conj()), turned(s['dk'], turn.conj())] if case['step'] else [])
    if case['op'] == 'loss':
        h, w, tg = s['hidden'].detach().double(), s['weight'].detach().double(), s['targets']
        b = None if s['bias'] is None else s['bias'].detach().double()
        n_kept = int((tg != IGNORE).sum())
        losses, dh, dw, db = [], [], torch.zeros_like(w), torch.zeros(len(w), dtype=torch.float64, device='cuda')
        for i in range(0, len(h), 2048):
            hi, ti = h[i:i + 2048], tg[i:i + 2048]
            logp = torch.log_softmax(hi @ w.T if b is None else hi @ w.T + b, -1)
            rows = torch.nonzero(ti != IGNORE)[:, 0]
            nll = torch.zeros(len(hi), dtype=torch.float64, device='cuda')
            nll[rows] = -logp[rows, ti[rows]]
            losses.append(nll)
            if case['step']:
                d = torch.zeros_like(logp)
                d[rows] = logp[rows].exp()
                d[rows, ti[rows]] -= 1.0
                d /= max(n_kept, 1)
                dh.append(d @ w)
                dw += d.T @ hi
                db += d.sum(0)
        if not case['step']:
            return [torch.cat(losses)]
        return [torch.cat(losses).sum() / max(n_kept, 1), torch.cat(dh), dw] + ([] if b is None else [db])
    a, b, c = NS_COEFFICIENTS
    g = s['grad'].double()
    u = g
    if case['update']:
        buf = 0.95 * s['buffer'].double() + g
        u = g + 0.95 * buf if case['nesterov'] else buf
    x = u / (torch.linalg.matrix_norm(u, keepdim=True) + 1e-7)
    for _ in range(5):      # x (a + b x'x + c (x'x)^2), on the shorter side
        if case['m'] >= case['n']:
            y = x.mT @ x
            x = a * x + x @ (b * y + c * y @ y)
        else:
            y = x @ x.mT
            x = a * x + (b * y + c * y @ y) @ x
    if not case['update']:
        return [x]
    w = s['weight'].double() * (1 - 0.02 * 0.01) - 0.02 * max(1.0, case['m'] / case['n']) ** 0.5 * x
    return [w, buf]
