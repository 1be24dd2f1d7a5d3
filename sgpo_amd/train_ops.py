"""Training operators of a denoiser on the GPU: position rotation of query and key heads, the cross entropy of a linear
vocabulary head without its logits, and updates orthogonalised by Newton-Schulz products.

The reference trains its denoisers through torch autograd (models/pretraining/trainer.py:75-88) with these steps as chains of
torch kernels; here each is one call into libsgpo_hip.so.  PyTorch is plumbing (device memory, the current HIP stream, the autograd
tape).  Every tensor is fp32 or bf16 device memory on the process's one GPU; a call runs on the stream that is current on that
device, allocates its outputs and scratch from torch's allocator (so it can be captured into a graph and used on any stream), and
does not synchronise.  There is no CPU fallback: bad arguments and host tensors raise SgpoError.
"""
import ctypes as C
import math

import torch

from . import _lib as L
from .runtime import init

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # Newton-Schulz quintic: singular values into about [0.7, 1.2] within 5 steps
_DTYPES = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16}
_REDUCE = {'none': L.REDUCE_NONE, 'mean': L.REDUCE_MEAN, 'sum': L.REDUCE_SUM}


def _require(ok, text):
    if not ok:
        raise L.SgpoError(text)


def _dtype(t, what):
    _require(t.dtype in _DTYPES, f'{what} must be float32 or bfloat16, got {t.dtype}')
    return _DTYPES[t.dtype]


def _on_device(first, *others):
    """The device of a call's tensors, all on one GPU, which is the one this process is bound to."""
    for t in (first, *others):
        _require(t is None or isinstance(t, torch.Tensor), f'a tensor is expected, got {type(t).__name__}')
        if t is not None and not t.is_cuda:
            raise L.SgpoError(f'host tensor {tuple(t.shape)} {t.dtype} passed where the library expects device memory')
        _require(t is None or t.device == first.device, f'tensors on {first.device} and on another device')
    return init(first.device)


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _scratch(nbytes, device):
    """Scratch of one call, 256-byte aligned; from torch's allocator, which keeps streams and captured graphs apart."""
    buf = torch.empty(int(nbytes) + 256, dtype=torch.uint8, device=device)
    return buf, C.c_void_p((buf.data_ptr() + 255) & ~255)


# ---------------------------------------------------------------------------------------------------------------- rotation

def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0,
                       device='cuda'):
    """(frequencies float64 (rotary_dim / 2,), scale): the angle per position of each pair, base ** (-2 j / rotary_dim) as in the
    reference's Rotary (dit.py:81-107), stretched for contexts longer than the original one.

    scaling None; 'linear': every angle / factor; 'ntk': base * factor ** (rotary_dim / (rotary_dim - 2)), which keeps the fastest pair
    and divides the slowest by factor; 'yarn': pairs that turn more than beta_fast times within original_length positions stay, those
    below beta_slow turns are divided by factor, linearly in between, and rotated elements are scaled by 0.1 ln(factor) + 1."""
    _require(rotary_dim >= 0 and rotary_dim % 2 == 0, f'rotary_dim must be even, got {rotary_dim}')
    _require(base > 0 and factor >= 1, f'base must be positive and factor at least 1, got {base} and {factor}')
    _require(scaling in (None, 'linear', 'ntk', 'yarn'), f'unknown scaling {scaling!r}')
    out, scale = [], 1.0
    if scaling == 'ntk':
        base = base * factor ** (rotary_dim / max(rotary_dim - 2, 1))
    if scaling == 'yarn':
        _require(beta_fast > beta_slow, 'beta_fast must be larger than beta_slow')
        scale = 0.1 * math.log(factor) + 1.0
    for j in range(0, rotary_dim, 2):
        f = base ** (-j / rotary_dim)
        if scaling == 'linear':
            f /= factor
        elif scaling == 'yarn':
            keep = min(max((original_length * f / (2 * math.pi) - beta_slow) / (beta_fast - beta_slow), 0.0), 1.0)
            f = f * keep + f / factor * (1.0 - keep)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64).to(device), scale


def _rotate(q, k, frequencies, positions, interleaved, scale, inverse, in_place=False):
    dev = _on_device(q, k, frequencies, positions)
    _require(q.dim() == 4, f'heads are (batch, tokens, heads, head_dim), got {tuple(q.shape)}')
    B, Lq, Hq, D = q.shape
    dt = _dtype(q, 'q')
    if k is not None:
        _require(k.dim() == 4 and (k.shape[0], k.shape[1], k.shape[3]) == (B, Lq, D) and k.dtype == q.dtype,
                 f'k {tuple(k.shape)} {k.dtype} does not match q {tuple(q.shape)} {q.dtype}')
    _require(frequencies.dtype == torch.float64 and frequencies.dim() == 1 and frequencies.is_contiguous(), 'frequencies must be a contiguous float64 vector')
    rot = 2 * frequencies.numel()
    _require(rot <= D, f'{rot} rotated elements in heads of {D}')
    psb = psl = 0
    if positions is not None:
        _require(positions.dtype == torch.int64, f'positions must be int64, got {positions.dtype}')
        _require(tuple(positions.shape) in ((Lq,), (B, Lq), (1, Lq), (B, 1)), f'positions {tuple(positions.shape)} for {B} x {Lq} tokens')
        if positions.dim() == 1:
            psl = positions.stride(0)
        else:
            psb = positions.stride(0) if positions.shape[0] > 1 else 0
            psl = positions.stride(1) if positions.shape[1] > 1 else 0
            _require(positions.shape[1] == Lq, f'positions {tuple(positions.shape)} for {B} x {Lq} tokens')
    a = L.RotaryArgs()
    src, dst = [], []
    for t in (q, k):
        if t is None:
            src.append(None)
            dst.append(None)
            continue
        s = t if t.stride(3) == 1 or D == 1 or not t.numel() else t.contiguous()
        if in_place:
            _require(s is t, 'in place, the elements of a head must be contiguous')
            _require(all(st > 0 or n <= 1 for st, n in zip(t.stride(), t.shape)), 'in place, heads must not be broadcast')
        src.append(s)
        dst.append(s if in_place else torch.empty(t.shape, dtype=t.dtype, device=dev))
    for name, s, d in (('q', src[0], dst[0]), ('k', src[1], dst[1])):
        if s is None:
            continue
        setattr(a, name, s.data_ptr())
        setattr(a, name + '_out', d.data_ptr())
        for i in range(3):
            getattr(a, name + '_stride')[i] = s.stride(i)
            getattr(a, name + '_out_stride')[i] = d.stride(i)
    a.positions = None if positions is None else positions.data_ptr()
    a.pos_stride_b, a.pos_stride_l = psb, psl
    a.frequencies = frequencies.data_ptr()
    a.B, a.L, a.heads_q, a.heads_k, a.head_dim, a.rot = B, Lq, Hq, 0 if k is None else k.shape[2], D, rot
    a.interleaved, a.inverse, a.dtype, a.scale = int(interleaved), int(inverse), dt, float(scale)
    L.check(L.load().sgpo_rotary(C.byref(a), _stream(dev)), 'sgpo_rotary')
    return dst


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, frequencies, positions, interleaved, scale):
        ctx.save_for_backward(frequencies, positions)
        ctx.how = interleaved, scale
        out = _rotate(q, k, frequencies, positions, interleaved, scale, False)
        return out[0], out[1]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        frequencies, positions = ctx.saved_tensors
        got = _rotate(dq, dk, frequencies, positions, *ctx.how, True)
        return got[0], got[1], None, None, None, None


def rotary_positions(q, k, frequencies, positions=None, interleaved=False, scale=1.0):
    """q (B, L, Hq, D) and k (B, L, Hk, D) (or None) with the first 2 * len(frequencies) elements of every head turned by their
    token's position; differentiable in q and k.  Returns new contiguous (q, k).

    frequencies and scale as rotary_frequencies gives them; positions int64 (L,), (B, L), (1, L) or None for 0 .. L - 1, of any size up to 2 ** 50; pairs are
    (j, j + rot / 2), or (2 j, 2 j + 1) if interleaved.  q and k may be views with any strides (of one packed projection, or of
    (B, H, L, D) tensors); only heads that are not contiguous in memory are copied first."""
    if not (torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad)):
        out = _rotate(q, k, frequencies, positions, interleaved, scale, False)
        return out[0], out[1]
    return _Rotary.apply(q, k, frequencies, positions, bool(interleaved), float(scale))


def rotary_positions_(q, k, frequencies, positions=None, interleaved=False, scale=1.0):
    """rotary_positions written over q and k (as the reference's apply_rotary_emb_qkv_, dit.py:112-115); not differentiable."""
    _require(not (torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad)), 'rotary_positions_ has no gradient: use rotary_positions')
    _rotate(q, k, frequencies, positions, interleaved, scale, False, in_place=True)
    return q, k


# -------------------------------------------------------------------------------------------------------------------- loss

def _loss_args(hidden, weight, targets, bias, ignore_index, reduction):
    a = L.LinearCeArgs()
    a.hidden, a.weight, a.targets = hidden.data_ptr(), weight.data_ptr(), targets.data_ptr()
    a.bias = None if bias is None else bias.data_ptr()
    (a.N, a.H), a.V = hidden.shape, weight.shape[0]
    a.ld_hidden = hidden.stride(0) if a.N > 1 else a.H
    a.ld_weight = weight.stride(0) if a.V > 1 else a.H
    a.ignore_index, a.dtype, a.reduction = ignore_index, _DTYPES[hidden.dtype], _REDUCE[reduction]
    return a


def _rows(t):
    """A matrix with contiguous rows that do not overlap."""
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _loss_forward(hidden, weight, targets, bias, ignore_index, reduction):
    dev = hidden.device
    lib = L.load()
    a = _loss_args(hidden, weight, targets, bias, ignore_index, reduction)
    need = lib.sgpo_linear_ce_workspace_bytes(C.byref(a), 0)
    buf, ws = _scratch(need, dev)
    out = torch.empty(2 * a.N + 2, dtype=torch.float32, device=dev)
    nll, lse, loss, inv = out[:a.N], out[a.N:2 * a.N], out[2 * a.N], out[2 * a.N + 1]
    L.check(lib.sgpo_linear_ce_forward(C.byref(a), L.ptr(nll), L.ptr(lse), L.ptr(loss), L.ptr(inv), ws, need, _stream(dev)),
            'sgpo_linear_ce_forward')
    return nll if reduction == 'none' else loss, lse, inv


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, bias, ignore_index, reduction):
        out, lse, inv = _loss_forward(hidden, weight, targets, bias, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, targets, bias, lse, inv)
        ctx.how = ignore_index, reduction
        return out.clone()      # its own storage: lse and inv live behind it

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, targets, bias, lse, inv = ctx.saved_tensors
        dev = hidden.device
        lib = L.load()
        a = _loss_args(hidden, weight, targets, bias, *ctx.how)
        grad = grad.to(torch.float32).contiguous()
        want = ctx.needs_input_grad
        dh = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if want[0] else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if want[1] else None
        db = torch.empty(bias.shape, dtype=torch.float32, device=dev) if want[3] else None
        need = lib.sgpo_linear_ce_workspace_bytes(C.byref(a), 1)
        buf, ws = _scratch(need, dev)
        L.check(lib.sgpo_linear_ce_backward(C.byref(a), L.ptr(lse), L.ptr(grad), L.ptr(inv), L.ptr(dh), L.ptr(dw), L.ptr(db), ws, need,
                                            _stream(dev)), 'sgpo_linear_ce_backward')
        return dh, dw, None, db, None, None


def linear_cross_entropy(hidden, weight, targets, bias=None, ignore_index=-100, reduction='mean'):
    """Cross entropy of softmax(hidden weight^T + bias) at targets without storing the logits; differentiable in hidden, weight
    and bias (once).

    hidden (..., H) and weight (V, H), both fp32 or both bf16; targets int64 of hidden's leading shape; bias fp32 (V,) or None, where -inf
    closes a class (the mask class of an absorbing-state model, mdlm_diffusion.py:325-341).  reduction 'none' gives fp32 losses of
    targets' shape; 'sum' and 'mean' (over the targets that are not ignore_index; 0 if there are none) give a scalar.  An ignored token has loss
    and gradients 0 whatever its features hold; a target outside [0, V) gives NaN, as no check on the host waits for the GPU."""
    dev = _on_device(hidden, weight, targets, bias)
    _dtype(hidden, 'hidden')
    _require(hidden.dim() >= 1 and weight.dim() == 2 and hidden.shape[-1] == weight.shape[1] and weight.numel() > 0,
             f'hidden {tuple(hidden.shape)} does not match weight {tuple(weight.shape)}')
    _require(weight.dtype == hidden.dtype, f'hidden is {hidden.dtype} and weight {weight.dtype}')
    _require(targets.dtype == torch.int64 and targets.shape == hidden.shape[:-1], f'targets {tuple(targets.shape)} {targets.dtype} for hidden {tuple(hidden.shape)}')
    _require(bias is None or bias.dtype == torch.float32 and tuple(bias.shape) == (weight.shape[0],), 'bias must be float32 with one value per class')
    _require(reduction in _REDUCE, f'unknown reduction {reduction!r}')
    h, w = _rows(hidden.reshape(-1, hidden.shape[-1])), _rows(weight)
    t = targets.reshape(-1).contiguous()
    b = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (hidden, weight, bias)):
        out = _LinearCrossEntropy.apply(h, w, t, b, int(ignore_index), reduction)
    else:
        out = _loss_forward(h, w, t, b, int(ignore_index), reduction)[0]
    return out.view(targets.shape) if reduction == 'none' else out


# ----------------------------------------------------------------------------------------------------------------- updates

def _coefficients(coefficients, steps):
    c = [float(v) for row in (coefficients if isinstance(coefficients[0], (tuple, list)) else [coefficients] * steps) for v in row]
    _require(len(c) == 3 * steps and steps >= 1, f'{steps} steps need {steps} coefficient triples')
    return (C.c_float * len(c))(*c)


def newton_schulz(update, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """The update (..., m, n) with every singular value moved towards 1 and its singular vectors kept: X = U / (|U|_F + eps), then
    X <- a X + (b X X^T + c (X X^T)^2) X per coefficient triple (one triple for all steps, or one each).  Leading dimensions are independent matrices.
    update fp32 or bf16; returns bf16, contiguous.  Iterates carry 16 bits of mantissa, sums 32 bits, the norm 64.  Not differentiable."""
    dev = _on_device(update)
    dt = _dtype(update, 'update')
    _require(update.dim() >= 2, f'an update is a matrix or a batch of them, got {tuple(update.shape)}')
    m, n = update.shape[-2:]
    u = update.detach().reshape(-1, m, n) if update.numel() else update.detach().new_empty(0, m, n)
    if u.numel() and (u.stride(2) != 1 and n > 1 or m > 1 and u.stride(1) < n):
        u = u.contiguous()
    out = torch.empty(update.shape, dtype=torch.bfloat16, device=dev)
    lib = L.load()
    need = lib.sgpo_newton_schulz_workspace_bytes(u.shape[0], m, n)
    buf, ws = _scratch(need, dev)
    L.check(lib.sgpo_newton_schulz(L.ptr(u), dt, u.shape[0], m, n, u.stride(0), u.stride(1), _coefficients(coefficients, steps), steps, float(eps),
                                   L.ptr(out), ws, need, _stream(dev)), 'sgpo_newton_schulz')
    return out


def muon_step(weight, grad, momentum_buffer, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NS_COEFFICIENTS,
              eps=1e-7):
    """One optimiser step of weight (..., m, n), in place, with an orthogonalised momentum update; leading dimensions are
    independent matrices.

    buffer = momentum * buffer + grad;  U = grad + momentum * buffer (nesterov) or buffer;  weight = (1 - lr * weight_decay) * weight -
    lr * sqrt(max(1, m / n)) * newton_schulz(U), the last product not rounded before it is applied.  weight and grad fp32 or bf16,
    momentum_buffer fp32 (the caller's state, zeros at first), all contiguous.  Returns weight."""
    dev = _on_device(weight, grad, momentum_buffer)
    wd, gd = _dtype(weight, 'weight'), _dtype(grad, 'grad')
    _require(weight.dim() >= 2 and weight.shape == grad.shape == momentum_buffer.shape, f'weight {tuple(weight.shape)}, grad {tuple(grad.shape)} and buffer {tuple(momentum_buffer.shape)} must agree')
    _require(momentum_buffer.dtype == torch.float32, 'momentum_buffer must be float32')
    _require(weight.is_contiguous() and momentum_buffer.is_contiguous(), 'weight and momentum_buffer are updated in place and must be contiguous')
    g = grad.detach().contiguous()
    m, n = weight.shape[-2:]
    batch = weight.numel() // (m * n) if m * n else 0
    lib = L.load()
    need = lib.sgpo_newton_schulz_workspace_bytes(batch, m, n)
    buf, ws = _scratch(need, dev)
    L.check(lib.sgpo_muon_step(L.ptr(weight), wd, L.ptr(g), gd, L.ptr(momentum_buffer), batch, m, n, float(lr), float(momentum), int(bool(nesterov)),
                               float(weight_decay), _coefficients(coefficients, steps), steps, float(eps), ws, need, _stream(dev)), 'sgpo_muon_step')
    return weight
