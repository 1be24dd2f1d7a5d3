"""Training operators of a denoiser on the GPU: position rotation of query and key heads, the cross entropy of a linear
vocabulary head without its logits, and updates orthogonalised by Newton-Schulz products.

The reference trains its denoisers through torch autograd (models/pretraining/trainer.py:75-88) with these steps as chains of
torch kernels; here each is one call into libsgpo_hip.so.  PyTorch is plumbing (device memory, the current HIP stream, the autograd
tape).  Every tensor is fp32 or bf16 device memory on the process's one GPU; a call runs on the stream that is current on that
device, allocates its outputs and scratch from torch's allocator (so it can be captured into a graph and used on any stream), and
does not synchronise.  There is no CPU fallback: bad arguments and host tensors raise SgpoError.
"""
import math
import struct

import torch

from . import _lib as L
from . import runtime

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # Newton-Schulz quintic: singular values into about [0.7, 1.2] within 5 steps
_DTYPES = {torch.float32: L.DTYPE_F32, torch.bfloat16: L.DTYPE_BF16}
_REDUCE = {'none': L.REDUCE_NONE, 'mean': L.REDUCE_MEAN, 'sum': L.REDUCE_SUM}
# The argument blocks of the C calls, packed in one go: filling a ctypes structure field by field takes longer than the smallest of
# these kernels.  Same order and padding as L.RotaryArgs and L.LinearCeArgs (checked below).
_ROTARY = struct.Struct('=4Q12qQ2qQ9if')
_LOSS = struct.Struct('=4Q3q5i4x')
assert _ROTARY.size == L.C.sizeof(L.RotaryArgs) and _LOSS.size == L.C.sizeof(L.LinearCeArgs)


def _refuse(text):
    raise L.SgpoError(text)


def _dtype(t, what):
    if t.dtype not in _DTYPES:
        _refuse(f'{what} must be float32 or bfloat16, got {t.dtype}')
    return _DTYPES[t.dtype]


def _on_device(first, *others):
    """The device of a call's tensors, all on one GPU, which is the one this process is bound to."""
    for t in (first, *others):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            _refuse(f'a tensor is expected, got {type(t).__name__}')
        if not t.is_cuda:
            _refuse(f'host tensor {tuple(t.shape)} {t.dtype} passed where the library expects device memory')
        if t.device != first.device:
            _refuse(f'tensors on {first.device} and on {t.device}')
    dev = first.device
    if dev.index not in runtime._initialised:
        runtime.init(dev)
    return dev


def _call(dev, name, *args):
    """One C call on the stream that is current on the tensors' device, which need not be the current device."""
    fn = getattr(L.load(), name)
    if torch._C._cuda_getDevice() == dev.index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))    # torch.cuda.current_stream(dev).cuda_stream without the object
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if rc:
        L.check(rc, name)


def _scratch(nbytes, dev):
    """(tensor, address, bytes) of one call's scratch, 256-byte aligned; from torch's allocator, which keeps streams and captured graphs apart."""
    buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=dev)
    return buf, (buf.data_ptr() + 255) & ~255


# ---------------------------------------------------------------------------------------------------------------- rotation

def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0,
                       device='cuda'):
    """(frequencies float64 (rotary_dim / 2,), scale): the angle per position of each pair, base ** (-2 j / rotary_dim) as in the
    reference's Rotary (dit.py:81-107), stretched for contexts longer than the original one.

    scaling None; 'linear': every angle / factor; 'ntk': base * factor ** (rotary_dim / (rotary_dim - 2)), which keeps the fastest pair
    and divides the slowest by factor; 'yarn': pairs that turn more than beta_fast times within original_length positions stay, those
    below beta_slow turns are divided by factor, linearly in between, and rotated elements are scaled by 0.1 ln(factor) + 1."""
    if rotary_dim < 0 or rotary_dim % 2:
        _refuse(f'rotary_dim must be even, got {rotary_dim}')
    if not (base > 0 and factor >= 1):
        _refuse(f'base must be positive and factor at least 1, got {base} and {factor}')
    if scaling not in (None, 'linear', 'ntk', 'yarn'):
        _refuse(f'unknown scaling {scaling!r}')
    out, scale = [], 1.0
    if scaling == 'ntk':
        base = base * factor ** (rotary_dim / max(rotary_dim - 2, 1))
    if scaling == 'yarn':
        if beta_fast <= beta_slow:
            _refuse('beta_fast must be larger than beta_slow')
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
    dt = _dtype(q, 'q')
    if q.dim() != 4:
        _refuse(f'heads are (batch, tokens, heads, head_dim), got {tuple(q.shape)}')
    B, Lq, Hq, D = q.shape
    Hk = 0
    if k is not None:
        if k.dim() != 4 or k.dtype != q.dtype or (k.shape[0], k.shape[1], k.shape[3]) != (B, Lq, D):
            _refuse(f'k {tuple(k.shape)} {k.dtype} does not match q {tuple(q.shape)} {q.dtype}')
        Hk = k.shape[2]
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        _refuse('frequencies must be a contiguous float64 vector')
    rot = 2 * frequencies.numel()
    if rot > D:
        _refuse(f'{rot} rotated elements in heads of {D}')
    pos = psb = psl = 0
    if positions is not None:
        ps = tuple(positions.shape)
        if positions.dtype != torch.int64 or ps not in ((Lq,), (B, Lq), (1, Lq)):
            _refuse(f'positions must be int64 for {B} x {Lq} tokens, got {ps} {positions.dtype}')
        pos, psl = positions.data_ptr(), positions.stride(-1)
        psb = positions.stride(0) if len(ps) == 2 and ps[0] > 1 else 0
    if in_place:
        for t in (q, k):
            if t is not None and (t.stride(3) != 1 and D > 1 or any(st == 0 and n > 1 for st, n in zip(t.stride(), t.shape))):
                _refuse('in place, the elements of a head must be contiguous and heads must not be broadcast')
        qo, ko = q, k
    else:
        if D > 1 and q.stride(3) != 1:
            q = q.contiguous()
        qo, ko = q.new_empty((B, Lq, Hq, D)), None
        if k is not None:
            if D > 1 and k.stride(3) != 1:
                k = k.contiguous()
            ko = k.new_empty((B, Lq, Hk, D))
    if k is None:
        kp = kop = 0
        ks = kos = (0, 0, 0)
    else:
        kp, kop, ks, kos = k.data_ptr(), ko.data_ptr(), k.stride()[:3], ko.stride()[:3]
    args = _ROTARY.pack(q.data_ptr(), qo.data_ptr(), kp, kop, *q.stride()[:3], *qo.stride()[:3], *ks, *kos, pos, psb, psl, frequencies.data_ptr(),
                        B, Lq, Hq, Hk, D, rot, interleaved, inverse, dt, scale)
    _call(dev, 'sgpo_rotary', args)
    return qo, ko


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, frequencies, positions, interleaved, scale):
        ctx.save_for_backward(frequencies, positions)
        ctx.how = interleaved, scale
        return _rotate(q, k, frequencies, positions, interleaved, scale, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        frequencies, positions = ctx.saved_tensors
        return (*_rotate(dq, dk, frequencies, positions, *ctx.how, True), None, None, None, None)


def rotary_positions(q, k, frequencies, positions=None, interleaved=False, scale=1.0):
    """q (B, L, Hq, D) and k (B, L, Hk, D) (or None) with the first 2 * len(frequencies) elements of every head turned by their
    token's position; differentiable in q and k.  Returns new contiguous (q, k).

    frequencies and scale as rotary_frequencies gives them; positions int64 (L,), (B, L), (1, L) or None for 0 .. L - 1, of any size up to 2 ** 50; pairs are
    (j, j + rot / 2), or (2 j, 2 j + 1) if interleaved.  q and k may be views with any strides (of one packed projection, or of
    (B, H, L, D) tensors); only heads that are not contiguous in memory are copied first."""
    if not (torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad)):
        return _rotate(q, k, frequencies, positions, interleaved, scale, False)
    return _Rotary.apply(q, k, frequencies, positions, interleaved, scale)


def rotary_positions_(q, k, frequencies, positions=None, interleaved=False, scale=1.0):
    """rotary_positions written over q and k (as the reference's apply_rotary_emb_qkv_, dit.py:112-115); not differentiable."""
    if torch.is_grad_enabled() and (q.requires_grad or k is not None and k.requires_grad):
        _refuse('rotary_positions_ has no gradient: use rotary_positions')
    _rotate(q, k, frequencies, positions, interleaved, scale, False, in_place=True)
    torch.autograd.graph.increment_version(q if k is None else (q, k))     # what autograd saved of them is stale now
    return q, k


# -------------------------------------------------------------------------------------------------------------------- loss

def _loss_args(hidden, weight, targets, bias, ignore_index, reduction):
    N, H = hidden.shape
    V = weight.shape[0]
    return _LOSS.pack(hidden.data_ptr(), weight.data_ptr(), 0 if bias is None else bias.data_ptr(), targets.data_ptr(), hidden.stride(0) if N > 1 else H,
                      weight.stride(0) if V > 1 else H, ignore_index, N, H, V, _DTYPES[hidden.dtype], reduction)


def _rows(t):
    """A matrix with contiguous rows that do not overlap."""
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _loss_forward(hidden, weight, targets, bias, ignore_index, reduction):
    """(loss or losses, state for the backward pass: the tokens' log-sums, the gradient's factor, and losses that are only summed)."""
    dev = hidden.device
    N = hidden.shape[0]
    args = _loss_args(hidden, weight, targets, bias, ignore_index, reduction)
    need = L.load().sgpo_linear_ce_workspace_bytes(args, 0)
    buf, ws = _scratch(need, dev)
    state = torch.empty(2 * N + 1 if reduction else N + 1, dtype=torch.float32, device=dev)
    out = torch.empty((N,) if reduction == 0 else (), dtype=torch.float32, device=dev)
    lse = state.data_ptr()
    inv, o = lse + 4 * N, out.data_ptr()
    _call(dev, 'sgpo_linear_ce_forward', args, inv + 4 if reduction else o, lse, o, inv, ws, need)
    return out, state


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, bias, ignore_index, reduction):
        out, state = _loss_forward(hidden, weight, targets, bias, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, targets, bias, state)
        ctx.how = ignore_index, reduction
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, targets, bias, state = ctx.saved_tensors
        dev = hidden.device
        args = _loss_args(hidden, weight, targets, bias, *ctx.how)
        grad = grad.contiguous()
        want = ctx.needs_input_grad
        dh = hidden.new_empty(hidden.shape) if want[0] else None
        dw = weight.new_empty(weight.shape) if want[1] else None
        db = bias.new_empty(bias.shape) if want[3] else None
        need = L.load().sgpo_linear_ce_workspace_bytes(args, 1)
        buf, ws = _scratch(need, dev)
        lse = state.data_ptr()
        _call(dev, 'sgpo_linear_ce_backward', args, lse, grad.data_ptr(), lse + 4 * hidden.shape[0], None if dh is None else dh.data_ptr(),
              None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(), ws, need)
        return dh, dw, None, db, None, None


def linear_cross_entropy(hidden, weight, targets, bias=None, ignore_index=-100, reduction='mean'):
    """Cross entropy of softmax(hidden weight^T + bias) at targets without storing the logits; differentiable in hidden, weight
    and bias (once).

    hidden (..., H) and weight (V, H), both fp32 or both bf16; targets int64 of hidden's leading shape; bias fp32 (V,) or None, where -inf
    closes a class (the mask class of an absorbing-state model, mdlm_diffusion.py:325-341).  reduction 'none' gives fp32 losses of
    targets' shape; 'sum' and 'mean' (over the targets that are not ignore_index; 0 if there are none) give a scalar.  An ignored token has loss
    and gradients 0 whatever its features hold; a target outside [0, V) gives NaN, as no check on the host waits for the GPU."""
    _on_device(hidden, weight, targets, bias)
    _dtype(hidden, 'hidden')
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or weight.numel() == 0:
        _refuse(f'hidden {tuple(hidden.shape)} does not match weight {tuple(weight.shape)}')
    if weight.dtype != hidden.dtype:
        _refuse(f'hidden is {hidden.dtype} and weight {weight.dtype}')
    if targets.dtype != torch.int64 or targets.shape != hidden.shape[:-1]:
        _refuse(f'targets {tuple(targets.shape)} {targets.dtype} for hidden {tuple(hidden.shape)}')
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (weight.shape[0],)):
        _refuse('bias must be float32 with one value per class')
    if reduction not in _REDUCE:
        _refuse(f'unknown reduction {reduction!r}')
    red = _REDUCE[reduction]
    h = _rows(hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1]))
    w = _rows(weight)
    t = targets if targets.dim() == 1 and targets.is_contiguous() else targets.reshape(-1).contiguous()
    b = None if bias is None else bias.contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or bias is not None and bias.requires_grad):
        out = _LinearCrossEntropy.apply(h, w, t, b, int(ignore_index), red)
    else:
        out = _loss_forward(h, w, t, b, int(ignore_index), red)[0]
    return out.view(targets.shape) if red == 0 and targets.dim() != 1 else out


# ----------------------------------------------------------------------------------------------------------------- updates

_tables = {}     # coefficients -> their C array


def _coefficients(coefficients, steps):
    key = (tuple(map(tuple, coefficients)) if isinstance(coefficients[0], (tuple, list)) else tuple(coefficients), steps)
    table = _tables.get(key)
    if table is None:
        rows = key[0] if isinstance(key[0][0], tuple) else (key[0],) * max(steps, 0)
        flat = [float(v) for row in rows for v in row]
        if steps < 1 or len(rows) != steps or len(flat) != 3 * steps:
            _refuse(f'{steps} steps need {steps} coefficient triples')
        if len(_tables) >= 64:
            _tables.clear()
        table = _tables[key] = (L.C.c_float * len(flat))(*flat)
    return table


def newton_schulz(update, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """The update (..., m, n) with every singular value moved towards 1 and its singular vectors kept: X = U / (|U|_F + eps), then
    X <- a X + (b X X^T + c (X X^T)^2) X per coefficient triple (one triple for all steps, or one each).  Leading dimensions are independent matrices.
    update fp32 or bf16; returns bf16, contiguous.  Iterates carry 17 bits, sums 32, the norm 64.  Not differentiable."""
    dev = _on_device(update)
    dt = _dtype(update, 'update')
    if update.dim() < 2:
        _refuse(f'an update is a matrix or a batch of them, got {tuple(update.shape)}')
    u = update.detach()
    m, n = u.shape[-2:]
    out = torch.empty(u.shape, dtype=torch.bfloat16, device=dev)
    table = _coefficients(coefficients, steps)
    if not u.numel():
        return out
    if u.dim() == 2:
        batch, sb, ld = 1, 0, u.stride(0)
    else:
        u = u.reshape(-1, m, n)
        batch, sb, ld = u.shape[0], u.stride(0), u.stride(1)
    if u.stride(-1) != 1 and n > 1 or m > 1 and ld < n:
        u = u.contiguous()
        sb, ld = m * n, n
    need = L.load().sgpo_newton_schulz_workspace_bytes(batch, m, n)
    buf, ws = _scratch(need, dev)
    _call(dev, 'sgpo_newton_schulz', u.data_ptr(), dt, batch, m, n, sb, ld, table, steps, eps, out.data_ptr(), ws, need)
    return out


def muon_step(weight, grad, momentum_buffer, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NS_COEFFICIENTS,
              eps=1e-7):
    """One optimiser step of weight (..., m, n), in place, with an orthogonalised momentum update; leading dimensions are
    independent matrices.

    buffer = momentum * buffer + grad;  U = grad + momentum * buffer (nesterov) or buffer;  weight = (1 - lr * weight_decay) * weight -
    lr * sqrt(max(1, m / n)) * newton_schulz(U), the last product not rounded before it is applied.  weight and grad fp32 or bf16,
    momentum_buffer fp32 (the caller's state, zeros at first); weight and buffer contiguous.  Returns weight."""
    dev = _on_device(weight, grad, momentum_buffer)
    wd, gd = _dtype(weight, 'weight'), _dtype(grad, 'grad')
    if weight.dim() < 2 or not weight.shape == grad.shape == momentum_buffer.shape:
        _refuse(f'weight {tuple(weight.shape)}, grad {tuple(grad.shape)} and buffer {tuple(momentum_buffer.shape)} must agree')
    if momentum_buffer.dtype != torch.float32:
        _refuse('momentum_buffer must be float32')
    if not (weight.is_contiguous() and momentum_buffer.is_contiguous()):
        _refuse('weight and momentum_buffer are updated in place and must be contiguous')
    if torch.is_grad_enabled() and weight.requires_grad and not weight.is_leaf:
        _refuse('weight is part of a graph: a step updates leaves')
    table = _coefficients(coefficients, steps)
    if not weight.numel():
        return weight
    g = grad.detach().contiguous()
    m, n = weight.shape[-2:]
    batch = weight.numel() // (m * n)
    need = L.load().sgpo_newton_schulz_workspace_bytes(batch, m, n)
    buf, ws = _scratch(need, dev)
    _call(dev, 'sgpo_muon_step', weight.data_ptr(), wd, g.data_ptr(), gd, momentum_buffer.data_ptr(), batch, m, n, lr, momentum, bool(nesterov), weight_decay,
                            table, steps, eps, ws, need)
    torch.autograd.graph.increment_version((weight, momentum_buffer))     # what autograd saved of them is stale now
    return weight
