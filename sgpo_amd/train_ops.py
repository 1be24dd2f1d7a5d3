"""Training operators of a denoiser on the GPU: position rotation of query and key heads, the cross entropy of a linear
vocabulary head without its logits, and updates orthogonalised by Newton-Schulz products.

The reference trains its denoisers through torch autograd (models/pretraining/trainer.py:75-88) with these steps as chains of
torch kernels; here each is one call into libsgpo_hip.so.  PyTorch is plumbing (device memory, the current HIP stream, the autograd
tape).  Every tensor is fp32 or bf16 device memory on the process's one GPU; a call runs on the stream that is current on that
device, allocates its outputs and scratch from torch's allocator (so it can be captured into a graph and used on any stream), and
does not synchronise.  There is no CPU fallback: bad arguments and host tensors raise SgpoError, and so do inputs with a forward-mode tangent
everywhere but in rotary_positions.
"""
import importlib
import math

import torch

from . import _lib as L

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # Newton-Schulz quintic: singular values into about [0.7, 1.2] within 5 steps
_ops = None


def _load():
    """The host side of the operators (csrc/torch_ops.cpp), bound to the library that _lib loaded."""
    global _ops
    if _ops is None:
        lib = L.load()
        try:
            ops = importlib.import_module('sgpo_amd._sgpo_torch')
        except ImportError as e:
            raise L.SgpoError(f'sgpo_amd/_sgpo_torch.so is not built or does not match this torch ({e}): build it with '
                              f'`make -C sgpo_amd/csrc`. There is no fallback.') from e
        ops.bind({n: L.C.cast(getattr(lib, n), L.C.c_void_p).value for n in (
            'sgpo_init', 'sgpo_last_error', 'sgpo_rotary', 'sgpo_linear_ce_workspace_bytes', 'sgpo_linear_ce_forward', 'sgpo_linear_ce_backward',
            'sgpo_newton_schulz_workspace_bytes', 'sgpo_newton_schulz', 'sgpo_muon_step')}, L.SgpoError)
        _ops = ops
    return _ops


def _refuse(text):
    raise L.SgpoError(text)


# ---------------------------------------------------------------------------------------------------------------- rotation

def rotary_frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0,
                       device='cuda'):
    """(frequencies float64 (rotary_dim / 2,), scale): the angle per position of each pair, base ** (-2 j / rotary_dim) as in the
    reference's Rotary (dit.py:81-107), stretched for contexts longer than the original one.

    scaling None; 'linear': every angle / factor; 'ntk': base * factor ** (rotary_dim / (rotary_dim - 2)), which keeps the fastest pair
    and divides the slowest by factor; 'yarn': pairs that turn more than beta_fast times within original_length positions stay, those
    below beta_slow turns are divided by factor, in between linearly in the number of turns, and rotated elements are scaled by 0.1 ln(factor) + 1.
    That is the published formula.  Programs that ramp linearly in the pair's index, between the rounded indices of the two bounds, give the pairs
    in between other frequencies: for a model trained so, pass its own float64 tensor to rotary_positions."""
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


def rotary_positions(q, k, frequencies, positions=None, interleaved=False, scale=1.0):
    """q (B, L, Hq, D) and k (B, L, Hk, D) (or None) with the first 2 * len(frequencies) elements of every head turned by their
    token's position; differentiable in q and k any number of times, in reverse and forward mode.  Returns new contiguous (q, k).

    frequencies and scale as rotary_frequencies gives them; positions int64 (L,), (B, L), (1, L) or None for 0 .. L - 1, up to 2 ** 50: an
    angle is position * frequency rounded to 64 bits, off by up to 2 ** -53 of itself (2 ** -24 radian at 2 ** 29, 2 ** -13 at 2 ** 40).
    Pairs are (j, j + rot / 2), or (2 j, 2 j + 1) if interleaved.  q and k may be views with any strides (of one packed projection, or of
    (B, H, L, D) tensors); only heads that are not contiguous in memory are copied first."""
    return (_ops or _load()).rotary_positions(q, k, frequencies, positions, interleaved, scale)


def rotary_positions_(q, k, frequencies, positions=None, interleaved=False, scale=1.0):
    """rotary_positions written over q and k (as the reference's apply_rotary_emb_qkv_, dit.py:112-115); not differentiable."""
    (_ops or _load()).rotary_positions_(q, k, frequencies, positions, interleaved, scale)
    return q, k


# -------------------------------------------------------------------------------------------------------------------- loss

def linear_cross_entropy(hidden, weight, targets, bias=None, ignore_index=-100, reduction='mean'):
    """Cross entropy of softmax(hidden weight^T + bias) at targets without storing the logits; differentiable in hidden, weight
    and bias (once).

    hidden (..., H) and weight (V, H), both fp32 or both bf16; targets int64 of hidden's leading shape; bias (V,), fp32 or of weight's type, or None,
    where -inf closes a class (the mask class of an absorbing-state model, mdlm_diffusion.py:325-341).  reduction 'none' gives fp32 losses of
    targets' shape; 'sum' and 'mean' (over the targets that are not ignore_index; 0 if there are none) give a scalar.  An ignored token has loss
    and gradients 0 whatever its features hold; a target outside [0, V) gives NaN, as no check on the host waits for the GPU."""
    return (_ops or _load()).linear_cross_entropy(hidden, weight, targets, bias, ignore_index, reduction)


# ----------------------------------------------------------------------------------------------------------------- updates

_tables = {}     # coefficients -> one flat list


def _coefficients(coefficients, steps):
    if len(coefficients) == 0:
        _refuse(f'{steps} steps need {steps} coefficient triples')
    key = (tuple(map(tuple, coefficients)) if isinstance(coefficients[0], (tuple, list)) else tuple(coefficients), steps)
    table = _tables.get(key)
    if table is None:
        rows = key[0] if isinstance(key[0][0], tuple) else (key[0],) * max(steps, 0)
        flat = [float(v) for row in rows for v in row]
        if steps < 1 or len(rows) != steps or len(flat) != 3 * steps:
            _refuse(f'{steps} steps need {steps} coefficient triples')
        if len(_tables) >= 64:
            _tables.clear()
        table = _tables[key] = flat
    return table


def newton_schulz(update, steps=5, coefficients=NS_COEFFICIENTS, eps=1e-7):
    """The update (..., m, n) with every singular value moved towards 1 and its singular vectors kept: X = U / (|U|_F + eps), then
    X <- a X + (b X X^T + c (X X^T)^2) X per coefficient triple (one triple for all steps, or one each).  Leading dimensions are independent matrices.
    update fp32 or bf16; returns bf16, contiguous.  Iterates carry at least 17 bits, sums 32, the norm 64.  Not differentiable."""
    return (_ops or _load()).newton_schulz(update, steps, _coefficients(coefficients, steps), eps)


def muon_step(weight, grad, momentum_buffer, lr, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=NS_COEFFICIENTS,
              eps=1e-7):
    """One optimiser step of weight (..., m, n), in place, with an orthogonalised momentum update; leading dimensions are
    independent matrices.

    buffer = momentum * buffer + grad;  U = grad + momentum * buffer (nesterov) or buffer;  weight = (1 - lr * weight_decay) * weight -
    lr * sqrt(max(1, m / n)) * newton_schulz(U), the last product not rounded before it is applied.  weight and grad fp32 or bf16,
    momentum_buffer fp32 (the caller's state, zeros at first); weight and buffer contiguous.  Returns weight."""
    (_ops or _load()).muon_step(weight, grad, momentum_buffer, lr, momentum, nesterov, weight_decay, steps, _coefficients(coefficients, steps), eps)
    return weight
