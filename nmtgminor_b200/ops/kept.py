"""Activations that wait for the backward pass in 8 bits.

Blocks of 32 elements along a row share a power of two, the smallest that brings the block's largest magnitude to 448 or less; an element is a
number of 4 exponent and 3 mantissa bits (33 bytes for 32 elements).  A restored element is off by at most 2^-4 of itself, or 2^-10 of the
block's unit where it is smaller than 2^-6 of it.  Infinities and NaN come back as NaN.

* ``quantise`` / ``restore``   the codes of a matrix (bf16, fp16, fp32) and their values;
* ``activation``              ``dropout(act(z))`` that keeps ``z`` so: the forward pass uses ``z`` itself, only the slope of the backward pass is that of
  the kept value;
* ``ops.linear(..., keep8=True)`` and ``ops.mlp(..., keep8=True)`` keep their inputs so (see there).

On a GPU ``csrc/kept8.cu``, one pass each; the plain PyTorch restatements below run on the CPU and are the tests' oracle.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

BLOCK = 32
_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_ACTS = {"none": 0, None: 0, "relu": 1, "gelu": 2, "silu": 3, "swish": 3}


class Kept:
    """A matrix in 8 bits: ``codes`` [rows, 32 * blocks] and ``scales`` [rows, blocks] (bytes: exponent + 127)."""

    __slots__ = ("codes", "scales", "width", "dtype")

    def __init__(self, codes, scales, width, dtype):
        self.codes, self.scales, self.width, self.dtype = codes, scales, width, dtype

    @property
    def shape(self):
        return (self.codes.shape[0], self.width)

    def nbytes(self):
        return self.codes.numel() + self.scales.numel()


# ---------------------------------------------------------------------------------------------------
# plain restatements
# ---------------------------------------------------------------------------------------------------
def quantise_reference(x):
    rows, width = x.shape
    full = F.pad(x.detach().float(), (0, -width % BLOCK)).view(rows, -1, BLOCK)
    finite = torch.isfinite(full)
    fraction, exponent = torch.frexp(torch.where(finite, full, torch.zeros_like(full)).abs().amax(-1, keepdim=True))
    exponent = torch.where(fraction > 0.875, exponent - 8, exponent - 9).clamp(min=-127)         # 448 = 0.875 * 2^9
    exponent = torch.where(fraction == 0, torch.full_like(exponent, -127), exponent)
    scaled = torch.where(finite, torch.ldexp(full.double(), -exponent), torch.full_like(full, float("nan"), dtype=torch.float64))
    codes = scaled.float().to(torch.float8_e4m3fn).view(torch.uint8)
    return Kept(codes.view(rows, -1), (exponent + 127).to(torch.uint8).view(rows, -1), width, x.dtype)


def restore_reference(kept, dtype=None):
    dtype = kept.dtype if dtype is None else dtype
    rows, blocks = kept.scales.shape
    v = kept.codes.view(torch.float8_e4m3fn).float().view(rows, blocks, BLOCK).double()
    v = torch.ldexp(v, kept.scales.int()[..., None] - 127).view(rows, -1)[:, :kept.width]
    most = torch.finfo(dtype).max
    return torch.where(torch.isnan(v), v, v.clamp(-most, most)).to(dtype)


def straight_through(x):
    """The kept value of ``x`` as autograd sees ``x``: the gradient passes unchanged."""
    held = restore_reference(quantise_reference(x)).to(x.dtype)
    return x + (held - x).detach()


def linear_reference(x, weight, bias):
    """``x W^T + b`` with the weight's gradient taken from the kept ``x``."""
    y = F.linear(x, weight.detach(), bias)
    if not (torch.is_grad_enabled() and weight.requires_grad):
        return y
    kept = F.linear(restore_reference(quantise_reference(x)).to(x.dtype), weight)
    return y + (kept - kept.detach())


def act_reference(z, act_id):
    """``act(z)`` with the slope taken at the kept ``z``."""
    from .reference import _act
    if not (torch.is_grad_enabled() and z.requires_grad):
        return _act(z, act_id)
    kept = _act(straight_through(z), act_id)
    return _act(z.detach(), act_id) + (kept - kept.detach())


# ---------------------------------------------------------------------------------------------------
# codes
# ---------------------------------------------------------------------------------------------------
def _check(x, name):
    if x.dim() != 2:
        raise ValueError("%s must be a matrix, got %s" % (name, tuple(x.shape)))
    if x.dtype not in _TYPES:
        raise TypeError("%s must be bfloat16, float16 or float32, not %s" % (name, x.dtype))


def _rows(x):
    return x if x.stride(1) == 1 and (x.shape[0] <= 1 or x.stride(0) >= x.shape[1]) else x.contiguous()


def _ext(launches=1):
    from . import LAUNCHES, ext
    LAUNCHES[0] += launches
    return ext()


def quantise(x) -> Kept:
    """The codes of a matrix."""
    _check(x, "x")
    if not x.is_cuda:
        return quantise_reference(x)
    codes, scales = _ext().kept_quantise(_rows(x.detach()))
    return Kept(codes, scales, x.shape[1], x.dtype)


def restore(kept: Kept, dtype=None):
    """The values of codes, in the type that was kept or another."""
    dtype = kept.dtype if dtype is None else dtype
    if dtype not in _TYPES:
        raise TypeError("the type must be bfloat16, float16 or float32, not %s" % dtype)
    if not kept.codes.is_cuda:
        return restore_reference(kept, dtype)
    return _ext().kept_restore(kept.codes, kept.scales, kept.width, dtype, True, -1, 0.0, 0, 0)[0]


def restore_activated(kept: Kept, act_id: int, p: float, seed: int, stream_id: int, plain: bool):
    """(x' where ``plain``, dropout(act(x'))) on a GPU, with the mask that ``dropout_add`` draws for the seed and stream."""
    return _ext().kept_restore(kept.codes, kept.scales, kept.width, kept.dtype, plain, act_id, p, seed, stream_id)


# ---------------------------------------------------------------------------------------------------
# activation
# ---------------------------------------------------------------------------------------------------
def activation(z, act="gelu", dropout_p: float = 0.0, training: bool = True):
    """``dropout(act(z))`` of a matrix whose backward pass takes the slope at the kept ``z``; nothing is kept where no gradient is asked for.
    ``act``: "none", "relu", "gelu" (erf) or "silu"."""
    _check(z, "z")
    if act not in _ACTS:
        raise ValueError("unknown activation %r" % (act,))
    p = float(dropout_p) if training else 0.0
    if not 0.0 <= p < 1.0:
        raise ValueError("dropout must be in [0, 1)")
    act_id = _ACTS[act]
    if not z.is_cuda:
        y = act_reference(z, act_id)
        return F.dropout(y, p, True) if p > 0 else y
    from . import _Rng, next_stream
    sid = next_stream() if p > 0 else 0
    x = _rows(z)
    if torch.is_grad_enabled() and z.requires_grad:
        return _ext(2).activation_node(x, act_id, p, _Rng.seed, sid)
    return _ext().kept_forward(x, act_id, False, p, _Rng.seed, sid)[0]
