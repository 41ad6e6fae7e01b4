"""Rotary positions of queries and keys over the HIP kernels.

``rotary_embedding(q, k, positions, frequencies, *, interleaved=False, magnitude=1.0, out_q=None, out_k=None)`` turns
pair i of the first ``2 * len(frequencies)`` values of every head by the angle ``positions[t] * frequencies[i]``:
(a, b) -> (a cos - b sin, b cos + a sin) * magnitude. Pairs are (i, i + r/2), or (2i, 2i + 1) when ``interleaved``; the
other values pass through. Angles are taken in 64 bits, so they are right at any position; the rotation is in fp32,
rounded once. The reference has no such op in this library's scope.

  q, k: bf16, fp16 or fp32 [tokens, heads, head_dim]; k may be None. Views serve as long as the last dimension is
  contiguous and everything else lies on 16 bytes, so the rotated part of a wider head is ``q[..., 128:]``.
  positions: int32 or int64 [tokens]; frequencies: fp64 [rotary_dim / 2] (``rotary_frequencies``), rotary_dim a
  multiple of 16. ``out_q``/``out_k``: where results go, q and k themselves for in place.

``rotary_frequencies`` builds the frequencies, plain or scaled for contexts longer than those a model was trained on.

Calls it does not serve return a ``FallbackReason``; so does a call that wants gradients or
tangents: these ops are for inference.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch.autograd import forward_ad

from . import _lib
from .dispatch import FallbackReason, aligned, api, on_gpu

_OOC = FallbackReason.OUT_OF_CONTRACT
_DTYPES = {torch.bfloat16: _lib.OUT_BF16, torch.float16: _lib.OUT_F16, torch.float32: _lib.F32}
_MAX_HEADS = 32768


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None, beta_fast=32.0,
                       beta_slow=1.0, device=None):
    """fp64 [rotary_dim / 2]: radians a position turns each pair by, ``base ** (-2 i / rotary_dim)``, and for contexts
    ``factor`` times longer than ``original_length``, the one trained on, by ``scaling``:

    - ``"linear"``: every frequency divided by the factor;
    - ``"ntk"``: a larger base, so that the slowest frequency is divided by the factor and the fastest stays;
    - ``"yarn"``: by parts. Pairs that turn ``beta_fast`` times or more over the original length stay, those that turn
      ``beta_slow`` times or less are divided by the factor, and a ramp over the pairs' index lies between.
      ``rotary_magnitude`` gives its factor of cos and sin."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim has to be even and positive, got {rotary_dim}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling is None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if not (base > 1 and factor >= 1):
        raise ValueError(f"base has to be above 1 and factor at least 1, got {base} and {factor}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = base ** -(i / rotary_dim)
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        if not original_length or original_length <= 0:
            raise ValueError("scaling 'yarn' needs the original_length")

        def index(turns):  # of the pair that turns this often over the original length
            return rotary_dim * math.log(original_length / (2 * math.pi * turns)) / (2 * math.log(base))

        low = max(math.floor(index(beta_fast)), 0)
        high = min(math.ceil(index(beta_slow)), rotary_dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
    return f.to(device) if device is not None else f


def rotary_magnitude(factor, scale=1.0):
    """The factor of cos and sin that belongs to ``"yarn"`` frequencies: 0.1 * scale * ln(factor) + 1."""
    return 0.1 * scale * math.log(factor) + 1.0 if factor > 1 else 1.0


# ---------------------------------------------------------------------------------------------
# checks shared with the cache ops
def wants_grad(*tensors) -> bool:
    """Whether a gradient, or the tangent of forward mode, would be lost."""
    given = [t for t in tensors if t is not None]
    return (torch.is_grad_enabled() and any(t.requires_grad for t in given)) or any(
        forward_ad.unpack_dual(t).tangent is not None for t in given)


def tensors_ok(*tensors) -> bool:
    """Whether all are tensors with memory of their own: a function transform's (vmap, jvp, grad) have none to name."""
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            return False
        try:
            t.data_ptr()
        except RuntimeError:
            return False
    return True


def vectors_ok(t, tokens, heads, head_dim, dtype) -> bool:
    """A [tokens, heads, head_dim] tensor the kernels can read: 16-byte pieces along the last dimension."""
    if t.dim() != 3 or tuple(t.shape) != (tokens, heads, head_dim) or t.dtype != dtype or t.layout != torch.strided:
        return False
    if t.stride(2) != 1 or not aligned(t):
        return False
    size = t.element_size()
    return t.stride(0) * size % 16 == 0 and t.stride(1) * size % 16 == 0


def no_inner_overlap(t) -> bool:
    """Whether no two elements of a strided tensor share memory (a sufficient test)."""
    span = 1
    for size, stride in sorted(((s, st) for s, st in zip(t.shape, t.stride()) if s > 1), key=lambda p: p[1]):
        if stride < span:
            return False
        span += (size - 1) * stride
    return True


def _span(t, dims) -> int:
    return (1 + sum((t.shape[d] - 1) * t.stride(d) for d in dims)) * t.element_size()


def apart(a, b) -> bool:
    """Whether two tensors share no memory: their ranges do not meet, or they are pieces of the same rows (queries and
    keys of one projection, keys and values of one allocation of pages) that do not meet within a row."""
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return True
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + _span(a, range(a.dim())) <= pb or pb + _span(b, range(b.dim())) <= pa:
        return True
    row = a.stride(0) * a.element_size()
    if a.dim() < 2 or b.dim() < 2 or row == 0 or row != b.stride(0) * b.element_size():
        return False
    gap = (pb - pa) % row
    return _span(a, range(1, a.dim())) <= gap and gap + _span(b, range(1, b.dim())) <= row


def same_place(a, b) -> bool:
    return a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype


def flag_ok(x) -> bool:
    return not hasattr(x, "__len__") and x in (True, False)


def number_ok(x) -> bool:
    """A number that fp32 holds, with room for the kernels' factor of log2(e)."""
    return isinstance(x, (int, float)) and abs(x) <= 2.0**127


def rotary_ok(positions, frequencies, interleaved, magnitude, tokens, head_dim) -> bool:
    if not flag_ok(interleaved) or not number_ok(magnitude):
        return False
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) != (tokens,) or not positions.is_contiguous():
        return False
    if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous() or wants_grad(frequencies):
        return False
    rot = 2 * frequencies.numel()
    return 16 <= rot <= head_dim and rot % 16 == 0


def stream(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


# ---------------------------------------------------------------------------------------------
@dataclass
class _RotaryPlan:
    q: torch.Tensor
    k: torch.Tensor | None
    positions: torch.Tensor
    frequencies: torch.Tensor
    interleaved: bool
    magnitude: float
    out_q: torch.Tensor | None
    out_k: torch.Tensor | None
    variant: str
    kernel_ref: str = "aklr_rotary_embedding"


def _run_rotary(p: _RotaryPlan):
    q, k = p.q, p.k
    out_q = p.out_q if p.out_q is not None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    out_k = p.out_k
    if k is not None and out_k is None:
        out_k = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    tokens, heads, head_dim = q.shape
    if tokens:
        kt = (None, 0, 0, None, 0, 0, 0)
        if k is not None:
            kt = (k.data_ptr(), k.stride(0), k.stride(1), out_k.data_ptr(), out_k.stride(0), out_k.stride(1), k.shape[1])
        with torch.cuda.device(q.device):
            st = _lib.lib().aklr_rotary_embedding(
                q.data_ptr(), q.stride(0), q.stride(1), out_q.data_ptr(), out_q.stride(0), out_q.stride(1), heads, *kt,
                p.positions.data_ptr(), int(p.positions.dtype == torch.int64), p.frequencies.data_ptr(), tokens, head_dim,
                2 * p.frequencies.numel(), int(p.interleaved), p.magnitude, _DTYPES[q.dtype], stream(q.device))
        _lib.check(st, "rotary_embedding")
    return out_q, out_k


@api("rotary_embedding@1.0", _run_rotary, native="rotary")
def rotary_embedding(q, k, positions, frequencies, *, interleaved=False, magnitude=1.0, out_q=None, out_k=None):
    given = [q, positions, frequencies] + [t for t in (k, out_q, out_k) if t is not None]
    if not tensors_ok(*given):
        return _OOC
    if q.dim() != 3 or q.dtype not in _DTYPES or (k is None and out_k is not None):
        return _OOC
    tokens, heads, head_dim = q.shape
    if not (1 <= heads <= _MAX_HEADS and 16 <= head_dim <= 1024 and head_dim % 16 == 0 and tokens < 2**31):
        return _OOC
    if not vectors_ok(q, tokens, heads, head_dim, q.dtype):
        return _OOC
    if k is not None and (k.dim() != 3 or not 1 <= k.shape[1] <= _MAX_HEADS or not vectors_ok(k, tokens, k.shape[1], head_dim, q.dtype)):
        return _OOC
    if not rotary_ok(positions, frequencies, interleaved, magnitude, tokens, head_dim):
        return _OOC
    if not on_gpu(*given) or wants_grad(q, k, out_q, out_k):
        return _OOC
    for out, like, other in ((out_q, q, k), (out_k, k, q)):
        if out is None:
            continue
        if not vectors_ok(out, tokens, like.shape[1], head_dim, q.dtype) or not no_inner_overlap(out):
            return _OOC
        if not all(apart(out, t) for t in (other, positions, frequencies)) or not (same_place(out, like) or apart(out, like)):
            return _OOC
    if not apart(out_q, out_k):
        return _OOC
    return _RotaryPlan(q, k, positions, frequencies, interleaved, float(magnitude), out_q, out_k,
                       "interleaved" if interleaved else "half")
