"""Operators around the products of a training step: layer norm, rotary positions, and the global gradient norm with clipping.

On a GPU each runs on the kernels of `csrc/layernorm.cu`, `csrc/rotary.cu` and `csrc/clip.cu` (current stream of the tensors' device; capturable into a
CUDA graph; first derivatives only, backward; fake and wrapped tensors are refused, so a sharded one goes in as its local part); tensors in host memory take the plain
PyTorch formulas below, which are the specification.
"""
import math

import torch

from . import load

FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _require(ok, message):
    if not ok:
        raise ValueError(message)


# ---- layer norm ---------------------------------------------------------------------------------------------------------------
def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension (biased variance), statistics and sums in fp32.

    x: fp32, bf16 or fp16, any leading dimensions and strides.  weight, bias: vectors of the last dimension's length in any of these types, either may be
    absent.  The result has x's type, or bf16 (`out_dtype`) for an fp32 x.  Gradients of x, weight and bias come in their types; the sums over rows
    are fp32 and have the same bits in every run."""
    if x.is_cuda:                                # checked there
        return load().layer_norm(x, weight, bias, eps, out_dtype)
    dim = x.shape[-1] if x.dim() else 0
    _require(dim > 0, "layer_norm: an input with a last dimension that is not empty is required")
    _require(x.dtype in FLOATS, f"layer_norm: fp32, bf16 or fp16 input required, got {x.dtype}")
    _require(out_dtype is None or out_dtype == x.dtype or (x.dtype == torch.float32 and out_dtype == torch.bfloat16),
             "layer_norm: out_dtype is the input's type, or bf16 for an fp32 input")
    _require(eps >= 0, "layer_norm: eps must not be negative")
    for p in (weight, bias):
        if p is not None:
            _require(p.dim() == 1 and p.shape[0] == dim and p.device == x.device and p.dtype in FLOATS,
                     "layer_norm: weight and bias are fp32, bf16 or fp16 vectors of the last dimension's length on the input's device")
    xf = x.float()
    centred = xf - xf.mean(-1, keepdim=True)
    y = centred * torch.rsqrt(centred.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(out_dtype or x.dtype)


# ---- rotary positions ------------------------------------------------------------------------------------------------------------
def rotary_frequencies(rotary_dim, theta=10000.0, scaling=None, device=None):
    """Angles per position of the ``rotary_dim / 2`` rotated pairs (64 bits) and the factor on the rotated values, as `rotary` takes them.

    ``f_i = theta ** (-2 i / rotary_dim)``.  `scaling` stretches them for contexts beyond the trained length, a dict with ``rope_type`` and ``factor`` s:

    * ``"linear"``: every angle divided by s (position interpolation);
    * ``"ntk"``: theta grows to ``theta * s ** (r / (r - 2))``, so the slowest pair turns s times slower and the fastest as before;
    * ``"yarn"``: pairs that make more than ``beta_fast`` turns (32) in ``original_max_position_embeddings`` positions stay, those below
      ``beta_slow`` (1) are divided by s (Peng et al., "YaRN", 2023).  The ramp between is linear in the pair's index, as published models use it, where the paper's
      is linear in the number of turns; its ends are rounded outwards to whole pairs unless ``truncate`` is false.  The factor is ``attention_factor``, or ``0.1 ln s + 1``."""
    _require(rotary_dim > 0 and rotary_dim % 2 == 0, "rotary_frequencies: an even number of rotated dimensions is required")
    _require(theta > 1, "rotary_frequencies: theta must be above 1")
    scaling = dict(scaling or {})
    kind, s = scaling.pop("rope_type", "default"), float(scaling.pop("factor", 1.0))
    length, fast, slow = scaling.pop("original_max_position_embeddings", None), float(scaling.pop("beta_fast", 32.0)), float(scaling.pop("beta_slow", 1.0))
    truncate, magnitude = scaling.pop("truncate", True), scaling.pop("attention_factor", None)
    _require(not scaling, f"rotary_frequencies: unknown scaling fields {sorted(scaling)}")
    _require(kind in ("default", "linear", "ntk", "yarn"), f"rotary_frequencies: unknown rope_type {kind!r}")
    _require(math.isfinite(s) and s >= 1, "rotary_frequencies: the factor must be finite and at least 1")
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    if kind == "ntk" and rotary_dim > 2:
        theta = theta * s ** (rotary_dim / (rotary_dim - 2))
    f = torch.exp(pair * (-2.0 / rotary_dim * math.log(theta)))
    if kind == "linear":
        f = f / s
    elif kind == "yarn":
        _require(length is not None and length > 0, "rotary_frequencies: yarn needs original_max_position_embeddings")
        _require(fast > slow > 0, "rotary_frequencies: yarn needs beta_fast > beta_slow > 0")
        at = lambda turns: rotary_dim * math.log(length / (2 * math.pi * turns)) / (2 * math.log(theta))       # the pair that makes `turns` turns
        first, last = at(fast), at(slow)
        if truncate:
            first, last = math.floor(first), math.ceil(last)
        first, last = max(first, 0), min(last, rotary_dim - 1)
        slowed = ((pair - first) / max(last - first, 1e-3)).clamp(0, 1)
        f = f * (1 - slowed) + f / s * slowed
    if magnitude is None:
        magnitude = 0.1 * math.log(s) + 1.0 if kind == "yarn" else 1.0
    return f.to(device or "cpu"), float(magnitude)


def _rotate(x, cos, sin, interleaved):
    r = 2 * cos.shape[-1]
    xf = x.float()
    a, b = (xf[..., 0:r:2], xf[..., 1:r:2]) if interleaved else (xf[..., :r // 2], xf[..., r // 2:r])
    pair = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
    return torch.cat([turned, xf[..., r:]], -1).to(x.dtype)


def rotary(q, k, positions, frequencies, magnitude=1.0, interleaved=False):
    """Rotary positions of queries and keys: each pair of a head turned by ``position * frequency`` and scaled by `magnitude`.

    q: ``[batch, seq, heads, dim]`` or ``[tokens, heads, dim]``; k: the same with a head count of its own, or None.  bf16, fp16 or fp32, any strides (a head-major
    tensor goes in as ``x.transpose(1, 2)``, a packed projection as slices); results have the layout of their input.  positions: whole numbers ``[seq]``
    or ``[batch, seq]`` (``[tokens]``), of any size and sign; angles are formed in 64 bits.  frequencies: ``rotary_dim / 2`` values in 64 bits
    (`rotary_frequencies`), which get no gradient: ones that want it are refused.  Dimensions from rotary_dim on pass through.  A pair is
    ``(x[i], x[i + rotary_dim / 2])``, interleaved ``(x[2 i], x[2 i + 1])``."""
    if q.dim() == 3:
        _require(k is None or k.dim() == 3, "rotary: queries and keys have the same number of dimensions")
        q2, k2 = rotary(q.unsqueeze(0), None if k is None else k.unsqueeze(0), positions, frequencies, magnitude, interleaved)
        return q2.squeeze(0), None if k2 is None else k2.squeeze(0)
    if q.is_cuda:                                # checked there
        out = load().rotary(q, k, positions, frequencies, magnitude, interleaved)
        return (out[0], out[1]) if k is not None else (out[0], None)
    _require(q.dim() == 4 and q.dtype in FLOATS, "rotary: fp32, bf16 or fp16 queries [batch, seq, heads, dim] required")
    B, S, _, D = q.shape
    if k is not None:
        _require(k.dim() == 4 and k.dtype == q.dtype and k.device == q.device and k.shape[:2] == (B, S) and k.shape[3] == D,
                 "rotary: keys have the type, device, batch, length and head size of the queries")
    _require(positions.dtype in (torch.int64, torch.int32) and positions.device == q.device and positions.shape in ((S,), (1, S), (B, S)),
             "rotary: whole positions [seq] or [batch, seq] on the queries' device required")
    _require(frequencies.dtype == torch.float64 and frequencies.device == q.device and frequencies.dim() == 1 and 2 * frequencies.shape[0] <= D,
             "rotary: 64-bit frequencies on the queries' device, at most half a head of them, required")
    _require(not (torch.is_grad_enabled() and not torch.is_inference_mode_enabled() and frequencies.requires_grad), "rotary: a gradient of the frequencies is not available; detached ones are required")
    angle = positions.double()[..., None, None] * frequencies
    cos, sin = (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()
    return _rotate(q, cos, sin, interleaved), None if k is None else _rotate(k, cos, sin, interleaved)


# ---- gradient norm and clipping ------------------------------------------------------------------------------------------------------
def _gradients(grads, out=None):
    if type(grads) is list and (out is None or type(out) is list and len(out) == len(grads)) and grads and all([g is not None for g in grads]):
        return grads, out
    grads = [grads] if torch.is_tensor(grads) else list(grads)
    if out is not None:
        out = [out] if torch.is_tensor(out) else list(out)
        _require(len(out) == len(grads), "clip_grad_norm: as many results as gradients required")
        out = [o for o, g in zip(out, grads) if g is not None]
    grads = [g for g in grads if g is not None]
    _require(grads, "clip_grad_norm: at least one gradient required")
    return grads, out


def _check_host(grads, out):
    """What the kernels' host side checks for CUDA tensors, for tensors in host memory."""
    _require(all(g.device == grads[0].device for g in grads), "clip_grad_norm: gradients on one device required")
    _require(all(g.dtype in FLOATS for g in grads), "clip_grad_norm: fp32, bf16 or fp16 gradients required")
    span = lambda t: (t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
    _require(all(torch.ops.aten.is_non_overlapping_and_dense(g) for g in grads), "clip_grad_norm: gradients without gaps or overlaps in memory required")
    if out is not None:
        _require(all(o.device == g.device and o.dtype == g.dtype and o.shape == g.shape and (o.stride() == g.stride() or (o.is_contiguous() and g.is_contiguous()))
                     for o, g in zip(out, grads)), "clip_grad_norm: a result has its gradient's device, type, shape and layout")
    written = sorted(span(t) for t in (grads if out is None else out) if t.numel())
    _require(all(a[1] <= b[0] for a, b in zip(written, written[1:])), "clip_grad_norm: a tensor, or a part of one, is listed twice")
    if out is not None:
        for o, g in zip(out, grads):
            if g.numel() and span(o) != span(g):
                _require(all(w[1] <= span(g)[0] or w[0] >= span(g)[1] for w in written), "clip_grad_norm: a result overlaps a gradient that is not its own")


def grad_norm(grads):
    """Global 2-norm of a list of fp32, bf16 and fp16 tensors (entries that are None are left out): a 0-dim fp32 tensor on their device.

    Squares are added in 64 bits in a fixed order (on a GPU those of 16-bit values by fours in fp32 first, where they are exact).  Tensors are dense in memory, in any layout and at any offset."""
    grads, _ = _gradients(grads)
    if grads[0].is_cuda:
        return load().grad_norm(grads)
    _require(all(g.device == grads[0].device and g.dtype in FLOATS for g in grads), "grad_norm: fp32, bf16 or fp16 gradients on one device required")
    return torch.stack([g.detach().double().square().sum() for g in grads]).sum().sqrt().float()


def clip_grad_norm(grads, max_norm, out=None):
    """Scale tensors by ``min(1, max_norm / (norm + 1e-6))`` with their global 2-norm, which is returned (before clipping, 0-dim fp32).

    In place, or into `out`: as many tensors of the same types, shapes and layouts (the views of an optimizer's flat buffer, say), each
    its own gradient or apart from all of them.  No tensor may be listed twice.  Where the factor is 1, nothing is written in place.  The device is not
    waited for: a norm that is not finite shows in the result and makes the scaled values NaN or zero, as the formula says."""
    grads, out = _gradients(grads, out)
    if grads[0].is_cuda:                         # checked there
        return load().clip_grad_norm_(grads, max_norm) if out is None else load().clip_grad_norm_out(grads, out, max_norm)
    _require(max_norm > 0, "clip_grad_norm: max_norm must be positive")
    _check_host(grads, out)
    with torch.no_grad():
        norm = grad_norm(grads)
        factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
        for o, g in zip(grads if out is None else out, grads):
            o.copy_(g.float() * factor)
    return norm
