"""What stands between two blocks of a decoder layer, in one launch.

The reference's model runs its modules one after the other between two blocks (the Hugging Face layer loop behind
nanoPD/engine/model_runner.py:75-212: a residual sum, then a norm).  ``residual_norms`` does that pass once over the rows,
together with what some models put around it: a norm behind the block, a gate, a scale of the residual branch.  The
decode harness calls it for layers of that shape (``decoder_step.DecoderShape.post_norms``).
"""
from __future__ import annotations

import struct
from typing import Dict, Optional

import torch

from ._lib import NPD_OP_RESIDUAL_NORMS
from .paged_kernels import _DTYPE_CODE, _packed_op, _raw_stream, _remember, _require

MAX_HIDDEN = 32768
_plans: Dict[tuple, tuple] = {}
_pack = struct.Struct("<q7Q3d8qQ").pack                # device, then the entry point's arguments


def _rows(t: torch.Tensor, name: str, T: int, H: int) -> int:
    """Row stride of ``t`` seen as [T, H]; the leading dims must fold into one."""
    _require(t.dim() == 2 and t.shape == (T, H), f"residual_norms: {name} must be [{T}, {H}], got {tuple(t.shape)}")
    _require(H == 1 or t.stride(1) == 1, f"residual_norms: the rows of {name} must be contiguous")
    return t.stride(0) if T > 1 else H           # the stride of a single row means nothing


def _apart(a: int, a_bytes: int, a_stride: int, b: int, b_bytes: int, b_stride: int, row: int) -> bool:
    """Whether rows of ``row`` bytes at ``a`` and at ``b`` (addresses, extents and strides in bytes) share none: one behind
    the other, or columns of one buffer."""
    if a + a_bytes <= b or b + b_bytes <= a:
        return True
    return a_stride == b_stride and row <= (a - b) % a_stride <= a_stride - row


def _clear_of(w: int, po: int, eo: int, to: int, ph: int, eh: int, th: int, row: int) -> bool:
    """Whether the ``row`` bytes of a weight at ``w`` lie beside both outputs: outside their extent or between their rows."""
    return ((po + eo <= w or w + row <= po or row <= (w - po) % to <= to - row)
            and (ph + eh <= w or w + row <= ph or row <= (w - ph) % th <= th - row))


def residual_norms(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                   gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0,
                   residual_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """The residual sum behind a block and the norm in front of the next one; returns ``(residual_out, out)``.

    ``y = x``; with ``post_weight`` ``y = y * rsqrt(mean(y^2) + eps) * (post_weight + weight_offset)``; with ``gate`` ``y = gate * y``;
    ``residual_out = residual + residual_scale * y``; ``out = r * rsqrt(mean(r^2) + eps) * (weight + weight_offset)`` of that sum
    ``r`` before it is rounded.  Everything is computed in fp32 and each output rounded once.

    ``x``, ``residual``: ``[T, H]`` of one dtype (fp16, bf16, fp32) with contiguous rows, H a multiple of 8 up to 32768; ``weight``,
    ``post_weight``: ``[H]``; ``gate``: ``[H]`` or ``[T, H]``.  ``residual_out`` and ``out`` are allocated when absent; each may be
    the very rows of ``x`` or of ``residual`` (in place), other overlaps (with the weights and the gate too) are refused.
    """
    try:
        # one flat key: what the checks look at (the launches are short, and nested tuples cost as much as the checks)
        key = (x.shape, x.stride(), x.dtype, x.device, residual.shape, residual.stride(), residual.dtype, residual.device, weight.shape,
               weight.stride(), weight.dtype, weight.device,
               None if post_weight is None else (post_weight.shape, post_weight.stride(), post_weight.dtype, post_weight.device),
               None if gate is None else (gate.shape, gate.stride(), gate.dtype, gate.device),
               None if residual_out is None else (residual_out.shape, residual_out.stride(), residual_out.dtype, residual_out.device),
               None if out is None else (out.shape, out.stride(), out.dtype, out.device))
    except AttributeError:
        raise RuntimeError("residual_norms takes tensors") from None
    plan = _plans.get(key)
    if plan is None:
        _require(x.is_cuda, "residual_norms: x must be a CUDA tensor (this library has no CPU path)")
        _require(x.dim() == 2, "residual_norms: x must be [T, H]")
        _require(x.dtype in _DTYPE_CODE, f"residual_norms: unsupported dtype {x.dtype}")
        T, H = x.shape
        _require(H % 8 == 0 and 0 < H <= MAX_HIDDEN, f"residual_norms: H must be a multiple of 8 up to {MAX_HIDDEN}, got {H}")
        strides = [_rows(x, "x", T, H), _rows(residual, "residual", T, H)]
        for name, w in (("weight", weight), ("post_weight", post_weight)):
            _require(w is None or (w.shape == (H,) and w.stride(0) == 1), f"residual_norms: {name} must be a contiguous [{H}] tensor")
        if gate is None or gate.dim() == 1:
            _require(gate is None or (gate.shape == (H,) and gate.stride(0) == 1), f"residual_norms: gate must be [{H}] or [{T}, {H}]")
            strides.append(0)
        elif T > 1 and gate.dim() == 2 and gate.stride(0) == 0:          # an expanded row
            _rows(gate, "gate", T, H)
            strides.append(0)
        else:
            strides.append(_rows(gate, "gate", T, H))
        for name, o in (("residual_out", residual_out), ("out", out)):
            strides.append(H if o is None else _rows(o, name, T, H))
        for t in (residual, weight, post_weight, gate, residual_out, out):
            _require(t is None or (t.dtype == x.dtype and t.device == x.device), "residual_norms: tensors must share x's dtype and device")
        e = x.element_size()
        spans = tuple([(((T - 1) * st + H) * e, st * e) for st in strides])     # extent and stride in bytes
        plan = (x.device.index, H * e, spans, (T, H, *strides, _DTYPE_CODE[x.dtype]))
        if T > 0:
            _remember(_plans, key, plan)
    dev_index, row, (sx, sr, sg, so, sh), args = plan
    given = residual_out is not None or out is not None
    if residual_out is None:
        residual_out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out is None:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if args[0] == 0:
        return residual_out, out
    px, pr, po, ph, pg = x.data_ptr(), residual.data_ptr(), residual_out.data_ptr(), out.data_ptr(), 0 if gate is None else gate.data_ptr()
    pw, pp = weight.data_ptr(), 0 if post_weight is None else post_weight.data_ptr()
    if given:
        # a row's values are all read before its outputs are written: an output may be the very rows of x or of the residual
        (ex, tx), (er, tr), (eo, to), (eh, th) = sx, sr, so, sh
        if not ((po + eo <= px or px + ex <= po or (po == px and to == tx) or _apart(po, eo, to, px, ex, tx, row))
                and (po + eo <= pr or pr + er <= po or (po == pr and to == tr) or _apart(po, eo, to, pr, er, tr, row))
                and (ph + eh <= px or px + ex <= ph or (ph == px and th == tx) or _apart(ph, eh, th, px, ex, tx, row))
                and (ph + eh <= pr or pr + er <= ph or (ph == pr and th == tr) or _apart(ph, eh, th, pr, er, tr, row))
                and (po + eo <= ph or ph + eh <= po or _apart(po, eo, to, ph, eh, th, row))
                and (pg == 0 or (_apart(po, eo, to, pg, *sg, row) and _apart(ph, eh, th, pg, *sg, row)))
                and _clear_of(pw, po, eo, to, ph, eh, th, row) and (pp == 0 or _clear_of(pp, po, eo, to, ph, eh, th, row))):
            raise RuntimeError("residual_norms: an output overlaps another tensor without being the same rows of x or residual")
    _packed_op(NPD_OP_RESIDUAL_NORMS, _pack, dev_index, po, ph, px, pr, pw, pp, pg, residual_scale, eps, weight_offset, *args, _raw_stream(dev_index))
    return residual_out, out
