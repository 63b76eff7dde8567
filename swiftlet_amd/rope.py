"""Rotary positions: tables of cos and sin for contexts of any length (swq_rope_table) and queries and keys turned by
them (swq_rope), for what QwenCPUModel.applyRope (QwenCPUModel.swift:308-343) does inside swq_attention_step.  A table
is also what AttentionQ4GPU takes as `rope_table`.  torch supplies device memory and streams only."""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _lib
from ._lib import SWQ_ROPE_HALF, SWQ_ROPE_INTERLEAVED, RopeHeads, RopeScalingDesc, SwqError, check
from .engine import _code, _elsewhere, _i32, _ptr, _stream_handle, _torch

_KINDS = {"none": _lib.SWQ_ROPE_PLAIN, "default": _lib.SWQ_ROPE_PLAIN, "linear": _lib.SWQ_ROPE_LINEAR, "ntk": _lib.SWQ_ROPE_NTK,
          "yarn": _lib.SWQ_ROPE_YARN}
_LAYOUTS = {"half": SWQ_ROPE_HALF, "interleaved": SWQ_ROPE_INTERLEAVED}


@dataclass(frozen=True)
class RopeScaling:
    """How a model reads contexts longer than it was trained on (swq_rope_scaling): "linear", "ntk" or "yarn"."""

    kind: str
    factor: float
    original_positions: int = 0
    beta_fast: float = 32.0
    beta_slow: float = 1.0
    magnitude: float | None = None

    def desc(self) -> RopeScalingDesc:
        if self.kind not in _KINDS:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "RopeScaling: " + str(self.kind))
        if self.magnitude is not None and not self.magnitude > 0:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "RopeScaling: magnitude")
        return RopeScalingDesc(_KINDS[self.kind], self.original_positions, self.beta_fast, self.beta_slow, self.magnitude or 0.0, self.factor, 0)


class RopeGPU:
    """Rotary positions of heads whose first `rotary_dims` elements turn, in pairs of the two halves ("half") or of
    neighbours ("interleaved")."""

    def __init__(self, rotary_dims: int, rope_theta: float, layout: str = "half", scaling: RopeScaling | None = None, device="cuda"):
        self.lib = _lib.load()
        if layout not in _LAYOUTS:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "RopeGPU: layout")
        self.rot, self.theta, self.scaling, self.device = rotary_dims, rope_theta, scaling, device
        self._layout = _LAYOUTS[layout]
        self._desc = scaling.desc() if scaling is not None else None
        self._ref = ctypes.byref(self._desc) if scaling is not None else None

    @classmethod
    def from_config(cls, config: dict, device="cuda") -> "RopeGPU":
        """The rotary positions of a model's config.json, as attention_from_checkpoint reads them, with the scaling
        that its "rope_scaling" or "rope_parameters" names."""
        c = config.get("text_config", config)
        rp = c.get("rope_parameters") or {}
        theta = float(rp.get("rope_theta", c.get("rope_theta", 10_000_000)))
        part = float(rp.get("partial_rotary_factor", c.get("partial_rotary_factor", 0.25)))
        sc = c.get("rope_scaling") or rp
        kind = sc.get("rope_type", sc.get("type", "default"))
        if kind not in _KINDS:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "RopeGPU: rope_type " + str(kind))
        scaling = None
        if _KINDS[kind] != _lib.SWQ_ROPE_PLAIN:
            sc = {k: v for k, v in sc.items() if v is not None}
            if "factor" not in sc:
                raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "RopeGPU: rope_type " + str(kind) + " without a factor")
            # what would change the angles or the magnitude and is not in RopeScaling
            odd = [k for k, plain in (("mscale", None), ("mscale_all_dim", None), ("truncate", True)) if sc.get(k, plain) != plain]
            if odd:
                raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "RopeGPU: " + ", ".join(odd))
            scaling = RopeScaling(kind, float(sc["factor"]), int(sc.get("original_max_position_embeddings", c.get("max_position_embeddings", 0))),
                                  float(sc.get("beta_fast", 32.0)), float(sc.get("beta_slow", 1.0)), sc.get("attention_factor"))
        return cls(int(c["head_dim"] * part), theta, scaling=scaling, device=device)

    def table(self, positions=None, first: int = 0, count: int | None = None, out=None, stream=None):
        """cos and sin, f32 [n, rotary_dims / 2, 2]: of positions (int32 device [n]), or of first .. first + count - 1."""
        torch = _torch()
        n = count if positions is None else positions.numel()
        if n is None or n < 0 or (count is not None and count != n):
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "rope_table: count")
        _i32(n, "rope_table: count")
        if out is None:
            if stream is not None and _elsewhere(stream):
                with torch.cuda.stream(stream):
                    return self.table(positions, first, count)
            out = torch.empty((n, self.rot // 2, 2), dtype=torch.float32, device=self.device if positions is None else positions.device)
        at = _here(out, "rope_table")
        if out.numel() != n * (self.rot // 2) * 2:
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope_table: out")
        check(self.lib.swq_rope_table(self.rot, self.theta, self._ref, _ptr(positions, 0, "rope_table: positions", at, torch.int32), first, n,
                                      _ptr(out, 0, "rope_table: out", at, torch.float32), _stream_handle(stream)), "rope_table")
        return out

    def apply(self, xs, table, rows=None, norm_weights=None, eps: float = 1e-6, inverse: bool = False, out=None, stream=None):
        """Tensors [N, heads, hd] of the same tokens (f32 or bf16; any strides, elements side by side) turned by
        `table`: token t by row rows[t] (int32 device [N]), or by row t.  norm_weights: for each tensor the f32 weight
        [hd] with which its heads are RMS-normalised first, or None.  inverse turns back.  out: tensors for the
        results, which may be the inputs; made if not given.  Returns the results in a list."""
        torch = _torch()
        if out is None:
            if stream is not None and _elsewhere(stream):
                with torch.cuda.stream(stream):
                    return self.apply(xs, table, rows, norm_weights, eps, inverse)
            out = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs]
        if not xs or len(out) != len(xs) or (norm_weights is not None and len(norm_weights) != len(xs)):
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: tensors")
        at, dtype, shape = _here(table, "rope"), xs[0].dtype, xs[0].shape
        if len(shape) != 3:
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: tensors")
        N, _, hd = shape
        _i32(N, "rope: tokens")
        parts = (RopeHeads * len(xs))()
        for part, x, y, w in zip(parts, xs, out, norm_weights or (None,) * len(xs)):
            shape = x.shape
            if x.get_device() != at or y.get_device() != at:
                raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "rope: not on the table's device")
            if x.dtype != dtype or y.dtype != dtype:
                raise SwqError(_lib.SWQ_ERR_UNSUPPORTED_DTYPE, "rope: tensors of two types")
            if len(shape) != 3 or shape[0] != N or shape[2] != hd or y.shape != shape:
                raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: tensors")
            heads, (part.token_stride, part.head_stride, e), (to, ho, eo) = shape[1], x.stride(), y.stride()
            if hd > 1 and (e != 1 or eo != 1):
                raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: tensors")
            if (to == 0 and N > 1) or (ho == 0 and heads > 1):
                raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: out")
            if w is not None:
                if w.numel() != hd:
                    raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: norm_weights")
                part.norm_weight = _ptr(w, hd, "rope: norm_weights", at, torch.float32)
            part.x, part.out, part.heads, part.out_token_stride, part.out_head_stride = x.data_ptr(), y.data_ptr(), heads, to, ho
        if table.shape[1:] != (self.rot // 2, 2):
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "rope: table")
        check(self.lib.swq_rope(parts, len(xs), N, hd, self.rot, self._layout, int(inverse), eps, _ptr(table, 1, "rope: table", at, torch.float32),
                                _i32(len(table), "rope: table"), _ptr(rows, N, "rope: rows", at, torch.int32), _code(xs[0], "rope"), _stream_handle(stream)), "rope")
        return out


def _here(t, what):
    """The tensor's device, if it is the current one, to which streams and launches belong."""
    if t.get_device() < 0 or t.get_device() != _torch().cuda.current_device():
        raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, what + ": not on the current device")
    return t.get_device()
