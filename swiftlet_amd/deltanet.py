"""The gated DeltaNet block (linear_attn) on the device: the input
projections (swq_encode_gemv), the decode step (swq_deltanet_step) and
out_proj — QwenMetalModel.encDeltaLayer (QwenMetalModel.swift:989-1084) for
one token, numerics of QwenCPUModel.deltaNetForward (QwenCPUModel.swift:
371-496); and the block between its projections for the tokens of many
sequences (swq_deltanet_tokens), prompts (`prefill`) or one token each
(`step_batch`).  torch supplies device memory and streams only."""

from __future__ import annotations

import ctypes

from . import _lib
from ._lib import SWQ_DELTA_INTERLEAVED, SWQ_DELTA_SPLIT, DeltaNetBatch, DeltaNetLayer, SwqError, check
from .engine import DescArray, GPULinear, HipEngine, _code, _elsewhere, _i32, _norm_arg, _ptr, _stream_handle, _torch, own_launches


def _row_stride(t, rows, width, what, device):
    """Elements between the rows of a tensor [rows, width] (or wider) whose rows are contiguous."""
    if t.get_device() != device:
        raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, what + ": not on the block's device")
    if t.dim() != 2:
        raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, what)
    (n, w), (row, element) = t.shape, t.stride()
    if n != rows or w < width or element != 1 or (rows > 1 and row < width):
        raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, what)
    return row if rows > 1 else 0


def _most(max_tokens, tokens):
    """The most tokens of one sequence, no more than the call has."""
    return max(min(max_tokens or tokens, tokens), -1) or 1


class DeltaNetGPU:
    """One linear_attn block: shapes, small f32 parameters on the device,
    and (optionally) its projections.

    INTERLEAVED (qwen3_next): projections = (in_proj_qkvz, in_proj_ba).
    SPLIT (qwen3_5): projections = (in_proj_qkv, in_proj_z, in_proj_b,
    in_proj_a), whose outputs land as [q|k|v|z] and [b|a]."""

    def __init__(self, nk: int, nv: int, dk: int, dv: int, conv_kernel: int, layout: int, eps: float,
                 conv_weight, a_log, dt_bias, norm_weight, projections=(), out_proj: GPULinear | None = None,
                 device="cuda"):
        torch = _torch()
        self.lib = _lib.load()
        self.nk, self.nv, self.dk, self.dv, self.K = nk, nv, dk, dv, conv_kernel
        self.layout, self.eps = layout, eps
        self.key_dim, self.value_dim = nk * dk, nv * dv
        self.conv_dim = 2 * self.key_dim + self.value_dim
        f32 = dict(dtype=torch.float32, device=device)
        self.conv_weight = torch.as_tensor(conv_weight, **f32).reshape(-1).contiguous()
        self.a_log = torch.as_tensor(a_log, **f32).contiguous()
        self.dt_bias = torch.as_tensor(dt_bias, **f32).contiguous()
        self.norm_weight = torch.as_tensor(norm_weight, **f32).contiguous()
        assert self.conv_weight.numel() == self.conv_dim * conv_kernel and self.a_log.numel() == nv
        self.projections, self.out_proj = tuple(projections), out_proj
        self._c = DeltaNetLayer(
            num_key_heads=nk, num_value_heads=nv, key_head_dim=dk, value_head_dim=dv, conv_kernel=conv_kernel,
            layout=layout, norm_eps=eps, reserved=0, conv_weight=self.conv_weight.data_ptr(),
            a_log=self.a_log.data_ptr(), dt_bias=self.dt_bias.data_ptr(), norm_weight=self.norm_weight.data_ptr())
        self._projs = DescArray()
        self._ref = ctypes.byref(self._c)
        self._scratch = self.lib.swq_deltanet_scratch_floats(self._ref)
        self._slot_bytes = self.lib.swq_deltanet_slot_bytes(self._ref)

    @property
    def state_bytes(self) -> int:
        n = self.lib.swq_deltanet_state_bytes(ctypes.byref(self._c))
        if n == 0:
            raise _lib.SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "deltanet_state_bytes")
        return n

    def new_state(self):
        """A fresh session's state (zeros), as a flat uint8 device tensor."""
        torch = _torch()
        return torch.zeros(self.state_bytes, dtype=torch.uint8, device=self.conv_weight.device)

    def state_views(self, state):
        """(conv ring [K, convD], recurrent state [nv, dv, dk]) views of a state buffer."""
        torch = _torch()
        ring_bytes = (self.K * self.conv_dim * 4 + 255) // 256 * 256
        ring = state[:self.K * self.conv_dim * 4].view(torch.float32).reshape(self.K, self.conv_dim)
        rec = state[ring_bytes:ring_bytes + self.nv * self.dv * self.dk * 4].view(torch.float32)
        return ring, rec.reshape(self.nv, self.dv, self.dk)

    @property
    def slot_bytes(self) -> int:
        if self._slot_bytes == 0:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "deltanet_slot_bytes")
        return self._slot_bytes

    def new_states(self, slots: int):
        """Fresh states (zeros) of `slots` sequences, as a flat uint8 device tensor."""
        torch = _torch()
        return torch.zeros(slots * self.slot_bytes, dtype=torch.uint8, device=self.conv_weight.device)

    def states_views(self, states):
        """(conv rings [slots, K, convD], recurrent states [slots, nv, dv, dk]) views of a buffer of many states."""
        torch = _torch()
        n, at = self.slot_bytes, (self.K * self.conv_dim * 4 + 255) // 256 * 256
        slots = states.numel() // n
        whole = states[:slots * n].view(slots, n)
        return (whole[:, :self.K * self.conv_dim * 4].view(torch.float32).view(slots, self.K, self.conv_dim),
                whole[:, at:at + self.nv * self.dv * self.dk * 4].view(torch.float32).view(slots, self.nv, self.dv, self.dk))

    def new_batch_workspace(self, sequences: int, tokens: int | None = None, max_tokens: int | None = None):
        """For calls of up to `sequences` sequences, `tokens` tokens (one each if not given) and
        `max_tokens` of one sequence (any number of the call's if not given)."""
        torch = _torch()
        tokens = sequences if tokens is None else tokens
        b = DeltaNetBatch(sequences=_i32(sequences, "deltanet_tokens: sequences"), tokens=_i32(tokens, "deltanet_tokens: tokens"),
                          max_tokens=_most(max_tokens, tokens), slots=sequences, starts=1)
        n = self.lib.swq_deltanet_tokens_workspace_bytes(ctypes.byref(self._c), ctypes.byref(b))
        if n == 0:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "deltanet_tokens_workspace_bytes")
        return torch.empty(n, dtype=torch.uint8, device=self.conv_weight.device)

    def prefill(self, qkvz, ba, states, positions, ws, starts=None, slots=None, max_tokens: int | None = None, out=None,
                stream=None):
        """The tokens of many sequences from their projection outputs (swq_deltanet_tokens): qkvz [N, convD +
        nv*dv], ba [N, 2*nv], f32 or bf16, rows as far apart as they may be; returns out [N, nv*dv] of qkvz's
        type and updates `states` (new_states).  positions (int32 device [B]): tokens in each state already.
        starts (int32 device [B + 1]) where sequences bring different numbers of tokens, then max_tokens, the most
        that one brings (default: N).  slots (int32 device [B]): each sequence's state, none twice; one that is out
        of range leaves its sequence out (default: the b-th)."""
        torch = _torch()
        if out is None:
            if stream is not None and _elsewhere(stream):
                with torch.cuda.stream(stream):
                    return self.prefill(qkvz, ba, states, positions, ws, starts, slots, max_tokens)
            out = torch.empty((qkvz.shape[0], self.value_dim), dtype=qkvz.dtype, device=qkvz.device)
        at, B, N, dtype, i32, u8 = self.conv_weight.get_device(), positions.numel(), len(qkvz), qkvz.dtype, torch.int32, torch.uint8
        if at < 0 or at != torch.cuda.current_device():
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "deltanet_tokens: the block is not on the current device")
        if ba.dtype != dtype:
            raise SwqError(_lib.SWQ_ERR_UNSUPPORTED_DTYPE, "deltanet_tokens: ba")
        if out.numel() != N * self.value_dim:
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "deltanet_tokens: out")
        states_bytes = states.numel()
        b = DeltaNetBatch(B, _i32(N, "deltanet_tokens: tokens"), _most(max_tokens, N), _i32(states_bytes // self.slot_bytes, "deltanet_tokens: states"),
                          None if starts is None else _ptr(starts, B + 1, "deltanet_tokens: starts", at, i32),
                          _ptr(positions, 1, "deltanet_tokens: positions", at, i32),
                          None if slots is None else _ptr(slots, B, "deltanet_tokens: slots", at, i32),
                          _row_stride(qkvz, N, self.conv_dim + self.value_dim, "deltanet_tokens: qkvz", at),
                          _row_stride(ba, N, 2 * self.nv, "deltanet_tokens: ba", at), 0)
        check(self.lib.swq_deltanet_tokens(
            self._ref, ctypes.byref(b), qkvz.data_ptr(), ba.data_ptr(), _code(qkvz, "deltanet_tokens"),
            _ptr(states, 1, "deltanet_tokens: states", at, u8), states_bytes, _ptr(out, 0, "deltanet_tokens: out", at),
            _code(out, "deltanet_tokens"), _ptr(ws, 1, "deltanet_tokens: ws", at, u8), ws.numel(), _stream_handle(stream)), "deltanet_tokens")
        return out

    def step_batch(self, qkvz, ba, states, positions, ws, slots=None, out=None, stream=None):
        """One token of each of positions.numel() sequences, as `prefill`."""
        if qkvz.shape[0] != positions.numel():
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "deltanet_tokens: qkvz")
        return self.prefill(qkvz, ba, states, positions, ws, None, slots, 1, out, stream)

    def step(self, qkvz, ba, state, position: int, out=None, stream=None):
        """One token from its projection outputs; returns the gated-normed
        output [nv*dv] (f32) and updates `state`."""
        torch = _torch()
        assert qkvz.dtype == torch.float32 and ba.dtype == torch.float32
        assert qkvz.numel() >= self.conv_dim + self.value_dim and ba.numel() >= 2 * self.nv
        if out is None:
            out = torch.empty(self.value_dim, dtype=torch.float32, device=qkvz.device)
        check(self.lib.swq_deltanet_step(ctypes.byref(self._c), qkvz.data_ptr(), ba.data_ptr(), state.data_ptr(),
                                         state.numel(), position, out.data_ptr(), _stream_handle(stream)),
              "deltanet_step")
        return out

    def forward_token(self, engine: HipEngine, x, state, position: int, norm_weight=None, eps: float = 1e-6,
                      stream=None):
        """x [H] f32 -> the block's output [H]: the input projections in one
        launch (with norm_weight, x is the un-normalised hidden state and the
        input RMSNorm runs inside that launch), the step, out_proj.  One native
        call, or the launches one by one where `step` or one of the engine's
        has been overridden."""
        if stream is not None and _elsewhere(stream):
            with _torch().cuda.stream(stream):
                return DeltaNetGPU.forward_token(self, engine, x, state, position, norm_weight, eps)
        if not own_launches(engine, self.step, _OWN_STEP):
            return self._forward_launches(engine, x, state, position, norm_weight, eps, stream)
        empty, f32, dev = _torch().empty, _torch().float32, x.device
        scratch = empty(self._scratch, dtype=f32, device=dev)
        r = empty(self.out_proj.out_dim, dtype=f32, device=dev)
        wdt, wptr = _norm_arg(norm_weight)
        check(self.lib.swq_deltanet_token(
            ctypes.byref(self._c), self._projs.of(self.projections), len(self.projections), self.out_proj.desc(),
            x.data_ptr(), wptr, wdt, eps, state.data_ptr(), state.numel(), position, scratch.data_ptr(), self._scratch,
            r.data_ptr(), _stream_handle(stream)), "deltanet_token")
        return r

    def _forward_launches(self, engine, x, state, position, norm_weight, eps, stream):
        torch = _torch()
        qkvz = torch.empty(self.conv_dim + self.value_dim, dtype=torch.float32, device=x.device)
        ba = torch.empty(2 * self.nv, dtype=torch.float32, device=x.device)
        if self.layout == SWQ_DELTA_INTERLEAVED:
            ys = [qkvz, ba]
        else:
            ys = [qkvz.data_ptr(), qkvz.data_ptr() + 4 * self.conv_dim, ba.data_ptr(), ba.data_ptr() + 4 * self.nv]
        engine.encode_gemv_multi(list(self.projections), x, ys, norm_weight=norm_weight, eps=eps, stream=stream)
        y = self.step(qkvz, ba, state, position, stream=stream)
        r = torch.empty(self.out_proj.out_dim, dtype=torch.float32, device=x.device)
        engine.encode_gemv(self.out_proj, y, r, stream=stream)
        return r


_OWN_STEP = DeltaNetGPU.step


def deltanet_from_checkpoint(ckpt, layer: int, config: dict, device="cuda", stream=None) -> DeltaNetGPU:
    """Layer `layer`'s linear_attn block from a checkpoint (swiftlet_amd.
    checkpoint.Checkpoint): the projections resident, the small parameters
    as f32.  The layout follows QwenConfig (QwenConfig.swift:103): split when
    the checkpoint holds in_proj_qkv, interleaved otherwise."""
    torch = _torch()
    p = f"model.layers.{layer}.linear_attn."
    split = ckpt.contains(p + "in_proj_qkv.weight")
    names = ("in_proj_qkv", "in_proj_z", "in_proj_b", "in_proj_a") if split else ("in_proj_qkvz", "in_proj_ba")
    projs = [ckpt.gpu_linear(p + n, device=device, stream=stream) for n in names]

    def f32(name):
        return ckpt.load(p + name, device=device, stream=stream).to(torch.float32)

    c = config
    return DeltaNetGPU(c["linear_num_key_heads"], c["linear_num_value_heads"], c["linear_key_head_dim"],
                       c["linear_value_head_dim"], c["linear_conv_kernel_dim"],
                       SWQ_DELTA_SPLIT if split else SWQ_DELTA_INTERLEAVED, c.get("rms_norm_eps", 1e-6),
                       f32("conv1d.weight"), f32("A_log"), f32("dt_bias"), f32("norm.weight"),
                       projections=projs, out_proj=ckpt.gpu_linear(p + "out_proj", device=device, stream=stream),
                       device=device)
