"""Gated GQA attention over a KV cache held in 4 bits (swq_attention_q4): what
AttentionGPU does for one token and an f32 cache (QwenMetalModel.swift:922-951,
:1086-1134; numerics of QwenCPUModel.swift:285-367), for the tokens of many
sequences, one each (`step`) or prompts (`prefill`), at a seventh of the cache
bytes; and the cache's own calls: rows in (`append`), out as values
(`Q4Cache.read`), and the most attended ones into a smaller cache (`evict`).
torch supplies device memory and streams only."""

from __future__ import annotations

import ctypes

from . import _lib
from ._lib import AttentionLayer, Q4Batch, Q4CacheDesc, SwqError, check
from .engine import GPULinear, HipEngine, _code, _elsewhere, _ptr, _stream_handle, _torch


class Q4Cache:
    """Keys and values of `sequences` sequences in 4-bit codes (swq_q4_cache).
    data: a uint8 tensor of at least swq_q4_cache_bytes bytes, 256-byte
    aligned; made here if not given."""

    def __init__(self, sequences: int, num_kv_heads: int, head_dim: int, max_positions: int, data=None, device="cuda"):
        torch = _torch()
        self.lib = _lib.load()
        self.sequences, self.KVH, self.hd, self.max_positions = sequences, num_kv_heads, head_dim, max_positions
        n = self.lib.swq_q4_cache_bytes(sequences, num_kv_heads, head_dim, max_positions)
        if n == 0:
            raise SwqError(_lib.SWQ_ERR_LIMIT if min(sequences, num_kv_heads, head_dim, max_positions) > 0
                           else _lib.SWQ_ERR_INVALID_ARGUMENT, "q4_cache_bytes")
        if data is None:
            data = torch.zeros(n, dtype=torch.uint8, device=device)
        elif data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() < n:
            raise SwqError(_lib.SWQ_ERR_WORKSPACE, "Q4Cache")
        self.data = data
        self.desc = Q4CacheDesc(data=data.data_ptr(), bytes=data.numel(), sequences=sequences, num_kv_heads=num_kv_heads,
                                head_dim=head_dim, max_positions=max_positions)
        self.ref = ctypes.byref(self.desc)
        self.device_index = data.get_device()

    def here(self, what):
        """The cache's device, if it is the current one, to which streams and launches belong."""
        if self.device_index < 0 or self.device_index != _torch().cuda.current_device():
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, what + ": the cache is not on the current device")
        return self.device_index

    def views(self):
        """(k words int32 [B, KVH, R, hd/8], v words int32 [B, KVH, R/8, hd], params f16 [B, KVH, 4, hd/64, R])
        over the cache's memory; R: max_positions rounded up to 32."""
        torch = _torch()
        B, kvh, hd, R = self.sequences, self.KVH, self.hd, (self.max_positions + 31) // 32 * 32
        n, p = B * kvh * R * hd // 2, B * kvh * R * hd // 8
        at = (n + 255) // 256 * 256
        return (self.data[:n].view(torch.int32).view(B, kvh, R, hd // 8),
                self.data[at:at + n].view(torch.int32).view(B, kvh, R // 8, hd),
                self.data[2 * at:2 * at + p].view(torch.float16).view(B, kvh, 4, hd // 64, R))

    def read(self, first, count: int, dtype=None, starts=None, tokens: int | None = None, rows=None, sequences: int | None = None,
             stream=None):
        """Rows as values (swq_q4_read): k and v [B, count, KVH, hd] f32 (or dtype bfloat16), rows
        first[b] .. of each sequence (first int32 device [B] or None: 0); with starts (int32 device
        [B + 1]) and tokens, starts[b + 1] - starts[b] of them, packed: [tokens, KVH, hd].  rows (int32
        device [B]): those from rows[b] on come as zeros."""
        torch = _torch()
        if stream is not None and _elsewhere(stream):
            with torch.cuda.stream(stream):
                return self.read(first, count, dtype, starts, tokens, rows, sequences)
        B, at = sequences or self.sequences, self.here("q4_read")
        shape = (B, count, self.KVH, self.hd) if starts is None else (tokens, self.KVH, self.hd)
        if starts is not None and tokens is None:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "q4_read: starts without tokens")
        k, v = torch.empty((2, *shape), dtype=dtype or torch.float32, device=self.data.device).unbind(0)
        check(self.lib.swq_q4_read(self.ref, B, _ptr(first, B, "q4_read: first", at, torch.int32),
                                   _ptr(starts, B + 1, "q4_read: starts", at, torch.int32),
                                   _ptr(rows, B, "q4_read: rows", at, torch.int32),
                                   shape[0] if starts is not None else count, k.data_ptr(), v.data_ptr(),
                                   _code(k, "q4_read"), _stream_handle(stream)), "q4_read")
        return k, v


class AttentionQ4GPU:
    """One self_attn block over a 4-bit cache: AttentionGPU's shapes, q/k norm
    weights (f32, device) and, optionally, projections and o_proj.  rope_table:
    f32 device [positions, rotary_dims / 2, 2], cos and sin, 16-byte aligned, which
    layers may share; made for `max_positions` positions by the first workspace or
    call if not given (before a graph is captured, then)."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, rotary_dims: int, rope_theta: float,
                 eps: float, max_positions: int, q_norm_weight, k_norm_weight, projections=(),
                 o_proj: GPULinear | None = None, device="cuda", rope_table=None):
        torch = _torch()
        self.lib = _lib.load()
        self.H, self.KVH, self.hd = num_heads, num_kv_heads, head_dim
        self.rot, self.theta, self.eps, self.max_positions = rotary_dims, rope_theta, eps, max_positions
        f32 = dict(dtype=torch.float32, device=device)
        self.q_norm = torch.as_tensor(q_norm_weight, **f32).contiguous()
        self.k_norm = torch.as_tensor(k_norm_weight, **f32).contiguous()
        if self.q_norm.numel() != head_dim or self.k_norm.numel() != head_dim:
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "AttentionQ4GPU: norm weights")
        self.projections, self.o_proj = tuple(projections), o_proj
        self.device = device
        if rope_table is not None and rotary_dims and (
                rope_table.dtype != torch.float32 or not rope_table.is_contiguous()
                or tuple(rope_table.shape[1:]) != (rotary_dims // 2, 2) or not len(rope_table)):
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "AttentionQ4GPU: rope_table")
        if rope_table is not None and rotary_dims and rope_table.get_device() != self.q_norm.get_device():
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "AttentionQ4GPU: rope_table on another device than the norm weights")
        self._table = rope_table
        self._rope = None if rotary_dims else (None, 0)
        self._c = AttentionLayer(num_heads=num_heads, num_kv_heads=num_kv_heads, head_dim=head_dim,
                                 rotary_dims=rotary_dims, rope_theta=rope_theta, norm_eps=eps,
                                 max_positions=max_positions, reserved=0, q_norm_weight=self.q_norm.data_ptr(),
                                 k_norm_weight=self.k_norm.data_ptr())
        self._ref = ctypes.byref(self._c)

    @property
    def rope_table(self):
        """cos and sin of every position, made when first asked for (a block that only evicts needs none)."""
        if self._table is None and self.rot:
            host = _torch().empty((self.max_positions, self.rot // 2, 2), dtype=_torch().float32)
            check(self.lib.swq_q4_rope_table(self.rot, self.theta, 0, self.max_positions, host.data_ptr()), "q4_rope_table")
            self._table = host.to(self.device)
        return self._table if self.rot else None

    def _rope_args(self):
        if self._rope is None:
            self._rope = (self.rope_table.data_ptr(), len(self._table))
        return self._rope

    @classmethod
    def of(cls, block, rope_table=None) -> "AttentionQ4GPU":
        """The same layer as an AttentionGPU, over a 4-bit cache."""
        return cls(block.H, block.KVH, block.hd, block.rot, block.theta, block.eps, block.max_positions, block.q_norm,
                   block.k_norm, block.projections, block.o_proj, block.device, rope_table)

    def new_cache(self, sequences: int = 1, max_positions: int | None = None) -> Q4Cache:
        return Q4Cache(sequences, self.KVH, self.hd, max_positions or self.max_positions, device=self.device)

    def new_weights(self, cache: Q4Cache):
        """Gathered attention of every row, none yet: f32 [sequences, KVH, max_positions]."""
        torch = _torch()
        return torch.zeros((cache.sequences, self.KVH, cache.max_positions), dtype=torch.float32, device=self.device)

    def new_workspace(self, cache: Q4Cache, tokens: int | None = None, max_tokens: int = 1, weights: bool = False):
        """For calls of up to `tokens` tokens (one per sequence if not given), `max_tokens` of one sequence."""
        torch = _torch()
        self._rope_args()
        b = Q4Batch(sequences=cache.sequences, tokens=tokens or cache.sequences, max_tokens=max_tokens, starts=1)
        n = self.lib.swq_attention_q4_workspace_bytes(self._ref, cache.ref, ctypes.byref(b), int(weights))
        if n == 0:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "attention_q4_workspace_bytes")
        return torch.empty(n, dtype=torch.uint8, device=self.device)

    def _batch(self, cache, rows, tokens, starts, max_tokens, max_rows, positions, what):
        torch = _torch()
        B, at = rows.numel(), cache.here(what)
        if self.q_norm.get_device() != at:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, what + ": the cache is not on the block's device")
        return Q4Batch(B, tokens, max_tokens, max_rows, _ptr(starts, B + 1, what + ": starts", at, torch.int32),
                       _ptr(rows, 1, what + ": rows", at, torch.int32), _ptr(positions, B, what + ": positions", at, torch.int32),
                       *self._rope_args(), 0)

    def append(self, k, v, cache: Q4Cache, rows, starts=None, max_tokens: int | None = None, positions=None, stream=None):
        """k, v [N, KVH*hd] (f32 or bf16) of the sequences' next tokens into `cache`, the first of
        sequence b at row rows[b] (int32 device [B]).  starts (int32 device [B + 1]) where sequences
        bring different numbers of tokens, then max_tokens, at most that many of one (default: N)."""
        N = k.numel() // (self.KVH * self.hd)
        b = self._batch(cache, rows, N, starts, max_tokens or N, 0, positions, "q4_append")
        n, at = N * self.KVH * self.hd, cache.device_index
        if k.dtype != v.dtype:
            raise SwqError(_lib.SWQ_ERR_UNSUPPORTED_DTYPE, "q4_append")
        check(self.lib.swq_q4_append(self._ref, cache.ref, ctypes.byref(b), _ptr(k, n, "q4_append: k", at),
                                     _ptr(v, n, "q4_append: v", at),
                                     _code(k, "q4_append"), _stream_handle(stream)), "q4_append")

    def prefill(self, q, k, v, cache: Q4Cache, rows, ws, starts=None, max_tokens: int | None = None, out=None, weights=None,
                positions=None, max_rows: int = 0, stream=None):
        """The tokens' k, v appended and their attention (swq_attention_q4): q [N, H*2*hd] (per head the
        query, then the gate), k, v [N, KVH*hd] (both None: the cache has them), f32 or bf16; returns
        out [N, H*hd] of q's type.  rows, starts, max_tokens, positions as in `append`; weights:
        gathers the rows' attention; max_rows: about how many rows a sequence has after the call
        (0: as many as the cache), which only sets how the work is split."""
        torch = _torch()
        N = q.numel() // (2 * self.H * self.hd)
        if out is None:
            if stream is not None and _elsewhere(stream):
                with torch.cuda.stream(stream):
                    out = torch.empty((N, self.H * self.hd), dtype=q.dtype, device=q.device)
            else:
                out = torch.empty((N, self.H * self.hd), dtype=q.dtype, device=q.device)
        b = self._batch(cache, rows, N, starts, max_tokens or N, max_rows, positions, "attention_q4")
        if (k is None) != (v is None):
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "attention_q4: k and v")
        if k is not None and (k.dtype != q.dtype or v.dtype != q.dtype):
            raise SwqError(_lib.SWQ_ERR_UNSUPPORTED_DTYPE, "attention_q4: k and v")
        n, val, at = N * self.KVH * self.hd, N * self.H * self.hd, cache.device_index
        check(self.lib.swq_attention_q4(
            self._ref, cache.ref, ctypes.byref(b), _ptr(q, 2 * val, "attention_q4: q", at), _ptr(k, n, "attention_q4: k", at),
            _ptr(v, n, "attention_q4: v", at), _code(q, "attention_q4"),
            _ptr(weights, rows.numel() * self.KVH * cache.max_positions, "attention_q4: weights", at, torch.float32),
            _ptr(out, val, "attention_q4: out", at), _code(out, "attention_q4"), _ptr(ws, 1, "attention_q4: ws", at, torch.uint8),
            ws.numel(), _stream_handle(stream)), "attention_q4")
        return out

    def step(self, q, k, v, cache: Q4Cache, rows, ws, out=None, weights=None, positions=None, max_rows: int = 0, stream=None):
        """One token of each of rows.numel() sequences, as `prefill`."""
        if q.numel() != 2 * self.H * self.hd * rows.numel():
            raise SwqError(_lib.SWQ_ERR_BAD_SHAPE, "attention_q4: q")
        return self.prefill(q, k, v, cache, rows, ws, None, None, out, weights, positions, max_rows, stream)

    def evict(self, cache: Q4Cache, weights, rows, into: Q4Cache, budget: int, sink: int = 0, recent: int = 0,
              new_weights=None, stream=None):
        """The rows worth keeping into another cache (swq_q4_evict): the first `sink`, the last `recent`
        and the heaviest between, `budget` in all.  Returns (kept int32 [B, KVH, budget], their rows in
        `cache`, -1 past the last; new_rows int32 [B])."""
        torch = _torch()
        if stream is not None and _elsewhere(stream):
            with torch.cuda.stream(stream):
                return self.evict(cache, weights, rows, into, budget, sink, recent, new_weights)
        B, at = rows.numel(), cache.here("q4_evict")
        if into.device_index != at:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "q4_evict: caches on two devices")
        if budget <= 0:
            raise SwqError(_lib.SWQ_ERR_INVALID_ARGUMENT, "q4_evict: budget")
        kept = torch.empty((B, self.KVH, budget), dtype=torch.int32, device=rows.device)
        new_rows = torch.empty(B, dtype=torch.int32, device=rows.device)
        check(self.lib.swq_q4_evict(
            cache.ref, B, _ptr(weights, B * self.KVH * cache.max_positions, "q4_evict: weights", at, torch.float32),
            _ptr(rows, B, "q4_evict: rows", at, torch.int32), into.ref, budget, sink, recent,
            _ptr(new_weights, B * self.KVH * into.max_positions, "q4_evict: new_weights", at, torch.float32),
            new_rows.data_ptr(), kept.data_ptr(), _stream_handle(stream)), "q4_evict")
        return kept, new_rows

    def forward_token(self, engine: HipEngine, x, cache: Q4Cache, rows, ws, norm_weight=None, eps: float = 1e-6,
                      weights=None, positions=None, max_rows: int = 0, stream=None):
        """x [H_model] f32 of one sequence's next token -> the block's output, as AttentionGPU's: q/k/v_proj
        in one launch (with norm_weight, behind the input RMSNorm), `step`, o_proj."""
        torch = _torch()
        if stream is not None and _elsewhere(stream):
            with torch.cuda.stream(stream):
                return self.forward_token(engine, x, cache, rows, ws, norm_weight, eps, weights, positions, max_rows)
        q, k, v = (torch.empty(p.out_dim, dtype=torch.float32, device=x.device) for p in self.projections)
        engine.encode_gemv_multi(list(self.projections), x, [q, k, v], norm_weight=norm_weight, eps=eps, stream=stream)
        val, kv = 2 * self.H * self.hd, self.KVH * self.hd
        att = self.step(q[:val], k[:kv], v[:kv], cache, rows, ws, None, weights, positions, max_rows, stream)
        r = torch.empty(self.o_proj.out_dim, dtype=torch.float32, device=x.device)
        engine.encode_gemv(self.o_proj, att, r, stream=stream)
        return r
