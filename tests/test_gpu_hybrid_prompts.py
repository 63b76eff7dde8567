"""DeltaNet blocks over many tokens, rotary tables and the 4-bit cache's attention as a hybrid model runs them: prompts of
several sequences in one call, then a token of each at a time, eager and captured.

Bars: each operator's own, on the inputs that the ones before it made (tests of the DeltaNet block and of the long cache:
1e-5 of the largest in f32; queries turned by swq_rope are off by 16 * 2^-24, a tenth of what that bar lets a score be).
The tiny model's logits: 2e-3, as of its token after token run."""

import json
import math

import numpy as np
import pytest
import torch

from oracle import deltanet_tokens_ref as R
from swiftlet_amd._lib import SWQ_DELTA_INTERLEAVED, SWQ_DELTA_SPLIT
from swiftlet_amd.attention_q4 import AttentionQ4GPU
from swiftlet_amd.deltanet import DeltaNetGPU, deltanet_from_checkpoint
from swiftlet_amd.rope import RopeGPU, RopeScaling
from tests.deltanet_cases import off
from tests.test_gpu_deltanet import G

pytestmark = pytest.mark.gpu


class Stack:
    """A DeltaNet block and an attention block between projections, for B sequences that all begin with nothing."""

    width = 128

    def __init__(self, heads, split, B, most, seed):
        nk, nv, dk, dv = self.heads = heads
        g = torch.Generator(device="cuda").manual_seed(seed)
        n = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.n, self.conv, self.val, self.split = n, 2 * nk * dk + nv * dv, nv * dv, split
        self.params = dict(conv_w=n(self.conv, 4) * 0.5, a_log=n(nv) * 0.5, dt_bias=n(nv) * 0.5 - 2, norm_w=1 + 0.2 * n(dv))
        self.delta = DeltaNetGPU(nk, nv, dk, dv, 4, SWQ_DELTA_SPLIT if split else SWQ_DELTA_INTERLEAVED, 1e-6, *self.params.values())
        self.H, self.KVH, self.hd = 4, 2, 64
        self.rope = RopeGPU(32, 1e6, scaling=RopeScaling("yarn", 4.0, 64))
        self.table = self.rope.table(first=0, count=most)
        self.qw, kw = 1 + 0.2 * n(self.hd), 1 + 0.2 * n(self.hd)
        self.attention = AttentionQ4GPU(self.H, self.KVH, self.hd, 32, 1e6, 1e-6, most, self.qw, kw, rope_table=self.table)
        W = self.width
        self.into = [n(W, o) / math.sqrt(W) for o in (self.conv + self.val, 2 * nv, 2 * self.H * self.hd, self.KVH * self.hd, self.KVH * self.hd)]
        self.out_of = [n(self.val, W) / math.sqrt(self.val), n(self.H * self.hd, W) / math.sqrt(self.H * self.hd)]
        self.states = self.delta.new_states(B)
        self.cache = self.attention.new_cache(B)
        self.done = torch.zeros(B, dtype=torch.int32, device="cuda")
        self.seen = [[] for _ in range(B)]  # per sequence: qkvz, ba, what DeltaNet made of them, queries, attention

    def workspaces(self, tokens, most):
        return self.delta.new_batch_workspace(len(self.seen), tokens, most), self.attention.new_workspace(self.cache, tokens, most)

    def run(self, x, ws, starts=None, most=1):
        """A layer of each kind; positions move on."""
        qkvz, ba = x @ self.into[0], x @ self.into[1]
        kw = dict(starts=starts, max_tokens=most) if starts is not None else {}
        y = (self.delta.prefill if kw else self.delta.step_batch)(qkvz, ba, self.states, self.done, ws[0], **kw)
        x = x + y @ self.out_of[0]
        q, k, v = (x @ w for w in self.into[2:])
        a = (self.attention.prefill if kw else self.attention.step)(q, k, v, self.cache, self.done, ws[1], **kw)
        self.done += starts.diff() if kw else 1
        return x + a @ self.out_of[1], (qkvz, ba, y, q, a)

    def keep(self, parts, counts):
        n0 = 0
        for seen, t in zip(self.seen, counts):
            seen.append([p[n0:n0 + t].clone() for p in parts])
            n0 += t

    def check(self):
        nk, nv, dk, dv = self.heads
        kk, vv = self.cache.read(None, int(self.done.max()))
        for b, seen in enumerate(self.seen):
            qkvz, ba, y, q, a = (torch.cat(p) for p in zip(*seen))
            T = len(y)
            zero = lambda t: torch.zeros_like(t, dtype=torch.float64)  # noqa: E731
            ring, rec = (t[b] for t in self.delta.states_views(self.states))
            want, _, S, _ = R.tokens(qkvz, ba, zero(ring), zero(rec), 0, nk=nk, nv=nv, dk=dk, dv=dv, eps=1e-6, split=self.split, **self.params)
            print(f"sequence {b} of {T}: DeltaNet {off(y, want):.1e}, state {off(rec, S):.1e}", flush=True)
            assert off(y, want) < 1e-5 and off(rec, S) < 1e-5
            q = q.view(T, self.H, 2, self.hd)
            x = self.rope.apply([q[:, :, 0]], self.table, norm_weights=[self.qw])[0].double()
            hidden = torch.ones((T, T), dtype=torch.bool, device="cuda").triu(1)
            want = torch.empty((T, self.H, self.hd), dtype=torch.float64, device="cuda")
            for h in range(self.H):
                kv = h * self.KVH // self.H
                s = x[:, h] @ kk[b, :T, kv].double().T.contiguous() / math.sqrt(self.hd)
                want[:, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vv[b, :T, kv].double().contiguous()
            want = (want * torch.sigmoid(q[:, :, 1].double())).reshape(T, -1)
            print(f"  attention {off(a, want):.1e}", flush=True)
            assert off(a, want) < 1e-5


@pytest.mark.parametrize("heads,split", [((4, 8, 64, 64), False), ((2, 4, 128, 128), True), ((2, 4, 8, 8), False)], ids=str)
@pytest.mark.parametrize("counts", [[150, 3, 70], [1, 64], [200]], ids=str)
def test_prompts_and_tokens(heads, split, counts):
    B, N, steps = len(counts), sum(counts), 4
    m = Stack(heads, split, B, max(counts) + 2 * steps, seed=N)
    ws = m.workspaces(N, max(counts))
    starts = torch.tensor(np.cumsum([0, *counts]), dtype=torch.int32, device="cuda")
    x = m.n(N, m.width)
    x, parts = m.run(x, ws, starts, max(counts))
    m.keep(parts, counts)
    x = x[starts[1:].long() - 1].clone()
    for _ in range(steps):
        x, parts = m.run(x, ws)
        m.keep(parts, [1] * B)
    # the same step captured
    before = [t.clone() for t in (m.states, m.cache.data, m.done)]
    given = x.clone()
    m.run(given, ws)
    for t, was in zip((m.states, m.cache.data, m.done), before):
        t.copy_(was)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, parts = m.run(given, ws)
    for _ in range(steps - 1):
        given.copy_(x)
        graph.replay()
        m.keep(parts, [1] * B)
        x = out.clone()
    torch.cuda.synchronize()
    assert m.done.tolist() == [n + 2 * steps - 1 for n in counts]
    m.check()


@pytest.mark.parametrize("prompt", [1, 5, None])
def test_tiny_q4_model_by_prompt_matches_mlx(prompt):
    """The tiny 4-bit model with the prompt's first tokens through each DeltaNet block in one call, the others one by one."""
    from oracle.qwen_tiny import TinyQwen
    from safetensors.numpy import load_file
    from swiftlet_amd.checkpoint import Checkpoint, moe_layer_from_checkpoint
    from swiftlet_amd.engine import HipEngine
    eng, d = HipEngine(), G / "tiny-model-q4"
    cfg = json.loads((d / "config.json").read_text())
    ck, m = Checkpoint(d), TinyQwen(d)
    fx = load_file(str(G / "tiny_forward_q4.safetensors"))
    toks = fx["input_ids"][0]
    S = len(toks)
    n = min(prompt or S, S)
    emb = ck.gpu_linear("model.embed_tokens")
    hd = torch.cat([eng.dequantize(emb, int(t), 1) for t in toks])
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        xin = eng.rms_norm(hd.clone(), ck.load(p + "input_layernorm.weight"), m.eps)
        if m.is_linear(i):
            blk = deltanet_from_checkpoint(ck, i, cfg)
            qkvz, ba = torch.empty((S, blk.conv_dim + blk.value_dim), device="cuda"), torch.empty((S, 2 * blk.nv), device="cuda")
            for t in range(S):
                eng.encode_gemv_multi(list(blk.projections), xin[t], [qkvz[t], ba[t]])
            states, ws = blk.new_states(1), blk.new_batch_workspace(1, S)
            at = torch.zeros(1, dtype=torch.int32, device="cuda")
            ys = [blk.prefill(qkvz[:n], ba[:n], states, at, ws)]
            for t in range(n, S):
                ys.append(blk.step_batch(qkvz[t:t + 1], ba[t:t + 1], states, at.fill_(t), ws))
            y, att = torch.cat(ys), torch.empty_like(hd)
            for t in range(S):
                eng.encode_gemv(blk.out_proj, y[t], att[t])
        else:
            att = torch.from_numpy(m.attention_forward(xin.cpu().numpy(), i)).cuda()
        x2 = eng.rms_norm(hd, ck.load(p + "post_attention_layernorm.weight"), m.eps, residual=att.contiguous())
        moe_layer_from_checkpoint(ck, i, cfg).decode(x2, out=hd, accumulate=True)
    hn = eng.rms_norm(hd, ck.load("model.norm.weight"), m.eps)
    head = ck.gpu_linear("lm_head")
    logits = torch.empty((S, head.out_dim), dtype=torch.float32, device="cuda")
    for t in range(S):
        eng.encode_gemv(head, hn[t], logits[t])
    torch.cuda.synchronize()
    got = logits.cpu().numpy()
    diff = np.abs(got - fx["logits"][0]).max()
    print(f"max |logit - mlx| = {diff:.3g}", flush=True)
    assert diff < 2e-3, diff
    assert np.argmax(got, axis=-1).tolist() == json.loads((G / "tiny_forward_q4.json").read_text())["greedy_next_tokens"]
