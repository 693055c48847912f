"""Minimal bs=1 greedy decode harness on the HIP backend.

The step order and every rounding point mirror the reference runtime's Triton
paths, with the fused options the Triton backend provides:

* ``DenseDecoder`` follows ``_forward_token_triton`` (gpu_runtime.py:11429-11726)
  with fused residual+RMSNorm, fused RoPE, the fused Triton attention backend and
  Triton elementwise ops; the greedy token comes from ``next_token_tensor``
  (gpu_runtime.py:11130-11209) in its default lm_head mode;
* ``MoEDecoder`` follows ``_forward_token_moe`` and ``_packed_moe_forward``
  (gpu_runtime.py:8968-9908) for MXFP4 experts.

Differences from the reference, by design:

* a flat KV cache ``[layers, kv_heads, capacity, head_dim]`` replaces the paged
  cache (same values, same attention);
* the token id and the position live on the device, so one decode step is captured
  once in a HIP graph and replayed for every token (the reference disables its
  CUDA graph for causal KV because it hard-codes the position,
  gpu_runtime.py:12594-12601);
* QKV and gate/up projections are one multi-matrix launch each, the MoE experts
  run as two fused launches, and attention biases are fused into the GEMV
  epilogue -- each with the reference's rounding points, so outputs are unchanged;
* the post-attention add_rms_norm the MoE path issues twice per layer
  (gpu_runtime.py:9233-9252 and 9254-9275, idempotent) runs once.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .backend import HipDecodeBackend
from .kv_cache import Int4KvCache
from .rotary import rotary_frequencies
from .synth import DenseWeights, MoEWeights

_ACT = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _int4_segment(seg: _lib.FusedSegment, weight, out: torch.Tensor, rows: int, kind: int, weight2=None) -> None:
    packed, scales = weight
    seg.weight = packed.data_ptr()
    seg.w_row_bytes = packed.stride(0) * packed.element_size()
    seg.scales = scales.data_ptr()
    seg.s_row = scales.stride(0)
    if weight2 is not None:
        seg.weight2 = weight2[0].data_ptr()
        seg.scales2 = weight2[1].data_ptr()
    seg.out = out.data_ptr()
    seg.rows = rows
    seg.kind = kind


def _dense_segment(seg: _lib.FusedSegment, weight: torch.Tensor, bias: torch.Tensor | None, out: torch.Tensor | None,
                   kind: int) -> None:
    seg.weight = weight.data_ptr()
    seg.w_row_bytes = weight.stride(0) * weight.element_size()
    seg.bias = bias.data_ptr() if bias is not None else None
    seg.out = out.data_ptr() if out is not None else None
    seg.rows = int(weight.shape[0])
    seg.kind = kind


def _kv_context(d: _lib.FusedGemv, dec: "_GraphedDecoder", cos: torch.Tensor, sin: torch.Tensor, head_dim: int,
                cache: torch.Tensor) -> None:
    d.position = dec.position.data_ptr()
    d.capacity = dec.capacity
    d.cache_head = cache.stride(0)
    d.cos_table = cos.data_ptr()
    d.sin_table = sin.data_ptr()
    d.table_row = cos.stride(0)
    d.table_rows = int(cos.shape[0])
    d.head_dim = head_dim


class _GraphedDecoder:
    """Common state: device token / position, token history, graph capture."""

    def __init__(self, backend: HipDecodeBackend, device: torch.device, capacity: int, max_new: int,
                 fused: bool = False) -> None:
        self.be = backend
        self.fused = fused
        self.device = device
        self.capacity = capacity
        self.token = backend._argmax_out_idx               # int64 0-d, written by the lm_head argmax
        self.position = torch.zeros(1, device=device, dtype=torch.int32)
        self.history = torch.zeros(max_new, device=device, dtype=torch.int64)
        self.base = torch.zeros(1, device=device, dtype=torch.int32)   # position of the first generated step
        self.graph: torch.cuda.CUDAGraph | None = None
        self._graph_stream: torch.cuda.Stream | None = None

    def prime(self, token: int, position: int) -> None:
        """Set the next input token and its position (host -> device, outside graphs)."""
        if not 0 <= position < self.capacity:
            raise ValueError("position outside the KV cache")
        self.token.fill_(int(token))
        self.position.fill_(int(position))
        self.base.fill_(int(position))
        self.history.zero_()

    def step(self) -> None:  # pragma: no cover - implemented by subclasses
        raise NotImplementedError

    def _step_and_record(self) -> None:
        if self.fused:
            # the fused step logs the token and advances the position in its last kernel
            self.fused_step()
            return
        self.step()
        self.be.record_token(self.token, self.position, self.base, self.history)
        self.be.advance_position(self.position)

    def fused_step(self) -> None:  # pragma: no cover - implemented by subclasses
        raise NotImplementedError

    def _reserve_scratch(self) -> None:  # pragma: no cover - implemented by subclasses
        raise NotImplementedError

    def capture(self) -> None:
        """Record one decode step (including token logging and the position advance)
        into a HIP graph.  The graph reads token/position from device memory.  All
        scratch is reserved beforehand, so no step runs (and no state changes) here."""
        self._reserve_scratch()
        torch.cuda.synchronize(self.device)
        self._graph_stream = torch.cuda.Stream(self.device)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self._graph_stream):
            self._step_and_record()

    def generate(self, start_token: int, position: int, steps: int, use_graph: bool = True) -> list[int]:
        """Greedy-decode `steps` tokens; returns the generated ids."""
        if position + steps > self.capacity:
            raise ValueError("not enough KV capacity for the requested steps")
        if steps > self.history.numel():
            raise ValueError("history buffer too small")
        if use_graph and self.graph is None:
            self.capture()
        self.prime(start_token, position)
        for _ in range(steps):
            if use_graph:
                self.graph.replay()
            else:
                self._step_and_record()
        torch.cuda.synchronize(self.device)
        return self.history[:steps].cpu().tolist()


class DenseDecoder(_GraphedDecoder):
    """Llama-3.2-1B-shaped int4 g128 decoder.

    ``fused=True`` runs the step as five launches per layer (QKV GEMV with the
    residual add + RMSNorm prologue and the RoPE / KV-append epilogue, attention
    partials and combine, o_proj, gate/up GEMV with the add + RMSNorm prologue and the
    SiLU epilogue, down_proj) and a final lm_head launch whose prologue is the last
    add + RMSNorm and whose finishing kernel also logs the token and advances the
    position.  Every rounding point is the unfused operator's, so both modes give
    the same bits."""

    def __init__(self, backend: HipDecodeBackend, weights: DenseWeights, fused: bool = False) -> None:
        s = weights.shape
        super().__init__(backend, weights.embed.device, int(weights.k_cache.shape[2]), s.max_new_tokens, fused)
        self.w = weights
        self.s = s
        dev, dt = weights.embed.device, torch.float16
        self.hidden_a = torch.empty(s.hidden, device=dev, dtype=dt)
        self.hidden_b = torch.empty(s.hidden, device=dev, dtype=dt)
        self.normed = torch.empty(s.hidden, device=dev, dtype=dt)
        self.qkv = torch.empty(s.q_dim + 2 * s.kv_dim, device=dev, dtype=dt)
        self.attn = torch.empty(s.q_dim, device=dev, dtype=dt)
        self.attn_out = torch.empty(s.hidden, device=dev, dtype=dt)
        self.gate_up = torch.empty(2 * s.intermediate, device=dev, dtype=dt)
        self.act = torch.empty(s.intermediate, device=dev, dtype=dt)
        self.mlp = torch.empty(s.hidden, device=dev, dtype=dt)
        self.final = torch.empty(s.hidden, device=dev, dtype=dt)

    def _reserve_scratch(self) -> None:
        s = self.s
        self.be._attention_scratch(s.heads, self.capacity, s.head_dim)
        self.be._argmax_scratch(int(self.w.lm_head.shape[0]), s.hidden)
        self.be.logits_buffer(int(self.w.lm_head.shape[0]), torch.float16)

    def step(self) -> None:
        be, w, s = self.be, self.w, self.s
        q, k, v = self.qkv[: s.q_dim], self.qkv[s.q_dim: s.q_dim + s.kv_dim], self.qkv[s.q_dim + s.kv_dim:]
        gate, up = self.gate_up[: s.intermediate], self.gate_up[s.intermediate:]
        be.embedding(w.embed, self.token, self.hidden_a)
        be.rms_norm(self.hidden_a, w.layers[0].ln1, self.normed, s.eps)
        for li, L in enumerate(w.layers):
            be.multi_int4_scaled_matvec((L.q[0], L.k[0], L.v[0]), (L.q[1], L.k[1], L.v[1]),
                                        (s.q_dim, s.kv_dim, s.kv_dim), s.hidden, self.normed, self.qkv,
                                        group_size=s.group)
            be.rope_qk_inplace(q, k, w.cos, w.sin, s.heads, s.kv_heads, s.head_dim, position=self.position)
            be.kv_append(k, v, w.k_cache[li], w.v_cache[li], self.position, s.kv_heads, s.head_dim)
            be.single_token_gqa_attention(q, w.k_cache[li], w.v_cache[li], self.attn, s.heads, s.kv_heads,
                                          s.head_dim, active_tokens=(self.position, 1))
            be.int4_scaled_matvec(L.o[0], L.o[1], self.attn, self.attn_out, rows=s.hidden, cols=s.q_dim,
                                  group_size=s.group)
            be.add_rms_norm(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps)
            be.multi_int4_scaled_matvec((L.gate[0], L.up[0]), (L.gate[1], L.up[1]), (s.intermediate, s.intermediate),
                                        s.hidden, self.normed, self.gate_up, group_size=s.group)
            be.silu_mul(gate, up, self.act)
            be.int4_scaled_matvec(L.down[0], L.down[1], self.act, self.mlp, rows=s.hidden, cols=s.intermediate,
                                  group_size=s.group)
            if li + 1 < len(w.layers):
                be.add_rms_norm(self.hidden_b, self.mlp, self.hidden_a, w.layers[li + 1].ln1, self.normed, s.eps)
            else:
                be.add_rms_norm(self.hidden_b, self.mlp, self.hidden_a, w.final_norm, self.final, s.eps)
        be.matvec_argmax_tensor(w.lm_head, self.final)

    def _build_fused(self) -> None:
        w, s = self.w, self.s
        act = _ACT[self.hidden_a.dtype]
        q = self.qkv[: s.q_dim]
        self._qkv_desc, self._gu_desc = [], []
        for li, L in enumerate(w.layers):
            d = _lib.FusedGemv()
            d.weight_format, d.group_size, d.act_dtype, d.cols = _lib.FMT_INT4_G, s.group, act, s.hidden
            if li == 0:
                d.prologue = _lib.PRO_EMBED_NORM
                d.embed, d.embed_row, d.vocab = w.embed.data_ptr(), w.embed.stride(0), int(w.embed.shape[0])
                d.token = self.token.data_ptr()
            else:
                d.prologue = _lib.PRO_ADD_NORM
                d.left, d.right = self.hidden_b.data_ptr(), self.mlp.data_ptr()
            d.norm_weight, d.eps, d.residual_out = L.ln1.data_ptr(), s.eps, self.hidden_a.data_ptr()
            d.count = 3
            _int4_segment(d.seg[0], L.q, q, s.q_dim, _lib.SEG_ROPE_OUT)
            _int4_segment(d.seg[1], L.k, w.k_cache[li], s.kv_dim, _lib.SEG_ROPE_CACHE)
            _int4_segment(d.seg[2], L.v, w.v_cache[li], s.kv_dim, _lib.SEG_CACHE)
            _kv_context(d, self, w.cos, w.sin, s.head_dim, w.k_cache[li])
            self._qkv_desc.append(d)
            g = _lib.FusedGemv()
            g.weight_format, g.group_size, g.act_dtype, g.cols = _lib.FMT_INT4_G, s.group, act, s.hidden
            g.prologue = _lib.PRO_ADD_NORM
            g.left, g.right = self.hidden_a.data_ptr(), self.attn_out.data_ptr()
            g.norm_weight, g.eps, g.residual_out = L.ln2.data_ptr(), s.eps, self.hidden_b.data_ptr()
            g.count = 1
            _int4_segment(g.seg[0], L.gate, self.act, s.intermediate, _lib.SEG_SILU, weight2=L.up)
            self._gu_desc.append(g)
        h = _lib.FusedGemv()
        h.weight_format, h.weight_dtype, h.act_dtype, h.cols = _lib.FMT_DENSE, _ACT[w.lm_head.dtype], act, s.hidden
        h.prologue = _lib.PRO_ADD_NORM
        h.left, h.right = self.hidden_b.data_ptr(), self.mlp.data_ptr()
        h.norm_weight, h.eps = w.final_norm.data_ptr(), s.eps
        h.count = 1
        _dense_segment(h.seg[0], w.lm_head, None, self.be.logits_buffer(int(w.lm_head.shape[0]), self.hidden_a.dtype),
                       _lib.SEG_PLAIN)
        self._head_desc = h

    def fused_step(self) -> None:
        be, w, s = self.be, self.w, self.s
        if not hasattr(self, "_head_desc"):
            self._build_fused()
        q = self.qkv[: s.q_dim]
        # the o_proj GEMV combines the attention chunk partials itself (head_dim-64 caches
        # of whole 64-token chunks, at most 32 query heads, 1/2/4/8 per KV head)
        combine = (s.head_dim == 64 and s.heads <= 32 and s.group == 128 and s.heads // s.kv_heads in (1, 2, 4, 8)
                   and int(w.k_cache[0].shape[1]) % 64 == 0 and w.k_cache[0].stride(1) == 64
                   and w.v_cache[0].stride(1) == 64)
        for li, L in enumerate(w.layers):
            be.fused_gemv(self._qkv_desc[li])
            if combine:
                be.attention_then_int4_matvec(q, w.k_cache[li], w.v_cache[li], s.heads, s.kv_heads, s.head_dim,
                                              L.o[0], L.o[1], self.attn_out, active_tokens=(self.position, 1))
            else:
                be.single_token_gqa_attention(q, w.k_cache[li], w.v_cache[li], self.attn, s.heads, s.kv_heads,
                                              s.head_dim, active_tokens=(self.position, 1))
                be.int4_scaled_matvec(L.o[0], L.o[1], self.attn, self.attn_out, rows=s.hidden, cols=s.q_dim,
                                      group_size=s.group)
            be.fused_gemv(self._gu_desc[li])
            be.int4_scaled_matvec(L.down[0], L.down[1], self.act, self.mlp, rows=s.hidden, cols=s.intermediate,
                                  group_size=s.group)
        be.fused_lm_head_argmax(self._head_desc, position=self.position, base=self.base, history=self.history)


class MoEDecoder(_GraphedDecoder):
    """gpt-oss-20B-shaped decoder with MXFP4 experts, fp16 attention with sinks.

    ``fused=True`` folds the embedding / residual add + RMSNorm into the QKV launch,
    RoPE and the KV append into its epilogue, the post-attention add + RMSNorm into the
    router launch, and the final add + RMSNorm, token log and position advance into the
    lm_head launches, with the unfused rounding points."""

    def __init__(self, backend: HipDecodeBackend, weights: MoEWeights, fused: bool = False) -> None:
        s = weights.shape
        super().__init__(backend, weights.embed.device, int(weights.k_cache.shape[2]), s.max_new_tokens, fused)
        self.w = weights
        self.s = s
        dev, dt = weights.embed.device, torch.float16
        self.hidden_a = torch.empty(s.hidden, device=dev, dtype=dt)
        self.hidden_b = torch.empty(s.hidden, device=dev, dtype=dt)
        self.normed = torch.empty(s.hidden, device=dev, dtype=dt)
        self.qkv = torch.empty(s.q_dim + 2 * s.kv_dim, device=dev, dtype=dt)
        self.attn = torch.empty(s.q_dim, device=dev, dtype=dt)
        self.attn_out = torch.empty(s.hidden, device=dev, dtype=dt)
        self.router_idx = torch.empty(s.top_k, device=dev, dtype=torch.int32)
        self.router_scores = torch.empty(s.top_k, device=dev, dtype=dt)
        self.router_logits = torch.empty((1, s.experts), device=dev, dtype=torch.float32)
        # the fused step hands the router logits to the SwiGLU launch, which takes the top-k
        # itself (False: the norm + router launch finishes the top-k)
        self.router_in_swiglu = True
        self.act = torch.empty((s.top_k, s.intermediate), device=dev, dtype=dt)
        self.moe = torch.empty(s.hidden, device=dev, dtype=dt)
        self.final = torch.empty(s.hidden, device=dev, dtype=dt)

    def _reserve_scratch(self) -> None:
        s = self.s
        self.be._attention_scratch(s.heads, self.capacity, s.head_dim)
        self.be._argmax_scratch(int(self.w.lm_head.shape[0]), s.hidden)
        self.be.logits_buffer(int(self.w.lm_head.shape[0]), torch.float16)
        self.be.reserve_batch_workspaces(1)

    def step(self) -> None:
        be, w, s = self.be, self.w, self.s
        q, k, v = self.qkv[: s.q_dim], self.qkv[s.q_dim: s.q_dim + s.kv_dim], self.qkv[s.q_dim + s.kv_dim:]
        be.embedding(w.embed, self.token, self.hidden_a)
        be.rms_norm(self.hidden_a, w.layers[0].ln1, self.normed, s.eps)
        for li, L in enumerate(w.layers):
            be.multi_matvec_bias((L.q, L.k, L.v), (L.q_bias, L.k_bias, L.v_bias), self.normed, self.qkv)
            be.rope_qk_inplace(q, k, w.cos, w.sin, s.heads, s.kv_heads, s.head_dim, position=self.position)
            be.kv_append(k, v, w.k_cache[li], w.v_cache[li], self.position, s.kv_heads, s.head_dim)
            be.single_token_gqa_attention(q, w.k_cache[li], w.v_cache[li], self.attn, s.heads, s.kv_heads,
                                          s.head_dim, sinks=L.sinks, active_tokens=(self.position, 1))
            be.multi_matvec_bias((L.o,), (L.o_bias,), self.attn, self.attn_out)
            be.add_rms_norm(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps)
            be.moe_router_matvec_topk(L.router, self.normed, self.router_idx, self.router_scores, bias=L.router_bias,
                                      renormalize=True)
            be.mxfp_lowbit_selected_swiglu(L.gate_up_blocks, L.gate_up_scales, self.normed, self.router_idx, self.act,
                                           bits=4, alpha=s.swiglu_alpha, limit=s.swiglu_limit, bias=L.gate_up_bias)
            be.mxfp_lowbit_weighted_down(L.down_blocks, L.down_scales, self.act, self.router_idx, self.router_scores,
                                         self.moe, bits=4, bias=L.down_bias)
            if li + 1 < len(w.layers):
                be.add_rms_norm(self.hidden_b, self.moe, self.hidden_a, w.layers[li + 1].ln1, self.normed, s.eps)
            else:
                be.add(self.hidden_b, self.moe, self.hidden_a)
                be.rms_norm(self.hidden_a, w.final_norm, self.final, s.eps)
        be.matvec_argmax_tensor(w.lm_head, self.final)

    def _build_fused(self) -> None:
        w, s = self.w, self.s
        act = _ACT[self.hidden_a.dtype]
        q = self.qkv[: s.q_dim]
        self._qkv_desc = []
        for li, L in enumerate(w.layers):
            d = _lib.FusedGemv()
            d.weight_format, d.weight_dtype, d.act_dtype, d.cols = _lib.FMT_DENSE, _ACT[L.q.dtype], act, s.hidden
            if li == 0:
                d.prologue = _lib.PRO_EMBED_NORM
                d.embed, d.embed_row, d.vocab = w.embed.data_ptr(), w.embed.stride(0), int(w.embed.shape[0])
                d.token = self.token.data_ptr()
            else:
                d.prologue = _lib.PRO_ADD_NORM
                d.left, d.right = self.hidden_b.data_ptr(), self.moe.data_ptr()
            d.norm_weight, d.eps, d.residual_out = L.ln1.data_ptr(), s.eps, self.hidden_a.data_ptr()
            d.count = 3
            _dense_segment(d.seg[0], L.q, L.q_bias, q, _lib.SEG_ROPE_OUT)
            _dense_segment(d.seg[1], L.k, L.k_bias, w.k_cache[li], _lib.SEG_ROPE_CACHE)
            _dense_segment(d.seg[2], L.v, L.v_bias, w.v_cache[li], _lib.SEG_CACHE)
            _kv_context(d, self, w.cos, w.sin, s.head_dim, w.k_cache[li])
            self._qkv_desc.append(d)
        h = _lib.FusedGemv()
        h.weight_format, h.weight_dtype, h.act_dtype, h.cols = _lib.FMT_DENSE, _ACT[w.lm_head.dtype], act, s.hidden
        h.prologue = _lib.PRO_ADD_RMS_NORM
        h.left, h.right = self.hidden_b.data_ptr(), self.moe.data_ptr()
        h.norm_weight, h.eps = w.final_norm.data_ptr(), s.eps
        h.count = 1
        _dense_segment(h.seg[0], w.lm_head, None, self.be.logits_buffer(int(w.lm_head.shape[0]), self.hidden_a.dtype),
                       _lib.SEG_PLAIN)
        self._head_desc = h

    def fused_step(self) -> None:
        be, w, s = self.be, self.w, self.s
        if not hasattr(self, "_head_desc"):
            self._build_fused()
        q = self.qkv[: s.q_dim]
        for li, L in enumerate(w.layers):
            be.fused_gemv(self._qkv_desc[li])
            be.single_token_gqa_attention(q, w.k_cache[li], w.v_cache[li], self.attn, s.heads, s.kv_heads,
                                          s.head_dim, sinks=L.sinks, active_tokens=(self.position, 1))
            be.multi_matvec_bias((L.o,), (L.o_bias,), self.attn, self.attn_out)
            if self.router_in_swiglu:
                be.add_rms_norm_router_logits(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps,
                                              L.router, self.router_logits, bias=L.router_bias)
                be.mxfp_lowbit_selected_swiglu_router(L.gate_up_blocks, L.gate_up_scales, self.normed,
                                                      self.router_logits, self.router_idx, self.router_scores,
                                                      self.act, bits=4, alpha=s.swiglu_alpha, limit=s.swiglu_limit,
                                                      renormalize=True, bias=L.gate_up_bias)
            else:
                be.add_rms_norm_router_topk(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps,
                                            L.router, self.router_idx, self.router_scores, bias=L.router_bias,
                                            renormalize=True)
                be.mxfp_lowbit_selected_swiglu(L.gate_up_blocks, L.gate_up_scales, self.normed, self.router_idx,
                                               self.act, bits=4, alpha=s.swiglu_alpha, limit=s.swiglu_limit,
                                               bias=L.gate_up_bias)
            be.mxfp_lowbit_weighted_down(L.down_blocks, L.down_scales, self.act, self.router_idx, self.router_scores,
                                         self.moe, bits=4, bias=L.down_bias)
        be.fused_lm_head_argmax(self._head_desc, position=self.position, base=self.base, history=self.history)


class MoEBatchDecoder:
    """``batch`` independent gpt-oss-shaped sequences decoded in lockstep, one token of each
    per step (eight independent bs=1 routings at batch 8; the reference decodes one token
    per step and has no batched path).

    Every sequence has its own KV cache (``k_cache``/``v_cache`` [layers, batch * kv_heads,
    capacity, head_dim]: sequence b owns KV heads b * kv_heads ...) and token; the position
    is shared.  Every launch covers the whole batch: the fused QKV (norm prologue, RoPE /
    cache epilogue) and o_proj with a token grid dimension, attention (the batch's query
    and KV heads are the heads of one call, so each head's arithmetic is the bs=1
    arithmetic), add+RMSNorm+router (one workgroup per token), the expert SwiGLU and
    weighted down (token-indexed slots) and the M-row lm_head argmax; only the final
    add + RMSNorm runs per sequence.  Each sequence's tokens equal
    MoEDecoder's stream for that sequence bit for bit."""

    def __init__(self, backend: HipDecodeBackend, weights: MoEWeights, batch: int, k_cache: torch.Tensor,
                 v_cache: torch.Tensor) -> None:
        s = weights.shape
        if batch < 1:
            raise ValueError("batch must be at least 1")
        want = (s.layers, batch * s.kv_heads)
        if tuple(k_cache.shape[:2]) != want or k_cache.shape != v_cache.shape or k_cache.shape[3] != s.head_dim:
            raise ValueError(f"KV caches must be [{s.layers}, {batch * s.kv_heads}, capacity, {s.head_dim}]")
        self.be, self.w, self.s, self.batch = backend, weights, s, batch
        dev = weights.embed.device
        self.device = dev
        self.k_cache, self.v_cache = k_cache, v_cache
        self.capacity = int(k_cache.shape[2])
        self.tokens = torch.zeros(batch, device=dev, dtype=torch.int64)
        self.position = torch.zeros(1, device=dev, dtype=torch.int32)
        self.base = torch.zeros(1, device=dev, dtype=torch.int32)
        self.history = torch.zeros((batch, s.max_new_tokens), device=dev, dtype=torch.int64)
        dt = torch.float16
        self.q_all = torch.empty((batch, s.q_dim), device=dev, dtype=dt)
        self.attn_all = torch.empty((batch, s.q_dim), device=dev, dtype=dt)
        self.final_all = torch.empty((batch, s.hidden), device=dev, dtype=dt)
        self.hidden_a = torch.empty((batch, s.hidden), device=dev, dtype=dt)
        self.hidden_b = torch.empty((batch, s.hidden), device=dev, dtype=dt)
        self.normed = torch.empty((batch, s.hidden), device=dev, dtype=dt)
        self.attn_out = torch.empty((batch, s.hidden), device=dev, dtype=dt)
        self.moe = torch.empty((batch, s.hidden), device=dev, dtype=dt)
        self.router_idx = torch.empty((batch, s.top_k), device=dev, dtype=torch.int32)
        self.router_scores = torch.empty((batch, s.top_k), device=dev, dtype=dt)
        self.router_logits = torch.empty((batch, s.experts), device=dev, dtype=torch.float32)
        # as MoEDecoder.router_in_swiglu; off here: the top-k of every wave in the batched
        # SwiGLU launch measured 2215 -> 2131 tok/s at eight sequences (bs=1: 711 -> 717)
        self.router_in_swiglu = False
        self.act = torch.empty((batch * s.top_k, s.intermediate), device=dev, dtype=dt)
        self.sinks = [L.sinks.repeat(batch).contiguous() for L in weights.layers]
        self._build_qkv()
        self.graph: torch.cuda.CUDAGraph | None = None
        self._graph_stream: torch.cuda.Stream | None = None

    def _build_qkv(self) -> None:
        """One multi-token fused QKV descriptor per layer: MoEDecoder's descriptor with the
        batch's buffers and per-token strides (sequence t's KV heads follow sequence t-1's)."""
        w, s, B = self.w, self.s, self.batch
        act = _ACT[torch.float16]
        self._qkv_desc = []
        for li, L in enumerate(w.layers):
            d = _lib.FusedGemv()
            d.weight_format, d.weight_dtype, d.act_dtype, d.cols = _lib.FMT_DENSE, _ACT[L.q.dtype], act, s.hidden
            if li == 0:
                d.prologue = _lib.PRO_EMBED_NORM
                d.embed, d.embed_row, d.vocab = w.embed.data_ptr(), w.embed.stride(0), int(w.embed.shape[0])
                d.token = self.tokens.data_ptr()
            else:
                d.prologue = _lib.PRO_ADD_NORM
                d.left, d.right = self.hidden_b.data_ptr(), self.moe.data_ptr()
            d.norm_weight, d.eps, d.residual_out = L.ln1.data_ptr(), s.eps, self.hidden_a.data_ptr()
            d.count = 3
            _dense_segment(d.seg[0], L.q, L.q_bias, self.q_all, _lib.SEG_ROPE_OUT)
            _dense_segment(d.seg[1], L.k, L.k_bias, self.k_cache[li], _lib.SEG_ROPE_CACHE)
            _dense_segment(d.seg[2], L.v, L.v_bias, self.v_cache[li], _lib.SEG_CACHE)
            _kv_context(d, self, w.cos, w.sin, s.head_dim, self.k_cache[li])
            d.tokens, d.token_x, d.token_out = B, s.hidden, s.q_dim
            d.token_cache = s.kv_heads * self.k_cache[li].stride(0)
            self._qkv_desc.append(d)

    def _reserve_scratch(self) -> None:
        s = self.s
        self.be._attention_scratch(self.batch * s.heads, self.capacity, s.head_dim)
        self.be._batched_argmax_scratch(self.batch, int(self.w.lm_head.shape[0]), s.hidden)
        self.be.reserve_batch_workspaces(self.batch)

    def step(self) -> None:
        """One token of every sequence, logged at history[:, position - base]; advances the position."""
        be, w, s, B = self.be, self.w, self.s, self.batch
        for li, L in enumerate(w.layers):
            be.fused_gemv(self._qkv_desc[li])
            be.single_token_gqa_attention(self.q_all.view(-1), self.k_cache[li], self.v_cache[li],
                                          self.attn_all.view(-1), B * s.heads, B * s.kv_heads, s.head_dim,
                                          sinks=self.sinks[li], active_tokens=(self.position, 1))
            be.matvec_bias_rows(L.o, L.o_bias, self.attn_all, self.attn_out)
            if self.router_in_swiglu:
                be.add_rms_norm_router_logits(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps,
                                              L.router, self.router_logits, bias=L.router_bias)
                be.mxfp_lowbit_selected_swiglu_router(L.gate_up_blocks, L.gate_up_scales, self.normed,
                                                      self.router_logits, self.router_idx, self.router_scores,
                                                      self.act, bits=4, alpha=s.swiglu_alpha, limit=s.swiglu_limit,
                                                      renormalize=True, bias=L.gate_up_bias)
            else:
                be.add_rms_norm_router_topk(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps,
                                            L.router, self.router_idx, self.router_scores, bias=L.router_bias,
                                            renormalize=True)
                be.mxfp_lowbit_selected_swiglu_tokens(L.gate_up_blocks, L.gate_up_scales, self.normed,
                                                      self.router_idx, self.act, bits=4, alpha=s.swiglu_alpha,
                                                      limit=s.swiglu_limit, bias=L.gate_up_bias)
            be.mxfp_lowbit_weighted_down_tokens(L.down_blocks, L.down_scales, self.act, self.router_idx,
                                                self.router_scores, self.moe, bits=4, bias=L.down_bias)
        be.add_then_rms_norm_rows(self.hidden_b, self.moe, self.hidden_a, w.final_norm, self.final_all, s.eps)
        be.matvec_argmax_batched(w.lm_head, self.final_all, out=self.tokens)
        be.record_tokens_advance(self.tokens, self.position, self.base, self.history)

    def capture(self) -> None:
        """Record one batched step into a HIP graph (scratch reserved first)."""
        self._reserve_scratch()
        torch.cuda.synchronize(self.device)
        self._graph_stream = torch.cuda.Stream(self.device)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self._graph_stream):
            self.step()

    def prime(self, tokens: list[int], position: int) -> None:
        if len(tokens) != self.batch:
            raise ValueError("one start token per sequence")
        if not 0 <= position < self.capacity:
            raise ValueError("position outside the KV cache")
        self.tokens.copy_(torch.tensor(tokens, dtype=torch.int64))
        self.position.fill_(int(position))
        self.base.fill_(int(position))
        self.history.zero_()

    def generate(self, start_tokens: list[int], position: int, steps: int, use_graph: bool = True) -> list[list[int]]:
        """Greedy-decode `steps` tokens of every sequence; returns one id list per sequence."""
        if position + steps > self.capacity:
            raise ValueError("not enough KV capacity for the requested steps")
        if steps > self.history.shape[1]:
            raise ValueError("history buffer too small")
        if use_graph and self.graph is None:
            self.capture()
        self.prime(start_tokens, position)
        for _ in range(steps):
            if use_graph:
                self.graph.replay()
            else:
                self.step()
        torch.cuda.synchronize(self.device)
        return self.history[:, :steps].cpu().tolist()


class DenseBatchDecoder:
    """Requests of a dense int4 model decoded together, each at its own position over a KV cache of
    4 bits, their tokens sampled from given uniform numbers.

    Every launch covers the batch, but for the embedding, which is one per request: batched int4 GEMMs, rotary
    positions from frequencies (``rotary``: frequencies and amplitude of
    :func:`~thintensor_amd.rotary.rotary_frequencies`, by default the model's theta), the append to each layer's
    cache, attention (optionally a window of ``window`` tokens and ``first_tokens`` first ones, planned for the
    capacity), the lm_head's logits and ``sample_rows``.  Sampling settings are per request
    (:meth:`set_sampling`, greedy at first).  The model's head also leaves its argmax in ``greedy``.  A step of
    the 1B model takes 0.94 ms for one request, 1.37 for 8 and 2.36 for 64 in a graph (500 tokens each, capacity
    1024), 1.67, 1.67 and 2.39 launched one by one.  A request that has reached the capacity
    keeps decoding without storing further tokens; one whose logits leave nothing gets token -1 and stays
    there until it is primed again, the others' tokens are what they were."""

    def __init__(self, backend: HipDecodeBackend, weights: DenseWeights, batch: int, capacity: int, *,
                 group_size: int = 32, window: int = 0, first_tokens: int = 0,
                 rotary: tuple[torch.Tensor, float] | None = None) -> None:
        s = weights.shape
        if not 1 <= batch <= 64 or capacity < 1:
            raise ValueError("a batch is of 1 to 64 requests (of the batched GEMMs), the capacity at least 1")
        self.be, self.w, self.s, self.batch = backend, weights, s, batch
        dev = weights.embed.device
        self.device, dt = dev, torch.float16
        self.window, self.first_tokens = window, first_tokens
        self.inv_freq, self.amplitude = rotary or rotary_frequencies(s.head_dim, s.rope_theta, device=dev)
        self.caches = [Int4KvCache.allocate(batch, s.kv_heads, capacity, s.head_dim, group_size, dev)
                       for _ in weights.layers]
        self.capacity = self.caches[0].capacity
        self.tokens = torch.zeros(batch, device=dev, dtype=torch.int64)
        self.positions = torch.zeros(batch, device=dev, dtype=torch.int32)   # of the tokens to come
        self.lengths = torch.ones(batch, device=dev, dtype=torch.int32)      # positions + 1
        self.uniforms = torch.zeros(batch, device=dev)
        self.temperature = torch.zeros(batch, device=dev)
        self.top_k = torch.zeros(batch, device=dev, dtype=torch.int32)
        self.top_p = torch.ones(batch, device=dev)
        self.min_p = torch.zeros(batch, device=dev)
        self.probs = torch.zeros(batch, device=dev)
        empty = lambda n: torch.empty((batch, n), device=dev, dtype=dt)  # noqa: E731
        self.zeros = torch.zeros((batch, s.hidden), device=dev, dtype=dt)
        self.embedded, self.hidden_a, self.hidden_b = empty(s.hidden), empty(s.hidden), empty(s.hidden)
        self.normed, self.attn_out, self.mlp = empty(s.hidden), empty(s.hidden), empty(s.hidden)
        self.q, self.k, self.v, self.attn = empty(s.q_dim), empty(s.kv_dim), empty(s.kv_dim), empty(s.q_dim)
        self.gate, self.up, self.act = empty(s.intermediate), empty(s.intermediate), empty(s.intermediate)
        self.greedy = torch.zeros(batch, device=dev, dtype=torch.int64)
        self.logits = empty(int(weights.lm_head.shape[0]))
        self.graph: torch.cuda.CUDAGraph | None = None
        self._graph_stream: torch.cuda.Stream | None = None
        self._graph_scratch: torch.Tensor | None = None

    def set_sampling(self, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0) -> None:
        """Settings of every request: a number for all of them, or one per request."""
        for buf, value in ((self.temperature, temperature), (self.top_k, top_k), (self.top_p, top_p), (self.min_p, min_p)):
            buf.copy_(torch.as_tensor(value, dtype=buf.dtype).expand(self.batch))

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor,
               counts: torch.Tensor | None = None) -> None:
        """Tokens that the requests already hold (rotated k, v [batch, tokens, kv_heads, head_dim])."""
        self.be.kv_append_int4(self.caches[layer], k, v, starts, counts)

    def step(self) -> None:
        """One token of every request from ``uniforms``; advances the positions."""
        be, w, s, B = self.be, self.w, self.s, self.batch
        heads = self.q.view(B, s.heads, s.head_dim)
        k, v = self.k.view(B, s.kv_heads, s.head_dim), self.v.view(B, s.kv_heads, s.head_dim)
        # the embedding writes nothing for token -1, whose row then is NaN: no logits, token -1 again
        self.embedded.fill_(math.nan)
        for b in range(B):
            be.embedding(w.embed, self.tokens[b], self.embedded[b])
        left, right = self.embedded, self.zeros
        for li, L in enumerate(w.layers):
            be.add_then_rms_norm_rows(left, right, self.hidden_a, L.ln1, self.normed, s.eps)
            for (packed, scales), out in ((L.q, self.q), (L.k, self.k), (L.v, self.v)):
                be.int4_batched_matvec(packed, scales, self.normed, out, group_size=s.group)
            be.rotary_rows(heads, k, self.positions, self.inv_freq, amplitude=self.amplitude)
            be.kv_append_int4(self.caches[li], k, v, self.positions)
            be.gqa_attention_int4(heads, self.caches[li], self.attn.view(B, s.heads, s.head_dim), self.lengths,
                                  window=self.window, first_tokens=self.first_tokens)
            be.int4_batched_matvec(L.o[0], L.o[1], self.attn, self.attn_out, group_size=s.group)
            be.add_then_rms_norm_rows(self.hidden_a, self.attn_out, self.hidden_b, L.ln2, self.normed, s.eps)
            be.int4_batched_matvec(L.gate[0], L.gate[1], self.normed, self.gate, group_size=s.group)
            be.int4_batched_matvec(L.up[0], L.up[1], self.normed, self.up, group_size=s.group)
            be.silu_mul(self.gate, self.up, self.act)
            be.int4_batched_matvec(L.down[0], L.down[1], self.act, self.mlp, group_size=s.group)
            left, right = self.hidden_b, self.mlp
        be.add_then_rms_norm_rows(left, right, self.hidden_a, w.final_norm, self.normed, s.eps)
        be.matvec_argmax_batched(w.lm_head, self.normed, logits=self.logits, out=self.greedy)
        be.sample_rows(self.logits, self.uniforms, self.tokens, temperature=self.temperature, top_k=self.top_k,
                       top_p=self.top_p, min_p=self.min_p, probs=self.probs)
        self.positions.add_(1)
        self.lengths.add_(1)

    def capture(self) -> None:
        """Record one step into a HIP graph.  The lm_head's scratch belongs to the backend, which replaces
        it when a larger batch comes, and is held here for the graph (so graphs of decoders that share a
        backend replay one at a time); the other operators take theirs from the graph's own pool."""
        self._graph_scratch = self.be._batched_argmax_scratch(self.batch, int(self.w.lm_head.shape[0]), self.s.hidden)
        torch.cuda.synchronize(self.device)
        self._graph_stream = torch.cuda.Stream(self.device)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=self._graph_stream):
            self.step()

    def prime(self, tokens: list[int], positions: list[int]) -> None:
        """The requests' next input tokens and the positions that these take."""
        if len(tokens) != self.batch or len(positions) != self.batch:
            raise ValueError("one start token and position per request")
        if not all(0 <= t < int(self.w.embed.shape[0]) for t in tokens):
            raise ValueError("start token outside the vocabulary")
        if not all(0 <= p < self.capacity for p in positions):
            raise ValueError("position outside the KV cache")
        self.tokens.copy_(torch.tensor(tokens, dtype=torch.int64))
        self.positions.copy_(torch.tensor(positions, dtype=torch.int32))
        self.lengths.copy_(torch.tensor(positions, dtype=torch.int32) + 1)

    def generate(self, tokens: list[int], positions: list[int], uniforms: torch.Tensor, use_graph: bool = True) -> list[list[int]]:
        """One token per row of ``uniforms`` [steps, batch] for every request; one id list per request."""
        steps = int(uniforms.shape[0])
        if uniforms.ndim != 2 or uniforms.shape[1] != self.batch or uniforms.dtype != torch.float32:
            raise ValueError("uniforms must be float32 [steps, batch]")
        if max(positions) + steps > self.capacity:
            raise ValueError("not enough KV capacity for the requested steps")
        if use_graph and self.graph is None:
            self.capture()
        self.prime(tokens, positions)
        history = torch.empty((steps, self.batch), device=self.device, dtype=torch.int64)
        uniforms = uniforms.to(self.device)
        for i in range(steps):
            self.uniforms.copy_(uniforms[i])
            if use_graph:
                self.graph.replay()
            else:
                self.step()
            history[i].copy_(self.tokens)
        torch.cuda.synchronize(self.device)
        return history.t().cpu().tolist()
