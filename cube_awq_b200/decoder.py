"""A decoder layer on INT4 weights, from this library's operators alone.

The reference offers the quantised linears (``AWQGEMMLinear``,
src/modules/awq_gemm.rs:127-233) and leaves the layer around them to its host
framework. :class:`AWQDecoderLayer` is that layer for the pre-norm, gated-MLP,
rotary decoders that AutoAWQ checkpoints hold:

    h, r  = rms_norm(x + r)            residual stream r in F
    q,k,v = qkv(h)                     one fused INT4 GEMM
    q     = rope_append(q, k, v)       rotary, k and v into the paged cache
    a     = attention(q, cache)        one token per sequence, or prompts
    h, r  = rms_norm(o(a) + r)
    x     = down(silu(gate(h)) * up(h))

Eight to ten launches a layer: the attention is one of them, two where it splits
long caches and joins the parts, three where a batch of prompts and short runs
behind long caches takes both of its forms.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .errors import ShapeError
from .layer_ops import attention_decode, attention_prefill, rms_norm, rope_append
from .modules import AWQGateUpSiluMul, AWQGEMMLinear, AWQQKVLinear


class AWQDecoderLayer:
    """One decoder layer. ``input_norm`` and ``post_norm`` are the RMS norms'
    weights [hidden] in F; ``n_q`` query and ``n_kv`` key / value heads of
    ``head_dim``; ``window`` and ``sinks`` as in :func:`attention_decode`."""

    def __init__(self, input_norm: torch.Tensor, qkv: AWQQKVLinear, o: AWQGEMMLinear,
                 post_norm: torch.Tensor, gate_up: AWQGateUpSiluMul, down: AWQGEMMLinear,
                 n_q: int, n_kv: int, head_dim: int, eps: float = 1e-6,
                 window: Optional[int] = None, sinks: int = 0):
        hidden = input_norm.shape[0]
        for what, got, want in (
                ("post_norm", post_norm.shape[0], hidden),
                ("qkv's input", qkv.d_input, hidden),
                ("qkv's q output", qkv.n_q, n_q * head_dim),
                ("qkv's k and v outputs", qkv.n_kv, n_kv * head_dim),
                ("o's input", o.qweight.shape[0], n_q * head_dim),
                ("o's output", o.scales.shape[1], hidden),
                ("gate_up's input", gate_up.d_input, hidden),
                ("down's input", down.qweight.shape[0], gate_up.d_output),
                ("down's output", down.scales.shape[1], hidden)):
            if got != want:
                raise ShapeError(f"{what} must be {want}, got {got}", _lib.CAWQ_ERR_INVALID_SHAPE)
        self.input_norm, self.post_norm = input_norm, post_norm
        self.qkv, self.o, self.gate_up, self.down = qkv, o, gate_up, down
        self.n_q, self.n_kv, self.head_dim = n_q, n_kv, head_dim
        self.eps, self.window, self.sinks = eps, window, sinks

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor], rope: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                seq_lens: torch.Tensor, q_start: Optional[torch.Tensor] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
        """x [tokens, hidden]: the previous layer's output, ``residual`` its
        residual stream (None before the first layer: x is the stream). Returns
        (output, residual) for the next layer; after the last one, the stream
        is their sum (``rms_norm(x, norm, residual=residual)``). The batch is
        described as in :mod:`cube_awq_b200.layer_ops`; this layer's keys and
        values go to ``k_cache`` and ``v_cache``."""
        tokens = x.shape[0]
        h, stream = rms_norm(x, self.input_norm, self.eps, residual=residual)
        if stream is None:
            stream = x
        q, k, v = self.qkv(h)
        q = q.view(tokens, self.n_q, self.head_dim)
        heads = (tokens, self.n_kv, self.head_dim)
        q = rope_append(q, k.view(heads), v.view(heads), rope, k_cache, v_cache, block_table,
                        seq_lens, q_start=q_start, out=q)
        if q_start is None:
            a = attention_decode(q, k_cache, v_cache, block_table, seq_lens, window=self.window,
                                 sinks=self.sinks)
        else:
            a = attention_prefill(q, k_cache, v_cache, block_table, seq_lens, q_start,
                                  window=self.window, sinks=self.sinks)
        a = self.o(a.view(tokens, self.n_q * self.head_dim))
        h, stream = rms_norm(a, self.post_norm, self.eps, residual=stream)
        return self.down(self.gate_up(h)), stream

    __call__ = forward
