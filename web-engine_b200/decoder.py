"""A text decoder's layers, one token at a time: int4 weights, a 4-bit K/V cache, cross attention to another sequence's
states (the caption of an image, or a prompt rewritten from an image's tokens; no reference counterpart).

A layer, for the newest token x of each sequence (f32, one row per sequence):

    x += wo attention(rope(norm_q(wq h)), K, V),  h = norm1(x);  K, V: the cache, this token's k and v appended
    x += wo' cross_attention(wq' h', K', V'),     h' = norm2(x); K', V' = the states' projections, made once
    x += down(silu(gate h'') up h''),             h'' = norm3(x)

`step` runs every layer for one token of every sequence: the linears on `kernels.matvec` (the residual adds and the
SwiGLU in its epilogue), the cache on `kv4`, the states on `kernels.cross_attention`. Its launches are recorded once as
a CUDA graph; what changes from token to token (lengths, the RoPE rows) is read from device memory.
`prompt` runs many tokens of one sequence: the linears on `kernels.matmul`, causal attention over the rows of the cache
as it holds them, so that a prompt and its tokens one by one agree to rounding.
"""
from __future__ import annotations

from dataclasses import dataclass, replace

import numpy as np

from . import _lib as L
from . import kernels as K
from . import kv4, ops
from .graph import Binding, Buffer, Graph, addr


@dataclass
class DecoderConfig:
    """Sizes of a layer. hidden, mlp and heads * head_dim are multiples of 64 (int4 groups); head_dim 64, 128 or 256."""

    hidden: int
    mlp: int
    heads: int
    kv_heads: int
    head_dim: int
    eps: float = 1e-5
    norm_offset: float = 0.0  # 1: zero-centred norm weights
    theta: float = 10000.0
    pairing: str = "half"
    page: int = 64


@dataclass
class DecoderLayer:
    """One layer's weights: int4 linears (ops.Linear, no LoRA) and f32 norm weights. The cross_* linears and norm are all
    given or all None (a layer that sees no states); cross_k and cross_v project the states."""

    norm: object
    q: ops.Linear
    k: ops.Linear
    v: ops.Linear
    o: ops.Linear
    q_norm: object
    k_norm: object
    mlp_norm: object
    gate: ops.Linear
    up: ops.Linear
    down: ops.Linear
    cross_norm: object = None
    cross_q: ops.Linear | None = None
    cross_k: ops.Linear | None = None
    cross_v: ops.Linear | None = None
    cross_o: ops.Linear | None = None


class Decoder:
    """Layers, their caches and the buffers of a step for `batch` sequences (at most 16) of up to `tokens` tokens.

    x: the device buffer [batch, hidden] f32 that `step` reads the tokens' embeddings from and leaves the last layer's
    output in. lengths: tokens of each sequence so far (host copy of the caches' shared lengths)."""

    def __init__(self, graph: Graph, cfg: DecoderConfig, layers: list[DecoderLayer], batch: int, tokens: int):
        if not 1 <= batch <= L.MATVEC_MAX_ROWS:
            raise ValueError(f"a step takes 1 to {L.MATVEC_MAX_ROWS} sequences, got {batch}")
        if cfg.heads % cfg.kv_heads:
            raise ValueError("heads must be a multiple of kv_heads")
        qw, kw = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        for i, w in enumerate(layers):
            shapes = {"q": (qw, cfg.hidden), "k": (kw, cfg.hidden), "v": (kw, cfg.hidden), "o": (cfg.hidden, qw),
                      "gate": (cfg.mlp, cfg.hidden), "up": (cfg.mlp, cfg.hidden), "down": (cfg.hidden, cfg.mlp)}
            cross = [w.cross_norm, w.cross_q, w.cross_k, w.cross_v, w.cross_o]
            if any(p is not None for p in cross):
                if any(p is None for p in cross):
                    raise ValueError(f"layer {i}: all of the cross attention's weights or none")
                shapes |= {"cross_q": (qw, cfg.hidden), "cross_k": (kw, w.cross_k.k), "cross_v": (kw, w.cross_k.k),
                           "cross_o": (cfg.hidden, qw)}
            for name, (n, k) in shapes.items():
                m = getattr(w, name)
                if m.dtype != "int4" or m.lora is not None or (m.n, m.k) != (n, k):
                    raise ValueError(f"layer {i}: {name} must be an int4 linear [{n}, {k}] without LoRA")
        self.graph, self.cfg, self.layers, self.batch, self.tokens = graph, cfg, layers, batch, tokens
        self.lengths = [0] * batch
        self.x = graph.buffer(batch * cfg.hidden * 4)
        self.caches: list[kv4.Cache] = []
        for _ in layers:
            self.caches.append(kv4.Cache.create(graph, batch, tokens, cfg.kv_heads, cfg.head_dim, cfg.page,
                                                like=self.caches[0] if self.caches else None))
        pairs = cfg.head_dim // 2
        self._rope = graph.buffer(2 * batch * pairs * 4)  # cos rows, then sin rows
        self._states: list[tuple] = []
        self._state_lengths = None
        self._state_tokens = 0
        bf = lambda n: graph.buffer(batch * n * 2)  # noqa: E731
        self._h, self._q, self._k, self._v = bf(cfg.hidden), bf(qw), bf(kw), bf(kw)
        self._qr, self._kr, self._a, self._g, self._u = bf(qw), bf(kw), bf(qw), bf(cfg.mlp), bf(cfg.mlp)
        self._captured = None

    # ---- states ----
    def set_states(self, states, tokens: int, lengths=None) -> None:
        """Projects the states [batch, tokens, width] (bf16, on the device) to every layer's keys and values, once for all
        tokens to come. lengths: how many states of each sequence are real (default: all)."""
        g, kw = self.graph, self.cfg.kv_heads * self.cfg.head_dim
        if any(w.cross_k is not None for w in self.layers) and tokens < 1:
            raise ValueError("the layers attend to states: at least one token of them")
        n = [tokens] * self.batch if lengths is None else [int(v) for v in lengths]
        if len(n) != self.batch:
            raise ValueError(f"one length for each of {self.batch} sequences, got {len(n)}")
        self._drop()
        for pair in self._states:
            for b in pair or ():
                g.free(b)
        if self._state_lengths is not None:
            g.free(self._state_lengths)
        self._states, self._state_lengths = [], None  # (none, should what follows fail)
        made: list[Buffer] = []
        try:
            pairs = []
            for w in self.layers:
                if w.cross_k is None:
                    pairs.append(None)
                    continue
                for m in (w.cross_k, w.cross_v):
                    made.append(g.buffer(self.batch * tokens * kw * 2))
                    self._matmul(states, m, made[-1], self.batch * tokens)
                pairs.append((made[-2], made[-1]))
            of_each = g.buffer(np.asarray(n, np.int32))
        except BaseException:
            for b in made:
                g.free(b)
            raise
        self._states, self._state_tokens, self._state_lengths = pairs, tokens, of_each

    # ---- one token of every sequence ----
    def step(self, x=None) -> Buffer:
        """The next token of every sequence: x [batch, hidden] f32 (host array; None: `self.x` holds it already).
        Returns self.x, the last layer's output, in stream order. Every sequence takes part: a full one is an error for
        all of them, and `reset` empties them together."""
        g, cfg = self.graph, self.cfg
        self._ready()
        if max(self.lengths) >= self.tokens:
            raise ValueError(f"a sequence is full ({self.tokens} tokens)")
        if x is not None:
            x = np.ascontiguousarray(x, np.float32)
            if x.size != self.batch * cfg.hidden:
                raise ValueError(f"x must hold {self.batch} x {cfg.hidden} values, got {x.size}")
        cos, sin, _ = K.rope_tables(np.asarray(self.lengths), (cfg.head_dim,), cfg.theta)
        g.write(self._rope, np.concatenate([cos, sin]))
        if x is not None:
            g.write(self.x, x)
        if self._captured is None:
            with g.capture() as cap:
                self._layers_of_step()
            self._captured = cap
        self._captured.launch()
        self.lengths = [n + 1 for n in self.lengths]
        return self.x

    def _layers_of_step(self) -> None:
        g, cfg, m = self.graph, self.cfg, self.batch
        pairs = cfg.head_dim // 2
        cos, sin = self._rope, Binding(self._rope, m * pairs * 4, m * pairs * 4)
        to_bf16 = {"x_dtype": "bf16", "y_dtype": "bf16"}
        residual = {"x_dtype": "bf16", "y_dtype": "f32", "accumulate": True}
        for w, cache, states in zip(self.layers, self.caches, self._states or [None] * len(self.layers)):
            self._norm(self.x, w.norm, m, self._h)
            self._matvec(self._h, w.q, self._q, **to_bf16)
            self._matvec(self._h, w.k, self._k, **to_bf16)
            self._matvec(self._h, w.v, self._v, **to_bf16)
            self._rotate(self._q, w.q_norm, cos, sin, m, cfg.heads, self._qr)
            self._rotate(self._k, w.k_norm, cos, sin, m, cfg.kv_heads, self._kr)
            kv4.append(g, cache, self._kr, self._v, 1)
            kv4.attention(g, cache, self._qr, self._a, 1, cfg.heads)
            self._matvec(self._a, w.o, self.x, **residual)
            if states is not None:
                self._norm(self.x, w.cross_norm, m, self._h)
                self._matvec(self._h, w.cross_q, self._q, **to_bf16)
                K.cross_attention(g, self._q, *states, self._a, m, 1, self._state_tokens, cfg.heads, cfg.kv_heads, cfg.head_dim,
                                  key_lengths=self._state_lengths, dtype="bf16", out_dtype="bf16")
                self._matvec(self._a, w.cross_o, self.x, **residual)
            self._norm(self.x, w.mlp_norm, m, self._h)
            self._matvec(self._h, w.gate, self._g, **to_bf16)
            self._matvec(self._h, w.up, self._u, aux_op="swiglu", aux=self._g, aux_dtype="bf16", **to_bf16)
            self._matvec(self._u, w.down, self.x, **residual)
        if self.caches:
            kv4.advance(g, self.caches[0])

    # ---- many tokens of one sequence ----
    def prompt(self, sequence: int, x, tokens: int) -> Buffer:
        """Fills an empty sequence's caches with `tokens` tokens x [tokens, hidden] (f32, on the device), in place: x then
        holds the last layer's output."""
        g, cfg = self.graph, self.cfg
        self._ready()
        if not 0 <= sequence < self.batch:
            raise ValueError(f"sequence must be in 0..{self.batch - 1}, got {sequence}")
        if self.lengths[sequence]:
            raise ValueError(f"sequence {sequence} has {self.lengths[sequence]} tokens already")
        if not 0 < tokens <= self.tokens:
            raise ValueError(f"a prompt has 1 to {self.tokens} tokens, got {tokens}")
        qw, kw = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        residual = {"y_dtype": "f32", "accumulate": True}
        mark = g.mark()
        try:
            cos, sin, _ = K.rope_tables(np.arange(tokens), (cfg.head_dim,), cfg.theta)
            cos, sin = g.buffer(cos), g.buffer(sin)
            bf = lambda n: g.buffer(tokens * n * 2)  # noqa: E731
            h, q, k, v, qr, kr, a = bf(cfg.hidden), bf(qw), bf(kw), bf(kw), bf(qw), bf(kw), bf(qw)
            gate, u = bf(cfg.mlp), bf(cfg.mlp)
            for i, w in enumerate(self.layers):
                cache = self._of(self.caches[i], sequence)
                self._norm(x, w.norm, tokens, h)
                self._matmul(h, w.q, q, tokens)
                self._matmul(h, w.k, k, tokens)
                self._matmul(h, w.v, v, tokens)
                self._rotate(q, w.q_norm, cos, sin, tokens, cfg.heads, qr)
                self._rotate(k, w.k_norm, cos, sin, tokens, cfg.kv_heads, kr)
                kv4.append(g, cache, kr, v, tokens)
                kv4.unpack(g, cache, k, v, tokens)  # what later tokens will see of these
                K.attention(g, qr, k, v, tokens, cfg.heads, cfg.kv_heads, cfg.head_dim, a, causal=True, dtype="bf16",
                            out_dtype="bf16")
                self._matmul(a, w.o, x, tokens, **residual)
                if w.cross_q is not None:
                    self._norm(x, w.cross_norm, tokens, h)
                    self._matmul(h, w.cross_q, q, tokens)
                    each = self._state_tokens * kw * 2
                    ck, cv = (Binding(b, sequence * each, each) for b in self._states[i])
                    K.cross_attention(g, q, ck, cv, a, 1, tokens, self._state_tokens, cfg.heads, cfg.kv_heads, cfg.head_dim,
                                      key_lengths=Binding(self._state_lengths, sequence * 4, 4), dtype="bf16", out_dtype="bf16")
                    self._matmul(a, w.cross_o, x, tokens, **residual)
                self._norm(x, w.mlp_norm, tokens, h)
                self._matmul(h, w.gate, gate, tokens)
                self._matmul(h, w.up, u, tokens, aux_op="swiglu", aux=gate, aux_dtype="bf16")
                self._matmul(u, w.down, x, tokens, **residual)
            if self.caches:
                kv4.advance(g, self._of(self.caches[0], sequence), tokens)
        finally:
            g.release(mark)
        self.lengths[sequence] = tokens
        return x

    def reset(self) -> None:
        """Empties every sequence."""
        self.lengths = [0] * self.batch
        if self.caches:
            self.graph.write(self.caches[0].lengths, np.zeros(self.batch, np.int32))

    def destroy(self) -> None:
        """Frees the recorded step (the buffers go with the graph's context)."""
        self._drop()

    # ---- parts ----
    def _ready(self) -> None:
        if self._state_lengths is None and any(w.cross_q is not None for w in self.layers):
            raise ValueError("the layers attend to states: call set_states first")

    def _drop(self) -> None:
        if self._captured is not None:
            self._captured.destroy()
            self._captured = None

    @staticmethod
    def _of(cache: kv4.Cache, sequence: int) -> kv4.Cache:
        """One sequence of a cache: the same pages, its row of the page table."""
        table = addr(cache.page_table).value + sequence * cache.max_pages * 4
        return replace(cache, page_table=table, lengths=addr(cache.lengths).value + sequence * 4, batch=1)

    def _norm(self, x, weight, rows: int, out) -> None:
        K.rmsnorm(self.graph, x, weight, rows, self.cfg.hidden, out, eps=self.cfg.eps, offset=self.cfg.norm_offset,
                  out_dtype="bf16")

    def _rotate(self, x, weight, cos, sin, tokens: int, heads: int, out) -> None:
        K.qknorm_rope(self.graph, x, weight, cos, sin, tokens, heads, self.cfg.head_dim // 2, out, self.cfg.eps,
                      self.cfg.norm_offset, self.cfg.pairing, "bf16", "bf16")

    def _matvec(self, x, w: ops.Linear, y, **kw) -> None:
        K.matvec(self.graph, x, w.buffer, y, self.batch, w.n, w.k, group_scale=w.group_scale, bias=w.bias, **kw)

    def _matmul(self, x, w: ops.Linear, y, m: int, y_dtype: str = "bf16", **kw) -> None:
        K.matmul(self.graph, x, w.buffer, y, m, w.n, w.k, w_dtype="int4", group_scale=w.group_scale, bias=w.bias, x_dtype="bf16",
                 y_dtype=y_dtype, **kw)
