"""A decoder's steps and prompts (decoder.Decoder) against float64 on the same int4 weights.

The oracle attends to the rows that the caches hold (their codes are checked bit for bit elsewhere; here each is within
two steps of the oracle's own k and v), and rounds nothing. What is left are the path's bf16 roundings, 2^-9 of a value
each at most: up to 8 in series in a branch, in 2 layers of 3 branches, about sqrt(48) 2^-9 = 1.4% of what the layers add
to x if they are independent. The bound is twice that, 3% (root mean square).
"""
import numpy as np
import pytest

from oracle import oracle as O
from util import bf16, bf16_round, randn

pytestmark = pytest.mark.gpu

BOUND = 0.03


def make(we, graph, n, k, seed):
    packed, s = O.quant_int4_g64(randn(n * k, seed, k ** -0.5), n, k)
    b = np.asarray(packed, np.uint8).reshape(n, k // 2)
    q = np.empty((n, k), np.int64)
    q[:, 0::2], q[:, 1::2] = b & 15, b >> 4
    scales = np.asarray(s).view(np.float16).reshape(n, k // 64).astype(np.float64)
    w = ((q + 8) % 16 - 8) * np.repeat(scales, 64, 1)
    return w, we.Linear(graph.buffer(packed), "int4", 1.0, n, k, group_scale=graph.buffer(s))


class Model:
    def __init__(self, we, graph, cfg, layers, cross, width=128):
        self.cfg, self.host, self.dev = cfg, [], []
        qw, kw = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
        shapes = {"q": (qw, cfg.hidden), "k": (kw, cfg.hidden), "v": (kw, cfg.hidden), "o": (cfg.hidden, qw),
                  "gate": (cfg.mlp, cfg.hidden), "up": (cfg.mlp, cfg.hidden), "down": (cfg.hidden, cfg.mlp)}
        if cross:
            shapes |= {"cross_q": (qw, cfg.hidden), "cross_k": (kw, width), "cross_v": (kw, width), "cross_o": (cfg.hidden, qw)}
        norms = {"norm": cfg.hidden, "q_norm": cfg.head_dim, "k_norm": cfg.head_dim, "mlp_norm": cfg.hidden}
        if cross:
            norms["cross_norm"] = cfg.hidden
        for i in range(layers):
            h, d = {}, {}
            for j, (name, (n, k)) in enumerate(shapes.items()):
                h[name], d[name] = make(we, graph, n, k, 100 * i + j)
            for j, (name, n) in enumerate(norms.items()):
                w = 1 + randn(n, 100 * i + 50 + j, 0.1)
                h[name], d[name] = w.astype(np.float64), graph.buffer(w)
            self.host.append(h)
            self.dev.append(we.decoder.DecoderLayer(**d))


def norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def rotate(x, pos, theta):
    d = x.shape[-1]
    a = np.asarray(pos, np.float64)[:, None, None] * theta ** (-np.arange(0, d, 2) / d)
    lo, hi = x[..., : d // 2], x[..., d // 2:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)


def softmax(s):
    e = np.exp(s - s.max(-1, keepdims=True))
    return e / e.sum(-1, keepdims=True)


def attend(q, k, v, seen):
    """q [t, heads, d], k, v [n, kv_heads, d]; query i sees keys 0 .. seen[i] - 1."""
    t, heads, d = q.shape
    group = heads // k.shape[1]
    out = np.zeros((t, heads, d))
    for i in range(t):
        for h in range(heads):
            if seen[i]:
                kk, vv = k[: seen[i], h // group], v[: seen[i], h // group]
                out[i, h] = softmax(kk @ q[i, h] / d ** 0.5) @ vv
    return out.reshape(t, heads * d)


def rows(graph, cache, name, b, n):
    """The first n rows of a sequence as the cache holds them (its pages are b * max_pages and on): values and steps."""
    per = cache.page * cache.kv_heads * cache.dim
    pages = -(-n // cache.page)
    raw = graph.read(getattr(cache, name), cache.pages * per // 2).reshape(cache.pages, -1)[b * cache.max_pages:][:pages]
    raw = raw.reshape(pages, cache.kv_heads, cache.page, cache.dim // 2)
    q = np.empty((*raw.shape[:3], cache.dim), np.int64)
    q[..., 0::2], q[..., 1::2] = raw & 15, raw >> 4
    s = graph.read(getattr(cache, name + "_scale"), cache.pages * per // 64 * 2, np.float16).reshape(cache.pages, -1)
    s = s[b * cache.max_pages:][:pages].reshape(pages, cache.kv_heads, cache.page, cache.dim // 64).astype(np.float64)
    step = np.repeat(s, 64, -1)
    put = lambda a: a.transpose(0, 2, 1, 3).reshape(-1, cache.kv_heads, cache.dim)[:n]  # noqa: E731
    return put(((q + 8) % 16 - 8) * step), put(step)


def oracle(graph, model, dec, b, x, start, states, n_states):
    """The layers over tokens x [t, hidden] of sequence b from position `start`, attending to the caches' own rows."""
    cfg = model.cfg
    x = np.asarray(x, np.float64)
    t = len(x)
    pos = np.arange(start, start + t)
    for w, cache in zip(model.host, dec.caches):
        h = norm(x, w["norm"], cfg.eps)
        q = rotate(norm((h @ w["q"].T).reshape(t, cfg.heads, -1), w["q_norm"], cfg.eps), pos, cfg.theta)
        k = rotate(norm((h @ w["k"].T).reshape(t, cfg.kv_heads, -1), w["k_norm"], cfg.eps), pos, cfg.theta)
        v = (h @ w["v"].T).reshape(t, cfg.kv_heads, -1)
        ck, sk = rows(graph, cache, "k", b, start + t)
        cv, sv = rows(graph, cache, "v", b, start + t)
        for own, held, step in ((k, ck, sk), (v, cv, sv)):
            assert np.all(np.abs(own - held[start:]) <= 2 * step[start:] + 1e-6)
        x = x + attend(q, ck, cv, pos + 1) @ w["o"].T
        if "cross_q" in w:
            h = norm(x, w["cross_norm"], cfg.eps)
            q = (h @ w["cross_q"].T).reshape(t, cfg.heads, -1)
            k, v = ((states[b] @ w[n].T).reshape(states.shape[1], cfg.kv_heads, -1) for n in ("cross_k", "cross_v"))
            x = x + attend(q, k, v, [n_states[b]] * t) @ w["cross_o"].T
        h = norm(x, w["mlp_norm"], cfg.eps)
        g, u = h @ w["gate"].T, h @ w["up"].T
        x = x + (g / (1 + np.exp(-g)) * u) @ w["down"].T
    return x


def close(got, want, start):
    err = np.sqrt(((got - want) ** 2).mean()) / np.sqrt(((want - start) ** 2).mean())
    assert err <= BOUND, err


@pytest.mark.parametrize("heads,kv_heads,dim,cross,own_stream", [(4, 2, 64, True, False), (2, 2, 128, True, True),
                                                                (6, 1, 64, False, False)])
def test_steps_and_prompts(we, graph, heads, kv_heads, dim, cross, own_stream):
    """Three sequences, two with prompts of other lengths (one ends inside a page) and one from nothing, then steps."""
    import torch

    cfg = we.decoder.DecoderConfig(192, 320, heads, kv_heads, dim, page=16)
    stream = torch.cuda.Stream() if own_stream else None
    if stream:
        graph.set_stream(stream.cuda_stream)
    try:
        model = Model(we, graph, cfg, 2, cross)
        dec = we.decoder.Decoder(graph, cfg, model.dev, 3, 60)
        states, n_states = bf16_round(randn(3 * 21 * 128, 7)).reshape(3, 21, 128).astype(np.float64), [21, 0, 9]
        if cross:
            dec.set_states(graph.buffer(bf16(states)), 21, n_states)
        checks = []
        for b, n in ((0, 37), (1, 5)):
            x = randn(n * cfg.hidden, 20 + b).reshape(n, cfg.hidden)
            xb = graph.buffer(x)
            got = graph.read(dec.prompt(b, xb, n), x.nbytes, np.float32).reshape(x.shape)
            checks.append((b, x, 0, got.copy()))
        for s in range(4):
            x = randn(3 * cfg.hidden, 40 + s).reshape(3, cfg.hidden)
            before = list(dec.lengths)
            got = graph.read(dec.step(x), x.nbytes, np.float32).reshape(x.shape)
            checks += [(b, x[b:b + 1], before[b], got[b:b + 1].copy()) for b in range(3)]
        assert dec.lengths == [41, 9, 4]
        assert list(graph.read(dec.caches[0].lengths, 12, np.int32)) == dec.lengths
        for b, x, start, got in checks:
            close(got, oracle(graph, model, dec, b, x, start, states, n_states), x)
        assert graph.device_error() == 0
        # again from nothing, with other states: the recorded step follows
        dec.reset()
        if cross:
            states = bf16_round(randn(3 * 8 * 128, 8)).reshape(3, 8, 128).astype(np.float64)
            dec.set_states(graph.buffer(bf16(states)), 8)
        x = randn(3 * cfg.hidden, 60).reshape(3, cfg.hidden)
        got = graph.read(dec.step(x), x.nbytes, np.float32).reshape(x.shape)
        for b in range(3):
            close(got[b:b + 1], oracle(graph, model, dec, b, x[b:b + 1], 0, states, [8] * 3), x[b:b + 1])
        dec.destroy()
    finally:
        if stream:
            graph.sync()
            graph.set_stream(None)


def test_refusals(we, graph):
    cfg = we.decoder.DecoderConfig(64, 128, 2, 1, 64, page=16)
    model = Model(we, graph, cfg, 1, True, 64)
    for batch in (0, 17):
        with pytest.raises(ValueError, match="1 to 16 sequences"):
            we.decoder.Decoder(graph, cfg, model.dev, batch, 16)
    dec = we.decoder.Decoder(graph, cfg, model.dev, 1, 2)
    x = randn(64, 1).reshape(1, 64)
    with pytest.raises(ValueError, match="set_states"):
        dec.step(x)
    with pytest.raises(ValueError, match="at least one"):
        dec.set_states(graph.buffer(4), 0)
    dec.set_states(graph.buffer(bf16(randn(3 * 64, 2))), 3)
    with pytest.raises(ValueError, match="1 to 2 tokens"):
        dec.prompt(0, graph.buffer(3 * 64 * 4), 3)
    dec.step(x)
    with pytest.raises(ValueError, match="has 1 tokens"):
        dec.prompt(0, graph.buffer(64 * 4), 1)
    dec.step(x)
    with pytest.raises(ValueError, match="full"):
        dec.step(x)
    from dataclasses import replace

    with pytest.raises(ValueError, match="int4 linear"):
        we.decoder.Decoder(graph, cfg, [replace(model.dev[0], up=model.dev[0].down)], 1, 2)
    with pytest.raises(ValueError, match="all of the cross"):
        we.decoder.Decoder(graph, cfg, [replace(model.dev[0], cross_q=None)], 1, 2)
