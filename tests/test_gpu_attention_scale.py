"""The scale of the cached and of the cross attention: either sign, with hidden keys of every kind, and what is refused.

Bounds as in test_gpu_kv4 and test_gpu_cross_attention, with |scale|.
"""
import math

import numpy as np
import pytest

from test_gpu_kv4 import Cache, attend, slack
from test_gpu_matvec import bits, values
from util import bf16_round, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [-0.125, -0.6])
@pytest.mark.parametrize("tokens,length,heads,kvh,dim", [(1, 20, 4, 2, 64), (3, 33, 6, 2, 128), (20, 100, 4, 2, 64), (1, 9000, 8, 1, 64)])
def test_cached_attention_of_a_negative_scale(we, graph, tokens, length, heads, kvh, dim, scale, dtype):
    """Last tiles that are not full and the new tokens' causal limit."""
    mark = graph.mark()
    n = length + tokens
    c = Cache(we, graph, 1, n, kvh, dim, 16, 1)
    kv = [bf16_round(randn(n * kvh * dim, 2 + i)).reshape(1, n, kvh, dim) for i in range(2)]
    we.kv4.append(graph, c.c, *(graph.buffer(np.asarray(x, np.float32)) for x in kv), n, dtype="f32")
    c.set_lengths([length])
    q = bf16_round(randn(tokens * heads * dim, 4, 2.0)).reshape(tokens, heads, dim)
    es = 2 if dtype == "bf16" else 4
    out = graph.buffer(np.full(q.size * es, 0xFF, np.uint8))
    we.kv4.attention(graph, c.c, graph.buffer(bits(q, dtype)), out, tokens, heads, dtype=dtype, out_dtype=dtype, scale=scale)
    got = values(graph.read(out, q.size * es).copy(), dtype).reshape(q.shape)
    kk, vv = c.sequence("k", 0, n), c.sequence("v", 0, n)
    seen = np.arange(n)[None, :] <= length + np.arange(tokens)[:, None]
    for h in range(heads):
        j = h // (heads // kvh)
        qh = q[:, h].astype(np.float64)
        want = attend(qh, kk[:, j], vv[:, j], seen, scale)
        assert np.all(np.abs(got[:, h] - want) <= slack(qh, kk[:, j], vv[:, j], want, -scale, dtype, 2.0**-11))
    assert graph.device_error() == 0
    graph.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tq,tk,dim", [(1, 77, 64), (2, 300, 128), (150, 203, 128), (33, 400, 64), (40, 91, 72), (3, 6000, 64)])
def test_cross_attention_of_a_negative_scale(we, graph, tq, tk, dim, dtype):
    """Lengths, a mask with an entry that hides everything, and K of NaN and V of infinities where nothing is seen."""
    mark = graph.mark()
    batch, heads, kvh, scale = 4, 4, 2, -0.2
    q = randn(batch * tq * heads * dim, 5, 2.0).reshape(batch, tq, heads, dim)
    k, v = (randn(batch * tk * kvh * dim, 6 + i).reshape(batch, tk, kvh, dim) for i in range(2))
    if dtype == "bf16":
        q, k, v = (bf16_round(a).reshape(a.shape) for a in (q, k, v))
    lengths = np.array([tk, tk // 2, tk, 5], np.int32)
    mask = (np.random.default_rng(8).random((batch, tk)) < 0.7).astype(np.uint8)
    mask[0], mask[2] = 1, 0
    seen = (mask != 0) & (np.arange(tk)[None, :] < lengths[:, None])
    k[~seen], v[~seen] = np.nan, np.inf
    es = 2 if dtype == "bf16" else 4
    out = graph.buffer(np.full(q.size * es, 0xFF, np.uint8))
    we.kernels.cross_attention(graph, *(graph.buffer(bits(a, dtype)) for a in (q, k, v)), out, batch, tq, tk, heads, kvh, dim,
                               key_lengths=graph.buffer(lengths), key_mask=graph.buffer(mask), dtype=dtype, out_dtype=dtype, scale=scale)
    got = values(graph.read(out, q.size * es).copy(), dtype).reshape(q.shape)
    k, v = np.where(seen[..., None, None], k, 0), np.where(seen[..., None, None], v, 0)
    for b in range(batch):
        for h in range(heads):
            qh, kh, vh = (a.astype(np.float64) for a in (q[b, :, h], k[b, :, h // 2], v[b, :, h // 2]))
            want = attend(qh, kh, vh, np.broadcast_to(seen[b], (tq, tk)), scale)
            assert np.all(np.abs(got[b, :, h] - want) <= slack(qh, kh, vh, want, -scale, dtype, 2.0**-8))
    assert graph.device_error() == 0
    graph.release(mark)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_a_scale_that_is_not_finite_is_refused(we, graph, scale):
    b = graph.buffer(4096)
    cache = we.kv4.Cache(b, b, b, b, b, b, pages=1, max_pages=1, batch=1, kv_heads=1, page=16, dim=64)
    with pytest.raises(we._lib.WeError, match="finite"):
        we.kv4.attention(graph, cache, b, b, 1, 1, scale=scale)
    for tq in (1, 200):
        with pytest.raises(we._lib.WeError, match="finite"):
            we.kernels.cross_attention(graph, b, b, b, b, 1, tq, 1, 1, 1, 64, dtype="bf16", out_dtype="bf16", scale=scale)
