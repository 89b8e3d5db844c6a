"""Attention whose keys are shared by several clusters, which merge through memory: the same bits call after call, with
other work of the same counters and scratch in between."""
import numpy as np
import pytest

from test_gpu_kv4 import Cache
from test_gpu_matvec import bits
from util import randn

pytestmark = pytest.mark.gpu


def test_cached_attention_merges_the_same_bits_every_time(we, graph):
    mark = graph.mark()
    heads, kvh, dim, n = 4, 2, 64, 40000
    c = Cache(we, graph, 2, n, kvh, dim, 64, 1)
    x = graph.buffer(bits(randn(2 * n * kvh * dim, 2), "bf16"))
    we.kv4.append(graph, c.c, x, x, n)
    q, out = graph.buffer(bits(randn(2 * heads * dim, 3), "bf16")), graph.buffer(2 * heads * dim * 2)
    want = {}
    for i in range(200):
        lengths = [(n - 1, 12345), (30000, n - 1)][i % 2]
        c.set_lengths(lengths)
        we.kv4.attention(graph, c.c, q, out, 1, heads)
        got = graph.read(out).copy()
        assert np.array_equal(want.setdefault(lengths, got), got)
    assert graph.device_error() == 0
    graph.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cross_attention_merges_the_same_bits_every_time(we, graph, dtype):
    mark = graph.mark()
    heads, kvh, dim, tk = 4, 2, 64, 20000
    es = 2 if dtype == "bf16" else 4
    q, k, v = (graph.buffer(bits(randn(n, 4 + i), dtype)) for i, n in enumerate((2 * heads * dim, 2 * tk * kvh * dim, 2 * tk * kvh * dim)))
    out, lengths = graph.buffer(2 * heads * dim * es), graph.buffer(np.array([tk, tk // 2], np.int32))
    call = we.kernels.cross_attention_call(graph, q, k, v, out, 2, 1, tk, heads, kvh, dim, key_lengths=lengths, dtype=dtype, out_dtype=dtype)
    call()
    want = graph.read(out).copy()
    for _ in range(100):
        call()
        assert np.array_equal(graph.read(out), want)
    assert graph.device_error() == 0
    graph.release(mark)
