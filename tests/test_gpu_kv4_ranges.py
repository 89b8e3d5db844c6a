"""Cached attention over values of very different magnitudes: what a row gives no weight takes no accuracy from it.

Bound of one output value, from what the row itself sees: with p the weights and s the scales of v, the weights' errors as in
test_gpu_kv4 (2 E + 2^-20, and for a bf16 output two roundings of 2^-11 more) times sum p |v|; products of weights and scales are
held to an absolute 2^-17 (bf16 output) or 2^-23 (f32) of the row's largest one, times codes of at most 8, for every key that is
seen; and the rounding of a bf16 output.
"""
import numpy as np
import pytest

from test_gpu_kv4 import Cache
from test_gpu_matvec import bits, values
from util import bf16_round, randn

pytestmark = pytest.mark.gpu


def check(we, graph, k, v, q, length, dtype, page=16, scale=0.125):
    """k, v [n, kvh, dim] into a cache of one sequence of `length` tokens and the rest new ones, whose queries are q."""
    mark = graph.mark()
    n, kvh, dim = k.shape
    tokens, heads, _ = q.shape
    c = Cache(we, graph, 1, n, kvh, dim, page, 1)
    we.kv4.append(graph, c.c, graph.buffer(np.asarray(k[None], np.float32)), graph.buffer(np.asarray(v[None], np.float32)), n, dtype="f32")
    c.set_lengths([length])
    es = 2 if dtype == "bf16" else 4
    q = bf16_round(q).reshape(q.shape)
    out = graph.buffer(np.full(q.size * es, 0xFF, np.uint8))
    we.kv4.attention(graph, c.c, graph.buffer(bits(q, dtype)), out, tokens, heads, dtype=dtype, out_dtype=dtype, scale=scale)
    got = values(graph.read(out, q.size * es).copy(), dtype).reshape(q.shape)
    assert graph.device_error() == 0
    kk, vv = c.sequence("k", 0, n), c.sequence("v", 0, n)
    s = c.rows("v")[1][c.table[0]].astype(np.float64).transpose(0, 2, 1, 3).reshape(-1, kvh, dim // 64)[:n]
    for i in range(tokens):
        seen = length + i + 1
        for h in range(heads):
            j = h // (heads // kvh)
            qh, kh, vh, sh = q[i, h].astype(np.float64), kk[:seen, j], vv[:seen, j], np.repeat(s[:seen, j], 64, -1)
            x = kh @ qh * scale
            p = np.exp(x - x.max())
            p /= p.sum()
            e = 2.0**-20 * scale * np.linalg.norm(qh) * np.linalg.norm(kh, axis=-1)
            want = p @ vh
            low = dtype == "bf16"
            tol = (p * (2 * e.max() + 2.0**-20 + (2.0**-10 if low else 0))) @ np.abs(vh)
            tol = tol + 8 * seen * 2.0 ** (-17 if low else -23) * (p[:, None] * sh).max(0)
            tol = tol + (2.0**-8 * np.abs(want) if low else 0)
            assert np.all(np.abs(got[i, h] - want) <= tol), (i, h, float(np.max(np.abs(got[i, h] - want) / tol)))
    graph.release(mark)


def inputs(n, kvh, dim, heads, tokens, seed):
    k, v = (randn(n * kvh * dim, seed + i).reshape(n, kvh, dim) for i in range(2))
    return k, v, randn(tokens * heads * dim, seed + 2, 1.0).reshape(tokens, heads, dim)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kvh,dim,tokens", [(1, 1, 64, 1), (8, 2, 128, 1), (4, 1, 128, 3), (6, 2, 64, 2), (2, 1, 256, 1), (12, 1, 256, 1)])
@pytest.mark.parametrize("where", [0, 5, 150, 297])
def test_a_large_value_without_weight(we, graph, where, heads, kvh, dim, tokens, dtype):
    """One key's values are 10^7 and more above the others', and its score is so low that it does not count."""
    k, v, q = inputs(300, kvh, dim, heads, tokens, 10)
    v *= np.float32(3e-4)
    v[where] *= np.float32(1e8)
    direction = np.ones(dim, np.float32)
    q += 0.5 * direction
    k[where] = -30 * direction
    check(we, graph, k, v, q, 300 - tokens, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("first", [True, False])
def test_a_large_value_that_one_row_attends_to(we, graph, first, dtype):
    """Two heads of a group: the key of large values is all that one sees, and nothing to the other."""
    k, v, q = inputs(300, 1, 128, 4, 1, 20)
    v *= np.float32(1e-3)
    at = 3 if first else 250
    v[at] *= np.float32(1e7)
    direction = np.ones(128, np.float32)
    k[at] = 4 * direction
    q[0, 0], q[0, 1] = direction, -direction
    check(we, graph, k, v, q, 299, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_groups_of_a_row_with_scales_of_their_own(we, graph, dtype):
    """Every row's first 64 values are 10^7 times its others."""
    for dim in (128, 256):
        k, v, q = inputs(200, 2, dim, 4, 2, 30)
        v[..., :64] *= 1e4
        v[..., 64:] *= 1e-3
        check(we, graph, k, v, q, 198, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_large_value_that_loses_its_weight_to_later_keys(we, graph, dtype):
    """The key of large values comes first with all the weight so far; keys with scores far above follow."""
    k, v, q = inputs(400, 1, 64, 1, 1, 40)
    v *= np.float32(1e-3)
    v[0] *= np.float32(1e7)
    q[:] = 1
    k[0], k[200:] = 0, k[200:] + 8
    check(we, graph, k, v, q, 399, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_large_value_of_little_weight_that_counts(we, graph, dtype):
    """Weights of 2^-17 to 2^-27 times values of 2^24: a product as large as the others'."""
    for score in (-12.0, -15.0, -19.0):
        k, v, q = inputs(300, 1, 64, 2, 1, 50)
        v *= np.float32(1e-3)
        v[100] *= np.float32(2.0**24)
        q[:] = 1
        k -= k.mean(-1, keepdims=True)
        k[100] = score / 8
        check(we, graph, k, v, q, 299, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rising", [True, False])
def test_values_over_nine_decades(we, graph, rising, dtype):
    k, v, q = inputs(600, 2, 128, 8, 4, 60)
    f = np.logspace(-4, 5, 600) if rising else np.logspace(5, -4, 600)
    check(we, graph, k, v * f[:, None, None].astype(np.float32), q, 596, dtype)
