"""NaN in the 4-bit cache: a group of 64 that holds one stays NaN where it is read, and nothing else does."""
import numpy as np
import pytest

from test_gpu_kv4 import Cache, quantise
from test_gpu_matvec import bits, values
from util import bf16_round, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim,kvh,tokens", [(64, 1, 1), (128, 2, 5), (256, 3, 700)])
def test_append_keeps_nan(we, graph, dim, kvh, tokens, dtype):
    mark = graph.mark()
    c = Cache(we, graph, 2, tokens + 3, kvh, dim, 16, 1)
    c.set_lengths([3, 0])
    x = {n: bf16_round(randn(2 * tokens * kvh * dim, 2 + i)).reshape(2, tokens, kvh, dim) for i, n in enumerate("kv")}
    x["k"][0, -1, 0, 5] = np.nan              # one value, a whole group, one beside an infinity, one among zeros
    x["v"][1, 0, -1, -64:] = np.nan
    x["k"][1, -1, -1, 3], x["k"][1, -1, -1, 60] = np.inf, -np.nan
    x["v"][0, 0, 0, :64] = 0
    x["v"][0, 0, 0, 63] = np.nan
    dev = [graph.buffer(bits(x[n], dtype)) for n in "kv"]
    we.kv4.append(graph, c.c, *dev, tokens, dtype=dtype)
    size = 2 * tokens * kvh * dim
    for od in ("f32", "bf16"):
        es = 4 if od == "f32" else 2
        back = [graph.buffer(size * es) for _ in "kv"]
        we.kv4.unpack(graph, c.c, *back, tokens, dtype=od)
        for n, b in zip("kv", back):
            got = values(graph.read(b, size * es).copy(), od).reshape(x[n].shape)
            bad = np.isnan(x[n]).reshape(*x[n].shape[:-1], -1, 64).any(-1)
            assert bad.sum() == 2 and np.array_equal(np.isnan(got), np.repeat(bad, 64, -1))
            clean = np.where(np.repeat(bad, 64, -1), 0, x[n])
            q, s = quantise(clean)
            want = (q * np.repeat(s.astype(np.float32), 64, -1)).astype(np.float32)
            want = want if od == "f32" else bf16_round(want.ravel()).reshape(want.shape)
            assert np.array_equal(np.where(np.isnan(got), 0, got), want)
    assert graph.device_error() == 0
    graph.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("side", ["k", "v"])
@pytest.mark.parametrize("heads,kvh,dim,tokens,n", [(2, 1, 64, 4, 40), (8, 2, 128, 4, 300), (4, 1, 256, 3, 90), (24, 2, 128, 5, 50)])
def test_attention_keeps_nan_to_the_rows_that_see_it(we, graph, heads, kvh, dim, tokens, n, side, dtype):
    """The NaN is in the second newest token of kv head 0: the two newest queries see it, of v in its group of 64 only; the
    other outputs are what they are without it, to the rounding of the other sweep that such a cache takes."""
    mark = graph.mark()
    es = 2 if dtype == "bf16" else 4
    kv = {name: bf16_round(randn(n * kvh * dim, 5 + i)).reshape(1, n, kvh, dim) for i, name in enumerate("kv")}
    q = graph.buffer(bits(randn(tokens * heads * dim, 7), dtype))
    outs = []
    for broken in (False, True):
        if broken:
            kv[side][0, n - 2, 0, dim - 10] = np.nan
        c = Cache(we, graph, 1, n, kvh, dim, 16, 1)
        we.kv4.append(graph, c.c, *(graph.buffer(np.asarray(kv[x], np.float32)) for x in "kv"), n, dtype="f32")
        c.set_lengths([n - tokens])
        out = graph.buffer(tokens * heads * dim * es)
        we.kv4.attention(graph, c.c, q, out, tokens, heads, dtype=dtype, out_dtype=dtype)
        outs.append(values(graph.read(out).copy(), dtype).reshape(tokens, heads, dim))
    clean, got = outs
    want = np.zeros(got.shape, bool)
    want[tokens - 2:, : heads // kvh, dim - 64 if side == "v" else 0:] = True
    assert np.array_equal(np.isnan(got), want)
    # both within 2^-8 of |v| <= 5 (bf16), 2^-20 (f32), as test_gpu_kv4 bounds them
    assert np.all(np.abs(np.where(want, 0, got - clean)) <= 2 * 5 * (2.0**-8 if dtype == "bf16" else 2.0**-19))
    assert graph.device_error() == 0
    graph.release(mark)
