"""Key counts near 2^31, where places of keys are the last that 31 bits count: the most that are taken, and more.

One key of a score far above the others' has all the weight (e^40 against 2^31 ones of e^0: the rest is below 2^-26), and it is
the last: the output is its value to that and to the output's rounding.
"""
import numpy as np
import pytest

from test_gpu_kv4 import Cache
from test_gpu_matvec import bits, values
from util import randn

pytestmark = pytest.mark.gpu

MOST = 2**31 - 1 - 2**24


@pytest.mark.parametrize("rows", [1, 3])
def test_cross_attention_of_two_billion_keys(we, graph, rows):
    """Heads of one bf16 value: k and v of all these keys are 4 GB each."""
    import torch

    tk = MOST
    dev = torch.device("cuda")
    k, v = torch.zeros(tk, dtype=torch.bfloat16, device=dev), torch.ones(tk, dtype=torch.bfloat16, device=dev)
    k[-1], v[-1] = 40.0, -3.0
    q = torch.ones(rows, dtype=torch.bfloat16, device=dev)
    out = torch.zeros(rows, dtype=torch.float32, device=dev)
    torch.cuda.synchronize()
    for hidden in (0, 1):  # all keys, then all but the last
        lengths = torch.tensor([tk - hidden], dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        we.kernels.cross_attention(graph, q, k, v, out, 1, rows, tk, 1, 1, 1, key_lengths=lengths, dtype="bf16", out_dtype="f32", scale=1.0)
        graph.sync()
        want = 1.0 if hidden else -3.0
        # weights and values are exact here, sums of 2^31 ones are within 2^-10 of their number in any order of f32 parts
        assert np.allclose(out.cpu().numpy(), want, rtol=2.0**-9, atol=0)
    assert graph.device_error() == 0
    del k, v
    torch.cuda.empty_cache()


def test_cached_attention_of_two_billion_keys(we, graph):
    """A page table whose slots share one page, but for the last."""
    page, dim = 64, 64
    slots = MOST // page
    table = np.zeros(slots, np.int32)
    table[-1] = 1
    mark = graph.mark()
    kv = we.kv4.Cache(graph.buffer(2 * page * dim // 2), graph.buffer(2 * page * dim // 2), graph.buffer(2 * page * 2), graph.buffer(2 * page * 2),
                      graph.buffer(table), graph.buffer(np.zeros(1, np.int32)), 2, slots, 1, 1, page, dim)
    small = we.kv4.Cache(kv.k, kv.v, kv.k_scale, kv.v_scale, graph.buffer(np.array([0, 1], np.int32)), kv.lengths, 2, 2, 1, 1, page, dim)
    k, v = np.zeros((2 * page, dim), np.float32), np.ones((2 * page, dim), np.float32)
    k[-1], v[-1] = 7.0, -3.5
    we.kv4.append(graph, small, graph.buffer(k), graph.buffer(v), 2 * page, dtype="f32")
    graph.write(kv.lengths, np.array([slots * page - 1], np.int32))
    q = np.full(dim, 40 / (7 * 64), np.float32)
    out = graph.buffer(dim * 4)
    for dtype in ("f32", "bf16"):
        we.kv4.attention(graph, kv, graph.buffer(bits(q, dtype)), out, 1, 1, dtype=dtype, out_dtype="f32", scale=1.0)
        assert np.allclose(graph.read(out, dim * 4, np.float32), -3.5, rtol=2.0**-9, atol=0)
    assert graph.device_error() == 0
    graph.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_length_at_the_end_of_its_type(we, graph, dtype):
    """A length of 2^31 - 1 beside a small page table: every new token sees the table's keys, the rest is recorded."""
    n, tokens, dim = 32, 5, 64
    mark = graph.mark()
    c = Cache(we, graph, 1, n, 1, dim, 16, 23)
    x = graph.buffer(np.asarray(randn(n * dim, 24), np.float32))
    we.kv4.append(graph, c.c, x, x, n, dtype="f32")
    q = graph.buffer(bits(np.tile(randn(dim, 25), (tokens, 1)), dtype))
    es = 2 if dtype == "bf16" else 4
    outs = []
    for length in (1000, 2**31 - 1):
        c.set_lengths([length])
        out = graph.buffer(tokens * dim * es)
        we.kv4.attention(graph, c.c, q, out, tokens, 1, dtype=dtype, out_dtype=dtype)
        assert graph.device_error() == 7
        outs.append(values(graph.read(out).copy(), dtype).reshape(tokens, dim))
    assert np.any(outs[0] != 0) and np.array_equal(outs[0], outs[1])
    graph.release(mark)


def test_more_keys_are_refused(we, graph):
    E, b = we._lib.WeError, graph.buffer(4096)
    with pytest.raises(E, match="tokens per sequence"):
        we.kv4.attention(graph, we.kv4.Cache(b, b, b, b, b, b, 1, MOST // 16 + 1, 1, 1, 16, 64), b, b, 1, 1)
    for kw in ({"tk": MOST + 1}, {"tk": 2**31 - 1}, {"tq": MOST + 1}):
        with pytest.raises(E, match="tokens"):
            we.kernels.cross_attention(graph, b, b, b, b, 1, kw.get("tq", 1), kw.get("tk", 1), 1, 1, 1, dtype="bf16", out_dtype="bf16")
    assert graph.device_error() == 0


def test_advance_stops_at_the_end_of_its_type(we, graph):
    """A length that would pass 31 bits stays a length: a negative one would mark the sequence idle."""
    c = Cache(we, graph, 4, 16, 1, 64, 16, 3)
    c.set_lengths([2**31 - 10, 5, -1, 2**31 - 1])
    we.kv4.advance(graph, c.c, 100)
    assert graph.read(c.lengths, 16, np.int32).tolist() == [2**31 - 1, 105, -1, 2**31 - 1]
    we.kv4.advance(graph, c.c, 2**31 - 1)
    assert graph.read(c.lengths, 16, np.int32).tolist() == [2**31 - 1, 2**31 - 1, -1, 2**31 - 1]
