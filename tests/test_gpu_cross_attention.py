"""GPU parity of cross attention with a plain float64 softmax: key counts other than the query count, key lengths, byte
masks, rows that see nothing, hidden NaN and infinities, strides, every type.

The bound is the cached attention's (test_gpu_kv4), with weights rounded to bf16 (2^-8) for a bf16 input's second product.
"""
import math

import numpy as np
import pytest

from test_gpu_kv4 import attend, slack
from test_gpu_matvec import bits, values
from util import bf16_round, randn

pytestmark = pytest.mark.gpu


def run(we, graph, batch, tq, tk, heads, kvh, dim, dtype, lengths=None, mask=None, out_dtype=None, seed=0, q_std=2.0, poison=False,
        k_scale=None):
    od = out_dtype or dtype
    mark = graph.mark()
    q = randn(batch * tq * heads * dim, seed, q_std).reshape(batch, tq, heads, dim)
    k, v = (randn(batch * tk * kvh * dim, seed + i).reshape(batch, tk, kvh, dim) for i in (1, 2))
    if k_scale is not None:
        k = k * k_scale[None, :, None, None].astype(np.float32)
    if dtype == "bf16":
        q, k, v = (bf16_round(a).reshape(a.shape) for a in (q, k, v))
    seen = np.ones((batch, tk), bool)
    if lengths is not None:
        seen &= np.arange(tk)[None, :] < np.asarray(lengths)[:, None]
    if mask is not None:
        seen &= mask != 0
    if poison:
        k[~seen], v[~seen] = np.nan, np.inf
    size = q.size * (2 if od == "bf16" else 4)
    out = graph.buffer(np.full(max(4, size), 0xFF, np.uint8))
    we.kernels.cross_attention(graph, graph.buffer(bits(q, dtype)), graph.buffer(bits(k, dtype)) if tk else None,
                               graph.buffer(bits(v, dtype)) if tk else None, out, batch, tq, tk, heads, kvh, dim,
                               key_lengths=None if lengths is None else graph.buffer(np.asarray(lengths, np.int32)),
                               key_mask=None if mask is None else graph.buffer(np.asarray(mask, np.uint8)),
                               dtype=dtype, out_dtype=od)
    got = values(graph.read(out, size).copy(), od).reshape(q.shape)
    assert graph.device_error() == 0
    graph.release(mark)
    k, v = np.where(seen[..., None, None], k, 0), np.where(seen[..., None, None], v, 0)
    for b in range(batch):
        for h in range(heads):
            j = h // (heads // kvh)
            qh, kh, vh = (a.astype(np.float64) for a in (q[b, :, h], k[b, :, j], v[b, :, j]))
            want = attend(qh, kh, vh, np.broadcast_to(seen[b], (tq, tk)), 1 / math.sqrt(dim))
            tol = slack(qh, kh, vh, want, 1 / math.sqrt(dim), od, 2.0**-8)
            if dtype == "bf16" and od == "f32" and vh.size:
                tol = tol + 2 * 2.0**-8 * np.abs(vh).max()
            err = np.abs(got[b, :, h] - want)
            assert np.all(err <= tol), (b, h, float(np.nanmax(err)), float(np.min(tol)))
    return got


SHAPES = [(1, 1, 1, 1, 1, 64), (1, 1, 77, 4, 2, 128), (2, 300, 203, 4, 2, 64), (1, 129, 128, 2, 2, 128), (3, 5, 700, 6, 2, 128),
          (2, 257, 64, 2, 1, 128), (1, 1, 5000, 8, 1, 64), (2, 2, 1031, 16, 4, 128), (1, 700, 1, 2, 2, 128), (1, 64, 513, 3, 3, 128),
          (2, 16, 100, 20, 2, 64), (1, 1000, 333, 1, 1, 64)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=["x".join(map(str, s)) for s in SHAPES])
def test_cross_attention_matches_float64(we, graph, shape, dtype):
    run(we, graph, *shape, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tq", [1, 3, 150, 260])
def test_lengths_masks_and_hidden_values(we, graph, tq, dtype):
    """Ragged lengths (0 and beyond tk included), a mask with a hidden entry and hidden first tiles; K is NaN and V
    infinite where nothing may be seen."""
    tk = 400
    lengths = [400, 0, 129, 1000, 5, 400]
    mask = (np.random.default_rng(3).random((6, tk)) < 0.7).astype(np.uint8) * 255
    mask[3] = 0
    mask[5, :300] = 0
    run(we, graph, 6, tq, tk, 4, 2, 64 if tq == 3 else 128, dtype, lengths, mask, seed=5, poison=True)
    run(we, graph, 6, tq, tk, 2, 2, 128, dtype, lengths, None, seed=6, poison=True)
    run(we, graph, 6, tq, tk, 2, 1, 128, dtype, None, mask, seed=7, poison=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [1, 16, 40, 72, 80, 96, 160, 200, 256])
def test_other_head_sizes(we, graph, dim, dtype):
    run(we, graph, 2, 37, 91, 4, 2, dim, dtype, lengths=[91, 40], seed=8)


@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("tq", [1, 200])
def test_mixed_types(we, graph, tq, dtype, out_dtype):
    run(we, graph, 2, tq, 300, 4, 2, 128, dtype, out_dtype=out_dtype, seed=9)


@pytest.mark.parametrize("tq", [2, 140])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores_that_grow_along_the_keys(we, graph, tq, dtype):
    run(we, graph, 1, tq, 900, 2, 1, 128, dtype, seed=10, q_std=4.0, k_scale=np.linspace(0.1, 3, 900))


def test_no_keys_and_no_queries(we, graph):
    got = run(we, graph, 2, 3, 0, 2, 1, 128, "bf16")
    assert np.all(got == 0)
    b = graph.buffer(4)
    we.kernels.cross_attention(graph, b, b, b, b, 1, 0, 5, 2, 1, 128, dtype="bf16", out_dtype="bf16")
    we.kernels.cross_attention(graph, b, b, b, b, 0, 5, 5, 2, 1, 128, dtype="bf16", out_dtype="bf16")
    assert graph.device_error() == 0


@pytest.mark.parametrize("dtype,shift", [("bf16", 0), ("bf16", 1), ("f32", 0), ("f32", 1)])
@pytest.mark.parametrize("tq", [1, 150])
def test_strides_of_a_fused_projection(we, graph, tq, dtype, shift):
    """k and v interleaved in one projection's rows, q and out inside wider rows; shift 1: addresses and strides that
    are aligned to the element only."""
    batch, tk, heads, kvh, dim = 2, 133, 4, 2, 64
    es = 2 if dtype == "bf16" else 4
    rs, qs, os_ = 2 * kvh * dim + 8 + shift, heads * dim + 8 + shift, heads * dim + 16 + shift
    kv, q = randn(batch * tk * rs + shift, 11), randn(batch * tq * qs + shift, 12, 2.0)
    if dtype == "bf16":
        kv, q = bf16_round(kv), bf16_round(q)
    kvb, qb = graph.buffer(bits(kv, dtype)), graph.buffer(bits(q, dtype))
    out = graph.buffer(bits(np.full(batch * tq * os_, 3.0, np.float32), dtype))
    we.kernels.cross_attention(graph, qb.ptr + es * shift, kvb.ptr + es * shift, kvb.ptr + es * (shift + kvh * dim), out, batch, tq, tk,
                               heads, kvh, dim, q_stride=qs, k_stride=rs, v_stride=rs, out_stride=os_, dtype=dtype, out_dtype=dtype,
                               scale=0.2)
    got = values(graph.read(out, batch * tq * os_ * es).copy(), dtype).reshape(batch * tq, os_)
    assert np.all(got[:, heads * dim:] == 3.0)
    rows, qr = kv[shift:].reshape(batch, tk, rs).astype(np.float64), q[shift:].reshape(batch, tq, qs).astype(np.float64)
    for b in range(batch):
        for h in range(heads):
            j = h // 2
            kh, vh = rows[b, :, j * dim:(j + 1) * dim], rows[b, :, (kvh + j) * dim:(kvh + j + 1) * dim]
            qh = qr[b, :, h * dim:(h + 1) * dim]
            want = attend(qh, kh, vh, np.ones((tq, tk), bool), 0.2)
            tol = slack(qh, kh, vh, want, 0.2, dtype, 2.0**-8)
            assert np.all(np.abs(got[b * tq:(b + 1) * tq, h * dim:(h + 1) * dim] - want) <= tol)


def test_deterministic_and_replays_from_a_graph(we, graph):
    for tq in (1, 300):
        b, tk, heads, kvh, dim = 2, 3000, 4, 2, 128
        q, k, v = (graph.buffer(bits(randn(n, 13 + i), "bf16")) for i, n in
                   enumerate((b * tq * heads * dim, b * tk * kvh * dim, b * tk * kvh * dim)))
        out, lens = graph.buffer(b * tq * heads * dim * 2), graph.buffer(np.array([3000, 1500], np.int32))
        call = we.kernels.cross_attention_call(graph, q, k, v, out, b, tq, tk, heads, kvh, dim, key_lengths=lens, dtype="bf16",
                                               out_dtype="bf16")
        call()
        first = graph.read(out).copy()
        with graph.capture() as cap:
            call()
        for _ in range(2):
            graph.write(out, np.zeros(first.size, np.uint8))
            cap.launch()
            assert np.array_equal(graph.read(out), first)
        cap.destroy()


def test_op_form_and_self_attention_agree(we, graph):
    """With tk = tq and no mask it is we_attention's formula: the op form against ops.attention in f32."""
    t, heads, kvh, dim = 70, 4, 2, 64
    q, k, v = (graph.buffer(randn(t * h * dim, 20 + i)) for i, h in enumerate((heads, kvh, kvh)))
    a = graph.read(we.cross_attention(graph, q, k, v, 1, t, t, heads, kvh, dim), None, np.float32)
    b = graph.read(we.attention(graph, q, k, v, t, heads, kvh, dim), None, np.float32)
    assert np.max(np.abs(a - b)) < 1e-5


def test_refusals(we, graph):
    E, b = we._lib.WeError, graph.buffer(4096)

    def refused(words, batch=1, tq=1, tk=1, heads=2, kvh=1, dim=64, q=b, k=b, **kw):
        with pytest.raises(E, match=words):
            we.kernels.cross_attention(graph, q, k, b, b, batch, tq, tk, heads, kvh, dim, **kw)

    refused("multiple of kvHeads", heads=3, kvh=2)
    refused("1..256", dim=0)
    refused("1..256", dim=257)
    refused("negative", tq=-1)
    refused("missing", k=None)
    refused("aligned", q=b.ptr + 1)
    refused("shorter", q_stride=64)
    refused("shorter", k_stride=32)
    refused("f32 or bf16", dtype="fp8")
    refused("65535", batch=70000)


@pytest.mark.parametrize("dim,out_dtype", [(64, "bf16"), (128, "bf16"), (128, "f32"), (64, "f32")])
@pytest.mark.parametrize("tk", [100, 300, 1111])
def test_more_query_tiles_than_resident_blocks(we, graph, dim, out_dtype, tk):
    """Blocks that take several query tiles each: entries without keys, with hidden tiles and with whole ones in turn,
    and rows that end inside a tile."""
    lengths = [tk, 0, tk // 2, tk - 1, 1]
    mask = (np.random.default_rng(21).random((5, tk)) < 0.9).astype(np.uint8)
    mask[3] = 1
    run(we, graph, 5, 300, tk, 24, 8, dim, "bf16", lengths, mask, out_dtype=out_dtype, seed=22, poison=True)
    run(we, graph, 5, 300, tk, 24, 24, dim, "bf16", lengths, None, out_dtype=out_dtype, seed=23, poison=True)


@pytest.mark.parametrize("tq", [1, 3, 44, 131])
@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (12, 2), (40, 1), (128, 1), (260, 2)])
def test_groups_of_heads_that_share_keys(we, graph, heads, kv_heads, tq):
    """Groups that do not divide a tile of rows, that fill it, and one larger than it."""
    run(we, graph, 2, tq, 333, heads, kv_heads, 64, "bf16", lengths=[333, 130], seed=31, poison=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,tq,tk,heads,kv_heads,dim", [(2, 1, 20000, 6, 2, 64), (1, 4, 12001, 4, 2, 128), (2, 2, 5003, 4, 1, 256),
                                                            (1, 11, 9000, 2, 2, 64)])
def test_keys_shared_by_several_clusters(we, graph, batch, tq, tk, heads, kv_heads, dim, dtype):
    lengths = [tk, tk // 3][:batch]
    for seed in (41, 42):
        run(we, graph, batch, tq, tk, heads, kv_heads, dim, dtype, lengths=lengths, seed=seed)
