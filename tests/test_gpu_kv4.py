"""GPU parity of the paged 4-bit K/V cache: append and unpack bit for bit against numpy, attention against float64 over
the cache's own values.

Attention's bound, with |v| <= V over a row's keys: a score is a sum of products exact to 2^-22, so its error is at most
E = 2^-20 scale |q| |k|; a weight's relative error is at most 2 E + 2^-20, and 2^-11 more where the weight is rounded to
f16 for a bf16 output; the output, an average of v by those weights, is off by at most twice that times V, and a bf16
output by 2^-8 of itself (8 significant bits, to nearest).
"""
import math

import numpy as np
import pytest

from oracle import oracle as O
from test_gpu_matvec import bits, values
from util import bf16_round, randn

pytestmark = pytest.mark.gpu


def quantise(x):
    """int4 group-64 rows as the header defines them: codes and f16 scales, in the arithmetic of f32."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 64)
    with np.errstate(all="ignore"):
        s = np.minimum(np.abs(g).max(-1) / np.float32(7), np.float32(65504)).astype(np.float16)
        q = np.clip(np.rint(g / s.astype(np.float32)[..., None]), -8, 7)
    q = np.where(s[..., None] == 0, 0, q)
    return q.reshape(x.shape), s


class Cache:
    """A cache filled with garbage (NaN scales included) under random pages, and what its rows should hold."""

    def __init__(self, we, graph, batch, tokens, kvh, dim, page, seed=0):
        r = np.random.default_rng(seed)
        per = max(1, -(-tokens // page))
        pages = batch * per + 3
        self.table = r.permutation(pages)[: batch * per].astype(np.int32).reshape(batch, per)
        self.shape, self.per, self.page, self.graph = (pages, kvh, page, dim), per, page, graph
        raw = {n: r.integers(0, 256, pages * kvh * page * dim // 2, dtype=np.uint8) for n in "kv"}
        junk = np.full(pages * kvh * page * (dim // 64), 0x7E00, np.uint16)
        self.lengths = graph.buffer(np.zeros(batch, np.int32))
        self.c = we.kv4.Cache(graph.buffer(raw["k"]), graph.buffer(raw["v"]), graph.buffer(junk), graph.buffer(junk),
                              graph.buffer(self.table), self.lengths, pages, per, batch, kvh, page, dim)
        self.raw = raw

    def set_lengths(self, lengths):
        self.graph.write(self.lengths, np.asarray(lengths, np.int32))

    def rows(self, name):
        """(codes, scales) of the whole cache as it is: [pages, kvh, page, dim] and [..., dim / 64]."""
        p, kvh, page, dim = self.shape
        b = self.graph.read(getattr(self.c, name), p * kvh * page * dim // 2).reshape(p, kvh, page, dim // 2)
        q = np.empty(self.shape, np.int64)
        q[..., 0::2], q[..., 1::2] = b & 15, b >> 4
        s = self.graph.read(getattr(self.c, name + "_scale"), p * kvh * page * (dim // 64) * 2, np.float16)
        return (q + 8) % 16 - 8, s.reshape(p, kvh, page, dim // 64)

    def sequence(self, name, b, n):
        """Values of the first n tokens of sequence b: [n, kvh, dim] float64."""
        q, s = self.rows(name)
        ids = self.table[b]
        v = q[ids] * np.repeat(s[ids].astype(np.float64), 64, -1)
        return v.transpose(0, 2, 1, 3).reshape(-1, self.shape[1], self.shape[3])[:n]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,tokens,kvh,dim,page,lengths", [
    (1, 1, 1, 64, 16, [0]), (2, 5, 3, 128, 16, [14, 31]), (3, 17, 2, 64, 48, [0, 47, 100]), (4, 1, 8, 128, 64, [-1, 63, 64, 0]),
    (2, 130, 1, 256, 32, [7, 0]), (3, 3, 2, 128, 64, [-1, -5, -1])])
def test_append_and_unpack(we, graph, batch, tokens, kvh, dim, page, lengths, dtype):
    mark = graph.mark()
    c = Cache(we, graph, batch, max(lengths) + tokens, kvh, dim, page, 1)
    c.set_lengths(lengths)
    x = {n: randn(batch * tokens * kvh * dim, 2 + (n == "v"), 3.0).reshape(batch, tokens, kvh, dim) for n in "kv"}
    x["k"][0, 0, 0, :64] = 0                          # a group of zeros: scale 0, codes 0
    x["v"][-1, -1, -1, -64:] = 1e-9                   # a scale that rounds to 0
    x["v"][0, 0, 0, 3] = 5e4                          # an outlier
    if dtype == "bf16":
        x = {n: bf16_round(a).reshape(a.shape) for n, a in x.items()}
    before = {n: c.rows(n) for n in "kv"}
    dev = {n: graph.buffer(bits(a, dtype)) for n, a in x.items()}
    we.kv4.append(graph, c.c, dev["k"], dev["v"], tokens, dtype=dtype)
    size = batch * tokens * kvh * dim
    back = {n: graph.buffer(size * 4) for n in "kv"}
    we.kv4.unpack(graph, c.c, back["k"], back["v"], tokens, dtype="f32")
    low = {n: graph.buffer(size * 2) for n in "kv"}
    we.kv4.unpack(graph, c.c, low["k"], None, tokens, dtype="bf16")
    we.kv4.unpack(graph, c.c, None, low["v"], tokens, dtype="bf16")
    assert graph.device_error() == 0
    for n in "kv":
        q, s = quantise(x[n])
        want_q, want_s = before[n]
        idle = np.array(lengths) < 0
        for b in range(batch):
            for t in range(tokens):
                if idle[b]:
                    continue
                at = lengths[b] + t
                page_id, row = c.table[b, at // page], at % page
                want_q[page_id, :, row], want_s[page_id, :, row] = q[b, t], s[b, t]
        got_q, got_s = c.rows(n)
        assert np.array_equal(got_q, want_q)
        assert np.array_equal(got_s.view(np.uint16), want_s.view(np.uint16))
        val = (q * np.repeat(s.astype(np.float32), 64, -1)).astype(np.float32)
        val[idle] = 0
        assert np.array_equal(graph.read(back[n], size * 4, np.float32), val.ravel())
        assert np.array_equal(values(graph.read(low[n], size * 2), "bf16"), bf16_round(val.ravel()))
    graph.release(mark)


def test_append_from_a_fused_projection_and_advance(we, graph):
    """k and v cut out of rows [q | k | v], at addresses that are aligned to their element only; then advance, and a
    second append after the first."""
    batch, kvh, dim, page, heads = 2, 2, 64, 16, 3
    row = (heads + 2 * kvh) * dim + 1
    c = Cache(we, graph, batch, 40, kvh, dim, page, 3)
    lengths = np.array([15, -1], np.int32)
    c.set_lengths(lengths)
    for step, tokens in enumerate((2, 3)):
        x = bf16_round(randn(batch * tokens * row + 1, 4 + step))
        buf = graph.buffer(bits(x, "bf16"))
        k0, v0 = 1 + heads * dim, 1 + (heads + kvh) * dim
        we.kv4.append(graph, c.c, buf.ptr + 2 * k0, buf.ptr + 2 * v0, tokens, stride=row)
        q, s = c.rows("v")
        rows = np.stack([x[v0 + t * row: v0 + t * row + kvh * dim].reshape(kvh, dim) for t in range(tokens)])
        want, ws = quantise(rows)
        for t in range(tokens):
            at = lengths[0] + t
            assert np.array_equal(q[c.table[0, at // page], :, at % page], want[t])
            assert np.array_equal(s[c.table[0, at // page], :, at % page], ws[t])
        we.kv4.advance(graph, c.c, tokens)
        lengths = lengths + np.array([tokens, 0], np.int32)
        assert np.array_equal(graph.read(c.lengths, 8, np.int32), lengths)
    assert graph.device_error() == 0


def test_append_infinite_values_stay_finite(we, graph):
    c = Cache(we, graph, 1, 4, 1, 64, 16, 5)
    x = randn(64, 6).reshape(1, 1, 1, 64)
    x[..., 5], x[..., 6] = np.inf, -np.inf
    b = graph.buffer(np.asarray(x, np.float32))
    we.kv4.append(graph, c.c, b, b, 1, dtype="f32")
    q, s = c.rows("k")
    at = c.table[0, 0]
    assert s[at, 0, 0, 0] == 65504 and q[at, 0, 0, 5] == 7 and q[at, 0, 0, 6] == -8 and q[at, 0, 0, 0] == 0


def test_bad_pages_and_full_tables_are_skipped_and_recorded(we, graph):
    batch, kvh, dim, page = 2, 1, 64, 16
    c = Cache(we, graph, batch, 32, kvh, dim, page, 7)
    c.set_lengths([10, 30])
    bad = c.table.copy()
    bad[0, 1] = c.shape[0] + 5
    graph.write(c.c.page_table, bad)
    x = graph.buffer(bits(randn(batch * 8 * kvh * dim, 8), "f32"))
    before = c.rows("k")[0]
    we.kv4.append(graph, c.c, x, x, 8, dtype="f32")
    assert graph.device_error() in (6, 7)
    after = c.rows("k")[0]
    changed = {(p, r) for p, _, r, _ in np.argwhere(before != after)}
    allowed = {(c.table[0, 0], r) for r in range(10, 16)} | {(c.table[1, 1], r) for r in (14, 15)}
    assert changed <= allowed and changed
    back = graph.buffer(batch * 8 * kvh * dim * 4)
    we.kv4.unpack(graph, c.c, back, None, 8, dtype="f32")
    got = graph.read(back, None, np.float32).reshape(batch, 8, dim)
    assert graph.device_error() in (6, 7)
    assert np.all(got[0, 6:] == 0) and np.all(got[1, 2:] == 0) and np.any(got[0, 0] != 0)


def attend(q, k, v, seen, scale):
    """q [t, d], k, v [n, d], seen [t, n] in float64; rows that see nothing are zero."""
    s = np.where(seen, q @ k.T * scale, -np.inf)
    top = np.where(seen.any(1), s.max(1, initial=-np.inf), 0)[:, None]
    p = np.where(seen, np.exp(s - top), 0)
    total = p.sum(1, keepdims=True)
    return (p / np.where(total > 0, total, 1)) @ v


def slack(q, k, v, want, scale, dtype, rounding):
    e = 2.0**-20 * scale * np.linalg.norm(q, axis=-1).max() * (np.linalg.norm(k, axis=-1).max() if k.size else 0)
    top = np.abs(v).max() if v.size else 0
    return 2 * (2 * e + 2.0**-20 + (rounding if dtype == "bf16" else 0)) * top + (
        2.0**-8 * np.abs(want) if dtype == "bf16" else 0)


CASES = [
    # batch, tokens, lengths, heads, kv_heads, dim, page
    (1, 1, [0], 1, 1, 64, 16), (1, 1, [16], 4, 1, 128, 16), (2, 1, [15, 200], 8, 2, 128, 16), (1, 1, [517], 48, 12, 128, 64),
    (3, 1, [-1, 0, 1000], 8, 8, 64, 32), (4, 3, [5, -1, 64, 129], 12, 4, 128, 48), (2, 5, [0, 333], 16, 2, 64, 64),
    (1, 8, [1021], 32, 4, 128, 128), (2, 40, [3, 100], 6, 3, 128, 16), (1, 200, [0], 4, 4, 64, 64), (1, 2, [77], 4, 2, 256, 32),
    (2, 1, [300, 9], 40, 2, 128, 16), (1, 1, [20000], 2, 1, 128, 64), (1, 33, [5000], 2, 2, 64, 16), (1, 1, [3000], 24, 1, 256, 16),
    (2, 2, [-1, -7], 4, 2, 128, 16)]


def run_attention(we, graph, batch, tokens, lengths, heads, kvh, dim, page, dtype, q_scale=2.0, seed=0, out_dtype=None):
    od = out_dtype or dtype
    most = max(lengths)
    c = Cache(we, graph, batch, max(0, most) + tokens, kvh, dim, page, seed)
    c.set_lengths([0 if x >= 0 else -1 for x in lengths])
    n = max(1, max(0, most) + tokens)
    # every sequence is filled to the longest one's end: keys past its own end hold values, garbage lies in other pages
    k = bf16_round(randn(batch * n * kvh * dim, seed + 1)).reshape(batch, n, kvh, dim)
    v = bf16_round(randn(batch * n * kvh * dim, seed + 2)).reshape(batch, n, kvh, dim)
    for b in range(batch):
        if lengths[b] >= 0:
            own = [-1] * batch
            own[b] = 0
            c.set_lengths(own)
            upto = lengths[b] + tokens
            kb, vb = np.zeros((batch, upto, kvh, dim), np.float32), np.zeros((batch, upto, kvh, dim), np.float32)
            kb[b], vb[b] = k[b, :upto], v[b, :upto]
            we.kv4.append(graph, c.c, graph.buffer(bits(kb, "f32")), graph.buffer(bits(vb, "f32")), upto, dtype="f32")
    c.set_lengths(lengths)
    q = randn(batch * tokens * heads * dim, seed + 3, q_scale).reshape(batch, tokens, heads, dim)
    q = bf16_round(q).reshape(q.shape) if dtype == "bf16" else q
    out = graph.buffer(np.full(q.size * (2 if od == "bf16" else 4), 0xFF, np.uint8))
    we.kv4.attention(graph, c.c, graph.buffer(bits(q, dtype)), out, tokens, heads, dtype=dtype, out_dtype=od)
    got = values(graph.read(out, q.size * (2 if od == "bf16" else 4)).copy(), od).reshape(q.shape)
    assert graph.device_error() == 0
    for b in range(batch):
        if lengths[b] < 0:
            assert np.all(got[b] == 0)
            continue
        n = lengths[b] + tokens
        kk, vv = c.sequence("k", b, n), c.sequence("v", b, n)
        seen = np.arange(n)[None, :] <= lengths[b] + np.arange(tokens)[:, None]
        for h in range(heads):
            j = h // (heads // kvh)
            qh = q[b, :, h].astype(np.float64)
            want = attend(qh, kk[:, j], vv[:, j], seen, 1 / math.sqrt(dim))
            tol = slack(qh, kk[:, j], vv[:, j], want, 1 / math.sqrt(dim), od, 2.0**-11)
            err = np.abs(got[b, :, h] - want)
            assert np.all(err <= tol), (b, h, err.max(), np.min(tol))
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention_matches_float64(we, graph, case, dtype):
    mark = graph.mark()
    run_attention(we, graph, *case, dtype, seed=10)
    graph.release(mark)


@pytest.mark.parametrize("dtype,out_dtype", [("bf16", "f32"), ("f32", "bf16")])
def test_attention_mixed_types(we, graph, dtype, out_dtype):
    mark = graph.mark()
    run_attention(we, graph, 2, 3, [70, 20], 8, 2, 128, 32, dtype, seed=11, out_dtype=out_dtype)
    graph.release(mark)


def test_attention_large_scores(we, graph):
    """Scores over hundreds of units: a single key takes nearly all the weight, the running maximum moves often."""
    mark = graph.mark()
    run_attention(we, graph, 1, 1, [2000], 4, 1, 128, 64, "f32", q_scale=30.0, seed=12)
    graph.release(mark)


def test_attention_values_of_any_magnitude(we, graph):
    """v rows from 1e-4 to 1e4 in one sequence, and all rows near 1e-4 in another: scales keep their relative accuracy."""
    for factor in (np.logspace(-4, 4, 300), np.full(300, 1e-4), np.full(300, 5e3), np.logspace(4, -4, 300)):
        mark = graph.mark()
        c = Cache(we, graph, 1, 300, 2, 64, 32, 13)
        k = randn(300 * 2 * 64, 14).reshape(1, 300, 2, 64)
        v = randn(300 * 2 * 64, 15).reshape(1, 300, 2, 64) * factor[None, :, None, None].astype(np.float32)
        we.kv4.append(graph, c.c, graph.buffer(np.asarray(k, np.float32)), graph.buffer(np.asarray(v, np.float32)), 300, dtype="f32")
        c.set_lengths([299])
        q = bf16_round(randn(4 * 64, 16, 2.0)).reshape(1, 1, 4, 64)
        for dtype in ("f32", "bf16"):
            out = graph.buffer(1024)
            we.kv4.attention(graph, c.c, graph.buffer(bits(q, dtype)), out, 1, 4, dtype=dtype, out_dtype=dtype)
            got = values(graph.read(out, 4 * 64 * (2 if dtype == "bf16" else 4)).copy(), dtype).reshape(4, 64)
            kk, vv = c.sequence("k", 0, 300), c.sequence("v", 0, 300)
            for h in range(4):
                qh = q[0, :, h].astype(np.float64)
                want = attend(qh, kk[:, h // 2], vv[:, h // 2], np.ones((1, 300), bool), 0.125)
                tol = slack(qh, kk[:, h // 2], vv[:, h // 2], want, 0.125, dtype, 2.0**-11)
                assert np.all(np.abs(got[h] - want) <= tol)
        graph.release(mark)


def test_attention_strides_scale_and_a_bad_page(we, graph):
    """q inside wider rows, out too, an own scale; then a page id out of range takes its keys out and is recorded."""
    heads, kvh, dim, page, n = 4, 2, 64, 16, 50
    c = Cache(we, graph, 1, n + 2, kvh, dim, page, 17)
    kv = randn(2 * (n + 2) * kvh * dim, 18).reshape(2, 1, n + 2, kvh, dim)
    we.kv4.append(graph, c.c, graph.buffer(np.asarray(kv[0], np.float32)), graph.buffer(np.asarray(kv[1], np.float32)), n + 2,
                  dtype="f32")
    c.set_lengths([n])
    qs, os_ = heads * dim + 5, heads * dim + 3
    q = randn(2 * qs, 19)
    fill = np.full(2 * os_, 7.0, np.float32)
    kk, vv = c.sequence("k", 0, n + 2), c.sequence("v", 0, n + 2)
    for broken in (False, True):
        if broken:
            table = c.table.copy()
            table[0, 1] = -3
            graph.write(c.c.page_table, table)
        out = graph.buffer(fill)
        we.kv4.attention(graph, c.c, graph.buffer(q), out, 2, heads, dtype="f32", out_dtype="f32", q_stride=qs, out_stride=os_,
                         scale=0.3)
        got = graph.read(out, fill.nbytes, np.float32)
        assert graph.device_error() == (6 if broken else 0)
        for i in range(2):
            for h in range(heads):
                seen = np.arange(n + 2)[None, :] <= n + i
                if broken:
                    seen = seen & ~((np.arange(n + 2) >= page) & (np.arange(n + 2) < 2 * page))[None, :]
                qh = q[i * qs + h * dim: i * qs + (h + 1) * dim].astype(np.float64)[None]
                want = attend(qh, kk[:, h // 2], vv[:, h // 2], seen, 0.3)[0]
                tol = slack(qh, kk[:, h // 2], vv[:, h // 2], want, 0.3, "f32", 0)
                assert np.all(np.abs(got[i * os_ + h * dim: i * os_ + (h + 1) * dim] - want) <= tol)
            assert np.all(got[i * os_ + heads * dim: (i + 1) * os_] == 7.0)


def test_attention_is_deterministic_and_replays_from_a_graph(we, graph):
    """The same call gives the same bits, and a captured step reads the lengths that the device holds when it runs."""
    heads, kvh, dim, page = 8, 1, 128, 64
    c = Cache(we, graph, 2, 9000, kvh, dim, page, 20)
    x = randn(2 * 9000 * kvh * dim, 21).reshape(2, 9000, kvh, dim)
    b = graph.buffer(bits(x, "bf16"))
    we.kv4.append(graph, c.c, b, b, 9000)
    q, out = graph.buffer(bits(randn(2 * heads * dim, 22), "bf16")), graph.buffer(2 * heads * dim * 2)
    call = we.kv4.attention_call(graph, c.c, q, out, 1, heads)
    seen = {}
    for lengths in ([8999, 20], [400, 8999], [8999, 20]):
        c.set_lengths(lengths)
        call()
        r = graph.read(out).copy()
        assert np.array_equal(seen.setdefault(tuple(lengths), r), r)
    with graph.capture() as cap:
        call()
    for lengths, want in seen.items():
        c.set_lengths(list(lengths))
        cap.launch()
        assert np.array_equal(graph.read(out), want)
    cap.destroy()


def test_attention_past_the_page_table(we, graph):
    """Lengths beyond the table: its keys are attended, the rest recorded as missing."""
    c = Cache(we, graph, 1, 32, 1, 64, 16, 23)
    x = graph.buffer(np.asarray(randn(32 * 64, 24), np.float32))
    we.kv4.append(graph, c.c, x, x, 32, dtype="f32")
    c.set_lengths([1000])
    q = randn(64, 25).reshape(1, 64)
    out = graph.buffer(256)
    we.kv4.attention(graph, c.c, graph.buffer(q), out, 1, 1, dtype="f32", out_dtype="f32")
    assert graph.device_error() == 7
    kk, vv = c.sequence("k", 0, 32)[:, 0], c.sequence("v", 0, 32)[:, 0]
    want = attend(q.astype(np.float64), kk, vv, np.ones((1, 32), bool), 0.125)
    got = graph.read(out, 256, np.float32)
    assert np.all(np.abs(got - want[0]) <= slack(q, kk, vv, want, 0.125, "f32", 0))


def test_refusals(we, graph):
    E, k4 = we._lib.WeError, we.kv4
    b = graph.buffer(4096)

    def cache(**kw):
        d = dict(k=b, v=b, k_scale=b, v_scale=b, page_table=b, lengths=b, pages=1, max_pages=1, batch=1, kv_heads=1, page=16, dim=64)
        return k4.Cache(**{**d, **kw})

    for words, kw in (("64, 128 or 256", {"dim": 96}), ("multiple of 16", {"page": 20}), ("missing", {"lengths": None}),
                      ("16-byte", {"k": b.ptr + 4}), ("31 bits", {"max_pages": 1 << 30}), ("negative", {"batch": -1})):
        with pytest.raises(E, match=words):
            k4.append(graph, cache(**kw), b, b, 1)
    with pytest.raises(E, match="multiple of kvHeads"):
        k4.attention(graph, cache(kv_heads=2), b, b, 1, 3)
    with pytest.raises(E, match="shorter"):
        k4.append(graph, cache(kv_heads=2), b, b, 1, stride=64)
    with pytest.raises(E, match="shorter"):
        k4.attention(graph, cache(), b, b, 1, 2, q_stride=64)
    with pytest.raises(E, match="tokens"):
        k4.append(graph, cache(), b, b, -1)
    with pytest.raises(E, match="f32 or bf16"):
        k4.attention(graph, cache(), b, b, 1, 1, dtype="fp8")
    k4.attention(graph, cache(batch=0), b, b, 1, 1)
    k4.append(graph, cache(), b, b, 0)
    with pytest.raises(ValueError, match="share a page table"):
        k4.Cache.create(graph, 1, 64, 1, 64, like=cache(batch=2))
    assert graph.device_error() == 0


def test_create_and_a_decoding_loop(we, graph):
    """Two layers that share lengths: prompt, then single tokens, each step's attention against float64."""
    batch, heads, kvh, dim = 2, 4, 2, 64
    mark = graph.mark()
    first = we.kv4.Cache.create(graph, batch, 40, kvh, dim, page=16)
    layers = [first, we.kv4.Cache.create(graph, batch, 40, kvh, dim, page=16, like=first)]
    have = 0
    hist = [[], []]
    for step, tokens in enumerate((19, 1, 1, 2)):
        for i, c in enumerate(layers):
            k, v = (randn(batch * tokens * kvh * dim, 100 + 10 * step + 2 * i + j).reshape(batch, tokens, kvh, dim) for j in (0, 1))
            q = randn(batch * tokens * heads * dim, 200 + 10 * step + i).reshape(batch, tokens, heads, dim)
            we.kv4.append(graph, c, graph.buffer(k), graph.buffer(v), tokens, dtype="f32")
            out = graph.buffer(q.nbytes)
            we.kv4.attention(graph, c, graph.buffer(q), out, tokens, heads, dtype="f32", out_dtype="f32")
            got = graph.read(out, q.nbytes, np.float32).reshape(q.shape)
            hist[i].append([a * np.repeat(s.astype(np.float64), 64, -1) for a, s in (quantise(k), quantise(v))])
            kk, vv = (np.concatenate([h[j] for h in hist[i]], 1) for j in (0, 1))
            n = have + tokens
            seen = np.arange(n)[None, :] <= have + np.arange(tokens)[:, None]
            for b in range(batch):
                for h in range(heads):
                    want = attend(q[b, :, h].astype(np.float64), kk[b, :, h // 2], vv[b, :, h // 2], seen, 0.125)
                    tol = slack(q[b, :, h], kk[b, :, h // 2], vv[b, :, h // 2], want, 0.125, "f32", 0)
                    assert np.all(np.abs(got[b, :, h] - want) <= tol)
        we.kv4.advance(graph, first, tokens)
        have += tokens
    assert graph.read(first.lengths, 8, np.int32).tolist() == [have, have]
    graph.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", [(2, 1, [30000, 9000], 8, 2, 64, 64), (1, 4, [24000], 16, 2, 128, 32), (3, 12, [9001, -1, 20], 6, 2, 64, 16),
                                  (1, 1, [8300], 3, 1, 256, 48)], ids=str)
def test_attention_over_several_runs(we, graph, case, dtype):
    """Sequences long enough that clusters share one, beside short and idle ones; twice, to see the counters left at zero."""
    mark = graph.mark()
    for seed in (30, 40):
        run_attention(we, graph, *case, dtype, seed=seed)
    graph.release(mark)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shift", [0, 1])
def test_append_of_a_long_prompt(we, graph, dtype, shift):
    """Enough tokens for more blocks than two an SM, with rows of whole 16 bytes and (shift) without."""
    tokens, kvh, dim, page = 2500, 3, 128, 32
    stride = kvh * dim + shift
    x = [bf16_round(randn(tokens * stride, 50 + i)) for i in range(2)]
    mark = graph.mark()
    c = Cache(we, graph, 1, tokens + 40, kvh, dim, page)
    c.set_lengths([33])
    we.kv4.append(graph, c.c, *(graph.buffer(bits(v, dtype)) for v in x), tokens, dtype=dtype, stride=stride)
    for name, v in zip("kv", x):
        rows = v.reshape(tokens, stride)[:, : kvh * dim].reshape(tokens, kvh, dim)
        q, s = quantise(rows)
        want = q * np.repeat(s.astype(np.float64), 64, -1).reshape(rows.shape)
        assert np.array_equal(c.sequence(name, 0, tokens + 33)[33:], want)
    assert graph.device_error() == 0
    graph.release(mark)
