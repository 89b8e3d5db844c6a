"""GPU parity of we_matvec (few rows times int4 group-64 weights) with a plain float64 product of the same codes.

Bound of one value, for any order of summation by groups of 64: every product is exact or within 2^-22 of itself (an f32
x is held as two terms), a group's sum has at most 64 additions and the sum over groups at most k / 64 + 16 more, each
within 2^-24 of a partial sum that is at most sum |w x|: (k / 64 + 84) 2^-24 sum |w x|. A bf16 output adds its own
rounding, at most 2^-8 |y| (8 significant bits, to nearest).
"""
import numpy as np
import pytest

from oracle import oracle as O
from util import bf16, bf16_round, randn

pytestmark = pytest.mark.gpu


def codes(packed, n, k):
    """Two's complement codes [n, k] of packed bytes, low nibble first."""
    b = packed.reshape(n, k // 2)
    q = np.empty((n, k), np.int64)
    q[:, 0::2], q[:, 1::2] = b & 15, b >> 4
    return (q + 8) % 16 - 8


def weights(n, k, seed, std=0.02):
    packed, scales = O.quant_int4_g64(randn(n * k, seed, std), n, k)
    s = np.asarray(scales, np.uint16).view(np.float16).reshape(n, k // 64)
    return np.asarray(packed, np.uint8), s, codes(np.asarray(packed, np.uint8), n, k) * np.repeat(s.astype(np.float64), 64, 1)


def bits(x, dtype):
    return bf16(x) if dtype == "bf16" else np.asarray(x, np.float32)


def values(raw, dtype):
    return O.bf16_to_f32(raw.view(np.uint16)) if dtype == "bf16" else raw.view(np.float32)


def bound(x, w, y, dtype):
    k = w.shape[1]
    slack = (k / 64 + 84) * 2.0**-24 * (np.abs(x) @ np.abs(w).T)
    return slack + (2.0**-8 * np.abs(y) if dtype == "bf16" else 0) + 1e-45


def product(we, graph, x, packed, s, m, n, k, x_dtype, y_dtype, **kw):
    mark = graph.mark()
    try:
        y = graph.buffer(max(4, m * n * (2 if y_dtype == "bf16" else 4)))
        we.kernels.matvec(graph, graph.buffer(bits(x, x_dtype)), graph.buffer(packed), y, m, n, k,
                          group_scale=graph.buffer(s), x_dtype=x_dtype, y_dtype=y_dtype, **kw)
        got = values(graph.read(y, m * n * (2 if y_dtype == "bf16" else 4)).copy(), y_dtype)
        assert graph.device_error() == 0
        return got.reshape(m, n).astype(np.float64)
    finally:
        graph.release(mark)


SHAPES = [(1, 1, 64), (1, 16, 64), (1, 17, 128), (2, 33, 192), (3, 100, 320), (4, 15, 2496), (5, 257, 1088),
          (7, 48, 6144), (8, 129, 4096), (9, 65, 704), (13, 31, 1984), (16, 1003, 512), (16, 8, 16384), (1, 4099, 448),
          (1, 1536, 6144), (8, 6144, 1024)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matvec_matches_float64(we, graph, m, n, k, dtype):
    packed, s, w = weights(n, k, n + k)
    x = randn(m * k, m).reshape(m, k)
    if dtype == "bf16":
        x = bf16_round(x).reshape(m, k)
    want = x.astype(np.float64) @ w.T
    got = product(we, graph, x, packed, s, m, n, k, dtype, dtype)
    assert np.all(np.abs(got - want) <= bound(x.astype(np.float64), w, want, dtype))


@pytest.mark.parametrize("x_dtype,y_dtype", [("bf16", "f32"), ("f32", "bf16")])
def test_matvec_mixed_types(we, graph, x_dtype, y_dtype):
    m, n, k = 6, 70, 640
    packed, s, w = weights(n, k, 3)
    x = randn(m * k, 4).reshape(m, k)
    x = bf16_round(x).reshape(m, k) if x_dtype == "bf16" else x
    want = x.astype(np.float64) @ w.T
    got = product(we, graph, x, packed, s, m, n, k, x_dtype, y_dtype)
    assert np.all(np.abs(got - want) <= bound(x.astype(np.float64), w, want, y_dtype))


@pytest.mark.parametrize("dtype,scale", [("f32", 1e30), ("f32", 1e-30), ("bf16", 1e30), ("bf16", 1e-30), ("f32", 1e-40),
                                         ("bf16", 1e-39)])
def test_matvec_extreme_magnitudes(we, graph, dtype, scale):
    """Rows far outside f16's range, and rows whose groups differ by 9 decades: each group's terms keep their bits."""
    m, n, k = 3, 40, 512
    packed, s, w = weights(n, k, 5, 1.0)
    x = randn(m * k, 6).reshape(m, k) * np.float32(scale)
    x[1] *= np.repeat(10.0 ** np.linspace(-9, 0, k // 64), 64).astype(np.float32)
    x[2, ::7] = 0
    if dtype == "bf16":
        x = bf16_round(x).reshape(m, k)
    want = x.astype(np.float64) @ w.T
    got = product(we, graph, x, packed, s, m, n, k, dtype, "f32")
    # below the normal range of f32 the terms are multiples of 2^-149
    slack = bound(x.astype(np.float64), w, want, "f32") + np.abs(w).sum(1) * 2.0**-148
    assert np.all(np.abs(got - want) <= slack)


def test_matvec_within_a_group_of_wide_range(we, graph):
    """One large value among small ones of the same group: a term's error is at most 2^-36 of the group's maximum."""
    m, n, k = 2, 24, 256
    packed, s, w = weights(n, k, 7)
    x = randn(m * k, 8, 1e-4).reshape(m, k)
    x[:, 5::64] = 300.0
    want = x.astype(np.float64) @ w.T
    got = product(we, graph, x, packed, s, m, n, k, "f32", "f32")
    slack = bound(x.astype(np.float64), w, want, "f32") + 300 * 2.0**-36 * np.abs(w).sum(1)
    assert np.all(np.abs(got - want) <= slack)


def test_matvec_all_codes_and_scales(we, graph):
    """Every code, -8 included, zero and subnormal scales, against an exact product."""
    n, k = 32, 128
    r = np.random.default_rng(1)
    packed = r.integers(0, 256, n * k // 2, dtype=np.uint8)
    s = (r.random((n, 2)) * 0.1).astype(np.float16)
    s[0], s[1], s[2], s[3] = 0, 2.0**-24, 2.0**-15, 65504
    w = codes(packed, n, k) * np.repeat(s.astype(np.float64), 64, 1)
    x = bf16_round(randn(k, 2)).reshape(1, k)
    want = x.astype(np.float64) @ w.T
    got = product(we, graph, x, packed, s, 1, n, k, "bf16", "f32")
    assert np.all(np.abs(got - want) <= bound(x.astype(np.float64), w, want, "f32"))
    assert got[0, 0] == 0


def test_matvec_non_finite_rows_stay_their_own(we, graph):
    m, n, k = 4, 50, 320
    packed, s, w = weights(n, k, 9)
    x = bf16_round(randn(m * k, 10)).reshape(m, k)
    clean = product(we, graph, x, packed, s, m, n, k, "bf16", "f32")
    bad = x.copy()
    bad[1, 70], bad[2, 3] = np.nan, np.inf
    got = product(we, graph, bad, packed, s, m, n, k, "bf16", "f32")
    assert np.array_equal(got[[0, 3]], clean[[0, 3]])
    assert np.all(np.isnan(got[1])) and not np.any(np.isfinite(got[2]))


def test_matvec_strides_offsets_and_epilogue(we, graph):
    """x and y inside wider rows, bias, SwiGLU against an aux tensor, a per-channel gate and accumulation into y."""
    m, n, k, xs, ys, xo, yo = 5, 37, 192, 232, 61, 8, 11
    packed, s, w = weights(n, k, 11, 0.3)
    x = randn(xo + m * xs, 12)
    y0, aux = randn(yo + m * ys, 13), randn(yo + m * ys, 14)
    bias, gate = randn(n, 15), randn(n, 16)
    yb = graph.buffer(y0)
    we.kernels.matvec(graph, graph.buffer(x), graph.buffer(packed), yb, m, n, k, group_scale=graph.buffer(s),
                      bias=graph.buffer(bias), x_stride=xs, y_stride=ys, x_offset=xo, y_offset=yo, accumulate=True,
                      aux_op="swiglu", aux=graph.buffer(aux), gate=graph.buffer(gate))
    got = graph.read(yb, y0.nbytes, np.float32)
    xi = np.stack([x[xo + i * xs: xo + i * xs + k] for i in range(m)]).astype(np.float64)
    want = y0.astype(np.float64).copy()
    v = xi @ w.T + bias
    for i in range(m):
        a = aux[yo + i * ys: yo + i * ys + n].astype(np.float64)
        want[yo + i * ys: yo + i * ys + n] += gate * (a / (1 + np.exp(-a))) * v[i]
    # the product's bound times the largest factor after it, plus 2^-21 relative for the exponential and the products
    slack = 4 * np.max(bound(xi, w, v, "f32")) * np.max(np.abs(gate)) * np.max(np.abs(aux)) + 2.0**-21 * np.abs(want)
    assert np.all(np.abs(got - want) <= slack + 2.0**-20)
    untouched = np.ones(y0.size, bool)
    for i in range(m):
        untouched[yo + i * ys: yo + i * ys + n] = False
    assert np.array_equal(got[untouched], y0[untouched])


@pytest.mark.parametrize("act", ["gelu_tanh", "silu"])
def test_matvec_activation_and_op_form(we, graph, act):
    m, n, k = 2, 48, 256
    packed, s, w = weights(n, k, 17, 0.2)
    x = randn(m * k, 18).reshape(m, k)
    lin = we.Linear(graph.buffer(packed), "int4", 1.0, n, k, group_scale=graph.buffer(s))
    y = we.matvec(graph, graph.buffer(x), lin, m, act=act)
    got = graph.read(y, m * n * 4, np.float32).reshape(m, n)
    v = x.astype(np.float64) @ w.T
    want = v / (1 + np.exp(-v)) if act == "silu" else 0.5 * v * (1 + np.tanh(0.7978845608028654 * (v + 0.044715 * v**3)))
    assert np.max(np.abs(got - want)) <= 1.2 * np.max(bound(x.astype(np.float64), w, v, "f32")) + 2.0**-20 * np.max(np.abs(v))


def test_matvec_is_deterministic_and_replays_from_a_graph(we, graph):
    m, n, k = 3, 700, 4096
    packed, s, _ = weights(n, k, 19)
    x, y = graph.buffer(bf16(randn(m * k, 20))), graph.buffer(m * n * 2)
    call = we.kernels.matvec_call(graph, x, graph.buffer(packed), y, m, n, k, group_scale=graph.buffer(s),
                                  x_dtype="bf16", y_dtype="bf16")
    call()
    first = graph.read(y).copy()
    with graph.capture() as cap:
        call()
    for _ in range(3):
        graph.write(y, np.zeros(m * n, np.uint16))
        cap.launch()
        assert np.array_equal(graph.read(y), first)
    cap.destroy()


def test_matvec_refusals(we, graph):
    K, E = we.kernels, we._lib.WeError
    b = graph.buffer(1 << 16)

    def refused(words, m=1, n=8, k=64, w=b, **kw):
        with pytest.raises((E, ValueError), match=words):
            K.matvec(graph, b, w, b, m, n, k, group_scale=kw.pop("group_scale", b), **kw)

    refused("1 to 16 rows", m=0)
    refused("1 to 16 rows", m=17)
    refused("multiple of 64", k=96)
    refused("16-byte aligned", w=b.ptr + 8)
    refused("group scales", group_scale=None)
    refused("xOffset must be a multiple of 4", x_offset=9)
    refused("stride is shorter", x_stride=32)
    refused("stride is shorter", y_stride=4)
    refused("aux tensor", aux_op="swiglu")
    with pytest.raises(ValueError, match="int4"):
        we.matvec(graph, b, we.Linear(b, "fp8", 1.0, 8, 64), 1)
    K.matvec(graph, b, b, b, 1, 0, 64, group_scale=b)  # no channels: nothing to do
    assert graph.device_error() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,n,k", [(16, 37, 28736), (16, 21, 40000), (16, 19, 60032), (3, 9, 300032)])
def test_matvec_long_rows(we, graph, m, n, k, dtype):
    """x that leaves room for one block an SM, for a whole SM's shared memory, and (the last two, but for three bf16 rows) that does not fit 8 SMs':
    there a lane sums k / 32 products in turn, each rounded, and 32 lanes join in 5 more additions."""
    packed, s, w = weights(n, k, n + k)
    x = randn(m * k, m).reshape(m, k)
    if dtype == "bf16":
        x = bf16_round(x).reshape(m, k)
    x = x.astype(np.float64)
    want = x @ w.T
    got = product(we, graph, x.astype(np.float32), packed, s, m, n, k, dtype, dtype)
    slack = (k / 32 + 84) * 2.0**-24 * (np.abs(x) @ np.abs(w).T) + (2.0**-8 * np.abs(want) if dtype == "bf16" else 0)
    assert np.all(np.abs(got - want) <= slack)


def test_matvec_non_finite_rows(we, graph):
    """A row of x that holds a NaN or an infinity is NaN; the rows beside it are what they are without it."""
    m, n, k = 4, 40, 320
    packed, s, w = weights(n, k, 9)
    for dtype in ("bf16", "f32"):
        x = bf16_round(randn(m * k, 10)).reshape(m, k)
        clean = product(we, graph, x, packed, s, m, n, k, dtype, "f32")
        bad = x.copy()
        bad[1, 77], bad[3, 319] = np.nan, np.inf
        got = product(we, graph, bad, packed, s, m, n, k, dtype, "f32")
        assert np.all(np.isnan(got[[1, 3]]))
        assert np.array_equal(got[[0, 2]], clean[[0, 2]])
