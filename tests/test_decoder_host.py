"""Host side of the decoder's operators without a GPU: what the op forms and decoder.Decoder refuse before anything is
allocated, written or queued. The graph here hands out addresses and records calls."""
import numpy as np
import pytest


class HostGraph:
    """Addresses in place of device memory; `fail_at` makes that allocation (counted from 0) raise."""

    ctx = None

    def __init__(self, we):
        self.Buffer, self.next, self.owned, self.log, self.fail_at = we.Buffer, 1 << 20, {}, [], None

    def buffer(self, data):
        if self.fail_at == 0:
            raise MemoryError("no room")
        if self.fail_at is not None:
            self.fail_at -= 1
        n = int(data) if isinstance(data, (int, np.integer)) else np.asarray(data).nbytes
        b = self.Buffer(self.next, n)
        self.next += (n + 511) // 256 * 256
        self.owned[b.ptr] = n
        self.log.append(("buffer", n))
        return b

    def free(self, b):
        del self.owned[b.ptr]
        self.log.append(("free", b.size))

    def write(self, dst, data):
        self.log.append(("write", np.asarray(data).nbytes))


@pytest.fixture
def host(we):
    return HostGraph(we)


@pytest.mark.parametrize("kw", [{"y_stride": 128}, {"y_offset": 4}])
def test_matvec_op_has_an_output_of_its_own_layout(we, host, kw):
    """The op form's buffer holds m x n values: rows further apart would be written past its end."""
    lin = we.Linear(host.buffer(64 * 32), "int4", 1.0, 64, 64, group_scale=host.buffer(128))
    before = list(host.log)
    with pytest.raises(TypeError):
        we.matvec(host, 1 << 20, lin, 2, **kw)
    assert host.log == before


def test_cross_attention_op_has_an_output_of_its_own_layout(we, host):
    with pytest.raises(TypeError):
        we.cross_attention(host, 1 << 20, 1 << 20, 1 << 20, 1, 2, 3, 2, 1, 64, out_stride=256)
    assert host.log == []


def layer(we, host, cfg, width=None):
    """Weights of a layer by their shapes alone; width: of the states, None for a layer without cross attention."""
    def lin(n, k):
        return we.Linear(host.buffer(n * k // 2), "int4", 1.0, n, k, group_scale=host.buffer(n * k // 32))

    qw, kw = cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
    cross = {} if width is None else {"cross_norm": host.buffer(cfg.hidden * 4), "cross_q": lin(qw, cfg.hidden), "cross_k": lin(kw, width),
                                      "cross_v": lin(kw, width), "cross_o": lin(cfg.hidden, qw)}
    return we.decoder.DecoderLayer(host.buffer(cfg.hidden * 4), lin(qw, cfg.hidden), lin(kw, cfg.hidden), lin(kw, cfg.hidden), lin(cfg.hidden, qw),
                                   host.buffer(256), host.buffer(256), host.buffer(cfg.hidden * 4), lin(cfg.mlp, cfg.hidden),
                                   lin(cfg.mlp, cfg.hidden), lin(cfg.hidden, cfg.mlp), **cross)


def decoder(we, host, batch=3, width=None, layers=1):
    cfg = we.decoder.DecoderConfig(64, 128, 2, 1, 64, page=16)
    d = we.decoder.Decoder(host, cfg, [layer(we, host, cfg, width) for _ in range(layers)], batch, 32)
    host.log.clear()
    return d


@pytest.mark.parametrize("sequence", [-1, -3, 3, 100])
def test_a_prompt_names_a_sequence_of_the_batch(we, host, sequence):
    """A negative index would put the page table's row and the length before their buffers."""
    d = decoder(we, host)
    with pytest.raises(ValueError, match="sequence must be in 0..2"):
        d.prompt(sequence, 1 << 20, 4)
    assert host.log == [] and d.lengths == [0, 0, 0]


@pytest.mark.parametrize("lengths", [[], [3], [3, 3], [3, 3, 3, 3], np.array([1, 2])])
def test_states_have_a_length_for_every_sequence(we, host, lengths):
    """The kernels read one length of each sequence from the device."""
    d = decoder(we, host, width=64)
    with pytest.raises(ValueError, match="one length for each of 3"):
        d.set_states(1 << 20, 3, lengths)
    assert host.log == []


@pytest.mark.parametrize("shape", [(4, 64), (1, 64), (3, 65), (0,)])
def test_a_step_takes_one_embedding_of_every_sequence(we, host, shape):
    """More values would be copied past the end of the step's buffer, fewer would leave the last step's output in it."""
    d = decoder(we, host)
    with pytest.raises(ValueError, match="x must hold 3 x 64 values"):
        d.step(np.zeros(shape, np.float32))
    assert host.log == [] and d.lengths == [0, 0, 0]


def test_states_that_fail_half_way_leave_none(we, host, monkeypatch):
    """The old states are gone by then: a step asks for new ones, and nothing is freed twice or kept."""
    monkeypatch.setattr(we.kernels, "matmul", lambda *a, **k: None)
    d = decoder(we, host, width=64, layers=2)
    owned = set(host.owned)
    d.set_states(1 << 20, 3)
    assert len(set(host.owned) - owned) == 5
    for fail_at in (0, 3, 4):
        host.fail_at = fail_at
        with pytest.raises(MemoryError):
            d.set_states(1 << 20, 5)
        assert set(host.owned) == owned
        with pytest.raises(ValueError, match="call set_states first"):
            d.step(np.zeros((3, 64), np.float32))
    host.fail_at = None
    d.set_states(1 << 20, 4, [4, 0, 2])
    assert len(set(host.owned) - owned) == 5 and d._state_tokens == 4


def test_a_prompt_needs_the_same_memory_whatever_the_layers(we, host, monkeypatch):
    """The residuals are added in place by the linears: a long prompt takes no new buffers layer by layer."""
    for name in ("rmsnorm", "matmul", "qknorm_rope", "attention", "cross_attention"):
        monkeypatch.setattr(we.kernels, name, lambda *a, **k: None)
    for name in ("append", "unpack", "advance"):
        monkeypatch.setattr(we.kv4, name, lambda *a, **k: None)
    monkeypatch.setattr(we.ops, "add", lambda g, x, y, n: g.buffer(n * 4))
    host.mark, host.release, host.copy = lambda: 0, lambda mark: None, lambda *a: None
    took = {}
    for layers in (1, 4):
        d = decoder(we, host, width=64, layers=layers)
        d.set_states(1 << 20, 3)
        host.log.clear()
        d.prompt(1, 1 << 20, 20)
        took[layers] = sum(n for what, n in host.log if what == "buffer")
        assert d.lengths == [0, 20, 0]
    assert took[1] == took[4]


def test_no_kernel_of_these_operators_is_chosen_by_the_environment(we):
    """Sizes, types and alignment decide: a variable would change a call's rounding behind its caller's back."""
    import os

    csrc = os.path.join(os.path.dirname(we.__file__), "csrc")
    for name in ("we_decode.cu", "k_matvec.cu", "k_kv4.cu", "k_cross.cu", "k_cross_flash.cu", "attn_merge.cuh"):
        with open(os.path.join(csrc, name)) as f:
            assert "getenv" not in f.read(), name
