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
