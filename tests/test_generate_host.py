"""What Decoder and its buffers do before anything runs on a device: refusals, copies, pages."""
import numpy as np
import pytest

from warpforge_b200 import _native as N

LIB = N.load()


class HostContext:
    """A context without a device: a copy has to fit the allocation that it begins in, kernels are not launched."""

    def __init__(self):
        self._lib, self.handle, self.room, self.copies, self._next = LIB, 0, {}, 0, 4096

    def _ck(self, what, status):
        pass

    def allocate(self, n):
        at = self._next
        self._next += -(-n // 256) * 256 + 256
        self.room[at] = n
        return at

    def free(self, p):
        del self.room[p]

    def copy_to_device(self, dptr, host, stream=0, sync=True):
        assert host.nbytes <= self.room[dptr], f"{host.nbytes} bytes into {self.room[dptr]}"
        self.copies += 1

    def copy_to_host(self, host, dptr, stream=0, sync=True):
        assert host.nbytes <= self.room[dptr]
        host[:] = 0

    def synchronize(self, stream=0):
        pass


@pytest.fixture
def model():
    from warpforge_b200.generate import Decoder, DecoderSpec
    from warpforge_b200.quant import QuantizationType

    m = Decoder(HostContext(), DecoderSpec(QuantizationType.Q8_0, 64, 2, 1, 32, 64, 1, 64, max_positions=100), pages=12, page_tokens=16, max_tokens=32, max_sequences=3)
    yield m
    m.close()


def test_more_new_tokens_than_there_is_room_for(model):
    seqs = [model.sequence() for _ in range(2)]
    with pytest.raises(ValueError):
        model.step(seqs, [list(range(30)), list(range(10))])
    with pytest.raises(ValueError):
        model.prefill(seqs, [np.arange(30), np.arange(10)])


def test_a_copy_has_to_fit_its_buffer(model):
    for name, dtype in (("ids", "i64"), ("positions", "i32"), ("slots", "i64"), ("ancestors", "i64"), ("offsets", "i32"), ("lens", "i32"), ("counts", "i32"), ("tables", "i32"),
                        ("kept", "i32")):
        size = {"i32": 4, "i64": 8}[dtype]
        room = model.ctx.room[model.buf[name]] // size
        assert model._send(name, np.zeros(room), dtype).shape() == (room,)
        with pytest.raises(ValueError):
            model._send(name, np.zeros(room + 1), dtype)
