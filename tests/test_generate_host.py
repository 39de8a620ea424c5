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


def state(model, seqs):
    return [s.tokens for s in seqs], [list(s.pages) for s in seqs], model.cache.free_pages(), model.ctx.copies


def test_a_refused_call_changes_nothing(model):
    a, b, c, d = seqs = [model.sequence() for _ in range(4)]
    model.prefill([a, b], [np.arange(20), np.arange(5)])
    for _ in range(3):
        model.prefill([b], [np.arange(30)])  # 95 tokens of 100
    before = state(model, seqs)
    one = [0]
    refused = [
        lambda: model.prefill([a, c], [np.arange(20), np.arange(13)]),        # 33 tokens, room for 32
        lambda: model.prefill([a, b], [one, np.arange(6)]),                   # position 100 of 100
        lambda: model.prefill(seqs, [one] * 4),                               # four sequences, room for three
        lambda: model.prefill([a, c], [one]),                                 # a prompt is missing
        lambda: model.prefill([a, a], [one, one]),                            # named twice
        lambda: model.step([a, c], [[0] * 16, [0] * 17]),
        lambda: model.step([a, b], [one, [0] * 6]),
        lambda: model.step([b], [[0] * 18], [[-1] * 18]),                     # few positions, but 113 tokens in pages for 112
        lambda: model.step(seqs, [one] * 4),
        lambda: model.step([a, c], [one]),
        lambda: model.step([a, a], [one, one]),
        lambda: model.step([a], [[0, 0]], [[0, 0]]),                          # its own parent
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
        assert state(model, seqs) == before, i
    model.step([b], [[0] * 17], [[-1] * 17])


def test_no_more_drafts_than_a_word_has_bits():
    from warpforge_b200.generate import Decoder, DecoderSpec
    from warpforge_b200.quant import QuantizationType

    m = Decoder(HostContext(), DecoderSpec(QuantizationType.Q8_0, 64, 2, 1, 32, 64, 1, 64, max_positions=100), pages=12, page_tokens=16, max_tokens=99)
    s = m.sequence()
    with pytest.raises(ValueError):
        m.step([s], [[0] * 65])
    assert s.tokens == 0 and m.cache.free_pages() == 12
    m.step([s], [[0] * 64])
    m.close()


def test_a_call_that_fails_leaves_the_sequences_as_long_as_they_were(model):
    a, b = model.sequence(), model.sequence()
    model.prefill([a, b], [np.arange(17), np.arange(3)])
    full = model.sequence()
    full.extend(16 * (model.cache.free_pages() - 1))
    before = state(model, [a, b])
    for call in (lambda: model.prefill([a, b], [np.arange(16), np.arange(14)]), lambda: model.step([a, b], [[0] * 16, [0] * 14])):
        with pytest.raises(N.WfError):  # one page is left, and each wants one
            call()
        assert state(model, [a, b]) == before

    def fails(stream=0):
        raise N.WfError("wf_stream_sync", N.WF_ERR_INDEX, "WF_ERR_INDEX")

    model.ctx.synchronize = fails
    for call in (lambda: model.prefill([a, b], [np.arange(15), [0]]), lambda: model.step([a, b], [[0] * 15, [0]])):
        with pytest.raises(N.WfError):
            call()
        assert state(model, [a, b])[:3] == before[:3]


def test_what_is_kept_has_been_drafted(model):
    a, b = model.sequence(), model.sequence()
    model.prefill([a, b], [np.arange(10), np.arange(3)])
    model.step([a, b], [[0] * 5, [0] * 5])
    before = state(model, [a, b])
    for drafted, kept in (([5, 5], [[0, 5], [0]]), ([5, 5], [[0], [-1]]), ([5, 5], [[2, 1], [0]]), ([5, 5], [[1, 1], [0]]), ([16, 5], [[15], [0]]), ([-1, 5], [[], [0]]),
                          ([5, 5], [[0]]), ([5], [[0]]), ([5, 5], [[0], [0], [0]])):
        with pytest.raises(ValueError):
            model.keep([a, b], drafted, kept)
        assert state(model, [a, b]) == before, (drafted, kept)
    with pytest.raises(ValueError):
        model.keep([a, a], [5, 5], [[0], [0]])
    assert state(model, [a, b]) == before
    model.keep([a, b], [5, 5], [[0, 2, 4], []])
    assert (a.tokens, b.tokens) == (13, 3)


def test_drafts_that_are_kept_do_not_move_in_shared_pages(model):
    """A fork between step and keep shares the pages of the drafts; keep moves tokens in them."""
    a, other = model.sequence(), model.sequence()
    model.prefill([a], [np.arange(10)])
    model.step([a], [[0] * 30], [[-1] * 30])
    fork = a.fork()
    shared = list(a.pages[:2])
    assert [model.cache.holders(p) for p in shared] == [2, 2]
    model.keep([a], [30], [list(range(20))])  # as they lie: nothing moves
    assert a.pages[:2] == shared and fork.pages[:2] == shared
    a.free()
    a = fork.fork()
    sent = {}
    model.cache.compact = lambda tables, lens, kept, counts: sent.update(pages=list(a.pages))
    model.keep([a], [30], [[0, 1, 5, 9]])  # rows 12 and 13 of page 0
    assert sent["pages"][0] == a.pages[0] != fork.pages[0] and fork.pages[:2] == shared
    assert a.tokens == 14 and model.cache.holders(a.pages[0]) == 1
