"""The page state as the host keeps it (batch.Pages): over the page calls restated
on the CPU (oracle/batch_oracle.py), and over the package's on the GPU."""

import numpy as np
import pytest

from lama32_mojo_amd import batch, q8hip
from oracle import batch_oracle as bo

I4 = np.dtype(np.int32).itemsize


class Memory:
    """A buffer in host memory."""

    def __init__(self, nbytes):
        self.data = np.zeros(nbytes, np.uint8)

    @classmethod
    def alloc(cls, ctx, nbytes):
        return cls(nbytes)

    def upload(self, arr, off=0):
        raw = np.ascontiguousarray(arr).view(np.uint8).reshape(-1)
        self.data[off:off + raw.size] = raw

    def download(self, shape, dtype, off=0):
        n = int(np.prod(shape)) * np.dtype(dtype).itemsize
        return self.data[off:off + n].copy().view(dtype).reshape(shape)

    def free(self):
        pass


class Calls:
    """The page calls on host memory."""

    def __init__(self):
        self.o = None

    def run(self, ix, otab, olen, oheld, oref, nslots, maxpages, npages, page, step):
        o = bo.Pages(nslots, maxpages, npages, page)
        table = ix.download((nslots, maxpages), np.int32, I4 * otab)
        held = ix.download((nslots,), np.int32, I4 * oheld)
        o.rows = [table[s, :held[s]].tolist() for s in range(nslots)]
        if olen is not None:
            o.len = ix.download((nslots,), np.int32, I4 * olen).tolist()
        assert o.refs() == ix.download((npages,), np.int32, I4 * oref).tolist()
        step(o)
        for name, off in (("table", otab), ("len", olen), ("held", oheld), ("ref", oref)):
            if off is not None:
                ix.upload(o.arrays()[name], I4 * off)

    def reserve(self, ctx, ix, otab, olen, oheld, oref, owant, nslots, maxpages, npages, page, *pool):
        want = ix.download((nslots,), np.int32, I4 * owant).tolist()
        self.run(ix, otab, olen, oheld, oref, nslots, maxpages, npages, page, lambda o: o.reserve(want))

    def set_len(self, ctx, ix, otab, olen, oheld, oref, onew, nslots, maxpages, npages, page):
        new = ix.download((nslots,), np.int32, I4 * onew).tolist()
        self.run(ix, otab, olen, oheld, oref, nslots, maxpages, npages, page, lambda o: o.set_len(new))

    def fork(self, ctx, ix, otab, olen, oheld, oref, osource, nslots, maxpages, npages):
        source = ix.download((nslots,), np.int32, I4 * osource).tolist()
        self.run(ix, otab, olen, oheld, oref, nslots, maxpages, npages, 1, lambda o: o.fork(source))


@pytest.fixture(params=["host", pytest.param("gpu", marks=pytest.mark.gpu)])
def pages(request, monkeypatch):
    """Pages(slots, npages, maxpages) of 16 tokens."""
    ctx, made = None, []
    if request.param == "host":
        calls = Calls()
        monkeypatch.setattr(batch, "Buffer", Memory)
        for name in ("reserve", "set_len", "fork"):
            monkeypatch.setattr(q8hip, "pages_" + name, getattr(calls, name))
    else:
        ctx = request.getfixturevalue("ctx")

    def make(slots, npages, maxpages):
        made.append(batch.Pages(ctx, slots, npages, maxpages, 16, 1, 1, 64))
        return made[-1]
    yield make
    for p in made:
        p.close()


def state(p):
    """table, lengths, held pages and counts."""
    return tuple(p.ix.download(shape, np.int32, I4 * p.at[name]).tolist() for name, shape in (
        ("table", (p.slots, p.maxpages)), ("len", (p.slots,)), ("held", (p.slots,)), ("ref", (p.npages,))))


def test_fork_of_reserved_pages(pages):
    """Two slots without tokens that share pages held ahead: either may grow only
    with a page of its own, whatever other slots do before."""
    p = pages(3, 4, 2)
    p.reserve([32, 0, 20])
    p.set_len([-1, -1, 20])
    p.fork([-1, 0, -1])
    assert state(p)[0][:2] == [[0, 1]] * 2
    p.set_len([-1, -1, 19])                                   # another slot's length
    with pytest.raises(RuntimeError, match="pages full"):
        p.reserve([10, 0, 19])
    assert p.length == [0, 0, 19]


def test_refusal_leaves_the_state(pages):
    """A refused reservation leaves what was there, pages held ahead and shared ones
    among them: what an earlier reservation promised is still there."""
    p = pages(3, 6, 5)
    p.reserve([40, 0, 20])
    p.set_len([-1, -1, 20])                                   # slot 0 holds 3 pages ahead
    before = state(p)
    for want in ([40, 32, 20], [70, 0, 64], [40, 0, 1000]):
        with pytest.raises(RuntimeError, match="pages full"):
            p.reserve(want)
        assert state(p) == before and p.length == [0, 0, 20]
    p.fork([-1, 0, -1])
    before = state(p)
    with pytest.raises(RuntimeError, match="pages full"):
        p.reserve([40, 40, 20])                               # each sharer lacks three
    assert state(p) == before
    p.set_len([0, -1, -1])                                    # slot 1 has them alone
    p.reserve([0, 48, 20])
    assert state(p)[0][1][:3] == before[0][0][:3]
    # nothing held ahead: the pages that slots got before the refused one are free again
    q = pages(3, 4, 4)
    q.reserve([16, 16, 0])
    q.set_len([16, 16, 0])
    before = state(q)
    with pytest.raises(RuntimeError, match="pages full"):
        q.reserve([32, 16, 64])
    assert state(q) == before
    # a copy of a shared page is given back too
    q = pages(3, 3, 2)
    q.reserve([10, 0, 0])
    q.set_len([10, 0, 0])
    q.fork([-1, 0, -1])
    before = state(q)
    with pytest.raises(RuntimeError, match="pages full"):
        q.reserve([11, 10, 32])
    assert state(q) == before
    q.reserve([10, 10, 32])
    assert state(q)[3] == [2, 1, 1]


def test_length_past_the_held_pages(pages):
    """A length that the slot's pages do not hold is refused: the host's lengths stay
    those of the device."""
    p = pages(3, 6, 4)
    p.reserve([20, 0, 64])
    p.set_len([20, -1, -1])
    before = state(p)
    for new in ([33, -1, -1], [-1, 1, -1], [20, 0, 65]):
        with pytest.raises(ValueError, match="set_len"):
            p.set_len(new)
        assert state(p) == before and p.length == before[1] == [20, 0, 0]
    p.set_len([32, -1, 50])
    p.fork([-1, 2, -1])
    with pytest.raises(ValueError, match="set_len"):
        p.set_len([-1, 65, -1])
    p.set_len([-1, 64, 0])
    assert p.length == state(p)[1] == [32, 64, 0]


def test_one_value_per_slot(pages):
    """Lists of another length than the slots (whose rest would be that of an earlier
    call) are refused."""
    p = pages(3, 6, 4)
    p.reserve([20, 20, 20])
    p.set_len([20, 20, 20])
    before = state(p)
    for call in (p.reserve, p.set_len, p.fork):
        for values in ([16], [1] * 4, []):
            with pytest.raises(ValueError, match="slot"):
                call(values)
            assert state(p) == before and p.length == [20, 20, 20]
