"""Calls of Q8Batch that are refused leave it as it was: slots' adapters, lengths, pages.
(No model and no device: the state and the calls it reaches are stand-ins.)"""

import numpy as np
import pytest

from lama32_mojo_amd import batch
from lama32_mojo_amd.batch import Q8Batch, Sampling
from lama32_mojo_amd.q8hip import Q8_ERR_HIP, Q8Error


class Touched(Exception):
    """A call went on to the device."""


class NoDevice:
    length = [3, 4, 0]
    forked = set()

    def fork(self, source):
        raise Q8Error(Q8_ERR_HIP, "refused")

    def reserve(self, want):
        raise Touched


def a_batch():
    b = object.__new__(Q8Batch)
    b.slots, b.max_rows, b.adapters, b.share, b.adapter = 3, 8, None, False, [-1] * 3
    b.pages = NoDevice()

    class m:
        class cfg:
            hidden, vocab = 64, 50
    b.m = m
    return b


def test_fork():
    b = a_batch()
    b.adapter = [0, 1, -1]
    with pytest.raises(Q8Error):
        b.fork({2: 0, 1: 0})
    assert b.adapter == [0, 1, -1]
    taken = []
    b.pages.fork = taken.append
    b.fork({2: 0, 0: 1})
    assert b.adapter == [1, 1, 0] and taken == [[1, -1, 0]]


@pytest.mark.parametrize("how,u", [(Sampling(top_k=1 << 31), 0.5), (Sampling(top_k=-(1 << 31) - 1), 0.5),
                                   (Sampling(top_k=[3, 4]), 0.5), (Sampling(temperature="warm"), 0.5),
                                   (Sampling(min_p=[1]), 0.5), (Sampling(), "x"), (Sampling(), [0.5, 0.5])])
def test_settings(how, u):
    """Settings that q8_sample cannot take are refused before pages are taken."""
    b = a_batch()
    with pytest.raises((ValueError, TypeError, OverflowError)):
        b.forward({0: [1], 1: [2]}, sample={0: how}, u=[0.5, u])


def test_settings_that_pass():
    for how in (Sampling(), Sampling(0, np.int32(7), np.float32(0.5)), Sampling(float("nan")), Sampling(1, -5),
                Sampling(top_k=(1 << 31) - 1)):
        with pytest.raises(Touched):
            a_batch().forward({0: [1], 1: [2]}, sample={0: how}, u=np.array([0.5, 0.25]))
        with pytest.raises(Touched):
            a_batch().forward({0: [1, 2], 1: [2]}, every=True, sample={1: how}, u=(0.5, 0, 1))
