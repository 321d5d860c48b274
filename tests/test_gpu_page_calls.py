"""Calls of the page operators and of attention that their documentation allows
beside the ordinary ones: with another call's error pending."""
import numpy as np
import pytest
import torch

from demo_b200 import pages as pg
from demo_b200._lib import lib
from tests.test_gpu_attention import Batch, close
from tests.test_gpu_pages import GEOMETRIES, Case, compact, fork, ints, resize

pytestmark = pytest.mark.gpu


@pytest.fixture
def pending_error():
    """leaves an error of the CUDA runtime on this thread: 2^50 bytes are asked
    for, which the host refuses"""
    ad = lib.cuda_adaptor_create()
    assert ad
    byte = np.zeros(1, np.uint8)

    def leave():
        assert not lib.wrapper_ptr(ad, 0, byte.ctypes.data, 1 << 50)

    yield leave
    lib.cuda_adaptor_destroy(ad)


def test_page_calls_with_an_error_of_another_call_pending(pending_error):
    """both kernels of a call run: tables, lengths and bytes belong together"""
    c = Case(GEOMETRIES["mixed"], 40, 6, 6)
    pending_error()
    resize(c, [0, 1], [20, 30])
    c.same()
    pending_error()
    fork(c, [0, 1], [2, 3])
    c.same()
    pending_error()
    compact(c, [2], [16], [[17, 19]])
    c.same()
    pending_error()
    c.pool.copy(ints([1]), ints([39]))
    c.model.copy([1], [39])
    c.same()


def test_attention_with_an_error_of_another_call_pending(pending_error):
    b = Batch([6000, 17], [1, 1], seed=30)       # rows that the second kernel joins
    args, _ = b.args()
    att = b.attention()
    att(*args)                      # loads the kernels
    pending_error()
    out, lse = att(*args, return_lse=True)
    att.check()
    close(out, lse, b.expected())


def test_a_device_that_is_not_there_leaves_no_error_behind():
    c = Case(GEOMETRIES["mixed"], 40, 6, 6)
    c.pool._state.device = 63
    with pytest.raises(pg.CacheError):
        c.pool.resize(ints([0]), ints([8]))
    c.pool._state.device = 0
    resize(c, [0], [20])
    fork(c, [0], [1])
    c.same()
