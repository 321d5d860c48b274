"""Calls of the page operators and of attention that their documentation allows
beside the ordinary ones: with another call's error pending, with arguments
that are dropped while another stream still has to read them, that are the state's
own arrays, or that only the device can refuse."""
import numpy as np
import pytest
import torch

from demo_b200 import cache as cc
from demo_b200 import pages as pg
from demo_b200._lib import KVPAGE_ANY_DEVICE, lib
from demo_b200.attention import TreeAttention
from oracle import attention as oa
from oracle import pages_model as pm
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


class Dropped:
    """Calls on a side stream that is still busy; the arguments are dropped when
    the call returns, and the current stream takes and fills what memory it can
    get in their sizes."""

    def __init__(self):
        self.side = torch.cuda.Stream()

    def __call__(self, call, *arguments):
        given = [t.clone() for t in arguments]
        others = [torch.full_like(t, 1) for t in given]
        sizes = [(t.shape, t.dtype) for t in given]
        self.side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(self.side):
            torch.cuda._sleep(100_000_000)
        result = call(*given, stream=self.side)
        del given
        taken = [torch.empty(shape, dtype=dt, device="cuda") for shape, dt in sizes for _ in range(2)]
        for t, o in zip(taken[::2] + taken[1::2], others * 2):
            t.copy_(o)
        torch.cuda.synchronize()
        return result


def test_page_calls_whose_arguments_are_dropped():
    c = Case(GEOMETRIES["mixed"], 60, 8, 6)
    m, drop = c.model, Dropped()
    assert drop(c.pool.resize, ints([0, 5, 3]), ints([41, 17, 30])).tolist() == m.resize([0, 5, 3], [41, 17, 30])
    c.same()
    assert drop(c.pool.fork, ints([0, 3]), ints([2, 6])).tolist() == m.fork([0, 3], [2, 6])
    c.same()
    got = drop(c.pool.compact, ints([5, 2]), ints([3, 40]), ints([5, 9, 16, 40]), ints([0, 3, 4]))
    assert got.tolist() == m.compact([5, 2], [3, 40], [5, 9, 16, 40], [0, 3, 4])
    c.same()
    drop(c.pool.copy, ints([0, 2, 7]), ints([50, 51, 52]), ints([8, 3, 5]))
    m.copy([0, 2, 7], [50, 51, 52], [8, 3, 5])
    c.same()


def test_attention_whose_arguments_are_dropped():
    b = Batch([300, 40, 77], [3, 2, 5], seed=31).tree(31)
    args, parents = b.args()
    att = b.attention()
    want = att(*args, parents=parents)
    call = lambda *a, stream: att(0, *a[:4], parents=a[4], rows=a[5], stream=stream)
    assert torch.equal(Dropped()(call, *args[1:], parents, ints([0, 1, 2])), want)
    att.check()


@pytest.mark.parametrize("n", [2, 700, 4096])
def test_lengths_taken_from_the_state_itself(n):
    """rows exchange their lengths: row n - 1 - i gets what row i had"""
    c = Case(("nhd", 1, 1, 8, torch.int16, 4), 6 * n, n, 5)
    rng = np.random.default_rng(n)
    resize(c, list(range(n)), rng.integers(0, 21, n).tolist())
    rows = list(range(n))[::-1]
    assert c.pool.resize(ints(rows), c.pool.seq_lens).tolist() == c.model.resize(rows, c.model.lens.tolist())
    c.same()


def test_lists_taken_from_the_state_itself():
    """children named by the table, a start that is the lengths"""
    c = Case(GEOMETRIES["mixed"], 30, 4, 6)
    resize(c, [0, 1], [8 * 3 + 1, 8])
    table = c.pool.block_table                              # pages 0, 1, 2, 3 and 4
    assert c.model.table[0, :4].tolist() == [0, 1, 2, 3]
    assert c.pool.fork(table[0, :2], table[0, 2:4]).tolist() == c.model.fork([0, 1], [2, 3])
    c.same()
    lens = c.pool.seq_lens
    got = c.pool.compact(ints([0, 1, 2, 3]), lens, ints([]), ints([0] * 5))     # nothing dropped, nothing kept behind
    assert got.tolist() == c.model.compact([0, 1, 2, 3], c.model.lens.tolist(), [], [0] * 5)
    c.same()


def test_every_refused_length_sets_a_bit():
    for length in (-1, -2 ** 31, 6 * 8 + 1, 2 ** 31 - 1):
        c = Case(GEOMETRIES["mixed"], 40, 6, 6)
        resize(c, [0, 1], [20, length])
        c.same(pm.ERR_ROW)
        with pytest.raises(ValueError, match="length"):
            c.pool.check()


def test_planes_that_no_kernel_may_follow_are_refused():
    pageable = torch.zeros(2, 4, 16, 2, 64, dtype=torch.bfloat16)
    pinned, device = pageable.pin_memory(), pageable.cuda()
    assert [lib.kv_page_device_of(t.data_ptr()) for t in (pageable, pinned, device)] == [-22, KVPAGE_ANY_DEVICE, 0]
    layout, k, v = cc.layout_from_kv_tensors([pageable], kv_layout="flash_attn")
    table = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="not memory that a GPU reaches"):
        pg.PagePool(layout, k, v, table, ints([0]))
    att = TreeAttention(layout, k, v, 4, 2)
    with pytest.raises(ValueError, match="not memory that a GPU reaches"):
        att(0, torch.zeros(1, 4, 64, dtype=torch.bfloat16, device="cuda"), table, ints([1]), ints([0, 1]))


def test_a_cache_in_pinned_memory():
    t = torch.randint(-9, 9, (2, 6, 4, 1, 8), dtype=torch.int16).pin_memory()
    layout, k, v = cc.layout_from_kv_tensors([t], kv_layout="flash_attn")
    pool = pg.PagePool(layout, k, v, ints([-1] * 4).view(1, 4), ints([0]))
    want = t.clone()
    want[:, 5] = want[:, 2]
    pool.copy(ints([2]), ints([5]))
    pool.check()
    assert torch.equal(t, want)


def test_a_cache_of_bytes_whose_type_is_said():
    b = Batch([90, 40], [3, 1], seed=32, kvt=torch.float8_e4m3fn)
    args, _ = b.args()
    want = b.attention()(*args)
    layout, k, v = cc.layout_from_kv_tensors([t.view(torch.uint8) for t in b.store], kv_layout="flash_attn")
    assert (k, v) == (b.k, b.v)
    att = TreeAttention(layout, k, v, b.heads, b.kv_heads, k_scale=b.scales[0], v_scale=b.scales[1], kv_dtype=torch.float8_e4m3fn)
    assert torch.equal(att(*args), want)


def test_a_pool_of_free_pages_refuses_rows_that_hold_some():
    store = torch.zeros(2, 8, 4, 1, 8, dtype=torch.int16, device="cuda")
    layout, k, v = cc.layout_from_kv_tensors([store], kv_layout="flash_attn")
    table = torch.full((3, 2), -1, dtype=torch.int32, device="cuda")
    for lens in ([0, 5, 0], [0, 0, -1]):
        with pytest.raises(ValueError, match="needs empty rows"):
            pg.PagePool(layout, k, v, table, ints(lens))
    table[1] = ints([3, 4])
    pool = pg.PagePool(layout, k, v, table, ints([0, 5, 0]), refs=ints([0, 0, 0, 1, 1, 0, 0, 0]), free_list=ints([7, 6, 5, 2, 1, 0, 0, 0]),
                       free_count=ints([6]))            # with the state that they belong to they are taken
    assert pool.resize(ints([1]), ints([0])).tolist() == [pg.OK]
    pool.check()
    assert pool.free_list.tolist() == [7, 6, 5, 2, 1, 0, 3, 4]


def held_and_free(c):
    """every page that a row holds, or that is free, once per holder"""
    m = c.model
    held = [int(p) for r in range(m.rows) for p in m.table[r, :m._npages(m.lens[r])] if 0 <= p < m.pages]
    assert not set(held) & set(m.free) and [held.count(p) for p in range(m.pages)] == m.refs.tolist()


@pytest.mark.parametrize("where", ["full", "tail", "last_full"])
@pytest.mark.parametrize("page", [-1, 60, 2 ** 31 - 1])
def test_children_of_a_row_with_a_bad_page_stay_empty(where, page):
    """the other children get their pages as if it had not been named"""
    c = Case(GEOMETRIES["mixed"], 60, 12, 6)
    resize(c, [0, 1, 2], [8 * 4 + 3, 8 * 5, 8 * 2 + 7])
    r, k = {"full": (0, 1), "tail": (0, 4), "last_full": (1, 4)}[where]
    was = int(c.model.table[r, k])
    c.pool.block_table[r, k] = page
    c.model.table[r, k] = page
    fork(c, [2, 0, 1, 2, 0, 1], [3, 4, 5, 6, 7, 8])
    c.same(pm.ERR_PAGE)
    c.model.table[r, k] = was
    held_and_free(c)
    assert (c.model.lens[[4, 7]] == 0).all() == (r == 0) and (c.model.lens[[5, 8]] == 0).all() == (r == 1)


def test_many_children_of_rows_with_bad_pages():
    """more children than the plan has warps"""
    c = Case(("nhd", 1, 1, 8, torch.int16, 16), 4000, 700, 40)
    rng = np.random.default_rng(4)
    resize(c, list(range(20)), rng.integers(1, 40 * 16, 20).tolist())
    was = c.model.table.copy()
    for r in (3, 11, 12):
        k = int(rng.integers(0, -(-int(c.model.lens[r]) // 16)))
        c.pool.block_table[r, k] = -5
        c.model.table[r, k] = -5
    fork(c, rng.integers(0, 20, 680).tolist(), rng.permutation(np.arange(20, 700)).tolist())
    c.same(pm.ERR_PAGE)
    c.model.table[:20] = was[:20]
    held_and_free(c)


def test_ids_of_the_free_list_that_are_no_pages():
    """fork refuses the child, resize hands them out as they stand"""
    c = Case(GEOMETRIES["mixed"], 60, 12, 6)
    resize(c, [0], [8 * 2 + 3])
    for at, bad in ((-2, 99), (-5, -1)):
        c.model.free[at] = bad
        c.pool.free_list[int(c.pool.free_count) + at] = bad
    fork(c, [0, 0, 0], [1, 2, 3])
    c.same(pm.ERR_PAGE)
    held_and_free(c)
    assert c.model.lens[:4].tolist() == [19, 19, 0, 19]
    c.model.error = 0
    with pytest.raises(ValueError, match="page id"):
        c.pool.check()
    resize(c, [4, 5], [8, 17])
    c.same(pm.ERR_PAGE)
    assert c.model.table[5, 0] == -1
    resize(c, [4, 5], [0, 0])
    c.same(pm.ERR_PAGE)
    held_and_free(c)


@pytest.mark.parametrize("base", ["null", "misaligned"])
def test_compact_with_a_bad_base_leaves_its_rows_alone(base):
    """the bytes that could not be moved in one plane are not given up in the others"""
    c = Case(GEOMETRIES["mixed"], 40, 4, 6)
    resize(c, [0, 1], [20, 30])
    k = c.pool._k.clone()
    c.pool._k[1] = 0 if base == "null" else int(k[1]) + 8
    got = c.pool.compact(ints([0, 1]), ints([3, 0]), ints([9, 17, 2]), ints([0, 2, 3]))
    assert got.tolist() == [pg.INVALID] * 2
    c.model.error = 16
    c.same(16)
    with pytest.raises(ValueError, match="layer base"):
        c.pool.check()
    c.model.error = 0
    c.pool._k.copy_(k)
    compact(c, [0, 1], [3, 0], [[9, 17], [2]])
    c.same()


@pytest.mark.parametrize("value", [float("nan"), float("inf")], ids=str)
@pytest.mark.parametrize("n", [40, 6000])
def test_scores_of_minus_infinity_over_values_that_are_not_finite(n, value):
    """are nothing seen all the same: 0 with lse -inf, joined from pieces or not"""
    b = Batch([n, 30], [1, 1], heads=2, kv_heads=1, dim=64, seed=33)
    b.q[0] = 1
    held = torch.tensor(b.table[0, :-(-n // 16)].astype(np.int64)).cuda()
    b.view[0, 0, held] = -float("inf")
    b.view[0, 1, held] = value
    args, _ = b.args()
    out, lse = b.attention()(*args, return_lse=True)
    assert not out[0].any() and (lse[0] == -float("inf")).all()
    want = oa.attention(b.q[1:], *(b.view[0, i].double() for i in range(2)), b.table.tolist(), b.lens, [0, 1], rows=[1])
    close(out[1:], lse[1:], want)
