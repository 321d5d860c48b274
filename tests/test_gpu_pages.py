"""The page operators on the device against oracle/pages_model.py: tables,
reference counts, the free stack's order and every byte of the cache."""
import numpy as np
import pytest
import torch

from demo_b200 import cache as cc
from demo_b200 import pages as pg
from oracle import pages_model as pm

pytestmark = pytest.mark.gpu

# (order, layers, heads, head_dim, element type, block)
GEOMETRIES = {
    "nhd": ("nhd", 2, 8, 128, torch.int16, 16),
    "hnd": ("hnd", 3, 8, 128, torch.int16, 16),
    "mixed": ("mixed", 2, 4, 64, torch.int16, 8),        # K and V of a block side by side, token-major
    "k_only": ("k", 3, 1, 576, torch.int16, 64),
    "bytes": ("hnd", 2, 3, 5, torch.uint8, 7),           # 5-byte heads: single-byte vectors
    "pairs": ("nhd", 1, 3, 10, torch.uint8, 24),         # 30-byte units: 2-byte vectors
    "prime": ("nhd", 2, 1, 8 * 37, torch.int16, 1),      # 37 vectors a token, one token a page
}


def make_cache(geometry, num_pages, seed=0):
    """(storage, view [planes, pages, block, heads, dim], tensors for layout_from_kv_tensors, kv_layout)"""
    order, L, H, D, dt, bs = geometry
    g = torch.Generator(device="cuda").manual_seed(seed)
    lo, hi = (0, 256) if dt == torch.uint8 else (-30000, 30000)
    shape = {"nhd": (L, 2, num_pages, bs, H, D), "hnd": (L, num_pages, 2, H, bs, D), "mixed": (L, num_pages, 2, bs, H, D),
             "k": (L, num_pages, bs, D)}[order]
    c = torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=dt)
    if order == "nhd":
        return c, c.reshape(L * 2, num_pages, bs, H, D), list(c), "flash_attn"
    if order == "hnd":
        t = c.permute(0, 1, 2, 4, 3, 5)
        return c, t.permute(0, 2, 1, 3, 4, 5), list(t), "flashinfer"
    if order == "mixed":
        return c, c.permute(0, 2, 1, 3, 4, 5), list(c), "flashinfer"
    return c, c[:, :, :, None], list(c), None


class Case:
    """A pool and its model with the same cache bytes."""

    def __init__(self, geometry, num_pages, rows, width, seed=0, pad=0):
        self.store, self.view, tensors, kvl = make_cache(geometry, num_pages, seed)
        layout, k, v = cc.layout_from_kv_tensors(tensors, kv_layout=kvl)
        table = torch.full((rows, width + pad), -1, dtype=torch.int32, device="cuda")[:, :width]
        self.pool = pg.PagePool(layout, k, v, table, torch.zeros(rows, dtype=torch.int32, device="cuda"))
        self.model = pm.Pages(rows, width, num_pages, geometry[5], self.bytes())

    def bytes(self):
        v = self.view.reshape(-1, *self.view.shape[-4:])        # [planes, pages, block, heads, dim], copied
        return v.contiguous().reshape(*v.shape[:3], -1).view(torch.uint8).cpu().numpy().copy()

    def same(self, error=0):
        p, m = self.pool, self.model
        torch.cuda.synchronize()
        assert p.block_table.cpu().numpy().tolist() == m.table.tolist()
        assert p.seq_lens.tolist() == m.lens.tolist()
        assert p.refs.tolist() == m.refs.tolist()
        n = int(p.free_count.item())
        assert p.free_list.tolist()[:n] == m.free
        assert not p._marks.any()
        assert np.array_equal(self.bytes(), m.cache)
        assert int(p.error.item()) == m.error == error


def ints(x):
    return torch.tensor(np.asarray(x, dtype=np.int32).reshape(-1), dtype=torch.int32, device="cuda")


def resize(c, rows, lens):
    assert c.pool.resize(ints(rows), ints(lens)).tolist() == c.model.resize(rows, lens)


def fork(c, parents, children):
    assert c.pool.fork(ints(parents), ints(children)).tolist() == c.model.fork(parents, children)


def compact(c, rows, start, keeps):
    flat = [x for k in keeps for x in k]
    off = np.cumsum([0] + [len(k) for k in keeps])
    got = c.pool.compact(ints(rows), ints(start), ints(flat), ints(off))
    assert got.tolist() == c.model.compact(rows, start, flat, off)


@pytest.mark.parametrize("name", GEOMETRIES)
def test_random_sequence_of_calls(name):
    """sixty calls in the order a random engine makes them"""
    geo = GEOMETRIES[name]
    bs = geo[5]
    rng = np.random.default_rng(sum(map(ord, name)))
    rows, width, num_pages = 13, 6, 50
    c = Case(geo, num_pages, rows, width, pad=3)
    for step in range(60):
        kind = rng.integers(0, 4)
        if kind == 0:
            n = int(rng.integers(1, rows + 1))
            resize(c, rng.permutation(rows)[:n].tolist(), rng.integers(0, width * bs + 1, n).tolist())
        elif kind == 1:
            empty = [r for r in range(rows) if c.model.lens[r] == 0]
            held = [r for r in range(rows) if c.model.lens[r] > 0]
            if empty and held:
                n = int(rng.integers(1, len(empty) + 1))
                fork(c, rng.choice(held, n).tolist(), rng.permutation(empty)[:n].tolist())
        elif kind == 2:
            n = int(rng.integers(1, num_pages // 2))
            ids = rng.permutation(num_pages)
            tok = None if rng.random() < 0.3 else rng.integers(-1, bs + 2, n).tolist()
            c.pool.copy(ints(ids[:n]), ints(ids[n:2 * n]), ints(tok) if tok is not None else None)
            c.model.copy(ids[:n].tolist(), ids[n:2 * n].tolist(), tok)
        else:
            rs, st, ks, error = [], [], [], c.model.error
            for r in rng.permutation(rows):
                L = int(c.model.lens[r])
                s = int(rng.integers(0, L + 1))
                shared = any(c.model.refs[p] != 1 for p in c.model.table[r, s // bs:-(-L // bs)])
                if shared:
                    continue
                rs.append(int(r))
                st.append(s)
                ks.append((s + np.flatnonzero(rng.random(L - s) < rng.choice([0.1, 0.6, 1.0]))).tolist())
            if rs:
                compact(c, rs, st, ks)
        c.same()


def test_resize_many_rows_and_shared_pages():
    """more rows than a CTA's warps; pages shared by many rows, dropped in one
    call: pushed once, where the last of them stands"""
    bs, width = 16, 40
    c = Case(("nhd", 1, 1, 8, torch.int16, bs), 4000, 300, width)
    resize(c, [0, 1], [33 * bs, 17 * bs + 5])
    fork(c, [i % 2 for i in range(200)], list(range(2, 202)))
    c.same()
    resize(c, list(range(202, 300)), [(7 * i) % (width * bs) for i in range(98)])
    c.same()
    order = np.random.default_rng(3).permutation(300).tolist()
    resize(c, order, [0 if i % 3 else 5 * bs for i in range(300)])
    c.same()
    resize(c, order[::-1], [0] * 300)
    c.same()
    assert int(c.pool.free_count.item()) == 4000 and not c.pool.refs.any()


def test_resize_gives_pages_back_before_it_takes():
    c = Case(GEOMETRIES["mixed"], 6, 3, 6)
    resize(c, [0], [6 * 8])
    resize(c, [1, 0], [5 * 8, 1])               # row 1 gets what row 0 gives back
    c.same()
    resize(c, [2, 0, 1], [8, 17, 40])           # one page too few for row 2, row 0 stands behind it
    c.same()


@pytest.mark.parametrize("n", [1, 31, 33, 1025, 4096])
def test_resize_sizes(n):
    c = Case(("nhd", 1, 1, 8, torch.int16, 4), 3 * n + 7, n, 5)
    rng = np.random.default_rng(n)
    for _ in range(3):
        resize(c, rng.permutation(n).tolist(), rng.integers(0, 21, n).tolist())
    c.same()


def test_calls_of_nothing():
    c = Case(GEOMETRIES["nhd"], 8, 2, 4)
    empty = ints([])
    assert c.pool.resize(empty, empty).numel() == 0
    assert c.pool.fork(empty, empty).numel() == 0
    c.pool.copy(empty, empty)
    assert c.pool.compact(empty, empty, empty, ints([0])).numel() == 0
    c.same()
    compact(c, [0, 1], [0, 0], [[], []])        # empty rows, nothing kept
    fork(c, [0], [1])                           # a child of an empty row
    c.same()


@pytest.mark.parametrize("name", ["nhd", "hnd", "k_only"])
def test_compact_long_lists(name):
    """lists of many batches, overlapping source and destination pages"""
    geo = GEOMETRIES[name]
    bs = geo[5]
    width = -(-3001 // bs)
    c = Case(geo, 3 * width + 2, 3, width)
    resize(c, [0, 1, 2], [3001, 1700, 2])
    rng = np.random.default_rng(5)
    compact(c, [2, 0, 1], [1, 3, 900], [[1], (3 + np.flatnonzero(rng.random(2998) < 0.5)).tolist(), [1699]])
    c.same()
    compact(c, [0], [0], [list(range(1, int(c.model.lens[0])))])        # every token one up
    c.same()


def test_errors_leave_the_other_rows_right():
    bs = 8
    c = Case(GEOMETRIES["mixed"], 40, 6, 6)
    resize(c, [0, 1, 2], [20, 30, 11])
    # twice, out of range, too long, negative; row 2 is served
    resize(c, [0, 0, 6, -1, 1, 2, 3], [1, 2, 3, 4, 6 * bs + 1, 12, -5])
    c.same(pm.ERR_ROW)
    # children: not empty, twice, also a parent, out of range; row 5 is served
    fork(c, [0, 0, 0, 4, 1, 2, 0], [1, 3, 3, 3, 4, 5, 99])
    c.same(pm.ERR_ROW)
    c.model.error = 0
    with pytest.raises(ValueError, match="named twice"):
        c.pool.check()
    c.pool.check()
    c.same()
    # not ascending, behind the end, before start, offsets out of order; row 5 is served
    keep, off = [3, 3, 30, 1, 5, 6], [0, 2, 3, 4, 6, 5]
    got = c.pool.compact(ints([0, 1, 2, 5, 3]), ints([0, 0, 2, 5, 0]), ints(keep), ints(off))
    assert got.tolist() == c.model.compact([0, 1, 2, 5, 3], [0, 0, 2, 5, 0], keep, off)
    c.same(pm.ERR_KEEP)
    c.model.error = 0
    with pytest.raises(ValueError, match="ascending"):
        c.pool.check()
    compact(c, [0, 0, 9], [0, 0, 0], [[1], [1], [0]])
    c.same(pm.ERR_ROW)


def test_compact_refuses_shared_destinations():
    bs = 8
    c = Case(GEOMETRIES["mixed"], 40, 4, 6)
    resize(c, [0], [20])
    fork(c, [0], [1])
    compact(c, [0, 1], [0, 16], [[1, 2], [18]])     # row 0's first page is row 1's too; row 1's last is its own
    c.same(pm.ERR_REFS)


def test_bad_pages_are_reported_and_skipped():
    c = Case(GEOMETRIES["mixed"], 10, 3, 4)
    c.pool.copy(ints([0, -1, 10, 3]), ints([1, 2, 4, 99]))
    c.model.copy([0, -1, 10, 3], [1, 2, 4, 99])
    c.same(pm.ERR_PAGE)
    c.model.error = 0
    c.pool.error.zero_()
    resize(c, [0], [20])
    c.pool.block_table[0, 1] = c.model.table[0, 1] = 77     # an engine's bug
    resize(c, [0], [0])
    c.same(pm.ERR_PAGE)


def test_a_page_freed_twice_is_pushed_once():
    c = Case(GEOMETRIES["mixed"], 10, 3, 4)
    resize(c, [0, 1], [20, 8])
    c.pool.block_table[1, 0] = c.model.table[1, 0] = int(c.model.table[0, 0])   # held by two rows, counted once
    resize(c, [1, 0], [0, 0])
    p = c.pool
    torch.cuda.synchronize()
    n = int(p.free_count.item())
    assert int(p.error.item()) == pm.ERR_REFS
    assert len(set(p.free_list.tolist()[:n])) == n and not (p.refs < 0).any()


def test_offsets_past_32_bits():
    """pages more than 4 GiB into a plane: 64 KiB pages of one K-only layer"""
    n, bs, w = 70000, 64, 512
    store = torch.zeros(n, bs, w, dtype=torch.int16, device="cuda")
    layout, k, v = cc.layout_from_kv_tensors([store])
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(n, dtype=torch.int32, device="cuda")             # the last pages first
    pool = pg.PagePool(layout, k, v, table, torch.zeros(3, dtype=torch.int32, device="cuda"),
                       refs=torch.zeros(n, dtype=torch.int32, device="cuda"), free_list=free,
                       free_count=torch.full((1,), n, dtype=torch.int32, device="cuda"))
    pool.resize(ints([0]), ints([100]))
    ids = table[0, :2].tolist()
    assert ids == [n - 1, n - 2]
    g = torch.Generator(device="cuda").manual_seed(1)
    store[ids] = torch.randint(-9, 9, (2, bs, w), generator=g, device="cuda", dtype=torch.int16)
    want = store[ids].reshape(-1, w)
    pool.fork(ints([0]), ints([1]))
    pool.copy(ints([n - 1]), ints([66000]))
    pool.compact(ints([1]), ints([64]), ints([70, 99]), ints([0, 2]))
    pool.check()
    assert torch.equal(store[66000], store[n - 1])
    got = store[table[1, :2].long()].reshape(-1, w)
    assert torch.equal(got[:66], torch.cat([want[:64], want[70:71], want[99:100]]))
    assert int(store[:60000].count_nonzero()) == 0


def test_captured_step_and_other_stream():
    """an engine step -- grow, fork, compact, free -- captured once and
    replayed, beside the same calls made eagerly on another stream"""
    def step(p, stream=None):
        p.resize(ints_d["rows"], ints_d["lens"], stream=stream)
        p.fork(ints_d["par"], ints_d["chi"], stream=stream)
        p.compact(ints_d["crow"], ints_d["start"], ints_d["keep"], ints_d["off"], stream=stream)
        p.resize(ints_d["chi"], ints_d["zero"], stream=stream)

    ints_d = {"rows": ints([0, 1]), "lens": ints([100, 37]), "par": ints([0, 1]), "chi": ints([3, 2]),
              "crow": ints([1]), "start": ints([33]), "keep": ints([34, 36]), "off": ints([0, 2]), "zero": ints([0, 0])}
    c = Case(GEOMETRIES["hnd"], 60, 4, 8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    step(c.pool, side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c.pool)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for _ in range(4):
        m = c.model
        m.resize([0, 1], [100, 37])
        m.fork([0, 1], [3, 2])
        m.compact([1], [33], [34, 36], [0, 2])
        m.resize([3, 2], [0, 0])
    c.same()


def test_same_results_every_time():
    out = []
    for _ in range(3):
        c = Case(("nhd", 1, 1, 8, torch.int16, 16), 3000, 128, 32)
        rows = ints(np.random.default_rng(1).permutation(128))
        for seed in range(4):
            c.pool.resize(rows, ints(np.random.default_rng(seed).integers(0, 512, 128)))
        out.append((c.pool.block_table.tolist(), c.pool.free_list.tolist()))
    assert out[0] == out[1] == out[2]


def test_misaligned_planes():
    """bases that only a narrower vector fits, and a base the layout hides"""
    raw = torch.randint(0, 256, (2 * 10 * 8 * 16 + 64,), device="cuda", dtype=torch.uint8)
    t = raw[4:4 + 2 * 10 * 8 * 16].view(2, 10, 8, 1, 16)
    layout, k, v = cc.layout_from_kv_tensors([t])
    pool = pg.PagePool(layout, k, v, torch.full((1, 4), -1, dtype=torch.int32, device="cuda"),
                       torch.zeros(1, dtype=torch.int32, device="cuda"))
    want = t.clone()
    want[:, 5] = want[:, 2]
    pool.copy(ints([2]), ints([5]))
    pool.check()
    assert torch.equal(t, want)


def test_results_on_a_side_stream():
    """are not in memory that the current stream has freed but still has to
    write"""
    c = Case(GEOMETRIES["hnd"], 60, 4, 8)
    rows, lens = ints([0, 1]), ints([100, 37])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    held = torch.empty(2, dtype=torch.int32, device="cuda")
    torch.cuda._sleep(200_000_000)
    held.fill_(7)
    del held
    got = c.pool.resize(rows, lens, stream=side)
    torch.cuda.synchronize()
    assert got.tolist() == [pg.OK, pg.OK]
    c.model.resize([0, 1], [100, 37])
    c.same()


def test_check_waits_for_every_stream():
    c = Case(GEOMETRIES["hnd"], 60, 4, 8)
    rows, lens = ints([9]), ints([16])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    got = c.pool.resize(rows, lens, stream=side)
    with pytest.raises(ValueError, match="row"):
        c.pool.check()
    c.pool.check()
    assert got.tolist() == [pg.INVALID]
