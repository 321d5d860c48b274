"""Attention over the pages of a cache against its definition in 64 bits
(oracle/attention.py, which also derives the tolerances)."""
import math

import numpy as np
import pytest
import torch

from demo_b200 import cache as cc
from demo_b200 import pages as pg
from demo_b200.attention import TreeAttention
from oracle import attention as oa

pytestmark = pytest.mark.gpu
BF16, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


class Batch:
    """A paged cache with sequences of the given lengths on scattered pages;
    everything that no sequence holds is NaN."""

    def __init__(self, lens, nodes, heads=8, kv_heads=2, dim=128, block=16, order="nhd", qt=BF16, kvt=None, seed=0,
                 layers=1, spare_rows=0):
        kvt = kvt or qt
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.nodes, self.block, self.order, self.heads, self.kv_heads = list(lens), list(nodes), block, order, heads, kv_heads
        used = [-(-n // block) for n in lens]
        pages = sum(used) + 3
        width = max(used + [1])
        ids = rng.permutation(pages)
        self.table = np.full((len(lens) + spare_rows, width), -7, np.int32)
        shape = (layers, 2, pages, block, kv_heads, dim) if order == "nhd" else (layers, pages, 2, kv_heads, block, dim)
        store = torch.full(shape, math.nan, device="cuda").to(kvt)
        view = store if order == "nhd" else store.permute(0, 2, 1, 4, 3, 5)
        at = 0
        raw = view.view(torch.uint8 if kvt == E4M3 else torch.int16)
        for r, n in enumerate(lens):
            self.table[r, :used[r]] = ids[at:at + used[r]]
            at += used[r]
            pos = np.arange(n)
            p, s = torch.tensor(self.table[r, pos // block].astype(np.int64)), torch.tensor(pos % block)
            x = torch.randn(layers, 2, n, kv_heads, dim, generator=g, device="cuda").to(kvt)
            raw[:, :, p.cuda(), s.cuda()] = x.view(raw.dtype)
        self.store, self.view = store, view
        tensors = list(store) if order == "nhd" else list(store.permute(0, 1, 2, 4, 3, 5))
        self.layout, self.k, self.v = cc.layout_from_kv_tensors(tensors, kv_layout="flash_attn" if order == "nhd" else "flashinfer")
        self.q = torch.randn(sum(nodes), heads, dim, generator=g, device="cuda").to(qt)
        self.off = np.cumsum([0] + list(nodes)).tolist()
        self.parents = None
        self.scales = (0.5, 1.5) if kvt == E4M3 else (1.0, 1.0)

    def tree(self, seed=0, padding=0.0):
        rng = np.random.default_rng(seed)
        self.parents = [int(rng.integers(-1, j)) if rng.random() >= padding else -2 for n in self.nodes for j in range(n)]
        return self

    def attention(self):
        return TreeAttention(self.layout, self.k, self.v, self.heads, self.kv_heads, k_scale=self.scales[0], v_scale=self.scales[1])

    def args(self, layer=0):
        i32 = lambda x: torch.tensor(np.asarray(x, np.int32), device="cuda")
        return (layer, self.q, i32(self.table), i32(self.lens + [0] * (len(self.table) - len(self.lens))), i32(self.off)), \
            i32(self.parents) if self.parents is not None else None

    def expected(self, layer=0):
        k, v = (self.view[layer, i].double() for i in range(2))
        return oa.attention(self.q, k, v, self.table.tolist(), self.lens, self.off, self.parents, k_scale=self.scales[0],
                            v_scale=self.scales[1])

    def check(self, layer=0):
        att = self.attention()
        args, parents = self.args(layer)
        out, lse = att(*args, parents=parents, return_lse=True)
        att.check()
        close(out, lse, self.expected(layer))


def close(out, lse, want):
    o, l, ot, lt = want
    assert out.shape == o.shape and torch.equal(torch.isinf(lse), torch.isinf(l))
    bad = ~((out.double() - o).abs() <= ot)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float(((out.double() - o).abs() - ot).nan_to_num(9e9).max()))
    fin = ~torch.isinf(l)
    bad = ~((lse.double() - l).abs()[fin] <= lt[fin])
    assert not bad.any(), (int(bad.sum()), float((lse.double() - l).abs()[fin].max()))


LENS = [1, 2, 63, 64, 65, 128, 129, 1000]


@pytest.mark.parametrize("order", ["nhd", "hnd"])
@pytest.mark.parametrize("types", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)], ids=["bf16", "fp16", "bf16-e4m3", "fp16-e4m3"])
def test_single_tokens(order, types):
    Batch(LENS, [1] * len(LENS), order=order, qt=types[0], kvt=types[1]).check()


@pytest.mark.parametrize("types", [(BF16, BF16), (FP16, FP16), (BF16, E4M3), (FP16, E4M3)], ids=["bf16", "fp16", "bf16-e4m3", "fp16-e4m3"])
@pytest.mark.parametrize("order", ["nhd", "hnd"])
def test_trees(order, types):
    nodes = [1, 2, 7, 31, 0, 16, 64, 33]
    Batch(LENS, nodes, order=order, qt=types[0], kvt=types[1], seed=1).tree().check()


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 160, 192, 256])
@pytest.mark.parametrize("kvt", [BF16, E4M3], ids=["16bit", "8bit"])
def test_head_dims(dim, kvt):
    Batch([70, 1, 333], [5, 1, 20], dim=dim, kvt=kvt, order="hnd", seed=dim).tree(dim).check()


@pytest.mark.parametrize("block", [1, 3, 8, 24, 64, 100, 256])
def test_block_sizes(block):
    for order in ("nhd", "hnd"):
        Batch([300, 5, 64, 257], [3, 5, 1, 40], block=block, order=order, seed=block).tree(block).check()


@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (32, 8), (5, 1), (12, 2), (71, 1), (128, 1)], ids=str)
def test_head_groups(heads):
    Batch([200, 3, 90], [7, 3, 30], heads=heads[0], kv_heads=heads[1], dim=64, seed=2).tree(2).check()


def test_chains_and_prompt_chunks():
    Batch([300, 130, 700, 40, 1], [300, 129, 257, 1, 1], dim=64, heads=6, seed=3).check()


def test_trees_over_many_row_tiles():
    Batch([1000, 513, 400], [400, 513, 65], dim=64, seed=4).tree(4).check()


def test_deep_trees():
    """a tree that is one path, out of another's middle"""
    b = Batch([500, 300], [200, 150], dim=64, seed=5)
    b.parents = list(range(-1, 199)) + [-1] + [0] * 2 + list(range(2, 149))
    b.check()


def test_padding_nodes_see_and_show_nothing():
    b = Batch([90, 40, 64, 5], [20, 33, 64, 5], seed=6, dim=64).tree(6, padding=0.4)
    for r, n in enumerate(b.lens):
        first = b.off[r]
        for j in range(b.nodes[r]):
            if b.parents[first + j] == -2:
                p = n - b.nodes[r] + j
                b.view[:, :, int(b.table[r, p // b.block]), p % b.block] = math.nan
    args, parents = b.args()
    out, lse = b.attention()(*args, parents=parents, return_lse=True)
    pad = torch.tensor([p == -2 for p in b.parents], device="cuda")
    assert not out[pad].any() and torch.isinf(lse[pad]).all()
    b.view.nan_to_num_(0.0)
    close(out, lse, b.expected())


@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=["nan", "inf"])
@pytest.mark.parametrize("kvt", [BF16, E4M3], ids=["16bit", "8bit"])
def test_masked_infinities_stay_masked(bad, kvt):
    """a node whose K and V are not finite spoils itself and its descendants only"""
    if kvt == E4M3 and bad == math.inf:
        pytest.skip("e4m3 has no infinities")
    b = Batch([90, 200], [20, 30], seed=7, dim=64, kvt=kvt).tree(7)
    spoilt = [4, 20 + 11]
    clean = b.expected()
    for i in spoilt:
        r = 0 if i < 20 else 1
        p = b.lens[r] - b.nodes[r] + i - b.off[r]
        b.view[:, 1, int(b.table[r, p // b.block]), p % b.block, :, 3] = torch.full((), bad, device="cuda").to(kvt)
    args, parents = b.args()
    out, lse = b.attention()(*args, parents=parents, return_lse=True)
    hit = torch.zeros(50, dtype=torch.bool)
    for r in range(2):
        sees = oa.visible(b.parents[b.off[r]:b.off[r + 1]], b.nodes[r])
        for j, s in enumerate(sees):
            hit[b.off[r] + j] = any(b.off[r] + x in spoilt for x in s)
    assert hit.any() and not hit.all()
    spoiled = ~torch.isfinite(out[:, :, 3]).cpu()
    assert torch.equal(spoiled.all(1), hit) and torch.equal(spoiled.any(1), hit)
    out[:, :, 3] = clean[0][:, :, 3].to(out.dtype)
    close(out, lse, clean)


@pytest.mark.parametrize("kvt", [BF16, E4M3], ids=["16bit", "8bit"])
@pytest.mark.parametrize("block", [16, 24], ids=["block16", "block24"])
def test_a_value_of_the_context_that_is_not_finite_reaches_every_row(kvt, block):
    """beside the nodes, in their tile, and in an earlier one"""
    for pos in (3, 85, 190, 199):
        b = Batch([90, 210], [4, 10], seed=15, dim=64, kvt=kvt, block=block).tree(15)
        r = 0 if pos < 86 else 1
        clean = b.expected()
        b.view[:, 1, int(b.table[r, pos // block]), pos % block, :, 3] = torch.full((), math.nan, device="cuda").to(kvt)
        args, parents = b.args()
        out, lse = b.attention()(*args, parents=parents, return_lse=True)
        hit = torch.zeros(14, dtype=torch.bool)
        hit[b.off[r]:b.off[r + 1]] = True
        spoiled = ~torch.isfinite(out[:, :, 3]).cpu()
        assert torch.equal(spoiled.all(1), hit) and torch.equal(spoiled.any(1), hit), pos
        out[:, :, 3] = clean[0][:, :, 3].to(out.dtype)
        close(out, lse, clean)


@pytest.mark.parametrize("qt", [BF16, FP16], ids=["bf16", "fp16"])
def test_every_8bit_value(qt):
    """one visible position: the output is its value, widened exactly"""
    b = Batch([1] * 2, [1] * 2, heads=2, kv_heads=1, dim=128, qt=qt, kvt=E4M3, order="hnd")
    codes = torch.arange(256, dtype=torch.int32, device="cuda").to(torch.uint8).view(E4M3)
    for r in range(2):
        b.view[0, 1].view(torch.uint8)[int(b.table[r, 0]), 0, 0] = codes[128 * r:128 * r + 128].view(torch.uint8)
    b.scales = (1.0, 1.0)
    args, parents = b.args()
    out = b.attention()(*args).double()
    want = codes.double().view(2, 1, 128).expand(2, 2, 128)
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(), want.nan_to_num())


def test_large_scores():
    """rows whose maximum climbs through the whole context, and scores that
    only a running maximum survives"""
    b = Batch([700, 640], [5, 64], dim=64, seed=8).tree(8)
    for r, n in enumerate(b.lens):
        pos = np.arange(n)
        p, s = torch.tensor(b.table[r, pos // 16].astype(np.int64)).cuda(), torch.tensor(pos % 16).cuda()
        ramp = torch.linspace(0.1, 40, n, device="cuda").to(BF16)[:, None, None]
        b.view[0, 0, p, s] = (b.view[0, 0, p, s] * ramp)
    b.check()


def test_rows_strides_layers_and_uncovered_queries():
    """rows picked out of a wider, strided table; q and out as slices of larger
    tensors; a layer behind the first; queries behind the last sequence"""
    b = Batch([100, 200, 50, 75], [3, 4, 2, 6], seed=9, layers=3, order="hnd", spare_rows=2).tree(9)
    args, parents = b.args(2)
    pick = [2, 0, 3]
    off = np.cumsum([0] + [b.nodes[r] for r in pick]).tolist()
    order = [i for r in pick for i in range(b.off[r], b.off[r + 1])]
    big = torch.zeros(len(order) + 4, 11, 3, 128, dtype=BF16, device="cuda")
    q = big[:, 2:10, 1]
    q[:len(order)] = b.q[order]
    out = torch.full((len(order) + 4, 8, 160), 7.0, dtype=BF16, device="cuda")[..., 16:144]
    wide = torch.full((6, 31), -9, dtype=torch.int32, device="cuda")
    wide[:, :args[2].shape[1]] = args[2]
    par = [b.parents[i] for i in order] + [0] * 4
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    att = b.attention()
    got, lse = att(2, q, wide[:, :args[2].shape[1]], args[3], i32(off), parents=i32(par), rows=i32(pick), out=out, return_lse=True)
    att.check()
    n = len(order)
    assert got.data_ptr() == out.data_ptr() and (got[n:] == 7).all()
    k, v = (b.view[2, i].double() for i in range(2))
    close(got[:n], lse[:n], oa.attention(b.q[order], k, v, b.table.tolist(), b.lens, off, [b.parents[i] for i in order], rows=pick))


def test_many_sequences():
    rng = np.random.default_rng(10)
    lens = rng.integers(1, 100, 700).tolist()
    Batch(lens, [int(rng.integers(0, min(n, 4) + 1)) for n in lens], heads=2, kv_heads=1, dim=32, block=8, seed=10).check()


def test_long_context_few_heads():
    """one K/V head, split over many CTAs, beside short rows"""
    Batch([40000, 17, 9000], [16, 17, 1], heads=8, kv_heads=1, dim=128, seed=11).tree(11).check()


def test_errors_void_their_own_rows():
    b = Batch([100, 200, 50], [3, 4, 2], seed=12, dim=64).tree(12)
    args, parents = b.args()
    want = b.expected()
    att = b.attention()

    def run(change, sequence, nodes, match):
        a = [x.clone() if torch.is_tensor(x) else x for x in args]
        p = parents.clone()
        change(a, p)
        out, lse = att(*a, parents=p, return_lse=True)
        with pytest.raises(ValueError, match=match):
            att.check()
        keep = torch.ones(9, dtype=torch.bool)
        keep[b.off[sequence]:b.off[sequence + 1]] = False
        for t in (out, lse):
            assert not t[~keep].isnan().any()
        if nodes is not None:
            for j in nodes:
                assert not out[b.off[sequence] + j].any() and torch.isinf(lse[b.off[sequence] + j]).all()
        close(out[keep.cuda()], lse[keep.cuda()], [w[keep.cuda()] for w in want])

    run(lambda a, p: a[3].__setitem__(1, 3), 1, range(4), "length")                    # shorter than its nodes
    run(lambda a, p: a[3].__setitem__(1, -5), 1, range(4), "length")
    run(lambda a, p: a[3].__setitem__(1, 13 * 16 + 1), 1, range(4), "length")          # longer than its row
    run(lambda a, p: p.__setitem__(3 + 2, 2), 1, [2], "parent")                        # its own parent
    run(lambda a, p: p.__setitem__(3 + 2, -3), 1, [2], "parent")
    run(lambda a, p: a[2].__setitem__((1, 4), 1 << 20), 1, None, "page id")
    run(lambda a, p: a[2].__setitem__((1, 4), -1), 1, None, "page id")


def test_capture_other_stream_and_repeats():
    b = Batch([3000, 17, 900], [16, 17, 1], heads=8, kv_heads=1, dim=128, seed=13).tree(13)
    args, parents = b.args()
    att = b.attention()
    want = b.expected()
    first, lse1 = att(*args, parents=parents, return_lse=True)
    close(first, lse1, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = att(*args, parents=parents, stream=side)
    side.synchronize()
    assert torch.equal(first, other)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = att(*args, parents=parents)
        graphs.append((g, res))
    for _ in range(2):
        for g, res in graphs:
            res.zero_()
            g.replay()
            assert torch.equal(res, first)
    # new lengths reach a captured graph
    args[3].copy_(torch.tensor([2900, 17, 800], dtype=torch.int32))
    graphs[0][0].replay()
    b.lens = [2900, 17, 800]
    now = b.expected()
    bad = ~((graphs[0][1].double() - now[0]).abs() <= now[2])
    assert not bad.any()
    att.check()


def test_a_step_over_the_pool_and_the_store():
    """room for a tree, its K and V written, attention over it, the accepted
    path kept, and the same attention for the next token; then the full blocks
    of the row go through the cache manager's records and come back"""
    L, H, D, bs, nb = 2, 2, 64, 16, 64
    g = torch.Generator(device="cuda").manual_seed(14)
    kv = [torch.randn(nb, 2, H, bs, D, generator=g, device="cuda").to(BF16).permute(0, 1, 3, 2, 4) for _ in range(L)]
    layout, k, v = cc.layout_from_kv_tensors(kv, kv_layout="flashinfer")
    table = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    pool = pg.PagePool(layout, k, v, table, lens)
    att = TreeAttention(layout, k, v, 8, H)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    pool.resize(i32([0, 2]), i32([256 + 3 + 5, 40 + 4]))
    parents = [-1, 0, 0, 1, 1, -1, 0, 0, 2]
    off = [0, 5, 9]
    q = torch.randn(9, 8, D, generator=g, device="cuda").to(BF16)
    for layer in range(L):
        out, lse = att(layer, q, table, lens, i32(off), parents=i32(parents), rows=i32([0, 2]), return_lse=True)
        kk, vv = kv[layer][:, 0].double(), kv[layer][:, 1].double()
        close(out, lse, oa.attention(q, kk, vv, table.tolist(), lens.tolist(), off, parents, rows=[0, 2]))
    # accepted: nodes 0, 1, 4 of row 0; nodes 0, 2 of row 2
    seq = []
    for r, keep in ((0, list(range(260)) + [260, 263]), (2, list(range(41)) + [42])):
        ids = table[r].long()
        seq.append([[kv[l][ids[p // bs], c, p % bs].clone() for p in keep] for l in range(L) for c in range(2)])
    pool.compact(i32([0, 2]), i32([259, 40]), i32([259, 260, 263, 40, 42]), i32([0, 3, 5]))
    pool.check()
    assert lens.tolist() == [262, 0, 42]
    for (r, n), want in zip(((0, 262), (2, 42)), seq):
        ids = table[r].tolist()
        for l in range(L):
            for c in range(2):
                have = [kv[l][ids[p // bs], c, p % bs] for p in range(n)]
                assert all(torch.equal(a, b) for a, b in zip(have, want[2 * l + c])), (r, l, c)
    # a fork decodes on: parent and child attend to the same tokens
    pool.fork(i32([0]), i32([1]))
    pool.resize(i32([0, 1]), i32([263, 263]))
    for r in (0, 1):
        p, s = int(table[r, 262 // bs]), 262 % bs
        for l in range(L):
            kv[l][p, :, s] = 0.25 * (l + 1)
    q1 = q[:2].clone()
    q1[1] = q1[0]
    out = att(1, q1, table, lens, i32([0, 1, 2]))
    att.check()
    assert torch.equal(out[0], out[1])
    assert int(table[0, 262 // bs]) != int(table[1, 262 // bs])
    # the record of row 0's first 256 tokens, stored and loaded into other pages
    cc.init(256, 8 << 20)
    try:
        w = cc.Worker("pages", layout, k, v)
        w.register()
        blocks = table[0, :16].tolist()
        assert w.store([b"k" * 32], blocks) == 0
        pool.resize(i32([2]), i32([256]))
        new = table[2, :16].tolist()
        for l in range(L):
            for b in new:
                kv[l][b] = 0
        torch.cuda.synchronize()
        assert w.load([b"k" * 32], new) == 0
        for l in range(L):
            assert torch.equal(kv[l][torch.tensor(new)], kv[l][torch.tensor(blocks)])
        w.unregister()
    finally:
        cc.exit()
    pool.resize(i32([0, 1, 2]), i32([0, 0, 0]))
    pool.check()
    assert int(pool.free_count.item()) == nb


def test_a_path_as_a_tree_is_a_chain():
    """3000 nodes, each the parent of the next: the bits of a call without
    parents, whose rows the oracle checks above"""
    b = Batch([3050, 700], [3000, 650], heads=4, kv_heads=2, dim=64, seed=15)
    args, _ = b.args()
    att = b.attention()
    chain = att(*args, return_lse=True)
    path = torch.cat([torch.arange(-1, n - 1, dtype=torch.int32, device="cuda") for n in b.nodes])
    for got, want in zip(att(*args, parents=path, return_lse=True), chain):
        assert torch.equal(got, want)
    att.check()


def test_positions_up_to_31_bits():
    """2^31 - 1 tokens on one page that the row names 2048 times: scores 0,
    values 1; each is exp(0) = 1, and sums of ones are exact up to 2^24, so
    that only the joined pieces' sums (at most 512 of them) round: 2^-15"""
    bs, w = 1 << 20, 2048
    k = torch.zeros(2, 1, bs, 1, 16, dtype=BF16, device="cuda")
    k[1] = 1
    layout, kp, vp = cc.layout_from_kv_tensors([k], kv_layout="flash_attn")
    att = TreeAttention(layout, kp, vp, 1, 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    out, lse = att(0, torch.ones(2, 1, 16, dtype=BF16, device="cuda"), i32([[0] * w]), i32([2 ** 31 - 1]), i32([0, 2]), return_lse=True)
    att.check()
    assert ((out.double() - 1).abs() <= 2.0 ** -8 + 2.0 ** -14).all()
    want = torch.tensor([math.log(2 ** 31 - 2), math.log(2 ** 31 - 1)], dtype=torch.float64, device="cuda")[:, None]
    assert ((lse.double() - want).abs() <= 2.0 ** -15 + 2.0 ** -21 * want).all()


@pytest.mark.parametrize("block, kvt", [(16, BF16), (24, BF16), (16, E4M3)], ids=["boxes", "copies", "8bit"])
def test_pages_past_32_bits(block, kvt):
    """pages more than 4 GiB into a plane"""
    esz, kv_heads, dim = (1 if kvt == E4M3 else 2), 8, 128
    pages = (1 << 32) // (block * kv_heads * dim * esz) + 9
    store = torch.empty(2, pages, block, kv_heads, dim, dtype=kvt, device="cuda")
    b = Batch([200, 61], [3, 61], heads=8, kv_heads=kv_heads, dim=dim, block=block, kvt=kvt, seed=16).tree(16)
    used = b.view.shape[2]
    for i in range(2):
        store.view(torch.uint8 if kvt == E4M3 else torch.int16)[i, -used:] = b.view[0, i].view(torch.uint8 if kvt == E4M3 else torch.int16)
    layout, k, v = cc.layout_from_kv_tensors([store], kv_layout="flash_attn")
    att = TreeAttention(layout, k, v, 8, kv_heads, k_scale=b.scales[0], v_scale=b.scales[1])
    args, parents = b.args()
    table = torch.where(args[2] >= 0, args[2] + (pages - used), args[2])
    out, lse = att(0, b.q, table, *args[3:], parents=parents, return_lse=True)
    att.check()
    close(out, lse, b.expected())


def test_rows_of_a_padded_batch():
    """sequences without nodes, whose rows are no rows: nothing of theirs is
    looked at"""
    b = Batch([100, 40], [3, 1], seed=17)
    args, _ = b.args()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    att = b.attention()
    out, lse = att(*args[:4], i32([0, 3, 3, 4, 4, 4]), rows=i32([0, -1, 1, 99, -5]), return_lse=True)
    att.check()
    close(out, lse, b.expected())


def test_a_long_sequence_that_does_not_fit():
    """its rows are voided by the whole grid, also where there are more
    sequences than threads look at in one go"""
    n, m = 20000, 400
    b = Batch([5] * (m - 1) + [n], [1] * (m - 1) + [n], heads=2, kv_heads=1, dim=16, seed=18)
    args, _ = b.args()
    args[3][m - 1] = n - 1
    att = b.attention()
    out, lse = att(*args, return_lse=True)
    with pytest.raises(ValueError, match="length"):
        att.check()
    assert not out[m - 1:].any() and torch.isinf(lse[m - 1:]).all()
    want = oa.attention(b.q[:m - 1], *(b.view[0, i].double() for i in range(2)), b.table.tolist(), b.lens, b.off[:m])
    close(out[:m - 1], lse[:m - 1], want)


def test_offsets_out_of_order_are_skipped():
    b = Batch([50, 60, 70], [2, 3, 4], seed=19)
    args, _ = b.args()
    att = b.attention()
    for off in ([0, 2, 1, 9], [0, 2, 2, 99], [-4, -1, 5, 9]):
        out = torch.full_like(b.q, 7.0)
        a = (*args[:4], torch.tensor(off, dtype=torch.int32, device="cuda"))
        att(*a, out=out)
        with pytest.raises(ValueError, match="offsets"):
            att.check()
        covered = {i for x, y in zip(off, off[1:]) if 0 <= x <= y <= 9 for i in range(x, y)}
        for i in range(9):
            assert (out[i] == 7).all() == (i not in covered), (off, i)


@pytest.mark.parametrize("n", [40, 6000])
def test_scores_of_minus_infinity_alone(n):
    """count as nothing seen, whether a row is joined from pieces or not"""
    b = Batch([n, 30], [1, 1], heads=2, kv_heads=1, dim=64, seed=20)
    b.q[0] = 1
    b.view[0, 0, torch.tensor(b.table[0, :-(-n // 16)].astype(np.int64)).cuda()] = -math.inf
    args, _ = b.args()
    out, lse = b.attention()(*args, return_lse=True)
    assert not out[0].any() and (lse[0] == -math.inf).all()
    want = oa.attention(b.q[1:], *(b.view[0, i].double() for i in range(2)), b.table.tolist(), b.lens, [0, 1], rows=[1])
    close(out[1:], lse[1:], want)


def test_memory_in_use_on_another_stream_is_left_alone():
    """what a call on a side stream allocates is not what the current stream has
    freed but still has to write"""
    b = Batch([300, 17], [2, 1], seed=21)
    args, _ = b.args()
    att = b.attention()
    want = att(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for shape, dt in ((want.shape, want.dtype), ((40 << 20,), torch.uint8)):
        held = torch.empty(shape, dtype=dt, device="cuda")
        torch.cuda._sleep(200_000_000)
        held.fill_(7)
        del held
        got = att(*args, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_check_waits_for_every_stream():
    b = Batch([30], [2], seed=24)
    args, _ = b.args()
    att = b.attention()
    att(*args)
    args[3].fill_(1)                    # shorter than its nodes
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    att(*args, stream=side)
    with pytest.raises(ValueError, match="length"):
        att.check()
    att.check()


def test_gradients_are_refused():
    b = Batch([30], [2], seed=23)
    args, _ = b.args()
    att = b.attention()
    want = att(*args)
    q = b.q.clone().requires_grad_()
    with pytest.raises(ValueError, match="no gradients"):
        att(0, q, *args[2:])
    with torch.no_grad():
        assert torch.equal(att(0, q, *args[2:]), want)


def test_the_first_call_is_captured():
    b = Batch([300, 17], [2, 1], seed=22)
    args, _ = b.args()
    b.attention()(*args)                # loads the kernels
    att = b.attention()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = att(*args, return_lse=True)
    att.check()
    g.replay()
    att.check()
    close(out, lse, b.expected())
