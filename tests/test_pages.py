"""Page operators without a GPU: what the C entry points and PagePool refuse
before anything is launched, and the structs' layout."""
import ctypes as C
import errno
import subprocess
from pathlib import Path

import pytest
import torch

from demo_b200 import pages as pg
from demo_b200._lib import (KVPAGE_MAX_CALL, KVPAGE_MAX_ROWS, KvPageCache, KvPageState, lib)
from demo_b200.cache import KVLayout
from oracle import pages_model as pm

INCLUDE = Path(__file__).resolve().parent.parent / "include"
X = 0x1000          # an address that is never followed


def state(**k):
    d = dict(table=X, lens=X, refs=X, free_list=X, free_count=X, marks=X, error=X, table_stride=8, width=8, num_rows=4,
             num_pages=32, block_size=16, device=0)
    return KvPageState(**{**d, **k})


def cache(**k):
    d = dict(layer_k=X, layer_v=X, error=X, block_stride=0, unit_bytes=256, head_bytes=0, block_size=16, num_layers=2,
             num_pages=32, base_align=16, device=0)
    return KvPageCache(**{**d, **k})


BAD_STATES = [dict(table=None), dict(lens=None), dict(refs=None), dict(free_list=None), dict(free_count=None),
              dict(marks=None), dict(error=None), dict(width=0), dict(table_stride=7), dict(num_rows=0), dict(num_pages=0),
              dict(num_pages=1 << 31), dict(block_size=0), dict(device=-1), dict(device=64)]
BAD_CACHES = [dict(layer_k=None), dict(error=None), dict(unit_bytes=0), dict(block_size=0), dict(num_layers=0),
              dict(num_pages=0), dict(base_align=12), dict(block_stride=100), dict(head_bytes=100),
              dict(unit_bytes=1 << 30), dict(device=-1), dict(device=64)]


@pytest.mark.parametrize("bad", BAD_STATES, ids=str)
def test_malformed_states_are_refused(bad):
    s = state(**bad)
    p = C.addressof(s)
    c = cache(device=bad.get("device", 0))
    assert lib.kv_page_resize_launch(p, X, X, 1, None, None) == -errno.EINVAL
    assert lib.kv_page_fork_launch(C.addressof(c), p, X, X, 1, X, None, None) == -errno.EINVAL
    assert lib.kv_page_compact_launch(C.addressof(c), p, X, X, X, X, 1, 1, X, None, None) == -errno.EINVAL


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
def test_malformed_caches_are_refused(bad):
    c = cache(**bad)
    s = state()
    p = C.addressof(c)
    assert lib.kv_page_copy_launch(p, X, X, None, 1, None) == -errno.EINVAL
    assert lib.kv_page_fork_launch(p, C.addressof(s), X, X, 1, X, None, None) == -errno.EINVAL
    assert lib.kv_page_compact_launch(p, C.addressof(s), X, X, X, X, 1, 1, X, None, None) == -errno.EINVAL


def test_arguments_and_limits():
    s, c = state(), cache()
    sp, cp = C.addressof(s), C.addressof(c)
    assert lib.kv_page_resize_launch(None, X, X, 1, None, None) == -errno.EINVAL
    assert lib.kv_page_copy_launch(None, X, X, None, 1, None) == -errno.EINVAL
    assert lib.kv_page_resize_launch(sp, None, X, 1, None, None) == -errno.EINVAL
    assert lib.kv_page_resize_launch(sp, X, None, 1, None, None) == -errno.EINVAL
    assert lib.kv_page_copy_launch(cp, None, X, None, 1, None) == -errno.EINVAL
    assert lib.kv_page_copy_launch(cp, X, None, None, 1, None) == -errno.EINVAL
    assert lib.kv_page_fork_launch(cp, sp, X, X, 1, None, None, None) == -errno.EINVAL
    assert lib.kv_page_compact_launch(cp, sp, X, X, None, X, 1, 1, X, None, None) == -errno.EINVAL
    assert lib.kv_page_compact_launch(cp, sp, X, X, X, X, 1, 1, None, None, None) == -errno.EINVAL
    assert lib.kv_page_resize_launch(sp, X, X, KVPAGE_MAX_CALL + 1, None, None) == -errno.E2BIG
    big = state(num_rows=KVPAGE_MAX_ROWS + 1)
    assert lib.kv_page_resize_launch(C.addressof(big), X, X, 1, None, None) == -errno.E2BIG
    wide = state(width=1 << 29, table_stride=1 << 29)
    assert lib.kv_page_resize_launch(C.addressof(wide), X, X, 2, None, None) == -errno.E2BIG
    for other in (cache(num_pages=31), cache(block_size=8), cache(device=1)):
        assert lib.kv_page_fork_launch(C.addressof(other), sp, X, X, 1, X, None, None) == -errno.EINVAL
    # nothing to do is no error, and nothing is launched
    n0 = lib.crosscache_kernel_launches()
    assert lib.kv_page_resize_launch(sp, None, None, 0, None, None) == 0
    assert lib.kv_page_copy_launch(cp, None, None, None, 0, None) == 0
    assert lib.kv_page_fork_launch(cp, sp, None, None, 0, None, None, None) == 0
    assert lib.kv_page_compact_launch(cp, sp, None, None, None, None, 0, 0, None, None, None) == 0
    assert lib.crosscache_kernel_launches() == n0


def test_pool_refuses_tensors_it_cannot_use():
    lay = KVLayout(1, 8, 16, 64, 2, 2)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="block_table"):
        pg.PagePool(lay, [X], [X], table, lens)                       # not on a CUDA device
    with pytest.raises(ValueError, match="contiguous int32"):
        pg._int32("x", lens.long(), -1)
    with pytest.raises(ValueError, match="contiguous int32"):
        pg._int32("x", torch.zeros(4, dtype=torch.int32)[::2], -1)
    with pytest.raises(ValueError, match="expected 3 values"):
        pg._int32("x", lens, -1, 3)
    with pytest.raises(ValueError, match="one pointer per layer"):
        pg.plane_bases(lay, [X, X], [X], lens.device)
    with pytest.raises(ValueError, match="kv must be 1"):
        pg.plane_bases(lay, [X], None, lens.device)
    with pytest.raises(ValueError, match="null"):
        pg.plane_bases(lay, [X], [0], lens.device)
    assert pg.plane_bases(lay, [X], [X + 4], lens.device)[2] == 4
    assert pg.plane_bases(lay, [X], [X + 64], lens.device)[2] == 16


PROBE = r"""
#include <stdio.h>
#include <stddef.h>
#include "kvpage.h"
#define F(s, f) printf(#s "." #f " %zu\n", offsetof(struct s, f))
int main(void) {
  printf("kv_page_state %zu\n", sizeof(struct kv_page_state));
  printf("kv_page_cache %zu\n", sizeof(struct kv_page_cache));
  F(kv_page_state, marks); F(kv_page_state, table_stride); F(kv_page_state, num_pages); F(kv_page_state, device);
  F(kv_page_cache, block_stride); F(kv_page_cache, head_bytes); F(kv_page_cache, base_align); F(kv_page_cache, device);
  return 0;
}
"""


def test_struct_layout(tmp_path):
    (tmp_path / "p.c").write_text(PROBE)
    subprocess.run(["gcc", "-std=c11", f"-I{INCLUDE}", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout
    mirror = {"kv_page_state": KvPageState, "kv_page_cache": KvPageCache}
    for line in out.splitlines():
        key, val = line.split()
        name, _, field = key.partition(".")
        assert (getattr(mirror[name], field).offset if field else C.sizeof(mirror[name])) == int(val), key


def test_the_model_keeps_its_invariants():
    """every page is free or held, and counted as often as it is held"""
    import numpy as np

    rng = np.random.default_rng(0)
    m = pm.Pages(6, 5, 20, 4, np.zeros((1, 20, 4, 2), np.uint8))
    for _ in range(200):
        if rng.random() < 0.6:
            n = int(rng.integers(1, 7))
            m.resize(rng.permutation(6)[:n], rng.integers(0, 21, n))
        else:
            empty = np.flatnonzero(m.lens == 0)
            if len(empty):
                m.fork([int(rng.integers(0, 6))], [int(empty[0])]) if m.lens.any() else None
        m.error = 0
        held = [int(p) for r in range(6) for p in m.table[r, :-(-int(m.lens[r]) // 4)]]
        assert sorted(set(held) | set(m.free)) == list(range(20)) and not set(held) & set(m.free)
        assert [held.count(p) for p in range(20)] == m.refs.tolist()


def test_copies_of_too_many_pages_are_refused():
    c = cache(num_layers=1)
    assert lib.kv_page_copy_launch(C.addressof(c), X, X, None, (1 << 31) + 5, None) == -errno.E2BIG
    c = cache(num_layers=1 << 30)
    assert lib.kv_page_copy_launch(C.addressof(c), X, X, None, 1, None) == -errno.EINVAL


def test_what_a_call_on_a_stream_was_given_is_recorded_there():
    class Tensor:
        def __init__(self):
            self.streams = []

        def record_stream(self, stream):
            self.streams.append(stream)

    a, b = Tensor(), Tensor()
    pg._used_on(None, a, b)
    pg._used_on("side", a, None, b)
    assert a.streams == b.streams == ["side"]


def test_planes_of_another_device_are_refused(monkeypatch):
    at = {X: 0, 2 * X: 1, 3 * X: -1, 4 * X: -errno.EINVAL}
    monkeypatch.setattr(lib, "kv_page_device_of", at.get)
    pg.planes_on(0, [X, 3 * X])             # its own memory, and pinned memory
    pg.planes_on(1, [2 * X])
    with pytest.raises(ValueError, match="cuda:1, not on cuda:0"):
        pg.planes_on(0, [X, 2 * X])
    with pytest.raises(ValueError, match="not memory that a GPU reaches"):
        pg.planes_on(0, [X, 4 * X])
