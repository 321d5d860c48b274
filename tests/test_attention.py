"""Tree attention without a GPU: what the C entry points and TreeAttention
refuse before anything is launched, the struct's layout, the oracle."""
import ctypes as C
import errno
import math
import subprocess
from pathlib import Path

import pytest
import torch

from demo_b200._lib import KVATTN_BF16, KVATTN_E4M3, KVATTN_FP16, KVATTN_MAX_SEQS, KvAttnDesc, lib
from demo_b200.attention import TreeAttention
from demo_b200.cache import KVLayout
from oracle import attention as oa

INCLUDE = Path(__file__).resolve().parent.parent / "include"
X = 0x1000          # an address that is never followed


def desc(**k):
    d = dict(q=X, out=X, lse=X, k=X, v=X, table=X, lens=X, q_offsets=X, error=X, workspace=X, workspace_bytes=1 << 40,
             table_stride=8, q_stride=1024, q_head_stride=128, out_stride=1024, out_head_stride=128, width=8, num_rows=4,
             num_seqs=4, total_q=4, num_pages=32, block_size=16, num_heads=8, num_kv_heads=2, head_dim=128,
             q_type=KVATTN_BF16, kv_type=KVATTN_BF16, scale=0.1, k_scale=1.0, v_scale=1.0)
    return KvAttnDesc(**{**d, **k})


SHAPES = [dict(num_heads=0), dict(num_kv_heads=0), dict(num_kv_heads=3), dict(head_dim=0), dict(head_dim=120),
          dict(head_dim=272), dict(num_heads=258), dict(block_size=0), dict(num_pages=0), dict(num_pages=1 << 31), dict(width=0),
          dict(table_stride=7), dict(num_rows=0), dict(q_type=KVATTN_E4M3), dict(q_type=5), dict(kv_type=KVATTN_FP16),
          dict(block_stride=4096), dict(block_stride=8200), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
          dict(k_scale=0.0), dict(k_scale=math.inf), dict(v_scale=math.nan), dict(device=-1), dict(device=64)]
POINTERS = [dict(q=None), dict(out=None), dict(k=None), dict(v=None), dict(table=None), dict(lens=None),
            dict(q_offsets=None), dict(error=None), dict(q=X + 8), dict(out=X + 2), dict(k=X + 8), dict(v=X + 4),
            dict(q_stride=1020), dict(q_head_stride=4), dict(q_stride=0), dict(q_head_stride=-128), dict(out_stride=1001), dict(out_head_stride=130)]


@pytest.mark.parametrize("bad", SHAPES, ids=str)
def test_malformed_shapes_are_refused(bad):
    p = C.addressof(d := desc(**bad))
    assert lib.kv_attn_workspace_bytes(p) == -errno.EINVAL
    assert lib.kv_attn_launch(p, None) == -errno.EINVAL, d


@pytest.mark.parametrize("bad", POINTERS, ids=str)
def test_malformed_pointers_are_refused(bad):
    p = C.addressof(d := desc(**bad))
    assert lib.kv_attn_workspace_bytes(p) >= 0
    assert lib.kv_attn_launch(p, None) == -errno.EINVAL, d


def test_limits_and_empty_calls():
    assert lib.kv_attn_launch(None, None) == -errno.EINVAL
    assert lib.kv_attn_workspace_bytes(None) == -errno.EINVAL
    d = desc(num_seqs=KVATTN_MAX_SEQS + 1)
    assert lib.kv_attn_launch(C.addressof(d), None) == -errno.E2BIG
    n0 = lib.crosscache_kernel_launches()
    for empty in (desc(num_seqs=0), desc(total_q=0, q=None, out=None)):
        assert lib.kv_attn_launch(C.addressof(empty), None) == 0
    assert lib.crosscache_kernel_launches() == n0


def layout(**k):
    return KVLayout(**{**dict(num_layers=1, num_blocks=8, block_size=16, hidden_dim_size=256, element_size=2, kv=2), **k})


@pytest.mark.parametrize("make, match", [
    (lambda: TreeAttention(layout(kv=1), [X], None, 8, 2), "K and V"),
    (lambda: TreeAttention(layout(), [X, X], [X], 8, 2), "one pointer"),
    (lambda: TreeAttention(layout(), [X], [X], 8, 3), "must divide"),
    (lambda: TreeAttention(layout(), [X], [X], 8, 0), "must divide"),
    (lambda: TreeAttention(layout(), [X], [X], 258, 2), "at most 128"),
    (lambda: TreeAttention(layout(hidden_dim_size=240), [X], [X], 8, 2), "multiple of 16"),
    (lambda: TreeAttention(layout(hidden_dim_size=1024), [X], [X], 8, 2), "multiple of 16"),
    (lambda: TreeAttention(layout(element_size=4), [X], [X], 8, 2), "1 or 2-byte"),
    (lambda: TreeAttention(layout(head_bytes=128), [X], [X], 8, 2), "head-major"),
    (lambda: TreeAttention(layout(), [X + 8], [X], 8, 2), "aligned"),
    (lambda: TreeAttention(layout(), [X], [0], 8, 2), "aligned"),
    (lambda: TreeAttention(layout(), [X], [X], 8, 2, scale=0.0), "above 0"),
    (lambda: TreeAttention(layout(), [X], [X], 8, 2, k_scale=-1.0), "above 0"),
    (lambda: TreeAttention(layout(), [X], [X], 8, 2, v_scale=math.inf), "finite"),
])
def test_construction_refuses(make, match):
    with pytest.raises(ValueError, match=match):
        make()


def test_calls_refuse_tensors_they_cannot_use():
    att = TreeAttention(layout(), [X], [X], 8, 2)
    i32 = torch.zeros(4, dtype=torch.int32)
    for q in (torch.zeros(4, 8, 128, dtype=torch.bfloat16), torch.zeros(4, 8, 128), torch.zeros(4, 1024)):
        with pytest.raises(ValueError, match="q: expected"):
            att(0, q, torch.zeros(4, 2, dtype=torch.int32), i32, torch.zeros(5, dtype=torch.int32))


PROBE = r"""
#include <stdio.h>
#include <stddef.h>
#include "kvattn.h"
#define F(f) printf(#f " %zu\n", offsetof(struct kv_attn_desc, f))
int main(void) {
  printf(" %zu\n", sizeof(struct kv_attn_desc));
  F(parents); F(workspace_bytes); F(table_stride); F(out_head_stride); F(width); F(head_major); F(kv_type); F(v_scale); F(device);
  return 0;
}
"""


def test_struct_layout(tmp_path):
    (tmp_path / "p.c").write_text(PROBE)
    subprocess.run(["gcc", "-std=c11", f"-I{INCLUDE}", str(tmp_path / "p.c"), "-o", str(tmp_path / "p")], check=True)
    out = subprocess.run([str(tmp_path / "p")], capture_output=True, text=True, check=True).stdout
    for line in out.splitlines():
        field, val = line.split(" ")
        assert (getattr(KvAttnDesc, field).offset if field else C.sizeof(KvAttnDesc)) == int(val), field


def test_packed_descriptor():
    """the descriptor that a call packs is the struct"""
    from demo_b200.attention import _DESC

    values = [*range(1, 13), *range(101, 108), *range(201, 211), 1, 2, 0.5, 0.25, 2.0, 7]
    d = KvAttnDesc.from_buffer_copy(_DESC.pack(*values))
    assert _DESC.size == C.sizeof(KvAttnDesc)
    assert [getattr(d, name) for name, _ in KvAttnDesc._fields_] == values


def test_the_oracle_on_a_case_worked_by_hand():
    """scores 0 everywhere: the mean of the values seen"""
    q = torch.zeros(4, 2, 16, dtype=torch.bfloat16)
    k = torch.randn(3, 2, 1, 16, dtype=torch.float64)
    v = torch.arange(6, dtype=torch.float64).reshape(3, 2, 1, 1).expand(3, 2, 1, 16)
    # one row, pages 2 and 0: values 4, 5, 0, 1; 1 cached token, then the path 0 - 2 and a padding node
    out, lse, _, _ = oa.attention(q[:3], k, v, [[2, 0]], [4], [0, 3], [-1, -2, 0])
    assert out[:, 0, 0].tolist() == [4.5, 0.0, 10 / 3]
    assert lse[:, 1].tolist() == pytest.approx([math.log(2), -math.inf, math.log(3)])
    assert oa.visible(None, 3) == [{0}, {0, 1}, {0, 1, 2}]
    assert oa.visible([-1, -2, 1, 0, 7], 5) == [{0}, None, {2}, {0, 3}, None]


@pytest.mark.parametrize("bad", [dict(out_stride=0), dict(out_stride=-1024), dict(out_head_stride=0), dict(out_head_stride=-128)], ids=str)
def test_results_that_would_lie_over_each_other_are_refused(bad):
    d = desc(**bad)
    assert lib.kv_attn_launch(C.addressof(d), None) == -errno.EINVAL


def test_too_many_queries_are_refused():
    d = desc(total_q=(1 << 27) + 1)
    assert lib.kv_attn_launch(C.addressof(d), None) == -errno.E2BIG


def test_a_stream_of_another_device_is_refused():
    from types import SimpleNamespace

    from demo_b200.pages import _on_stream

    with pytest.raises(ValueError, match="cuda:0"):
        _on_stream(SimpleNamespace(device_index=1), 0)


def typed(dtype, **k):
    return layout(dtype=dtype, element_size=dtype.itemsize, **k)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.float8_e5m2, torch.int16, torch.float8_e4m3fnuz], ids=str)
def test_caches_of_other_types_are_refused(dtype):
    with pytest.raises(ValueError, match="values, not"):
        TreeAttention(typed(dtype), [X], [X], 8, 2)


@pytest.mark.parametrize("held, said", [(torch.bfloat16, torch.float16), (torch.float8_e5m2, torch.float8_e4m3fn), (torch.float16, torch.float8_e4m3fn),
                                        (torch.uint8, torch.float8_e5m2), (torch.uint8, torch.bfloat16), (torch.int16, torch.float8_e4m3fn),
                                        (torch.int16, torch.float32)], ids=str)
def test_a_type_that_the_cache_does_not_hold_is_refused(held, said):
    with pytest.raises(ValueError, match="kv_dtype|values, not"):
        TreeAttention(typed(held), [X], [X], 8, 2, kv_dtype=said)


def test_what_a_cache_holds():
    make = lambda lay, said=None: TreeAttention(lay, [X], [X], 8, 2, kv_dtype=said).kv_dtype
    for t in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
        assert make(typed(t)) is make(typed(t), t) is make(layout(element_size=t.itemsize), t) is t
    assert make(typed(torch.uint8), torch.float8_e4m3fn) is torch.float8_e4m3fn
    assert make(typed(torch.int16), torch.bfloat16) is torch.bfloat16
    assert make(layout()) is None and make(layout(element_size=1)) is torch.float8_e4m3fn


class OnGpu:
    """stands for a CUDA tensor in the checks that come before anything is launched"""

    def __init__(self, shape, dtype, index=0):
        self.t, self.index = torch.zeros(shape, dtype=dtype), index

    def get_device(self):
        return self.index

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("held, queries", [(torch.bfloat16, torch.float16), (torch.float16, torch.bfloat16)], ids=str)
def test_queries_of_another_type_than_the_cache_are_refused(held, queries):
    att = TreeAttention(typed(held), [X], [X], 8, 2)
    i32 = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="over a cache of"):
        att(0, OnGpu((4, 8, 128), queries), i32.view(2, 2), i32, i32)


def test_layouts_know_what_their_tensors_hold():
    from demo_b200.cache import layout_from_kv_tensors

    for dtype in (torch.bfloat16, torch.float16, torch.uint8):
        lay, _, _ = layout_from_kv_tensors([torch.zeros(2, 4, 16, 2, 64, dtype=dtype)])
        assert lay.dtype is dtype
        assert lay == KVLayout(1, 4, 16, 128, dtype.itemsize, 2)       # two layouts are the same when their bytes are


@pytest.mark.parametrize("at, match", [(1, "cuda:1, not on cuda:0"), (-errno.EINVAL, "not memory that a GPU reaches")])
def test_queries_on_another_device_than_the_cache_are_refused(monkeypatch, at, match):
    monkeypatch.setattr(lib, "kv_page_device_of", lambda p: at)
    att = TreeAttention(typed(torch.bfloat16), [X], [X], 8, 2)
    i32 = torch.zeros(4, dtype=torch.int32)
    n0 = lib.crosscache_kernel_launches()
    with pytest.raises(ValueError, match=match):
        att(0, OnGpu((4, 8, 128), torch.bfloat16), OnGpu((2, 2), torch.int32), i32, i32[:3])
    assert lib.crosscache_kernel_launches() == n0


def test_gradients_of_every_kind_and_traces_are_refused():
    """before anything is looked at, so that the refusal shows without a GPU"""
    from torch.autograd import forward_ad

    att = TreeAttention(layout(), [X], [X], 8, 2)
    i32 = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    call = lambda x: att(0, x, torch.zeros(4, 2, dtype=torch.int32), i32, torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="no gradients"):
        call(q.clone().requires_grad_())
    for guard in (torch.enable_grad(), torch.no_grad()):
        with guard, forward_ad.dual_level():
            with pytest.raises(ValueError, match="no gradients"):
                call(forward_ad.make_dual(q, torch.ones_like(q)))
            with pytest.raises(ValueError, match="q: expected"):
                call(q)                             # a tensor without a tangent is no reason
    with pytest.raises(ValueError, match="no gradients"):
        torch.func.jvp(call, (q,), (torch.ones_like(q),))
    with pytest.raises(ValueError, match="no gradients"):
        torch.func.grad(lambda x: call(x).sum())(q.float())
    with pytest.raises(Exception, match="cannot be traced"):
        torch.jit.trace(call, (q,))
    with torch.no_grad(), pytest.raises(ValueError, match="q: expected"):
        call(q.clone().requires_grad_())


@pytest.mark.parametrize("dtype, half_step", [(torch.float16, 2.0 ** -25), (torch.bfloat16, 2.0 ** -134)], ids=str)
def test_the_bound_of_results_below_the_normal_range(dtype, half_step):
    """a result that is exact in 64 bits and halfway between two numbers of the type"""
    q = torch.zeros(1, 1, 16, dtype=dtype)
    v = torch.full((1, 1, 1, 16), 3 * half_step, dtype=torch.float64)
    out, _, tol, _ = oa.attention(q, torch.zeros(1, 1, 1, 16, dtype=torch.float64), v, [[0]], [1], [0, 1])
    off = (out.to(dtype).double() - out).abs()
    assert (off == half_step).all() and (off <= tol).all()
