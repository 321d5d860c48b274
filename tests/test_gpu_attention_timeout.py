"""Failure detection inside the attention kernel, without a GPU fault.

Every wait of kv_attn_kernel is bounded.  kv_attn_launch_stalled gives the
barrier of the first CTA's first tile of V one arrival that nobody makes: the
waits for it run out after some 20 milliseconds, every role leaves, the loads and
products in flight settle, the CTA frees its TMEM, and the host reads the error
bit.  The next call on the same context is right."""
import ctypes as C
import time

import pytest
import torch

from demo_b200._lib import KVATTN_BF16, KVATTN_E4M3, KVATTN_ERR_TIMEOUT, KvAttnDesc, lib
from tests.test_gpu_attention import BF16, E4M3, Batch, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("block, kvt", [(16, BF16), (24, BF16), (16, E4M3)], ids=["boxes", "copies", "8bit"])
def test_a_wait_runs_out_then_the_next_call_is_right(block, kvt, dim):
    # long enough for every CTA to have tiles: its beginning costs 3 of the 19 of a head
    b = Batch([1000] * 40, [2] * 40, heads=8, kv_heads=4, dim=dim, block=block, kvt=kvt, seed=dim)
    (_, q, table, lens, off), _ = b.args()
    total, heads, _ = q.shape
    out = torch.empty_like(q)
    lse = torch.empty(total, heads, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    d = KvAttnDesc(q=q.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), k=b.k[0], v=b.v[0], table=table.data_ptr(), lens=lens.data_ptr(),
                   q_offsets=off.data_ptr(), error=err.data_ptr(), block_stride=b.layout.block_stride, table_stride=table.stride(0),
                   q_stride=q.stride(0), q_head_stride=q.stride(1), out_stride=out.stride(0), out_head_stride=out.stride(1),
                   width=table.shape[1], num_rows=table.shape[0], num_seqs=len(b.lens), total_q=total, num_pages=b.layout.num_blocks,
                   block_size=block, num_heads=heads, num_kv_heads=4, head_dim=dim, q_type=KVATTN_BF16,
                   kv_type=KVATTN_E4M3 if kvt == E4M3 else KVATTN_BF16, scale=dim ** -0.5, k_scale=b.scales[0], v_scale=b.scales[1])
    need = lib.kv_attn_workspace_bytes(C.addressof(d))
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    d.workspace, d.workspace_bytes = work.data_ptr(), need
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.kv_attn_launch(C.addressof(d), stream) == 0      # loads the kernels
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    want = b.expected()
    took = []
    for _ in range(3):
        t0 = time.perf_counter()
        assert lib.kv_attn_launch_stalled(C.addressof(d), stream) == 0
        torch.cuda.synchronize()
        took.append(time.perf_counter() - t0)
        assert int(err.item()) == KVATTN_ERR_TIMEOUT
        err.zero_()
        out.fill_(7)
        assert lib.kv_attn_launch(C.addressof(d), stream) == 0
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        close(out, lse, want)
    # two waits one after the other, of a 64th of the ordinary limit each: the latter is about a second
    assert min(took) < 0.1
