"""Paged attention writes its workspace and nothing around it."""
import ctypes as C

import pytest
import torch

from test_gpu_paged import BF, DEV, Cache, zs
from test_paged_args import STRUCTS
from test_paged_workspace import formula

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


@pytest.mark.parametrize("lens,hq,hkv,D", [([70000], 4, 1, 128), ([70000, 3], 16, 2, 64), ([50000], 9, 1, 128), ([50000], 16, 1, 64),
                                           ([50001, 0], 20, 1, 128), ([9000] * 9, 32, 4, 128)])
def test_nothing_around_the_workspace_is_written(lens, hq, hkv, D):
    from zipserv_asplos26_b200._lib import lib
    f, need = lib().zs_paged_attention, lib().zs_paged_attention_workspace
    f.argtypes, f.restype, need.argtypes, need.restype = [C.c_char_p], C.c_int, [C.c_char_p], C.c_size_t
    c = Cache(lens, hkv, D, 64, BF, "heads", seed=hq)
    q = torch.randn(len(lens), hq, D, device=DEV).to(BF)
    want = zs().paged_attention(q, c.k, c.v, c.table, c.lens)
    out = torch.zeros_like(q)
    pools = [x for t in (c.k, c.v) for x in (t.data_ptr(), *t.stride()[:3], *t.shape, 0)]

    def args(ws, n):
        return STRUCTS["ZsPagedAttention"].pack(
            torch.cuda.current_stream().cuda_stream, q.data_ptr(), c.table.data_ptr(), c.table.stride(0), c.lens.data_ptr(), 0, 0,
            ws, n, out.data_ptr(), 0, 0, *pools, len(lens), hq, c.table.shape[1], 0, D ** -0.5, 0)

    n = need(args(0, 0))
    assert n == formula(len(lens), hq, hkv, D)
    block = torch.full((GUARD + n + GUARD,), 0x5A, dtype=torch.uint8, device=DEV)
    assert f(args(block.data_ptr() + GUARD, n)) == 0
    torch.cuda.synchronize()
    assert bool((block[:GUARD] == 0x5A).all() and (block[GUARD + n:] == 0x5A).all())
    assert torch.equal(out, want)
