"""Which kernel 4-bit attention takes, without a GPU: a call that needs no workspace gives each
unit a fixed number of warps, others deal runs of chunks. The sizes are ones that were timed in
both forms, beside the limits in paged_int4_attention.cu."""
import ctypes as C

import pytest

from test_int4_args import attention, pool, zlib  # noqa: F401


@pytest.mark.parametrize("batch,tokens,listed,runs", [
    (1, 2000, 0, False), (16, 1000, 0, False), (32, 1000, 0, False), (300, 600, 0, False), (512, 300, 0, False),
    (32, 1500, 0, True), (32, 2000, 0, True), (64, 2000, 0, True), (1, 4129, 0, True),
    (8, 8192, 16, False), (8, 8192, 64, False), (200, 2048, 8, False), (32, 8192, 64, True), (128, 2048, 16, True),
    (8, 32768, 256, True), (1, 8192, 64, True)])
def test_the_choice(zlib, batch, tokens, listed, runs):  # noqa: F811
    f = zlib.zs_paged_attention_int4_workspace
    f.restype = C.c_size_t
    p = dict(page_size=64, num_heads=8, codes_block=64 * 8 * 64, codes_head=64 * 64, params_block=64 * 8 * 4, params_head=64 * 4)
    width = -(-tokens // 64)
    more = dict(pages=256, counts=256, top=listed) if listed else {}
    a = attention(pool(**p), pool(**p), B=batch, Hq=32, width=width, table_stride=width, **more)
    assert (f(C.byref(a)) > 0) == runs
    if not listed:                        # a close bound counts as the table's width does
        a = attention(pool(**p), pool(**p), B=batch, Hq=32, width=4096, table_stride=4096, max_seqlen=tokens)
        assert (f(C.byref(a)) > 0) == runs
