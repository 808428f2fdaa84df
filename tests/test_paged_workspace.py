"""The attention workspace's size, by the formula of its parts: a plan (the chunks
a warp and each unit's first chunk, 8 bytes each, to whole 256 bytes), and for each
of the warps that the GPU holds two pieces of up to 16 heads, each head with its
maximum, sum and D outputs in 32 bits."""
import ctypes as C

import pytest

from test_paged_args import STRUCTS, _fn, zlib  # noqa: F401

CTAS = {(64, True): 4, (128, True): 3, (64, False): 3, (128, False): 2}     # an SM, by head dim and G <= 8
CASES = [(1, 32, 8, 128), (1, 8, 8, 64), (7, 56, 8, 128), (3, 64, 8, 64), (2, 9, 1, 128), (5, 16, 1, 64), (5, 16, 1, 128),
         (4, 20, 1, 128), (33, 128, 2, 64), (1000, 64, 8, 128)]


def formula(B, hq, hkv, D):
    G = hq // hkv
    units = B * hkv * -(-G // 16)
    warps = 148 * CTAS[D, G <= 8] * 4
    return -(-(1 + units) * 8 // 256) * 256 + 2 * warps * min(G, 16) * (D + 2) * 4


@pytest.mark.parametrize("B,hq,hkv,D", CASES)
def test_workspace_is_its_parts(zlib, B, hq, hkv, D):  # noqa: F811
    assert _fn(zlib, "zs_paged_attention_workspace_bytes", [C.c_int] * 4, C.c_size_t)(B, hq, hkv, D) == formula(B, hq, hkv, D)
    # a call in runs of chunks asks for as much (a table of 2^20 pages: no bound on the lengths); one token a row for none
    need = _fn(zlib, "zs_paged_attention_workspace", res=C.c_size_t)
    a, pool = 1 << 20, (1 << 20, 16 * hkv * D, hkv * D, D, 4, 16, hkv, D, 0)
    for width, most, want in ((1 << 20, 0, formula(B, hq, hkv, D)), (1, 0, 0), (1 << 20, 1, 0)):
        args = STRUCTS["ZsPagedAttention"].pack(0, a, a, width, a, 0, 0, 0, 0, a, 0, 0, *pool, *pool, B, hq, width, 0, 0.1, most)
        assert need(args) == want, (width, most)
