"""4-bit attention where the reference of the exponentials moves after tokens that only some
lanes of a warp hold: pages with few tokens that come first, outliers far above the rest.

Tolerances are test_gpu_int4.check_attention's."""
import numpy as np
import pytest
import torch

import int4_plain as plain
from test_gpu_int4 import BF, FP, U, TINY, check_attention, filled, i32, randn, rows_of, table_of, zs
from test_gpu_int4_references import shifted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rest", [1, 3, 7, 8, 9])
@pytest.mark.parametrize("page,pages", [(16, 5), (32, 5), (64, 6), (128, 4), (256, 3), (64, 400), (32, 300)])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("dtype,g,dim,group", [(BF, 4, 128, 64), (FP, 12, 128, 32), (FP, 8, 64, 64), (BF, 16, 64, 32)])
def test_a_short_last_page_anywhere_in_the_list(rest, page, pages, place, dtype, g, dim, group):
    """The last page's few tokens, then others of larger scores and values, and the reverse."""
    hkv, n = 2, (pages - 1) * page + rest
    table, blocks = table_of([n, n], page, seed=rest)
    kp, vp = filled(blocks, page, hkv, dim, group, seed=page)
    last = torch.arange(n - rest, n, device="cuda")
    for r in range(2):
        t = torch.as_tensor(table[r], device="cuda").long()
        at = t[torch.arange(n, device="cuda") // page] * page + torch.arange(n, device="cuda") % page
        scores = 4.0 * torch.arange(n, device="cuda") / n
        scores[last] = (-12.0, 9.0)[r]
        q1 = shifted((2, g * hkv, dim), kp, at, page, scores, dim, group, seed=3)
        vp.params[at[last] // page, at[last] % page] *= (2.0 ** -8, 1.0)[r]
    q = q1.to(dtype)
    order = np.arange(pages - 1)
    cut = {"first": 0, "middle": (pages - 1) // 2, "last": pages - 1}[place]
    order = np.concatenate([order[:cut], [pages - 1], order[cut:]]).astype(np.int32)
    lists = np.broadcast_to(order, (2, hkv, pages)).copy()
    lse = torch.empty(2, g * hkv, device="cuda")
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32([n, n]), pages=i32(lists),
                                  counts=i32(np.full((2, hkv), pages)), lse=lse)
    for r in range(2):
        k, v = (rows_of(p, table[r], n, page) for p in (kp, vp))
        want, sums = plain.attend(q[r], k, v, dim ** -0.5)
        bound = plain.attention_error(q[r], k, v, kp.params, dim ** -0.5, n)
        off = (o[r].double() - want).abs()
        assert bool((off <= U[dtype] * want.abs() + TINY[dtype] + bound * float(v.abs().max())).all()), (r, float(off.max()))
        assert float((lse[r].double() - sums).abs().max()) <= 2 * bound + 2.0 ** -20 * float(1 + sums.abs().max())


@pytest.mark.parametrize("n,width", [(200, None), (3000, None), (200, 1000), (20000, None)])
@pytest.mark.parametrize("peaks", [((10, 150.0), (70, 155.0)), ((3, 120.0), (100, 200.0)), ((0, 150.0), (33, 152.0), (90, 156.0)),
                                   ((17, 150.0), (65, 140.0), (127, 160.0))])
@pytest.mark.parametrize("dtype,g,dim,group", [(BF, 4, 64, 64), (FP, 12, 128, 32), (BF, 9, 128, 64), (FP, 1, 64, 32)])
def test_outliers_one_after_another(n, width, peaks, dtype, g, dim, group):
    """Scores far above the rest, each higher than those before it, in different steps of a warp."""
    page = 64
    table, blocks = table_of([n], page, width=width)
    kp, vp = filled(blocks, page, 1, dim, group, seed=n)
    i = torch.arange(n, device="cuda")
    at = torch.as_tensor(table[0], device="cuda").long()[i // page] * page + i % page
    scores = torch.zeros(n, device="cuda")
    for t, x in peaks:
        scores[t] = x
    q = shifted((1, g, dim), kp, at, page, scores, dim, group, seed=2).to(dtype)
    check_attention(q, kp, vp, table, [n], page)
    check_attention(q, kp, vp, table, [n], page, max_seqlen=n)
