"""4-bit attention and what its exponentials refer to: warps that attend nothing beside ones
whose scores are all far below zero. Softmax does not see a shift, so neither may the joins.

Tolerances are test_gpu_int4.check_attention's."""
import math

import numpy as np
import pytest
import torch

import int4_plain as plain
from test_gpu_int4 import BF, FP, U, TINY, check_attention, filled, i32, randn, rows_of, table_of, zs

pytestmark = pytest.mark.gpu


def shifted(q_shape, pool, at, page, scores, dim, group, seed=0):
    """q of ones and a little noise, and the rows at slots `at` of every head overwritten by keys
    whose scores, at 1 / sqrt(dim), are near `scores` (natural units)."""
    x = (scores / math.sqrt(dim)).view(-1, 1, 1) + 0.2 * randn(len(at), pool.codes.shape[2], dim, seed=seed)
    pool.codes[at // page, at % page], pool.params[at // page, at % page] = plain.quantise(x, group)
    return 1 + 0.05 * randn(*q_shape, seed=seed + 1)


def all_at(level, lens, hq, hkv, dim, page, group, dtype, width=None, layout="heads", seed=0):
    """A cache whose scores are all near `level`."""
    table, blocks = table_of(lens, page, seed=seed, width=width)
    kp, vp = filled(blocks, page, hkv, dim, group, layout, seed=seed)
    at = torch.arange(blocks * page, device="cuda")
    q = shifted((len(lens), hq, dim), kp, at, page, torch.full((len(at),), float(level), device="cuda"), dim, group, seed)
    return q.to(dtype), kp, vp, table


@pytest.mark.parametrize("level", [-300.0, -150.0, -100.0, -60.0, 0.0, 200.0])
@pytest.mark.parametrize("hq,hkv,dim,page,group,dtype", [
    (8, 2, 128, 64, 64, BF), (12, 1, 128, 16, 32, FP), (4, 4, 64, 16, 32, BF), (3, 1, 64, 64, 64, FP), (16, 1, 64, 32, 32, BF)])
def test_short_sequences_beside_longer_ones(level, hq, hkv, dim, page, group, dtype):
    """From 4 warps a sequence to 16, most of which have no tokens."""
    lens = [1, 2, 7, 15, 16, 17, 31, 33, 40, 300]
    for width in (None, 1024 // page, 4096 // page):
        q, kp, vp, table = all_at(level, lens, hq, hkv, dim, page, group, dtype, width=width)
        check_attention(q, kp, vp, table, lens, page)
    q, kp, vp, table = all_at(level, lens[:1], hq, hkv, dim, page, group, dtype)
    for most in (32, 128, 300, 700, 1500):
        wide = np.pad(table, ((0, 0), (0, 1500 // page)), constant_values=-1)
        check_attention(q, kp, vp, wide, lens[:1], page, max_seqlen=most)


@pytest.mark.parametrize("level", [-300.0, -80.0, -60.0])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_constant_values_at_low_scores(level, dtype):
    """Values without a range let weights go up to 2^55: an empty warp counted from some -50 on."""
    page, dim, lens = 16, 128, [1, 5, 40, 300]
    q, kp, vp, table = all_at(level, lens, 8, 2, dim, page, 64, dtype)
    codes, params = plain.quantise(torch.full((len(vp.codes), page, 2, dim), -3.0, device="cuda"), 64)
    vp.codes.copy_(codes)
    vp.params.copy_(params)
    check_attention(q, kp, vp, table, lens, page)


def kept_rows(table, n, page, blocks):
    """The tokens of a row of `table` whose pages are in the pool."""
    t = np.arange(n)
    ok = (table[t // page] >= 0) & (table[t // page] < blocks)
    return t[ok]


@pytest.mark.parametrize("level", [-200.0, 0.0])
@pytest.mark.parametrize("n,width", [(300, None), (20000, None), (9000, 4096)])
@pytest.mark.parametrize("g", [4, 12])
def test_pieces_whose_pages_are_all_refused(level, n, width, g):
    """Most of a sequence's pages lie outside the pool: whole warps have none."""
    page, dim, hkv = 16, 128, 2
    q, kp, vp, table = all_at(level, [n], g * hkv, hkv, dim, page, 64, BF, width=width)
    blocks = len(kp.codes)
    good = table.copy()
    pages = -(-n // page)
    table[0, :pages * 2 // 3] = blocks + 5
    err, lse = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(1, g * hkv, device="cuda")
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32([n]), lse=lse, err=err)
    assert int(err) == 2
    t = kept_rows(table[0], n, page, blocks)
    k, v = (rows_of(p, good[0], n, page)[t] for p in (kp, vp))
    want, sums = plain.attend(q[0], k, v, dim ** -0.5)
    bound = plain.attention_error(q[0], k, v, kp.params, dim ** -0.5, n)
    off = (o[0].double() - want).abs()
    assert bool((off <= U[BF] * want.abs() + bound * float(v.abs().max())).all()), float(off.max())
    assert float((lse[0].double() - sums).abs().max()) <= 2 * bound + 2.0 ** -20 * float(1 + sums.abs().max())


@pytest.mark.parametrize("level", [-200.0, -60.0])
@pytest.mark.parametrize("top,page", [(6, 64), (400, 16), (30, 32)])
@pytest.mark.parametrize("dtype,g", [(BF, 4), (FP, 9)])
def test_lists_whose_first_pages_are_refused(level, top, page, dtype, g):
    """Lists that begin with logical pages past the table and pages behind the length; lse too."""
    dim, hkv = 128, 2
    n = page * (top - top // 2) - 3
    width = top + 4
    q, kp, vp, table = all_at(level, [n, n], g * hkv, hkv, dim, page, 64, dtype, width=width)
    have = -(-n // page)
    pages = np.full((2, hkv, top), -1, np.int32)
    pages[..., :top // 2] = np.arange(width, width + top // 2)
    pages[..., top // 2:top // 2 + have] = np.arange(have)[::-1]
    pages[1, :, :min(4, top // 2)] = np.arange(have, have + min(4, top // 2))          # behind the length: no error
    counts = np.full((2, hkv), top // 2 + have, np.int32)
    err, lse = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.empty(2, g * hkv, device="cuda")
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32([n, n]), pages=i32(pages), counts=i32(counts), lse=lse, err=err)
    assert int(err) == 2
    for r in range(2):
        k, v = (rows_of(p, table[r], n, page) for p in (kp, vp))
        want, sums = plain.attend(q[r], k, v, dim ** -0.5)
        bound = plain.attention_error(q[r], k, v, kp.params, dim ** -0.5, n)
        off = (o[r].double() - want).abs()
        assert bool((off <= U[dtype] * want.abs() + TINY[dtype] + bound * float(v.abs().max())).all()), (r, float(off.max()))
        assert float((lse[r].double() - sums).abs().max()) <= 2 * bound + 2.0 ** -20 * float(1 + sums.abs().max())
