"""4-bit attention where its work is cut into runs: rows by token (heads side by side in a CTA
where their number allows), long lists of pages, pools of unlike layouts, many short units."""
import numpy as np
import pytest
import torch

import int4_plain as plain
from test_gpu_int4 import BF, FP, U, check_attention, filled, i32, randn, rows_of, table_of, zs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,dim,page,group,dtype", [
    (32, 8, 128, 16, 32, FP), (16, 4, 64, 64, 64, BF), (64, 2, 128, 32, 64, BF), (12, 12, 64, 16, 32, FP),
    (12, 3, 128, 64, 64, BF)])
@pytest.mark.parametrize("lens", [[4000, 0, 1, 1023, 2500], [9000], [700] * 40])
def test_rows_by_token(hq, hkv, dim, page, group, dtype, lens):
    table, blocks = table_of(lens, page, seed=3)
    kp, vp = filled(blocks, page, hkv, dim, group, "tokens", seed=hq)
    q = randn(len(lens), hq, dim, seed=1).to(dtype)
    a = check_attention(q, kp, vp, table, lens, page)
    # the same rows, each head's together: the same sums
    other = []
    for p in (kp, vp):
        x = zs().int4_pages(blocks, page, hkv, dim, group, "heads")
        x.codes.copy_(p.codes)
        x.params.copy_(p.params)
        other.append(x)
    b = check_attention(q, *other, table, lens, page)
    check_attention(q, kp, other[1], table, lens, page)
    assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -5 * float(a.double().abs().max())


@pytest.mark.parametrize("hq,hkv,page,group,dtype", [(8, 2, 64, 64, BF), (24, 2, 16, 32, FP)])
def test_long_lists_of_pages(hq, hkv, page, group, dtype):
    dim, lens, top = 128, [30001, 9000], 400
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, hkv, dim, group, seed=6)
    q = randn(len(lens), hq, dim, seed=2).to(dtype)
    rng = np.random.default_rng(0)
    pages, counts = np.full((len(lens), hkv, top), -1, np.int32), np.zeros((len(lens), hkv), np.int32)
    for r, n in enumerate(lens):
        for h in range(hkv):
            have = -(-n // page)
            counts[r, h] = min(have, top - 7 * h)
            pages[r, h, :counts[r, h]] = rng.permutation(have)[:counts[r, h]]
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens), pages=i32(pages), counts=i32(counts))
    g = hq // hkv
    for r, n in enumerate(lens):
        k, v = rows_of(kp, table[r], n, page), rows_of(vp, table[r], n, page)
        for h in range(hkv):
            t = (pages[r, h, :counts[r, h], None] * page + np.arange(page)).ravel()
            t = torch.as_tensor(t[t < n], device="cuda", dtype=torch.long)
            kk, vv, qq = k[t][:, h:h + 1], v[t][:, h:h + 1], q[r, h * g:(h + 1) * g]
            want, _ = plain.attend(qq, kk, vv, dim ** -0.5)
            err = plain.attention_error(qq, kk, vv, kp.params, dim ** -0.5, n)
            off = (o[r, h * g:(h + 1) * g].double() - want).abs()
            assert bool((off <= U[dtype] * want.abs() + err * float(vv.abs().max()) + 2.0 ** -25).all()), (r, h)


def test_a_wide_table_with_short_sequences():
    """The table's width, not the lengths, chooses runs; a close bound chooses units."""
    page, lens = 64, [97, 0, 300, 1, 64, 65]
    table, blocks = table_of(lens, page, width=700)
    kp, vp = filled(blocks, page, 2, 128, 64, seed=9)
    q = randn(len(lens), 8, 128, seed=2).to(BF)
    check_attention(q, kp, vp, table, lens, page)
    check_attention(q, kp, vp, table, lens, page, max_seqlen=300)
    check_attention(q, kp, vp, table, lens, page, max_seqlen=100000)


def test_two_graphs_replayed_side_by_side():
    """Each call's workspace is its own, in a graph too: attention and sampling of two graphs on
    two streams at once give what eager calls give."""
    page, graphs = 64, []
    for seed, lens in ((1, [9000, 100, 3000]), (2, [20000])):
        table, blocks = table_of(lens, page, seed=seed)
        kp, vp = filled(blocks, page, 2, 128, 64, seed=seed)
        q = randn(len(lens), 8, 128, seed=seed).to(BF)
        t, n = i32(table), i32(lens)
        x = randn(len(lens), 40000, seed=seed) * 3
        u = torch.rand(len(lens), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        want = zs().paged_attention_int4(q, kp, vp, t, n), zs().sample(x, u, 0.9, 0, 0.9)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            got = zs().paged_attention_int4(q, kp, vp, t, n), zs().sample(x, u, 0.9, 0, 0.9)
        graphs.append((g, side, got, want, (q, kp, vp, t, n, x, u)))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, side, *_ in graphs:
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for _, _, got, want, _ in graphs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
