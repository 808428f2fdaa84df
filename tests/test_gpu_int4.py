"""4-bit paged KV cache: quantising write, read back and attention against plain forms
(int4_plain.py), and PagedKVCache with bits=4.

Codes and parameters are equal: the kernel makes the formula's fp32 steps. A row read back
is the value rounded once. An attention output is the 64-bit one over the same values, off
by attention_error(...) max |v| and then rounded once (u relative, plus half of fp16's
smallest step)."""
import math

import numpy as np
import pytest
import torch

import int4_plain as plain

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
BF, FP = torch.bfloat16, torch.float16


def zs():
    import zipserv_asplos26_b200
    return zipserv_asplos26_b200


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=gen(seed))


def pools(blocks, page, heads, dim, group, layout="heads"):
    return [zs().int4_pages(blocks, page, heads, dim, group, layout) for _ in range(2)]


def filled(blocks, page, heads, dim, group, layout="heads", seed=0, offset=0.0):
    """Pools of quantised random rows, channels of unlike sizes."""
    out = []
    for i in range(2):
        x = randn(blocks, page, heads, dim, seed=seed + i) * torch.exp(randn(heads, dim, seed=seed + 7 + i)) + offset
        p = zs().int4_pages(blocks, page, heads, dim, group, layout)
        codes, params = plain.quantise(x, group)
        p.codes.copy_(codes)
        p.params.copy_(params)
        out.append(p)
    return out


def table_of(lens, page, seed=0, width=None):
    rng = np.random.default_rng(seed)
    pages = [-(-n // page) for n in lens]
    order = rng.permutation(sum(pages) + 3)
    t = np.full((len(lens), width or max(pages + [1])), -1, np.int32)
    at = 0
    for r, p in enumerate(pages):
        t[r, :p] = order[at:at + p]
        at += p
    return t, sum(pages) + 3


def rows_of(p, table, n, page):
    i = torch.arange(n, device="cuda")
    blk = torch.as_tensor(table, device="cuda").long()[i // page]
    return plain.values(p.codes[blk, i % page], p.params[blk, i % page])


def check_attention(q, kp, vp, table, lens, page, scale=None, out=None, lse=None, **more):
    hq, d = q.shape[1:]
    scale = 1 / math.sqrt(d) if scale is None else scale
    lse = torch.empty(q.shape[0], hq, device="cuda") if lse is None else lse
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens), scale, lse=lse, out=out, **more)
    for r, n in enumerate(lens):
        k, v = rows_of(kp, table[r], n, page), rows_of(vp, table[r], n, page)
        want, sums = plain.attend(q[r], k, v, scale)
        err = plain.attention_error(q[r], k, v, kp.params, scale, n)
        tol = U[q.dtype] * want.abs() + TINY[q.dtype] + err * (float(v.abs().max()) if n else 0.0)
        off = (o[r].double() - want).abs()
        assert bool((off <= tol).all()), (r, n, float((off - tol).max()))
        if n == 0:
            assert bool((lse[r] == -math.inf).all())
        else:
            assert float((lse[r].double() - sums).abs().max()) <= 2 * err + 2.0 ** -20 * float(1 + sums.abs().max()), r
    return o


# ------------------------------------------------------------------- write
def turned_inputs(n, hq, hkv, dim, rot, axes, dtype, seed=0):
    qkv = (randn(n, hq + 2 * hkv, dim, seed=seed) * torch.exp(randn(hq + 2 * hkv, dim, seed=seed + 1))).to(dtype)
    q, k, v = qkv.split([hq, hkv, hkv], 1)
    half = rot // 2
    ang = torch.arange(400, device="cuda")[:, None] * (1e4 ** (-torch.arange(half, device="cuda") / half))[None]
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
    pos = torch.randint(0, 400, (axes, n), device="cuda", generator=gen(seed + 2), dtype=torch.int32)
    sections = [half - (axes - 1) * (half // axes)] + [half // axes] * (axes - 1)
    rows = torch.repeat_interleave(torch.arange(axes), torch.tensor(sections)).cuda()
    at = pos.long()[rows].t()
    chan = torch.arange(half, device="cuda")
    return q, k, v, pos if axes > 1 else pos[0], cos_sin, sections, cos_sin[at, chan].unsqueeze(1), \
        cos_sin[at, half + chan].unsqueeze(1)


@pytest.mark.parametrize("n,hq,hkv,dim,rot,axes,page,group,dtype,layout,interleaved", [
    (1, 1, 1, 64, 64, 1, 16, 64, BF, "heads", False),
    (1, 32, 8, 128, 128, 1, 64, 64, BF, "heads", False),
    (33, 32, 8, 128, 128, 1, 64, 64, BF, "tokens", False),
    (33, 7, 1, 128, 128, 1, 16, 32, BF, "heads", False),
    (37, 24, 4, 128, 64, 3, 16, 32, FP, "tokens", True),
    (37, 6, 3, 128, 48, 2, 32, 64, FP, "heads", False),
    (129, 5, 5, 64, 32, 1, 32, 32, BF, "heads", True),
    (70, 4, 2, 64, 16, 1, 256, 64, FP, "tokens", False),
    (70, 4, 2, 64, 64, 4, 16, 32, FP, "heads", False),
    (5003, 9, 3, 128, 112, 1, 64, 32, BF, "heads", False),
])
def test_write_gives_the_formulas_codes(n, hq, hkv, dim, rot, axes, page, group, dtype, layout, interleaved):
    q, k, v, pos, cos_sin, sections, cos, sin = turned_inputs(n, hq, hkv, dim, rot, axes, dtype)
    blocks = n // page + 3
    kp, vp = pools(blocks, page, hkv, dim, group, layout)
    before = [t.clone() for t in (*kp, *vp)]
    slots = torch.randperm(blocks * page, device="cuda", generator=gen(5))[:n]
    if n > 2:
        slots[1] = -1
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = zs().rope_write_int4(q, k, v, pos, cos_sin, slots, kp, vp, sections, interleaved, err=err)
    dense = [torch.zeros(blocks, page, hkv, dim, dtype=dtype, device="cuda") for _ in range(2)]
    assert torch.equal(out, zs().rope_write(q, k, v, pos, cos_sin, slots, *dense, sections, interleaved))
    live = slots >= 0
    blk, row = slots[live] // page, slots[live] % page
    for x, p, old in ((plain.turn(k, cos, sin, interleaved), kp, before[:2]), (v.float(), vp, before[2:])):
        codes, params = plain.quantise(x[live], group)
        old[0][blk, row], old[1][blk, row] = codes, params
        assert torch.equal(p.codes, old[0])
        assert torch.equal(p.params, old[1])
        off = (plain.values(codes, params) - x[live].double()).abs().unflatten(-1, (-1, group))
        s, c = params.double().unbind(-2)
        assert bool((off <= (s / 2 + (15 * s + c.abs()) / 256).unsqueeze(-1)).all())
    assert int(err) == 0


def test_write_of_ties_flat_tiny_and_odd_groups():
    """Values in the middle of two codes go to the even one; groups without range, tiny ones
    and ones that are not finite have codes of 8, the last reading back as NaN."""
    n, dim, page, group = 12, 64, 16, 32
    v = torch.zeros(n, 1, dim, dtype=FP, device="cuda")
    v[0, 0, :32] = torch.arange(32) * 0.5 - 8.0              # scale 15.5 / 15: no ties, the ends
    v[1, 0, :16] = torch.arange(16) * 0.5
    v[1, 0, 16:32] = torch.arange(16) + 0.0                  # scale 1: halves are ties
    v[2] = 3.0                                               # flat
    v[3, 0, 5] = math.inf
    v[4, 0, 40] = math.nan
    v[5, 0, :32], v[5, 0, 32:] = 65504.0, -65504.0
    v[5, 0, 0], v[5, 0, 63] = -65504.0, 65504.0              # the type's whole range
    v[6] = 2.0 ** -24 * torch.arange(dim, device="cuda")     # fp16's smallest steps
    v[7, 0, 3] = -math.inf
    v[8] = -0.0
    v[9] = 1000.0 + torch.arange(dim, device="cuda") % 2     # the centre's rounding passes the step
    k = v.flip(0).contiguous()
    q = torch.zeros(n, 1, dim, dtype=FP, device="cuda")
    cos_sin = torch.cat([torch.ones(1, 32), torch.zeros(1, 32)], 1).cuda()
    kp, vp = pools(2, page, 1, dim, group)
    slots = torch.arange(n, device="cuda")
    pos = torch.zeros(n, dtype=torch.int32, device="cuda")
    zs().rope_write_int4(q, k, v, pos, cos_sin, slots, kp, vp)
    kk, vv = zs().read_int4(kp, vp, slots, FP)
    one = torch.ones(1, 1, 32, device="cuda")
    for x, p, back in ((plain.turn(k, one, 0 * one, False), kp, kk), (v, vp, vv)):
        codes, params = plain.quantise(x, group)
        assert torch.equal(p.codes[0, :n], codes)
        assert torch.equal(p.params[0, :n].isnan(), params.isnan())
        assert torch.equal(p.params[0, :n].nan_to_num(7.0), params.nan_to_num(7.0))
        assert torch.equal(back.isnan(), plain.values(codes, params).isnan())
    assert bool(vv[3, 0, :32].isnan().all()) and bool((vv[3, 0, 32:] == 0).all())
    assert bool((vv[2] == 3.0).all())
    # bf16 values whose range passes fp32's
    b = torch.zeros(1, 1, dim, dtype=BF, device="cuda")
    b[0, 0, 0], b[0, 0, 1], b[0, 0, 33] = 3.0e38, -3.0e38, 1e-39
    zs().rope_write_int4(b, b, b, pos[:1], cos_sin, slots[:1], kp, vp)
    back = zs().read_int4(kp, vp, slots[:1])[1]
    assert bool(back[0, 0, :32].isnan().all()) and bool((back[0, 0, 32:] == 0).all())


def test_write_in_place_and_bad_indexes():
    n, hkv, dim, page = 9, 2, 128, 16
    q, k, v, pos, cos_sin, _, cos, sin = turned_inputs(n, 4, hkv, dim, 128, 1, BF, seed=3)
    want = plain.turn(q, cos, sin, False)
    whole = q.contiguous()
    kp, vp = pools(2, page, hkv, dim, 64)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots = torch.arange(n, device="cuda")
    got = zs().rope_write_int4(whole, k, v, pos, cos_sin, slots, kp, vp, q_out=whole, err=err)
    assert got is whole and bool(((whole.double() - want.double()).abs() <=
                                  2.0 ** -8 * want.double().abs() + 2.0 ** -22 * q.double().abs().max()).all())
    assert int(err) == 0
    before = [t.clone() for t in (*kp, *vp)]
    for bad in (2 * page, 1 << 40, -2):
        err.zero_()
        s = torch.full((n,), bad, device="cuda")
        zs().rope_write_int4(q, k, v, pos, cos_sin, s, kp, vp, err=err)
        assert int(err) == 2
        assert all(torch.equal(x, y) for x, y in zip(before, (*kp, *vp)))
        err.zero_()
        a, b = zs().read_int4(kp, vp, s, err=err)
        assert int(err) == 2 and not a.any() and not b.any()
    err.zero_()
    a, _ = zs().read_int4(kp, vp, torch.full((3,), -1, device="cuda"), err=err)
    assert int(err) == 0 and not a.any()


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("n", [0, 1, 7, 1025, 3001])
@pytest.mark.parametrize("heads,dim,page,group,layout,dtype", [
    (1, 64, 16, 64, "heads", BF), (3, 64, 32, 32, "tokens", FP), (8, 128, 64, 64, "heads", BF),
    (5, 128, 256, 32, "tokens", BF)])
def test_read_rounds_the_values_once(n, heads, dim, page, group, layout, dtype):
    blocks = 9
    kp, vp = filled(blocks, page, heads, dim, group, layout, seed=n)
    slots = torch.randint(-1, blocks * page, (n,), device="cuda", generator=gen(n))       # some more than once
    k, v = zs().read_int4(kp, vp, slots, dtype)
    for got, p in ((k, kp), (v, vp)):
        blk, row = slots.clamp(min=0) // page, slots.clamp(min=0) % page
        want = plain.values(p.codes[blk, row], p.params[blk, row]).float()
        want[slots < 0] = 0
        assert got.shape == (n, heads, dim) and torch.equal(got, want.to(dtype))
    out = (torch.full_like(k, 9.0), torch.full_like(v, 9.0))
    assert zs().read_int4(kp, vp, slots, dtype, out=out) is out
    assert torch.equal(out[0], k) and torch.equal(out[1], v)


# --------------------------------------------------------------- attention
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17], [97], [255, 0, 300, 64, 31, 1], [4129, 700, 0, 2048]])
@pytest.mark.parametrize("hq,hkv,dim,page,group,layout,dtype", [
    (32, 8, 128, 64, 64, "heads", BF), (7, 1, 128, 16, 32, "tokens", FP), (4, 4, 64, 32, 64, "heads", FP),
    (18, 2, 64, 16, 32, "heads", BF), (16, 1, 128, 128, 64, "tokens", BF), (33, 1, 128, 16, 32, "heads", FP),
    (48, 2, 128, 256, 64, "heads", FP), (12, 1, 128, 16, 64, "heads", BF)])
def test_attention(lens, hq, hkv, dim, page, group, layout, dtype):
    table, blocks = table_of(lens, page, seed=len(lens))
    kp, vp = filled(blocks, page, hkv, dim, group, layout, seed=hq + len(lens))
    q = randn(len(lens), hq, dim, seed=1).to(dtype)
    a = check_attention(q, kp, vp, table, lens, page)
    b = check_attention(q, kp, vp, table, lens, page, max_seqlen=max(lens))
    assert torch.equal(a, zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens)))      # every run the same
    assert a.shape == q.shape and b.shape == q.shape


@pytest.mark.parametrize("lens,hkv,dim,group", [([131105], 1, 128, 64), ([70001, 5], 2, 64, 32), ([20011] * 9, 1, 128, 32)])
def test_attention_of_long_sequences(lens, hkv, dim, group):
    page = 64
    table, blocks = table_of(lens, page, seed=2)
    kp, vp = filled(blocks, page, hkv, dim, group, seed=4)
    q = randn(len(lens), 4 * hkv, dim, seed=1).mul_(0.3).to(FP)         # weights of many tokens
    check_attention(q, kp, vp, table, lens, page)


def test_attention_of_values_far_from_zero():
    """A common offset of keys and values is the centres' part: their scores and outputs."""
    page, lens = 16, [333, 90]
    table, blocks = table_of(lens, page)
    for offset in (40.0, -900.0):
        kp, vp = filled(blocks, page, 2, 128, 64, seed=3, offset=offset)
        check_attention((randn(2, 8, 128, seed=2) * 0.02).to(BF), kp, vp, table, lens, page)


def test_attention_of_large_and_small_numbers():
    page, lens = 16, [50]
    table, blocks = table_of(lens, page)
    for size in (2.0 ** -60, 2.0 ** -30, 2.0 ** 30, 2.0 ** 55):
        kp, vp = filled(blocks, page, 1, 64, 32, seed=3)
        kp.params.mul_(size)
        check_attention((randn(1, 3, 64, seed=2) / size).to(BF), kp, vp, table, lens, page)
        kp.params.div_(size)
        vp.params.mul_(size)
        check_attention(randn(1, 3, 64, seed=2).to(BF), kp, vp, table, lens, page)


def test_scores_that_grow_and_fall():
    """The reference of the exponentials moves late, or never."""
    page, lens = 16, [700]
    table, blocks = table_of(lens, page)
    n = lens[0]
    i = torch.arange(n, device="cuda")
    blk = torch.as_tensor(table[0], device="cuda").long()[i // page]
    for ramp in (torch.linspace(-30, 30, n), torch.linspace(30, -30, n), torch.linspace(0, 9, n), 0 * torch.ones(n),
                 torch.where(torch.arange(n) == 333, 200.0, -50.0)):
        kp, vp = filled(blocks, page, 1, 64, 64, seed=8)
        x = randn(n, 1, 64, seed=9) * 0.1 + ramp.cuda().view(-1, 1, 1)
        kp.codes[blk, i % page], kp.params[blk, i % page] = plain.quantise(x, 64)
        q = torch.full((1, 2, 64), 0.125, device="cuda", dtype=BF)
        check_attention(q, kp, vp, table, lens, page)


@pytest.mark.parametrize("group", [32, 64])
def test_odd_groups_reach_only_what_they_should(group):
    """A NaN key makes its head's outputs NaN, a NaN value its group's channels; rows behind the
    length are not read."""
    page, lens, dim, hkv = 16, [40, 40, 40], 128, 2
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, hkv, dim, group, seed=6)
    q = randn(3, 4, dim, seed=2).to(BF)
    clean = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens))
    kp.params[table[0, 1], 3, 1, 1, 0] = math.nan
    vp.params[table[1, 0], 5, 0, 1, dim // group - 1] = math.nan
    for p in (kp, vp):
        p.params[table[2, 2], 8:] = math.nan          # tokens 40 on
        p.codes[table[2, 2], 8:] = 255
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens))
    want = clean.clone()
    want[0, 2:] = math.nan
    want[1, :2, dim - group:] = math.nan
    assert torch.equal(o.isnan(), want.isnan())
    assert torch.equal(o.nan_to_num(0.0), want.nan_to_num(0.0))


def test_attention_over_lists_of_pages():
    page, hkv, dim, top = 32, 2, 128, 5
    lens = [500, 100, 0, 33]
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, hkv, dim, 64, seed=6)
    q = randn(len(lens), 8, dim, seed=2).to(BF)
    rng = np.random.default_rng(0)
    pages, counts = np.full((len(lens), hkv, top), -1, np.int32), np.zeros((len(lens), hkv), np.int32)
    for r, n in enumerate(lens):
        for h in range(hkv):
            have = -(-n // page)
            counts[r, h] = min(have, top - h)
            pages[r, h, :counts[r, h]] = np.sort(rng.permutation(have)[:counts[r, h]])
    o = zs().paged_attention_int4(q, kp, vp, i32(table), i32(lens), pages=i32(pages), counts=i32(counts))
    for r, n in enumerate(lens):
        k, v = rows_of(kp, table[r], n, page), rows_of(vp, table[r], n, page)
        for h in range(hkv):
            t = np.concatenate([np.arange(p * page, min(n, (p + 1) * page)) for p in pages[r, h, :counts[r, h]]] + [np.zeros(0, int)])
            t = torch.as_tensor(t, device="cuda", dtype=torch.long)
            kk, vv = k[t][:, h:h + 1], v[t][:, h:h + 1]
            qq = q[r, h * 4:h * 4 + 4]
            want, _ = plain.attend(qq, kk, vv, dim ** -0.5)
            err = plain.attention_error(qq, kk, vv, kp.params, dim ** -0.5, n)
            off = (o[r, h * 4:h * 4 + 4].double() - want).abs()
            assert bool((off <= U[BF] * want.abs() + err * (float(vv.abs().max()) if len(t) else 0.0)).all()), (r, h)


def test_bad_pages_are_skipped():
    page, lens = 16, [64]
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, 1, 128, 64, seed=6)
    q = randn(1, 4, 128, seed=2).to(BF)
    for bad in (-1, blocks, 1 << 30):
        t = table.copy()
        t[0, 2] = bad
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        o = zs().paged_attention_int4(q, kp, vp, i32(t), i32(lens), err=err)
        assert int(err) == 2
        keep = [i for i in range(64) if i // 16 != 2]
        k, v = rows_of(kp, table[0], 64, page)[keep], rows_of(vp, table[0], 64, page)[keep]
        want, _ = plain.attend(q[0], k, v, 128 ** -0.5)
        tol = U[BF] * want.abs() + plain.attention_error(q[0], k, v, kp.params, 128 ** -0.5, 64) * float(v.abs().max())
        assert bool(((o[0].double() - want).abs() <= tol).all())


def test_strided_pools_and_queries():
    """Pools that are parts of a larger one, q a slice, out given."""
    page, lens, hkv, dim = 16, [77, 30], 2, 128
    table, blocks = table_of(lens, page)
    big = [zs().int4_pages(blocks, page, 2 * hkv, dim, 64, layout) for layout in ("heads", "tokens")]
    kp, vp = [zs().Int4Pages(p.codes[:, :, h:h + hkv], p.params[:, :, h:h + hkv]) for p, h in zip(big, (0, 2))]
    src = filled(blocks, page, hkv, dim, 64, seed=11)
    for p, x in zip((kp, vp), src):
        p.codes.copy_(x.codes)
        p.params.copy_(x.params)
    q = randn(2, 12, dim, seed=2).to(BF)[:, 4:]
    out = torch.empty(2, 8, dim, dtype=BF, device="cuda")
    assert torch.equal(check_attention(q, kp, vp, table, lens, page, out=out), out)
    assert torch.equal(out, zs().paged_attention_int4(q, *src, i32(table), i32(lens)))
    slots = torch.arange(5, device="cuda")
    assert torch.equal(zs().read_int4(kp, vp, slots)[1], zs().read_int4(*src, slots)[1])


def test_streams_and_two_calls_at_once():
    page, lens = 64, [4000, 3000]
    table, blocks = table_of(lens, page)
    kp, vp = filled(blocks, page, 2, 128, 64, seed=6)
    q = randn(2, 8, 128, seed=2).to(BF)
    t, n = i32(table), i32(lens)
    want = zs().paged_attention_int4(q, kp, vp, t, n)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([zs().paged_attention_int4(q, kp, vp, t, n) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for g in got for o in g)


# ------------------------------------------------------------------- cache
@pytest.mark.parametrize("dtype,layout,group", [(BF, "heads", 64), (FP, "tokens", 32)])
def test_cache_steps_in_a_graph(dtype, layout, group):
    """Steps of a 4-bit cache, the last ones replayed: attention of each token over what the
    rows written so far stand for."""
    rows, hq, hkv, dim, page = 3, 8, 2, 64, 16
    cache = zs().PagedKVCache(40, rows, 12, hkv, dim, page, dtype, layout, bits=4, group=group)
    half = dim // 2
    ang = torch.arange(300, device="cuda")[:, None] * (1e4 ** (-torch.arange(half, device="cuda") / half))[None]
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()
    seen = [[] for _ in range(rows)]                      # (k, v) values of each row's tokens

    def step(new, n, seed):
        plan = cache.step(new, n)
        qkv = randn(n, hq + 2 * hkv, dim, seed=seed).to(dtype)
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        return plan, k, v, cache.write(q, k, v, cos_sin, plan)

    def record(plan, k, v):
        pos, who = plan.positions.long(), plan.token_seq.tolist()
        cos, sin = cos_sin[pos, :half].unsqueeze(1), cos_sin[pos, half:].unsqueeze(1)
        kk = plain.values(*plain.quantise(plain.turn(k, cos, sin, False), group))
        vv = plain.values(*plain.quantise(v, group))
        for i, r in enumerate(who):
            if r >= 0:
                seen[r].append((kk[i], vv[i]))
        back = cache.read(plan.slots)
        live = (plan.slots >= 0).view(-1, 1, 1)
        assert torch.equal(back[0], (kk * live).float().to(dtype)) and torch.equal(back[1], (vv * live).float().to(dtype))

    def check(q, o, lens):
        for r, n in enumerate(lens):
            k, v = (torch.stack([x[j] for x in seen[r][:n]]) for j in (0, 1))
            want, _ = plain.attend(q[r], k, v, dim ** -0.5)
            err = plain.attention_error(q[r], k, v, cache.k[0].params, dim ** -0.5, n)
            assert bool(((o[r].double() - want).abs() <= U[dtype] * want.abs() + TINY[dtype] + err * float(v.abs().max())).all())

    new = i32([33, 1, 16])
    plan, k, v, _ = step(new, 55, 1)                      # 50 tokens, padding behind them
    record(plan, k, v)
    ones = i32([1, 1, 1])
    qkv = torch.empty(rows, hq + 2 * hkv, dim, dtype=dtype, device="cuda")

    def decode():
        plan = cache.step(ones, rows)
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        q = cache.write(q, k, v, cos_sin, plan)
        return plan, q, cache.attention(q, rows=cache.token_rows(plan))

    state = [cache.seqlens, cache.free_count, cache.block_table, cache.free_blocks]
    kept = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        qkv.zero_()
        decode()
    torch.cuda.current_stream().wait_stream(side)
    for t, x in zip(state, kept):
        t.copy_(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, q, o = decode()
    for i in range(20):
        qkv.copy_(randn(rows, hq + 2 * hkv, dim, seed=50 + i).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        record(plan, qkv[:, hq:hq + hkv], qkv[:, hq + hkv:])
        check(q, o, cache.seqlens.tolist())
    assert cache.check_errors() == 0 and cache.seqlens.tolist() == [53, 21, 36]


def test_read_of_a_16_bit_cache():
    cache = zs().PagedKVCache(4, 1, 4, 2, 64, 16, BF)
    cache.k[0].copy_(randn(4, 16, 2, 64, seed=1))
    slots = torch.tensor([5, -1, 63], device="cuda")
    k, v = cache.read(slots)
    assert torch.equal(k[0], cache.k[0][0, 5]) and torch.equal(k[2], cache.k[0][3, 15]) and not k[1].any() and not v.any()


def test_refusals():
    z = zs()
    kp, vp = pools(4, 16, 2, 128, 64)
    q = torch.zeros(1, 4, 128, dtype=BF, device="cuda")
    t, n = i32([[0, 1]]), i32([3])
    ok = dict(q=q, k_pages=kp, v_pages=vp, block_table=t, seq_lens=n)
    z.paged_attention_int4(**ok)
    other = z.int4_pages(4, 16, 2, 128, 32)
    cut = z.Int4Pages(kp.codes[..., :32], kp.params)
    for bad in (dict(v_pages=other), dict(k_pages=cut), dict(k_pages=kp.codes), dict(q=q.float()), dict(q=q[:, :3]),
                dict(q=q[..., :64]), dict(k_pages=z.Int4Pages(kp.codes, kp.params.half())),
                dict(k_pages=z.Int4Pages(kp.codes.cpu(), kp.params.cpu())), dict(block_table=t.long()),
                dict(pages=i32([[[0], [0]]])), dict(max_seqlen=-1), dict(softmax_scale=math.inf),
                dict(k_pages=z.Int4Pages(kp.codes[:, :, :, 1:], kp.params)), dict(out=q[:, ::2])):
        with pytest.raises(ValueError):
            z.paged_attention_int4(**{**ok, **bad})
    with pytest.raises(ValueError):
        z.read_int4(kp, vp, torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        z.read_int4(kp, vp, torch.zeros(1, dtype=torch.long, device="cuda"), torch.float32)
    kv = torch.zeros(1, 2, 128, dtype=BF, device="cuda")
    cs = torch.zeros(1, 128, device="cuda")
    pos, slot = i32([0]), torch.zeros(1, dtype=torch.long, device="cuda")
    z.rope_write_int4(q, kv, kv, pos, cs, slot, kp, vp)
    for bad in ((q.float(), kv, kv), (q, kv.half(), kv), (q, kv[:, :1], kv), (q[:0], kv, kv)):
        with pytest.raises(ValueError):
            z.rope_write_int4(*bad, pos, cs, slot, kp, vp)
    with pytest.raises(ValueError):
        z.rope_write_int4(q, kv, kv, pos, cs[:, :120].contiguous(), slot, kp, vp)
    cache = z.PagedKVCache(4, 1, 4, 2, bits=4)
    with pytest.raises(RuntimeError):
        cache.sparse_attention(q, 2)
