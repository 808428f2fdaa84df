"""Infinite values in paged attention: where a value is infinite, so is the
weighted sum, as in the 64-bit form (every weight of a finite score is positive);
infinities of both signs and NaN give NaN. Finite channels are held to the
tolerance of test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import ATT, BF, DEV, HF, TINY, U, Cache, zs

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def put(c, b, t, h, d, value):
    """Value [t, h, d] of sequence b, in the cache and in its dense copy."""
    c.v[int(c.table[b, t // c.page]), t % c.page, h, d] = value
    c.dense[b][1][t, h, d] = value


def reference(q, dense, scale):
    """float64 output and the largest finite |v|."""
    B, hq, D = q.shape
    out, vmax = torch.zeros(B, hq, D, dtype=torch.float64), 0.0
    for b, (k, v) in enumerate(dense):
        if not k.shape[0]:
            continue
        G = hq // k.shape[1]
        for h in range(k.shape[1]):
            s = q[b, h * G:(h + 1) * G].double() @ k[:, h].double().t() * scale
            p, vv = torch.softmax(s, -1), v[:, h].double()
            fine = vv.isfinite()
            vmax = max(vmax, float(vv[fine].abs().max()))
            o = p @ torch.where(fine, vv, 0.0)
            up, down, nan = (p @ x.double() for x in (vv == INF, vv == -INF, vv.isnan()))
            o = torch.where(up > 0, INF, o)
            o = torch.where(down > 0, -INF, o)
            o = torch.where((nan > 0) | ((up > 0) & (down > 0)), NAN, o)
            out[b, h * G:(h + 1) * G] = o.cpu()
    return out, vmax


def check(out, ref, vmax, dtype):
    out = out.double().cpu()
    fine = ref.isfinite()
    assert torch.equal(out.isnan(), ref.isnan())
    assert torch.equal(out[~fine & ~ref.isnan()], ref[~fine & ~ref.isnan()])
    tol = U[dtype] * ref.abs() + ATT * vmax + TINY[dtype]
    assert bool(((out - ref).abs() <= tol)[fine].all())


def both_ways(q, c, ref, vmax, dtype, **kw):
    """The table as it is, and one so wide that the work goes in runs of chunks; a page list of all pages too."""
    wide = torch.nn.functional.pad(c.table, (0, 8192 - c.table.shape[1]), value=-1)
    n = c.table.shape[1]
    pages = torch.arange(n, device=DEV, dtype=torch.int32).repeat(q.shape[0], c.hkv, 1)
    counts = ((c.lens + c.page - 1) // c.page)[:, None].repeat(1, c.hkv).contiguous()
    for table in (c.table, wide):
        check(zs().paged_attention(q, c.k, c.v, table, c.lens, **kw), ref, vmax, dtype)
    for lists in (pages, torch.nn.functional.pad(pages, (0, 4096 - n), value=-1)):
        check(zs().paged_attention(q, c.k, c.v, c.table, c.lens, pages=lists.contiguous(), counts=counts, **kw), ref,
              vmax, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("value", [INF, -INF])
def test_one_token_with_an_infinite_value(dtype, value):
    """Its weight is 1: nothing is left for a remainder."""
    c = Cache([1, 1], 1, 64, 16, dtype, "heads", 3)
    put(c, 0, 0, 0, 5, value)
    q = torch.randn(2, 2, 64, device=DEV).to(dtype)
    ref, vmax = reference(q, c.dense, 0.125)
    assert ref[0, :, 5].tolist() == [value] * 2 and int(ref.isinf().sum()) == 2
    both_ways(q, c, ref, vmax, dtype)


@pytest.mark.parametrize("lens,hq,hkv,D,page,dtype,layout", [
    ([17, 40, 0], 2, 1, 64, 16, HF, "tokens"),
    ([700, 33, 129], 32, 8, 128, 64, BF, "heads"),          # four heads a KV head
    ([3000, 200], 16, 2, 128, 32, HF, "heads"),             # eight: as columns
    ([3000, 200], 18, 2, 128, 32, BF, "tokens"),            # nine: as rows
    ([2100, 65], 20, 1, 64, 16, HF, "heads"),               # two tiles of heads
])
def test_infinite_values_among_others(lens, hq, hkv, D, page, dtype, layout):
    c = Cache(lens, hkv, D, page, dtype, layout, seed=D + hq)
    q = torch.randn(len(lens), hq, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).to(dtype)
    last = lens[0] - 1
    put(c, 0, 0, 0, 0, INF)
    put(c, 0, last, 0, D - 1, -INF)
    put(c, 0, last // 2, hkv - 1, 7, INF)                   # the same sign twice
    put(c, 0, last, hkv - 1, 7, INF)
    put(c, 0, 3, 0, 9, INF)                                 # both signs, far apart
    put(c, 0, last, 0, 9, -INF)
    put(c, 0, 5, 0, 18, INF)                                # beside a NaN
    put(c, 0, 2, 0, 18, NAN)
    put(c, 1, 1, hkv - 1, 33, -INF)
    ref, vmax = reference(q, c.dense, 1 / math.sqrt(D))
    assert int(ref.isinf().sum()) == 4 * hq // hkv and int(ref.isnan().sum()) == 2 * hq // hkv
    both_ways(q, c, ref, vmax, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq", [2, 16])
@pytest.mark.parametrize("at", [0, 850])
def test_an_infinite_value_under_a_vanishing_weight(dtype, hq, at):
    """Scores 300 below the largest: weights that 32 bits do not hold, in one warp's share and in different ones."""
    T, D = 1200, 64
    c = Cache([T], 1, D, 16, dtype, "heads", 8)
    k = torch.zeros(T, 1, D, device=DEV, dtype=dtype)
    k[900:, 0, 0] = 1.0
    blk = c.table[0, :T // 16].long().repeat_interleave(16)
    c.k[blk, torch.arange(T, device=DEV) % 16] = k
    c.dense[0] = (k, c.dense[0][1])
    put(c, 0, at, 0, 11, INF)
    q = torch.zeros(1, hq, D, device=DEV, dtype=dtype)
    q[..., 0] = 1.0
    ref, vmax = reference(q, c.dense, 300.0)
    assert int(ref.isinf().sum()) == hq
    both_ways(q, c, ref, vmax, dtype, softmax_scale=300.0)


@pytest.mark.parametrize("T", [1, 20, 300])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scores_of_minus_infinity_weigh_nothing(T, dtype):
    """A key with an infinity: no weight where the score is -inf, and zeros where every score is."""
    c = Cache([T, T + 3], 1, 64, 16, dtype, "heads", 8)
    q = torch.randn(2, 2, 64, device=DEV).to(dtype)
    q[..., 4] = 1.0
    lost = range(T) if T < 300 else range(100, 220)
    for t in lost:
        c.k[int(c.table[0, t // 16]), t % 16, 0, 4] = -INF
    keep = torch.tensor([t for t in range(T) if t not in lost], device=DEV, dtype=torch.long)
    dense = [(c.dense[0][0][keep], c.dense[0][1][keep]), c.dense[1]]
    ref, vmax = reference(q, dense, 0.125)
    both_ways(q, c, ref, vmax, dtype)
    lse = torch.zeros(2, 2, device=DEV)
    zs().paged_attention(q, c.k, c.v, c.table, c.lens, lse=lse)
    assert bool((lse[0] == -INF).all()) == (T < 300) and bool(lse[1].isfinite().all())
