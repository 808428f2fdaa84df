"""Operators of the uncompressed paged KV cache against plain 64-bit forms:
step plan, rotary write, paged attention, page bounds, page choice and sparse
attention, and the cache class under a CUDA graph.

Tolerances. An output is the exact value rounded once to its type (half a unit
in the last place: u = 2^-8 relative for bf16's 8 bits, 2^-11 for fp16's 11, plus half of the
smallest subnormal step for fp16) after 32-bit arithmetic. The rotary write has two
fp32 products and a sum (3 * 2^-24 of |a| + |b|). Attention adds, relative to max
|v|: the remainder of P in two 16-bit parts (2^-17), and the scores' error
through the exponential, where |scale s| stays below 40 in base 2 and each score
sums up to 128 fp32 products: 40 * 2^-23 + 128 * 2^-24 * 40 * ln 2 < 2.3e-4
as a worst case. Whole numbers and choices are equal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
ATT = 2.3e-4
DEV = "cuda"


def zs():
    import zipserv_asplos26_b200
    return zipserv_asplos26_b200


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=DEV)


# -------------------------------------------------------------------- plan
def plan_ref(table, lens, new, free, count, page, room):
    table, lens, free = table.copy(), lens.copy(), free.copy()
    for r in range(len(new)):
        if new[r] < 0:
            for p in range(-(-lens[r] // page)):
                free[count] = table[r, p]
                count += 1
    asked = claimed = 0
    have, cu, refused, tok = count, [0], [], []
    for r in range(len(new)):
        if new[r] < 0:
            lens[r] = 0
            cu.append(cu[-1])
            refused.append(False)
            continue
        asked += new[r]
        old, now = -(-lens[r] // page), -(-(lens[r] + new[r]) // page)
        ok = asked <= room and now <= table.shape[1]
        if ok:
            claimed += now - old
            ok = now == old or claimed <= have
        refused.append(bool(not ok and new[r] > 0))
        if ok:
            for p in range(old, now):
                count -= 1
                table[r, p] = free[count]
            tok += [(table[r, t // page] * page + t % page, r, t) for t in range(lens[r], lens[r] + new[r])]
            lens[r] += new[r]
        cu.append(cu[-1] + (new[r] if ok else 0))
    tok += [(-1, -1, 0)] * (room - len(tok))
    tok = np.array(tok, np.int64).reshape(room, 3)
    return table, free, count, lens, np.array(cu), np.array(refused), tok


def plan_case(rng, R, page, width, longest, chunk, ended, spare):
    lens = rng.integers(0, min(longest, width * page) + 1, R)
    lens[rng.random(R) < 0.2] = 0
    new = rng.integers(0, chunk + 1, R)
    new[rng.random(R) < ended] = -1
    used = -(-lens // page)
    n = int(used.sum()) + spare
    order = rng.permutation(n)
    table = np.full((R, width), -1, np.int64)
    at = 0
    for r in range(R):
        table[r, :used[r]] = order[at:at + used[r]]
        at += used[r]
    free = np.full(n, -7, np.int64)
    free[:n - at] = order[at:]
    return table, lens, new, free, n - at


@pytest.mark.parametrize("R,page,width,longest,chunk,ended,spare,cut", [
    (1, 16, 4, 0, 1, 0.0, 3, 0),            # the first token of one request
    (1, 64, 1, 63, 0, 0.0, 0, 0),           # nothing to do, nothing free
    (5, 16, 3, 48, 40, 0.3, 9, 0),          # requests beyond the table's width
    (40, 32, 9, 200, 90, 0.2, 20, 0),       # too few pages
    (40, 32, 9, 200, 90, 0.2, 400, 700),    # too few tokens in the step
    (7, 256, 5, 1000, 300, 1.0, 0, 0),      # every request has ended
    (513, 16, 12, 150, 1, 0.1, 600, 0),     # one more request than threads
    (3000, 64, 3, 100, 5, 0.3, 200, 0),
    (8192, 16, 2, 20, 2, 0.05, 9000, 0),    # the most requests
])
def test_plan_step(R, page, width, longest, chunk, ended, spare, cut):
    rng = np.random.default_rng(R * 7 + page)
    table, lens, new, free, count = plan_case(rng, R, page, width, longest, chunk, ended, spare)
    room = max(0, int(np.maximum(new, 0).sum()) + 2 - cut)
    want = plan_ref(table, lens, new, free, count, page, room)
    wide = torch.full((R, width + 5), -9, dtype=torch.int32, device=DEV)     # a table with a row stride of its own
    wide[:, 2:2 + width] = i32(table)
    t, f = wide[:, 2:2 + width], i32(free)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(2):                                                        # repeating a step changes nothing
        p = zs().plan_step(t, i32(lens), i32(new), f, i32([count]), page, room, err=err)
        assert np.array_equal(t.cpu().numpy(), want[0])
        assert np.array_equal(f.cpu().numpy(), want[1])
        assert p.free_count.item() == want[2]
        assert np.array_equal(p.seq_lens.cpu().numpy(), want[3])
        assert np.array_equal(p.cu_tokens.cpu().numpy(), want[4])
        assert np.array_equal(p.refused.cpu().numpy(), want[5])
        assert np.array_equal(p.slots.cpu().numpy(), want[6][:, 0])
        assert np.array_equal(p.token_seq.cpu().numpy(), want[6][:, 1])
        assert np.array_equal(p.positions.cpu().numpy(), want[6][:, 2])
    assert err.item() == (4 if want[5].any() else 0)
    assert bool((wide[:, :2] == -9).all() and (wide[:, 2 + width:] == -9).all())


def test_plan_step_large_asks_are_refused():
    """Token counts whose sums pass 32 bits."""
    lens, new = i32([5, 0, 3]), i32([2 ** 31 - 1, 2 ** 31 - 1, 1])
    p = zs().plan_step(i32([[0, -1], [-1, -1], [1, -1]]), lens, new, i32([2, 3]), i32([2]), 16, 10)
    assert p.refused.tolist() == [True, True, True] and p.seq_lens.tolist() == [5, 0, 3]
    assert p.cu_tokens.tolist() == [0, 0, 0, 0] and p.free_count.item() == 2


def test_plan_step_lengths_end_below_31_bits():
    """A table of more than 2**31 tokens: a request grows up to the last whole page below that, and not past it."""
    page, width = 256, (1 << 23) + 4
    start = (1 << 31) - 300
    table = torch.zeros(2, width, dtype=torch.int32, device=DEV)
    table[0, start // page] = 7
    for new, refused in ((44, False), (45, True), (600, True)):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        p = zs().plan_step(table, i32([start, 0]), i32([new, 1]), i32(np.arange(64)), i32([64]), page, 1024, err=err)
        assert p.refused.tolist() == [refused, False]
        assert p.seq_lens.tolist() == [start + (0 if refused else new), 1]
        assert p.free_count.item() == 63 and err.item() == (4 if refused else 0)
        n = p.cu_tokens[-1].item()
        assert n == (1 if refused else new + 1)
        if not refused:
            assert p.positions[:new].tolist() == list(range(start, start + new))
            assert p.slots[:new].tolist() == [7 * page + x % page for x in range(start, start + new)]


def test_plan_step_free_list_overflow_is_flagged():
    """A free list that claims more entries than its buffer holds stays in bounds."""
    table, free = i32([[0, 1], [2, 3]]), i32([9, 8, 7])
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    p = zs().plan_step(table, i32([32, 32]), i32([-1, -1]), free, i32([2]), 16, 0, err=err)
    assert err.item() == 2 and p.free_count.item() == 3 and free.tolist() == [9, 8, 0]


# ------------------------------------------------------------ rotary write
def pool(nb, page, heads, dim, dtype, layout, fill=None):
    shape = (nb, heads, page, dim) if layout == "heads" else (nb, page, heads, dim)
    x = torch.full(shape, float("nan") if fill is None else fill, dtype=dtype, device=DEV)
    return x.transpose(1, 2) if layout == "heads" else x


def turn_ref(x, pos, cos_sin, sections, interleaved):
    """x [N, H, D]; float64."""
    x = x.double().cpu().numpy().copy()
    rot = cos_sin.shape[1]
    table = cos_sin.double().cpu().numpy()
    axis = np.repeat(np.arange(len(sections)), sections)
    pos = pos.reshape(len(sections), -1).cpu().numpy()
    out, mag = x.copy(), np.abs(x)
    for j in range(rot // 2):
        lo, hi = (2 * j, 2 * j + 1) if interleaved else (j, j + rot // 2)
        c, s = table[pos[axis[j]], j][:, None], table[pos[axis[j]], rot // 2 + j][:, None]
        a, b = x[:, :, lo], x[:, :, hi]
        out[:, :, lo], out[:, :, hi] = a * c - b * s, b * c + a * s
        mag[:, :, lo] = mag[:, :, hi] = np.abs(a) + np.abs(b)
    return torch.from_numpy(out), torch.from_numpy(mag)


@pytest.mark.parametrize("N,hq,hkv,D,rot,sections,interleaved,dtype,page,layout", [
    (1, 32, 8, 128, 128, None, False, torch.bfloat16, 64, "heads"),
    (5, 4, 4, 64, 32, None, True, torch.float16, 16, "tokens"),
    (33, 7, 1, 128, 128, [16, 24, 24], False, torch.bfloat16, 128, "tokens"),
    (33, 8, 2, 128, 96, [16, 17, 15], True, torch.float16, 32, "heads"),
    (19, 3, 3, 80, 80, [20, 20], False, torch.bfloat16, 16, "heads"),
    (300, 16, 2, 256, 64, [1, 2, 3, 26], False, torch.float16, 256, "tokens"),
    (4097, 8, 8, 64, 64, [0, 32], False, torch.bfloat16, 64, "heads"),
    (6000, 2, 1, 512, 512, None, True, torch.bfloat16, 64, "heads"),
])
def test_rope_write(N, hq, hkv, D, rot, sections, interleaved, dtype, page, layout):
    g = torch.Generator(device=DEV).manual_seed(N + D)
    rng = np.random.default_rng(N)
    qkv = torch.randn(N, (hq + 2 * hkv) * D, device=DEV, generator=g).to(dtype)
    q, k, v = (x.view(N, -1, D) for x in qkv.split([hq * D, hkv * D, hkv * D], 1))
    rows = 500
    ang = torch.rand(rows, rot // 2, device=DEV, generator=g) * 7 - 3
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1)
    axes = 1 if sections is None else len(sections)
    pos = torch.randint(0, rows, (axes, N), device=DEV, generator=g, dtype=torch.int32)
    nb = -(-N // page) + 2
    slots = torch.from_numpy(rng.permutation(nb * page)[:N].astype(np.int64)).to(DEV)
    if N > 4:
        slots[3] = -1
    kp, vp = pool(nb, page, hkv, D, dtype, layout), pool(nb, page, hkv, D, dtype, layout)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = zs().rope_write(q, k, v, pos[0] if axes == 1 else pos, cos_sin, slots, kp, vp, sections, interleaved, err=err)
    want, mag = turn_ref(q, pos, cos_sin, sections or [rot // 2], interleaved)
    tol = U[dtype] * want.abs() + 3 * 2.0 ** -24 * mag + TINY[dtype]
    assert bool(((out.double().cpu() - want).abs() <= tol).all())
    want, mag = turn_ref(k, pos, cos_sin, sections or [rot // 2], interleaved)
    tol = U[dtype] * want.abs() + 3 * 2.0 ** -24 * mag + TINY[dtype]
    live = (slots >= 0).cpu()
    s = slots[slots >= 0]
    assert bool(((kp[s // page, s % page].double().cpu() - want[live]).abs() <= tol[live]).all())
    assert torch.equal(vp[s // page, s % page], v[slots >= 0])
    # nothing else was written
    rest = torch.ones(nb, page, dtype=torch.bool, device=DEV)
    rest[s // page, s % page] = False
    assert bool(kp[rest].isnan().all() and vp[rest].isnan().all())
    assert err.item() == 0
    # in place
    qc = q.contiguous()
    assert zs().rope_write(qc, k, v, pos[0] if axes == 1 else pos, cos_sin, slots, kp, vp, sections, interleaved,
                           q_out=qc) is qc
    assert torch.equal(qc, out)


def test_rope_write_bad_indexes_are_skipped():
    dtype = torch.bfloat16
    q, k, v = (torch.randn(4, h, 64, device=DEV).to(dtype) for h in (2, 1, 1))
    kp, vp = pool(2, 16, 1, 64, dtype, "heads"), pool(2, 16, 1, 64, dtype, "heads")
    cos_sin = torch.cat([torch.ones(8, 32, device=DEV), torch.zeros(8, 32, device=DEV)], 1)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    pos, slots = i32([0, 7, 3, 1]), torch.tensor([31, 32, -5, 2 ** 40], device=DEV)
    zs().rope_write(q, k, v, pos, cos_sin, slots, kp, vp, err=err)
    assert err.item() == 2
    assert torch.equal(vp[1, 15], v[0]) and int(vp.isnan().all(-1).sum()) == 31
    err.zero_()
    zs().rope_write(q, k, v, i32([0, 8, -1, 1]), cos_sin, torch.full((4,), -1, device=DEV), kp, vp, err=err)
    assert err.item() == 2
    zs().rope_write(q[:0], k[:0], v[:0], pos[:0], cos_sin, slots[:0], kp, vp)          # no tokens


def test_rope_write_unaligned_inputs():
    dtype = torch.float16
    base = torch.randn(6 * (4 * 64 + 3) + 1, device=DEV).to(dtype)
    odd = base[1:].view(6, 4 * 64 + 3)
    q, k, v = odd[:, :128].view(6, 2, 64), odd[:, 128:192].view(6, 1, 64), odd[:, 192:256].view(6, 1, 64)
    ang = torch.rand(9, 32, device=DEV)
    cs, pos, slots = torch.cat([ang.cos(), ang.sin()], 1), i32(range(6)), torch.arange(6, device=DEV)
    a = [pool(1, 16, 1, 64, dtype, "heads", 0.0) for _ in range(2)]
    b = [pool(1, 16, 1, 64, dtype, "heads", 0.0) for _ in range(2)]
    x = zs().rope_write(q, k, v, pos, cs, slots, *a)
    y = zs().rope_write(q.contiguous(), k.contiguous(), v.contiguous(), pos, cs, slots, *b)
    assert torch.equal(x, y) and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# --------------------------------------------------------------- attention
class Cache:
    """A paged cache of given lengths over a shuffled pool; rows past a length and
    spare blocks hold NaN, table entries past a sequence's pages -1."""

    def __init__(self, lens, hkv, D, page, dtype, layout, seed, spare=3, k_scale=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device=DEV).manual_seed(seed)
        lens = np.asarray(lens)
        pages = -(-lens // page)
        n = int(pages.sum()) + spare
        self.k, self.v = pool(n, page, hkv, D, dtype, layout), pool(n, page, hkv, D, dtype, layout)
        order = rng.permutation(n)
        table = np.full((len(lens), max(1, pages.max(initial=0)) + 2), -1)
        at = 0
        self.dense = []
        for i, (p, t) in enumerate(zip(pages, lens)):
            table[i, :p] = order[at:at + p]
            at += p
            k = torch.randn(t, hkv, D, device=DEV, generator=g).mul_(k_scale).to(dtype)
            v = torch.randn(t, hkv, D, device=DEV, generator=g).to(dtype)
            self.dense.append((k, v))
            blk = torch.from_numpy(table[i, :p]).to(DEV).repeat_interleave(page)[:t]
            row = torch.arange(t, device=DEV) % page
            self.k[blk, row], self.v[blk, row] = k, v
        self.table, self.lens, self.page, self.hkv, self.D = i32(table), i32(lens), page, hkv, D


def attend_ref(q, dense, scale, rows=None):
    """q [B, Hq, D]; dense: per sequence (k, v) [T, Hkv, D]; rows(b, h): token indexes or None for all.
    float64 output, log-sum-exp and max |v|."""
    B, hq, D = q.shape
    out, lse = torch.zeros(B, hq, D, dtype=torch.float64), torch.full((B, hq), -math.inf, dtype=torch.float64)
    vmax = 0.0
    for b, (k, v) in enumerate(dense):
        hkv = k.shape[1]
        G = hq // hkv
        for h in range(hkv):
            idx = slice(None) if rows is None else rows(b, h)
            kk, vv = k[idx, h].double(), v[idx, h].double()
            if kk.shape[0] == 0:
                continue
            s = q[b, h * G:(h + 1) * G].double() @ kk.t() * scale
            out[b, h * G:(h + 1) * G] = (torch.softmax(s, -1) @ vv).cpu()
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(s, -1).cpu()
            vmax = max(vmax, float(vv.abs().max()))
    return out, lse, vmax


def close(out, ref, vmax, dtype):
    tol = U[dtype] * ref.abs() + ATT * vmax + TINY[dtype]
    return bool(((out.double().cpu() - ref).abs() <= tol).all())


BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("lens,hq,hkv,D,page,dtype,layout", [
    ([1], 8, 8, 64, 16, BF, "heads"),                                   # one token, one query a head
    ([0, 1, 15, 16, 17, 0], 8, 2, 128, 16, HF, "tokens"),               # empty rows first and last
    ([0, 0], 4, 1, 128, 64, BF, "heads"),                               # nothing at all
    ([63, 64, 65, 129, 1], 32, 8, 128, 64, BF, "heads"),
    ([300], 7, 1, 128, 32, BF, "tokens"),                               # seven heads a KV head
    ([511, 2, 300], 16, 1, 64, 128, HF, "heads"),                       # a full tile of heads
    ([100, 2049], 16, 2, 128, 64, HF, "heads"),                         # eight heads: as columns
    ([100, 2049], 9, 1, 128, 64, BF, "tokens"),                         # nine: as rows
    ([260, 33], 40, 2, 128, 256, BF, "heads"),                          # twenty heads: two tiles
    ([77, 1000], 64, 1, 64, 16, HF, "tokens"),                          # four tiles
    ([9001], 32, 8, 128, 64, BF, "heads"),                              # one long: split over its length
    ([5000, 1, 0, 700], 2, 1, 128, 16, HF, "tokens"),
    (list(range(150)), 2, 2, 64, 16, BF, "heads"),                      # more sequences than a CTA has threads
    ([40] * 700, 8, 8, 64, 32, HF, "heads"),                            # many short: several units a CTA
])
def test_paged_attention(lens, hq, hkv, D, page, dtype, layout):
    c = Cache(lens, hkv, D, page, dtype, layout, seed=len(lens) + D)
    q = torch.randn(len(lens), hq, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(dtype)
    scale = 1.0 / math.sqrt(D)
    lse = torch.full((len(lens), hq), 5.0, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = zs().paged_attention(q, c.k, c.v, c.table, c.lens, lse=lse, err=err)
    ref, ref_lse, vmax = attend_ref(q, c.dense, scale)
    assert close(out, ref, vmax, dtype)
    assert bool((out[c.lens == 0] == 0).all()) and err.item() == 0
    assert torch.allclose(lse.double().cpu(), ref_lse, rtol=1e-6, atol=ATT)
    again = zs().paged_attention(q.unsqueeze(1), c.k, c.v, c.table, c.lens)
    assert again.shape == (len(lens), 1, hq, D) and torch.equal(again.squeeze(1), out)      # bit for bit
    # a wide table: the same in runs of chunks, the way of long sequences
    wide = torch.nn.functional.pad(c.table, (0, 8192 - c.table.shape[1]), value=-1)
    out = zs().paged_attention(q, c.k, c.v, wide, c.lens, lse=lse.fill_(5.0), err=err)
    assert close(out, ref, vmax, dtype)
    assert bool((out[c.lens == 0] == 0).all()) and err.item() == 0
    assert torch.allclose(lse.double().cpu(), ref_lse, rtol=1e-6, atol=ATT)
    assert torch.equal(zs().paged_attention(q, c.k, c.v, wide, c.lens), out)
    # no result depends on the bound, a wrong one included
    for most in (max(lens), 1):
        out = zs().paged_attention(q, c.k, c.v, wide, c.lens, max_seqlen=most)
        assert close(out, ref, vmax, dtype)


def test_no_sequences():
    z = zs()
    c = Cache([40], 2, 64, 16, BF, "heads", 1)
    q, lens = torch.zeros(0, 4, 64, device=DEV, dtype=BF), c.lens[:0]
    assert z.paged_attention(q, c.k, c.v, c.table[:0], lens).shape == (0, 4, 64)
    codes = torch.zeros(c.k.shape[0], 2, 2, 64, dtype=torch.int8, device=DEV)
    scales = torch.zeros(c.k.shape[0], 2, device=DEV)
    z.page_bounds(c.k, c.table[:0], lens, lens, codes, scales, 5)
    out, pages, counts = z.sparse_attention(q, c.k, c.v, codes, scales, c.table[:0], lens, 4)
    assert out.shape == (0, 4, 64) and pages.shape == (0, 2, 4) and counts.shape == (0, 2)


def test_paged_attention_large_scores_and_scale():
    """Scores of some hundreds: the running maximum moves, all but a few weights vanish."""
    c = Cache([700, 90], 2, 128, 64, BF, "heads", 5, k_scale=4.0)
    q = torch.randn(2, 8, 128, device=DEV).mul_(4).to(BF)
    out = zs().paged_attention(q, c.k, c.v, c.table, c.lens, softmax_scale=0.05)
    ref, _, vmax = attend_ref(q, c.dense, 0.05)
    # base-2 scores stay below 64 here as for the common scale
    assert close(out, ref, 2 * vmax, BF)


def test_paged_attention_fp16_long_tail():
    """Weights of 2^-20 of the largest, many of them: fp16 probabilities keep them."""
    T = 40000
    c = Cache([T], 1, 64, 64, HF, "heads", 9)
    k = torch.zeros(T, 1, 64, device=DEV, dtype=HF)
    k[0, 0, 0] = 1.0
    v = torch.ones(T, 1, 64, device=DEV, dtype=HF)
    v[0] = -1.0
    blk = c.table[0, :-(-T // 64)].long().repeat_interleave(64)[:T]
    row = torch.arange(T, device=DEV) % 64
    c.k[blk, row], c.v[blk, row] = k, v
    q = torch.zeros(1, 1, 64, device=DEV, dtype=HF)
    q[0, 0, 0] = 1.0
    scale = 20 * math.log(2)
    out = zs().paged_attention(q, c.k, c.v, c.table, c.lens, softmax_scale=scale)
    w = (T - 1) * 2.0 ** -20
    want = (w - 1) / (w + 1)
    assert abs(float(out[0, 0, 0]) - want) <= U[HF] + ATT


@pytest.mark.parametrize("where", ["k", "v"])
def test_paged_attention_nan_stays_in_its_sequence(where):
    c = Cache([40, 50, 60], 2, 64, 16, BF, "tokens", 4)
    getattr(c, where)[int(c.table[1, 2]), 3, 1] = float("nan")       # sequence 1, KV head 1
    q = torch.randn(3, 4, 64, device=DEV).to(BF)
    out = zs().paged_attention(q, c.k, c.v, c.table, c.lens)
    bad = out.isnan()
    assert bool(bad[1, 2:].all()) and not bool(bad[0].any() or bad[2].any() or bad[1, :2].any())


def test_paged_attention_bad_table_entries_are_skipped():
    c = Cache([64, 64], 1, 64, 16, BF, "heads", 6)
    q = torch.randn(2, 2, 64, device=DEV).to(BF)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.table[0, 1], c.table[0, 3] = c.k.shape[0], -1
    out = zs().paged_attention(q, c.k, c.v, c.table, c.lens, err=err)
    ref, _, vmax = attend_ref(q, c.dense, 0.125, lambda b, h: [t for t in range(64) if b or t // 16 in (0, 2)])
    assert err.item() == 2 and close(out, ref, vmax, BF)


def test_paged_attention_lengths_beyond_the_table():
    """A length past the table's width counts the table's pages only; a negative one none."""
    c = Cache([64, 30], 1, 64, 16, BF, "heads", 6)
    lens = i32([10 ** 9, -4])
    q = torch.randn(2, 2, 64, device=DEV).to(BF)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = zs().paged_attention(q, c.k, c.v, c.table[:, :4], lens, err=err)
    ref, _, vmax = attend_ref(q, c.dense, 0.125, lambda b, h: [] if b else list(range(64)))
    assert close(out, ref, vmax, BF) and err.item() == 0


def test_paged_attention_offsets_past_32_bits():
    """Pages that begin beyond 2^32 elements of their pool."""
    page, hkv, D = 256, 8, 128
    nb = 2 ** 32 // (page * hkv * D) + 40
    k = torch.empty(nb, hkv, page, D, dtype=BF, device=DEV).transpose(1, 2)
    v = torch.empty(nb, page, hkv, D, dtype=BF, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    blocks = [nb - 1, 0, nb - 7]
    T = 2 * page + 33
    kd, vd = (torch.randn(T, hkv, D, device=DEV, generator=g).to(BF) for _ in range(2))
    for i, b in enumerate(blocks):
        n = min(page, T - i * page)
        k[b, :n], v[b, :n] = kd[i * page:i * page + n], vd[i * page:i * page + n]
    q = torch.randn(1, 16, D, device=DEV, generator=g).to(BF)
    out = zs().paged_attention(q, k, v, i32([blocks]), i32([T]))
    ref, _, vmax = attend_ref(q, [(kd, vd)], 1 / math.sqrt(D))
    assert close(out, ref, vmax, BF)
    # the rotary write and the bounds at the same offsets
    slot = torch.tensor([(nb - 1) * page + 255], device=DEV)
    one = torch.ones(1, hkv, D, device=DEV, dtype=BF)
    cs = torch.cat([torch.ones(1, 64, device=DEV), torch.zeros(1, 64, device=DEV)], 1)
    zs().rope_write(one, one * 3, one * 5, i32([0]), cs, slot, k, v)
    assert bool((k[nb - 1, 255] == 3).all() and (v[nb - 1, 255] == 5).all())
    codes, scales = torch.zeros(nb, hkv, 2, D, dtype=torch.int8, device=DEV), torch.zeros(nb, hkv, device=DEV)
    zs().page_bounds(k, i32([[nb - 1]]), i32([0]), i32([page]), codes, scales, page)
    kf = k[nb - 1].float()
    assert torch.equal(codes[nb - 1, :, 0].float(), (kf.amax(0) / scales[nb - 1, :, None]).ceil().clamp(-127, 127))
    del k, v
    torch.cuda.empty_cache()


def test_paged_attention_on_another_stream():
    c = Cache([3000, 100], 8, 128, 64, BF, "heads", 2)
    q = torch.randn(2, 32, 128, device=DEV).to(BF)
    want = zs().paged_attention(q, c.k, c.v, c.table, c.lens)
    side = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            big = big @ big * 1e-3
        q2 = q + (big.sum() * 0).nan_to_num(0.0).to(BF)         # ready late, on the side stream only
        got = zs().paged_attention(q2, c.k, c.v, c.table, c.lens)
    side.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------ bounds and choice
def bounds_ref(k):
    """[page, heads, D] float64 -> codes [heads, 2, D], scale [heads]."""
    hi, lo = k.max(0), k.min(0)
    most = np.maximum(np.abs(hi), np.abs(lo)).max(-1)
    codes, scale = np.zeros((k.shape[1], 2, k.shape[2]), np.int64), np.zeros(k.shape[1])
    for h in range(k.shape[1]):
        if not np.isfinite(most[h]):
            scale[h] = np.inf
        elif most[h] >= 2.0 ** -126:
            scale[h] = 2.0 ** (math.frexp(most[h])[1] - 7)
            codes[h, 0] = np.clip(np.ceil(hi[h] / scale[h]), -127, 127)
            codes[h, 1] = np.clip(np.floor(lo[h] / scale[h]), -127, 127)
    return codes, scale


@pytest.mark.parametrize("page,hkv,D,dtype,layout", [
    (16, 1, 64, BF, "heads"), (64, 8, 128, BF, "heads"), (32, 3, 128, HF, "tokens"), (256, 2, 256, HF, "heads"),
    (128, 5, 64, HF, "tokens")])
def test_page_bounds(page, hkv, D, dtype, layout):
    """Pages that became complete are described, no others."""
    before = [0, page - 1, page, 3 * page + 1, 5, 0]
    after = [3 * page + 2, page, 2 * page - 1, 4 * page, 5, page - 1]
    c = Cache(after, hkv, D, page, dtype, layout, seed=page + D)
    k = c.k
    b0 = int(c.table[0, 0])
    k[b0, 1, 0, 3] = 0.0
    k[b0, :, hkv - 1] = 0.0                                    # an all-zero head
    k[int(c.table[0, 1]), page - 1, 0, D - 1] = float("inf")
    k[int(c.table[0, 2]), 0, hkv - 1, 0] = float("nan")
    k[int(c.table[3, 3]), 5, 0, 7] = -60000.0                  # one outlier: codes of a few units
    n = k.shape[0]
    codes = torch.full((n, hkv, 2, D), 99, dtype=torch.int8, device=DEV)
    scales = torch.full((n, hkv), -3.0, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    zs().page_bounds(k, c.table, i32(before), c.lens, codes, scales, max(a - b for a, b in zip(after, before)),
                     err=err)
    done = set()
    for i, (a, z) in enumerate(zip(before, after)):
        done |= {int(c.table[i, p]) for p in range(a // page, z // page)}
    kd = k.double().cpu().numpy()
    for blk in range(n):
        if blk in done:
            wc, ws = bounds_ref(kd[blk])
            assert np.array_equal(codes[blk].cpu().numpy(), wc) and np.array_equal(scales[blk].cpu().numpy(), ws)
        else:
            assert bool((codes[blk] == 99).all() and (scales[blk] == -3).all())
    assert err.item() == 0


@pytest.mark.parametrize("B,prompts,page", [(3, {1: 700}, 16), (70, {0: 333, 69: 90}, 32), (300, {7: 5000}, 64),
                                            (1, {0: 129}, 128)])
def test_page_bounds_of_a_few_prompts_among_many_sequences(B, prompts, page):
    """The same bounds whether the tokens in all are bounded or not."""
    rng = np.random.default_rng(B)
    before = rng.integers(0, 3 * page, B)
    after = before + 1
    for b, n in prompts.items():
        after[b] = before[b] + n
    c = Cache(after, 2, 64, page, BF, "heads", seed=B)
    n = c.k.shape[0]
    got = []
    for total in (None, int((after - before).sum())):
        codes = torch.full((n, 2, 2, 64), 99, dtype=torch.int8, device=DEV)
        scales = torch.full((n, 2), -3.0, device=DEV)
        zs().page_bounds(c.k, c.table, i32(before), c.lens, codes, scales, max(prompts.values()), total)
        got.append((codes, scales))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert int((got[0][1][:, 0] > 0).sum()) == int((after // page - before // page).sum())


def select_ref(q, codes, scales, table, lens, page, top, sinks, local):
    q = q.double().cpu().numpy()
    codes, scales, table = codes.cpu().numpy().astype(np.int64), scales.double().cpu().numpy(), table.cpu().numpy()
    B, hq, D = q.shape
    hkv = codes.shape[1]
    G = hq // hkv
    pages, counts = np.full((B, hkv, top), -1), np.zeros((B, hkv), np.int64)
    for b in range(B):
        n = -(-int(lens[b]) // page)
        for h in range(hkv):
            if n <= top:
                pick = np.arange(n)
            else:
                qg = q[b, h * G:(h + 1) * G]
                most = np.abs(qg).max()
                step = 2.0 ** (math.frexp(most)[1] - 7) if most > 0 and np.isfinite(most) else 0.0
                q8 = np.clip(np.rint(qg / step), -127, 127).astype(np.int64) if step else np.zeros_like(qg, np.int64)
                cb = codes[table[b, :n], h]
                best = np.stack([np.where(x > 0, x * cb[:, 0], x * cb[:, 1]).sum(-1) for x in q8]).max(0)
                sc = scales[table[b, :n], h]
                key = np.where(np.isfinite(sc), best * np.where(np.isfinite(sc), sc, 0), np.inf)
                forced = (np.arange(n) < sinks) | (np.arange(n) >= n - local)
                pick = np.sort(np.lexsort((np.arange(n), -key, ~forced))[:top])
            counts[b, h] = len(pick)
            pages[b, h, :len(pick)] = pick
    return pages, counts


@pytest.mark.parametrize("lens,hq,hkv,D,page,top,sinks,local,dtype", [
    ([5000, 0, 1, 130], 32, 8, 128, 64, 8, 1, 1, BF),
    ([999], 7, 1, 64, 16, 5, 0, 1, HF),
    ([4000, 3333], 16, 1, 256, 32, 20, 2, 3, BF),
    ([1040, 1041], 4, 4, 64, 16, 64, 1, 1, HF),           # as many pages as chosen, one more
    ([1025 * 16], 2, 1, 128, 16, 2, 1, 1, BF),            # the forced pages alone
    ([90000], 64, 1, 64, 16, 700, 4, 16, HF),             # 5625 pages, 64 heads a KV head
    ([30000] * 3, 8, 2, 128, 32, 300, 1, 1, BF),
])
def test_select_pages(lens, hq, hkv, D, page, top, sinks, local, dtype):
    g = torch.Generator(device=DEV).manual_seed(D + top)
    rng = np.random.default_rng(top)
    n = [-(-t // page) for t in lens]
    nb = sum(n) + 2
    codes = torch.randint(-127, 128, (nb, hkv, 2, D), device=DEV, generator=g, dtype=torch.int32).to(torch.int8)
    codes = codes.sort(2, descending=True).values.contiguous()                          # upper above lower
    # a few scales, so that equal scores occur; a page without finite bounds among them
    scales = (2.0 ** torch.randint(-4, 1, (nb, hkv), device=DEV, generator=g)).float()
    scales[rng.integers(0, nb)] = float("inf")
    codes[rng.integers(0, nb, nb // 3)] = codes[0].clone()                              # ties
    order = rng.permutation(nb)
    table = np.full((len(lens), max(n) + 1), -1)
    at = 0
    for i, p in enumerate(n):
        table[i, :p] = order[at:at + p]
        at += p
    table, lt = i32(table), i32(lens)
    q = torch.randn(len(lens), hq, D, device=DEV, generator=g).to(dtype)
    pages, counts = zs().select_pages(q, codes, scales, table, lt, page, top, sinks, local)
    wp, wc = select_ref(q, codes, scales, table, lens, page, top, sinks, local)
    assert np.array_equal(counts.cpu().numpy(), wc) and np.array_equal(pages.cpu().numpy(), wp)


def test_select_pages_queries_without_numbers():
    """An all-zero, an infinite and a NaN query score every page alike: the lowest pages are chosen."""
    codes = torch.randint(-127, 128, (40, 1, 2, 64), device=DEV, dtype=torch.int32).to(torch.int8)
    scales = torch.ones(40, 1, device=DEV)
    q = torch.zeros(3, 2, 64, device=DEV, dtype=BF)
    q[1, 1, 5], q[2, 0, 9] = float("inf"), float("nan")
    table = torch.arange(40, device=DEV, dtype=torch.int32).repeat(3, 1)
    pages, counts = zs().select_pages(q, codes, scales, table, i32([640] * 3), 16, 6)
    assert pages.tolist() == [[[0, 1, 2, 3, 4, 39]]] * 3 and counts.tolist() == [[6]] * 3


@pytest.mark.parametrize("lens,hq,hkv,D,page,top,dtype,layout", [
    ([3000, 0, 17, 640], 16, 4, 128, 64, 6, BF, "heads"),
    ([2000], 7, 1, 64, 16, 9, HF, "tokens"),
    ([300, 5000, 64], 40, 2, 64, 32, 20, BF, "tokens"),
])
def test_sparse_attention(lens, hq, hkv, D, page, top, dtype, layout):
    c = Cache(lens, hkv, D, page, dtype, layout, seed=D + top)
    n = c.k.shape[0]
    codes = torch.zeros(n, hkv, 2, D, dtype=torch.int8, device=DEV)
    scales = torch.zeros(n, hkv, device=DEV)
    zs().page_bounds(c.k, c.table, torch.zeros_like(c.lens), c.lens, codes, scales, max(lens))
    q = torch.randn(len(lens), hq, D, device=DEV).to(dtype)
    out, pages, counts = zs().sparse_attention(q, c.k, c.v, codes, scales, c.table, c.lens, top)
    wp, wc = select_ref(q, codes, scales, c.table, lens, page, top, 1, 1)
    assert np.array_equal(pages.cpu().numpy(), wp) and np.array_equal(counts.cpu().numpy(), wc)

    def rows(b, h):
        t = (wp[b, h, :wc[b, h], None] * page + np.arange(page)).ravel()
        return torch.from_numpy(t[t < lens[b]]).to(DEV)

    ref, _, vmax = attend_ref(q, c.dense, 1 / math.sqrt(D), rows)
    assert close(out, ref, vmax, dtype)
    # the same list with room for many more pages: in runs of chunks
    wide = torch.nn.functional.pad(pages, (0, 4096 - top), value=-1)
    lse = torch.empty(len(lens), hq, device=DEV)
    out = zs().paged_attention(q, c.k, c.v, c.table, c.lens, pages=wide, counts=counts, lse=lse)
    assert close(out, ref, vmax, dtype)
    assert bool(((lse == -math.inf) == (c.lens == 0).unsqueeze(1)).all())


def test_calls_of_different_sizes_from_two_threads():
    """The shared memory that a call needs goes by its sizes; another thread's call must not take it away."""
    from concurrent.futures import ThreadPoolExecutor

    def select(width):
        torch.manual_seed(width)
        codes = torch.randint(-127, 128, (64, 1, 2, 64), dtype=torch.int8, device=DEV)
        scales = torch.ones(64, 1, device=DEV)
        table = torch.randint(0, 64, (1, width), dtype=torch.int32, device=DEV)
        q = torch.randn(1, 4, 64, dtype=torch.bfloat16, device=DEV)
        args = (q, codes, scales, table, i32([width * 16]), 16, 32)
        first = zs().select_pages(*args)[0].clone()
        same = [torch.equal(zs().select_pages(*args)[0], first) for _ in range(200)]
        return all(same)

    def plan(R):
        for _ in range(200):
            p = zs().plan_step(torch.zeros(R, 1, dtype=torch.int32, device=DEV), i32([0] * R), i32([1] * R),
                               i32(np.arange(R)), i32([R]), 16, 16)
        return p.cu_tokens[-1].item() == 16

    for f, sizes in ((select, (12000, 32768)), (plan, (3000, 8192))):
        with ThreadPoolExecutor(2) as pool:
            assert all(pool.map(f, sizes))


def test_listed_pages_out_of_range_are_skipped():
    """Entries of a caller's page list that name no page of the sequence count nothing."""
    c = Cache([100, 40], 1, 64, 16, BF, "heads", 8)
    q = torch.randn(2, 2, 64, device=DEV).to(BF)
    pages, counts = i32([[[6, -1, 2, 500]], [[7, 3, 1, 0]]]), i32([[4], [2]])
    ref, _, vmax = attend_ref(q, c.dense, 0.125,
                              lambda b, h: [] if b else list(range(32, 48)) + list(range(96, 100)))
    for p in (pages, torch.nn.functional.pad(pages, (0, 4092), value=3)):
        out = zs().paged_attention(q, c.k, c.v, c.table, c.lens, pages=p, counts=counts)
        assert close(out, ref, vmax, BF) and bool((out[1] == 0).all())


@pytest.mark.parametrize("page, flagged", ((-1, 2), (8, 2), (500, 2), (7, 0)))
def test_listed_pages_outside_the_table_are_flagged(page, flagged):
    """A page past the length but inside the table counts nothing and is no error."""
    c = Cache([100, 40], 1, 64, 16, BF, "heads", 8)
    table = c.table[:, :8]
    q = torch.randn(2, 2, 64, device=DEV).to(BF)
    for top in (4, 4096):
        err = torch.zeros(1, dtype=torch.int32, device=DEV)
        pages = torch.full((2, 1, top), page, dtype=torch.int32, device=DEV)
        out = zs().paged_attention(q, c.k, c.v, table, c.lens, pages=pages, counts=i32([[1], [1]]), err=err)
        assert bool((out == 0).all()) and err.item() == flagged


# --------------------------------------------------------------- the C ABI
def test_paged_attention_from_c():
    """The argument struct filled by a foreign caller; a workspace that is too small is refused."""
    import ctypes as C

    from test_paged_args import STRUCTS
    from zipserv_asplos26_b200._lib import lib
    L = lib()
    f, need = L.zs_paged_attention, L.zs_paged_attention_workspace
    f.argtypes, f.restype, need.argtypes, need.restype = [C.c_char_p], C.c_int, [C.c_char_p], C.c_size_t
    pack = STRUCTS["ZsPagedAttention"].pack
    for lens, wants in (([100, 33], False), ([40000], True)):
        c = Cache(lens, 2, 128, 64, BF, "heads", seed=31)
        q = torch.randn(len(lens), 8, 128, device=DEV).to(BF)
        want = zs().paged_attention(q, c.k, c.v, c.table, c.lens)
        out = torch.full_like(q, 7.0)
        pools = [x for t in (c.k, c.v) for x in (t.data_ptr(), *t.stride()[:3], *t.shape, 0)]

        def args(ws, n):
            return pack(torch.cuda.current_stream().cuda_stream, q.data_ptr(), c.table.data_ptr(), c.table.stride(0),
                        c.lens.data_ptr(), 0, 0, ws, n, out.data_ptr(), 0, 0, *pools, len(lens), 8, c.table.shape[1],
                        0, 128 ** -0.5, 0)

        n = need(args(0, 0))
        assert (n > 0) == wants
        if n:
            ws = torch.empty(n, dtype=torch.uint8, device=DEV)
            assert f(args(ws.data_ptr(), n - 1)) == 1 and f(args(0, n)) == 1
            torch.cuda.synchronize()
            assert bool((out == 7).all())
            assert f(args(ws.data_ptr(), n)) == 0
        else:
            assert f(args(0, 0)) == 0
        assert torch.equal(out, want)


# ----------------------------------------------------------------- the cache
def test_cache_steps_in_a_graph():
    """Prompts, then decode steps replayed from one CUDA graph, one request ending
    and another starting in its row, against attention on the kept keys."""
    z = zs()
    B, hq, hkv, D, page, rows = 3, 8, 2, 128, 16, 400
    g = torch.Generator(device=DEV).manual_seed(21)
    ang = torch.rand(rows, D // 2, device=DEV, generator=g) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1)
    cache = z.PagedKVCache(40, B, 12, hkv, D, page)

    def draw(n):
        x = torch.randn(n, (hq + 2 * hkv), D, device=DEV, generator=g).to(BF)
        return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]

    kept = [[], [], []]

    def keep(plan, k, v):
        for t, (r, p) in enumerate(zip(plan.token_seq.tolist(), plan.positions.tolist())):
            if r >= 0:
                kk, _ = turn_ref(k[t:t + 1], torch.tensor([[p]]), cs, [D // 2], False)
                kept[r].append((kk[0].to(BF).to(DEV), v[t].clone()))

    prompts = [33, 0, 70]
    q, k, v = draw(103)
    plan = cache.step(i32(prompts), 103)
    cache.write(q, k, v, cs, plan)
    keep(plan, k, v)
    new = i32([1, 1, 1])
    xq, xk, xv = (t.contiguous() for t in draw(B))

    def step():
        plan = cache.step(new, B)
        qt = cache.write(xq, xk, xv, cs, plan)
        order = plan.token_seq.clamp(min=0).long()
        ql = torch.zeros_like(qt).index_copy_(0, order, qt)
        return plan, ql, cache.attention(ql), cache.sparse_attention(ql, 4)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    state = [t.clone() for t in (cache.seqlens, cache.free_count, cache.block_table, cache.free_blocks)]
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, s in zip((cache.seqlens, cache.free_count, cache.block_table, cache.free_blocks), state):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, ql, out, (sout, pages, counts) = step()
    for i in range(40):
        if i == 20:                          # row 0 ends, then starts again
            p = cache.step(i32([-1, 0, 0]), 0)
            kept[0] = []
            assert cache.seqlens.tolist()[0] == 0
        a, b, c = draw(B)
        xq.copy_(a), xk.copy_(b), xv.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        assert plan.cu_tokens.tolist() == [0, 1, 2, 3]
        keep(plan, xk, xv)
        lens = cache.seqlens.tolist()
        assert lens == [len(x) for x in kept]
        if i % 7 and i != 20:
            continue
        dense = [(torch.stack([a for a, _ in x]), torch.stack([b for _, b in x])) for x in kept]
        # a kept key may differ from the cache's by one rounding of its type: half a unit of every channel
        ref, _, vmax = attend_ref(ql, dense, 1 / math.sqrt(D))
        assert close(out, ref, vmax, BF)
        pg, ct = pages.cpu().numpy(), counts.cpu().numpy()

        def picked(b, h):
            t = (pg[b, h, :ct[b, h], None] * page + np.arange(page)).ravel()
            return torch.from_numpy(t[t < lens[b]]).to(DEV)

        ref, _, vmax = attend_ref(ql, dense, 1 / math.sqrt(D), picked)
        assert close(sout, ref, vmax, BF)
        assert ct.max() <= 4
    assert cache.check_errors() == 0
    used = sum(-(-n // page) for n in cache.seqlens.tolist())
    assert cache.free_count.item() == 40 - used
    live = cache.free_blocks[:cache.free_count.item()].tolist() + [
        b for r, n in enumerate(cache.seqlens.tolist()) for b in cache.block_table[r, :-(-n // page)].tolist()]
    assert sorted(live) == list(range(40))


# ---------------------------------------------------------------- refusals
def test_refusals_on_the_gpu():
    z = zs()
    c = Cache([40], 2, 64, 16, BF, "heads", 1)
    q = torch.randn(1, 4, 64, device=DEV).to(BF)
    for bad in (dict(q=q.half()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(k_pages=c.k[:, :, :1]),
                dict(v_pages=c.v.half()), dict(block_table=c.table.long()), dict(block_table=c.table[:0]),
                dict(seq_lens=c.lens.long()), dict(seq_lens=c.lens.cpu()), dict(softmax_scale=float("nan")),
                dict(pages=i32([[[0], [0]]])), dict(out=torch.empty(1, 4, 32, device=DEV, dtype=BF)),
                dict(lse=torch.empty(1, 3, device=DEV)),
                dict(max_seqlen=-1)):
        args = dict(q=q, k_pages=c.k, v_pages=c.v, block_table=c.table, seq_lens=c.lens)
        args.update(bad)
        with pytest.raises(ValueError):
            z.paged_attention(**args)
    wide = torch.zeros(3, 16, 2, 192, device=DEV, dtype=BF)
    with pytest.raises(ValueError):
        z.paged_attention(torch.zeros(1, 4, 192, device=DEV, dtype=BF), wide, wide, c.table, c.lens)
    with pytest.raises(ValueError):
        z.paged_attention(q, c.k[..., 1:], c.v[..., 1:], c.table, c.lens)
    codes, scales = torch.zeros(c.k.shape[0], 2, 2, 64, dtype=torch.int8, device=DEV), torch.zeros(c.k.shape[0], 2, device=DEV)
    for kw in (dict(top_pages=1), dict(top_pages=4, sink_pages=4), dict(top_pages=4, local_pages=0)):
        with pytest.raises(ValueError):
            z.select_pages(q, codes, scales, c.table, c.lens, 16, **kw)
    with pytest.raises(ValueError):
        z.sparse_attention(q, c.k, c.v, codes[1:], scales[1:], c.table, c.lens, 4)
    with pytest.raises(ValueError):
        z.page_bounds(c.k, c.table, c.lens, c.lens, codes[..., :32], scales, 4)
    lens, one = i32([3, 3]), i32([1])
    table, free = i32([[0], [1]]), i32([2])
    for kw in (dict(page_size=24), dict(page_size=512), dict(max_tokens=-1), dict(new_lens=one),
               dict(free_blocks=free[:0]), dict(free_count=lens), dict(block_table=i32([[0, 1]]))):
        args = dict(block_table=table, seq_lens=lens, new_lens=lens, free_blocks=free, free_count=one, page_size=16,
                    max_tokens=4)
        args.update(kw)
        with pytest.raises(ValueError):
            z.plan_step(**args)
    p = z.plan_step(table, lens, lens, free, one, 16, 6)
    with pytest.raises(ValueError):
        z.plan_step(table, p.seq_lens, lens, free, one, 16, 6, out=p)          # lengths in place
    with pytest.raises(ValueError):
        z.plan_step(table, lens, p.seq_lens, free, one, 16, 6, out=p)          # over what is asked for
    cs = torch.zeros(5, 64, device=DEV)
    k = torch.zeros(1, 2, 64, device=DEV, dtype=BF)
    slot = torch.zeros(1, dtype=torch.int64, device=DEV)
    for kw in (dict(cos_sin=cs[:, :24].contiguous()), dict(cos_sin=cs.double()), dict(positions=i32([0, 1])),
               dict(sections=[16, 16]), dict(positions=i32([[0], [0]])), dict(slots=slot.int()), dict(k=k[:, :1]),
               dict(positions=i32([[0], [0]]), sections=[40, -8])):
        args = dict(q=q, k=k, v=k, positions=i32([0]), cos_sin=cs, slots=slot, k_pages=c.k, v_pages=c.v)
        args.update(kw)
        with pytest.raises(ValueError):
            z.rope_write(**args)
    with pytest.raises(RuntimeError):
        z.PagedKVCache(2, 1, 2, 1, bounds=False).sparse_attention(torch.zeros(1, 1, 128, device=DEV, dtype=BF), 2)
