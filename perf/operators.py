"""Operators of a decode step over an uncompressed paged KV cache: what is measured.

Four operators, all over one cache layout (page pools of `page` tokens, a block
table per request):

* plan       block tables, slots and positions of a step, from request lengths
* rope       rotary positions with one or several axes on q and k, k and v
             written to their slots
* attention  one new token per request over its pages
* sparse     bounds of complete pages in 8 bits, the choice of pages by those
             bounds, attention over the chosen pages

With `own` false, `run` computes an operator with elementary torch operations in
32 bits; with `own` true it calls the framework.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
GOLDEN = 0.6180339887498949


# ------------------------------------------------------------------- cases
def listed():
    return [
        # The smallest step of a server: three chats, one token each.
        {"name": "plan-3-requests", "op": "plan", "requests": 3, "page": 64, "kind": "decode", "longest": 700,
         "chunk": 1},
        # A busy server's mixed step: most requests decode, some end, some prompts come in by chunks.
        {"name": "plan-256-mixed", "op": "plan", "requests": 256, "page": 64, "kind": "mixed", "longest": 8192,
         "chunk": 1024},
        # A batch of new prompts admitted at once, small pages.
        {"name": "plan-prompts", "op": "plan", "requests": 37, "page": 16, "kind": "prompts", "longest": 8192,
         "chunk": 7013},
        # The decode step of 32 requests: latency.
        {"name": "rope-32-tokens", "op": "rope", "tokens": 32, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "axes": 1,
         "page": 64, "dtype": "bf16", "layout": "heads", "interleaved": False},
        # A prompt with images and video: three axes, an odd number of tokens.
        {"name": "rope-video-prompt", "op": "rope", "tokens": 16411, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "axes": 3, "page": 64, "dtype": "bf16", "layout": "heads", "interleaved": False},
        # A lone chat at its start: latency.
        {"name": "attention-1x97", "op": "attention", "requests": 1, "shortest": 97, "longest": 97, "hq": 32, "hkv": 8,
         "dim": 128, "page": 64, "dtype": "bf16", "layout": "heads"},
        # A batch in step at a common context.
        {"name": "attention-32x4129", "op": "attention", "requests": 32, "shortest": 4129, "longest": 4129, "hq": 32,
         "hkv": 8, "dim": 128, "page": 64, "dtype": "bf16", "layout": "heads"},
        # A server's ragged batch, empty rows among it, small pages with the tokens outermost.
        {"name": "attention-ragged-61", "op": "attention", "requests": 61, "shortest": 0, "longest": 16417, "hq": 64,
         "hkv": 8, "dim": 128, "page": 16, "dtype": "fp16", "layout": "tokens"},
        # One request with a long document: the split over the cache's length.
        {"name": "attention-1x131105", "op": "attention", "requests": 1, "shortest": 131105, "longest": 131105,
         "hq": 32, "hkv": 8, "dim": 128, "page": 64, "dtype": "bf16", "layout": "heads"},
        # The bounds of the pages that four prompts filled.
        {"name": "sparse-bounds", "op": "bounds", "requests": 4, "shortest": 16417, "longest": 32801, "hkv": 8,
         "dim": 128, "page": 64, "dtype": "bf16", "layout": "heads"},
        # One long request, 48 of its 513 pages attended: latency.
        {"name": "sparse-1x32801", "op": "sparse", "requests": 1, "shortest": 32801, "longest": 32801, "hq": 32,
         "hkv": 8, "dim": 128, "page": 64, "top": 48, "dtype": "bf16", "layout": "heads"},
        # Eight long documents, 64 of up to 2049 pages attended.
        {"name": "sparse-8x131105", "op": "sparse", "requests": 8, "shortest": 65553, "longest": 131105, "hq": 32,
         "hkv": 8, "dim": 128, "page": 64, "top": 64, "dtype": "bf16", "layout": "heads"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attention", "attention", "bounds", "sparse"])
    c = {"op": op, "page": rng.choice([16, 32, 64, 128])}
    if op == "plan":
        kind = rng.choice(["decode", "mixed", "prompts"])
        c.update(kind=kind, requests=_log(rng, 1, 1024), longest=_log(rng, 16, 16384), chunk=1)
        if kind != "decode":
            # the sum of the new tokens stays below the largest listed case's
            c["chunk"] = max(1, min(_log(rng, 2, 8192), 250000 // c["requests"]))
        return c
    c.update(dtype=rng.choice(["bf16", "bf16", "fp16"]), layout=rng.choice(["heads", "tokens"]),
             dim=rng.choice([64, 128, 128]))
    hkv = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 4, 4, 7, 8, 16])
    if op == "rope":
        c.update(tokens=_log(rng, 1, 16000), hkv=hkv, hq=min(hkv * group, 32) // hkv * hkv, axes=rng.choice([1, 2, 3]),
                 interleaved=rng.random() < 0.5)
        c["rot"] = c["dim"] if rng.random() < 0.6 else c["dim"] // 2
        return c
    longest = _log(rng, 1, 65536)
    kv_bytes = {"attention": 1.6e9 * min(1.0, 8 / group), "bounds": 0.4e9, "sparse": 3e9}[op]
    requests = max(1, min(_log(rng, 1, 128), int(kv_bytes / (longest * hkv * c["dim"] * 4.0))))
    c.update(requests=requests, shortest=int(longest * rng.choice([0.0, 0.3, 1.0])), longest=longest, hkv=hkv)
    if op != "bounds":
        c["hq"] = hkv * group
    if op == "sparse":
        pages = -(-longest // c["page"])
        c["top"] = _log(rng, 2, max(2, min(128, pages)))
        # the chosen pages' bytes stay below the largest listed case's
        c["top"] = max(2, min(c["top"], int(1.2e8 / (requests * hkv * c["page"] * c["dim"] * 4.0))))
    return c


# ------------------------------------------------------------ deterministic shapes
def _spread(n, lo, hi):
    """n lengths from lo to hi, the same for every seed (the seed permutes them)."""
    if n == 1:
        return np.array([hi], np.int64)
    f = np.modf((np.arange(n) + 1) * GOLDEN)[0]
    out = np.floor(lo + (hi - lo) * f + 0.5).astype(np.int64)
    out[int(f.argmax())] = hi
    out[int(f.argmin())] = lo
    return out


def _plan_lengths(case):
    """Length of each request before the step, and its new tokens (-1: it has ended)."""
    n, kind = case["requests"], case["kind"]
    before = _spread(n, 0 if kind != "decode" else 1, case["longest"])
    i = np.arange(n)
    if kind == "decode":
        new = np.where(i % 16 == 15, -1, 1)
    elif kind == "prompts":
        before = np.zeros(n, np.int64)
        new = _spread(n, 1, case["chunk"])
    else:
        f = _spread(n, 1, case["chunk"])
        new = np.where(i % 8 == 0, f, np.where(i % 16 == 3, -1, np.where(i % 16 == 7, 0, 1)))
    return before.astype(np.int64), new.astype(np.int64)


def work(case):
    op = case["op"]
    if op == "plan":
        before, new = _plan_lengths(case)
        n, page = case["requests"], case["page"]
        tokens = int(new.clip(0).sum())
        after = before + new.clip(0)
        blocks = int((-(-after // page) - -(-before // page))[new >= 0].sum())
        freed = int((-(-before // page))[new < 0].sum())
        # lengths in and out, offsets, per token a slot, its request and its position, per block taken or given
        # back one read and one write
        return {"bytes": 16 * n + 16 * tokens + 8 * (blocks + freed), "flops": 4 * n + 4 * tokens}
    e, d, hkv = 2, case["dim"], case["hkv"]
    if op == "rope":
        n, hq = case["tokens"], case["hq"]
        vals = n * (hq + 2 * hkv) * d
        return {"bytes": 2 * e * vals + n * (8 + 4 * case["axes"] + 4 * case["rot"]),
                "flops": 3 * n * (hq + hkv) * case["rot"]}
    lens = _spread(case["requests"], case["shortest"], case["longest"])
    page, table = case["page"], 4 * int((-(-lens // case["page"])).sum())
    if op == "bounds":
        full = int((lens // page).sum())
        return {"bytes": full * hkv * (page * d * e + 2 * d + 4) + table, "flops": 2 * full * page * hkv * d}
    hq, b = case["hq"], case["requests"]
    io = 2 * e * b * hq * d + 4 * b
    if op == "attention":
        t = int(lens.sum())
        return {"bytes": 2 * e * t * hkv * d + io + table, "flops": 4 * t * hq * d}
    pages = -(-lens // page)
    scored = int(np.where(pages > case["top"], pages - 2, 0).sum())
    taken = np.minimum(pages, case["top"])
    t = int(np.minimum(lens, taken * page - (pages * page - lens)).clip(0).sum())
    return {"bytes": 2 * e * t * hkv * d + io + table + scored * hkv * (2 * d + 4) + 4 * b * hkv * (case["top"] + 1),
            "flops": 4 * t * hq * d + 4 * scored * hq * d}


# ------------------------------------------------------------------ inputs
def _pool(shape, layout, dtype, gen, scale=None, drift=None):
    """A page pool [blocks, page, heads, dim]; layout "heads" keeps each head's rows of a page together."""
    blocks, page, heads, dim = shape
    if layout == "heads":
        x = torch.empty(blocks, heads, page, dim, dtype=dtype, device="cuda")
        step = max(1, (1 << 27) // (heads * page * dim))
        for i in range(0, blocks, step):
            part = torch.randn(min(step, blocks - i), heads, page, dim, dtype=torch.float32, device="cuda",
                               generator=gen)
            if drift is not None:
                part += drift[i:i + step].unsqueeze(2)
            if scale is not None:
                part *= scale.unsqueeze(1)
            x[i:i + step] = part
        return x.transpose(1, 2)
    x = torch.empty(blocks, page, heads, dim, dtype=dtype, device="cuda")
    step = max(1, (1 << 27) // (heads * page * dim))
    for i in range(0, blocks, step):
        part = torch.randn(min(step, blocks - i), page, heads, dim, dtype=torch.float32, device="cuda", generator=gen)
        if drift is not None:
            part += drift[i:i + step].unsqueeze(1)
        if scale is not None:
            part *= scale
        x[i:i + step] = part
    return x


def _tables(lens, page, rng, spare=5, width_slack=2):
    """A block table over a shuffled pool, -1 past each request's pages."""
    pages = -(-lens // page)
    total = int(pages.sum())
    order = rng.permutation(total + spare)
    width = max(1, int(pages.max(initial=0))) + width_slack
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = order[at:at + p]
        at += p
    return table, order[at:], total + spare


def _gpu(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device="cuda", dtype=dtype)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "plan":
        before, new = _plan_lengths(case)
        perm = rng.permutation(len(before))
        before, new = before[perm], new[perm]
        page = case["page"]
        after = before + new.clip(0)
        need = int((-(-after // page) - -(-before // page))[new >= 0].sum())
        table, free, blocks = _tables(before, page, rng, spare=need + 7)
        width = int((-(-after // page)).max(initial=1)) + 2
        if width > table.shape[1]:
            table = np.pad(table, ((0, 0), (0, width - table.shape[1])), constant_values=-1)
        free_list = np.full(blocks, -1, np.int32)
        free_list[:len(free)] = free
        s.update(table=_gpu(table), before=_gpu(before), new=_gpu(new), free=_gpu(free_list),
                 free_count=_gpu(np.array([len(free)])), tokens=int(new.clip(0).sum()) + 3)
        return s
    dtype, dim, hkv, page = TYPES[case["dtype"]], case["dim"], case["hkv"], case["page"]
    if op == "rope":
        n, hq, rot = case["tokens"], case["hq"], case["rot"]
        blocks = -(-n // page) + 3
        qkv = torch.randn(n, (hq + 2 * hkv) * dim, device="cuda", generator=gen).to(dtype)
        s["q"] = qkv[:, :hq * dim].view(n, hq, dim)
        s["k"] = qkv[:, hq * dim:(hq + hkv) * dim].view(n, hkv, dim)
        s["v"] = qkv[:, (hq + hkv) * dim:].view(n, hkv, dim)
        longest = 32768
        # text first, then frames of a grid: the axes are time, height and width
        pos = np.zeros((case["axes"], n), np.int64)
        start = int(rng.integers(0, longest // 4))
        i = np.arange(n)
        side = 24
        pos[0] = start + (i if case["axes"] == 1 else i // (side * side))
        if case["axes"] > 1:
            pos[1] = start + i // side % side
        if case["axes"] > 2:
            pos[2] = start + i % side
        s["positions"] = _gpu(pos[0] if case["axes"] == 1 else pos)
        inv = 500000.0 ** (-np.arange(rot // 2) * 2.0 / rot)
        ang = np.arange(longest)[:, None] * inv[None]
        s["cos_sin"] = _gpu(np.concatenate([np.cos(ang), np.sin(ang)], 1), torch.float32)
        s["sections"] = _sections(case)
        order = rng.permutation(blocks)
        slots = order[i // page] * page + i % page
        slots[rng.random(n) < 0.002] = -1          # padding of the step
        s["slots"] = _gpu(slots, torch.int64)
        s["k_pages"] = _pool((blocks, page, hkv, dim), case["layout"], dtype, gen)
        s["v_pages"] = _pool((blocks, page, hkv, dim), case["layout"], dtype, gen)
        return s
    lens = _spread(case["requests"], case["shortest"], case["longest"])
    lens = lens[rng.permutation(len(lens))]
    table, _, blocks = _tables(lens, page, rng)
    scale = torch.exp(torch.empty(hkv, dim, device="cuda").uniform_(math.log(0.1), math.log(4.0), generator=gen))
    s.update(table=_gpu(table), lens=_gpu(lens))
    # neighbouring tokens' keys are alike: pages differ by a mean of their own where pages are chosen
    drift = None
    if op != "attention":
        drift = torch.randn(blocks, hkv, dim, device="cuda", generator=gen).mul_(0.7)
    s["k_pages"] = _pool((blocks, page, hkv, dim), case["layout"], dtype, gen, scale, drift)
    if op == "bounds":
        s["before"] = torch.zeros_like(s["lens"])
        s["codes"] = torch.zeros(blocks, hkv, 2, dim, dtype=torch.int8, device="cuda")
        s["scales"] = torch.zeros(blocks, hkv, dtype=torch.float32, device="cuda")
        return s
    s["v_pages"] = _pool((blocks, page, hkv, dim), case["layout"], dtype, gen, scale)
    s["q"] = torch.randn(case["requests"], case["hq"], dim, device="cuda", generator=gen).to(dtype)
    if op == "sparse":
        codes, scales = [], []
        step = max(1, (1 << 27) // (hkv * page * dim))
        for i in range(0, blocks, step):
            c, t = _bounds_of(s["k_pages"][i:i + step])
            codes.append(c)
            scales.append(t)
        s["codes"], s["scales"] = torch.cat(codes), torch.cat(scales)
    return s


def _sections(case):
    half = case["rot"] // 2
    if case["axes"] == 1:
        return [half]
    rest = half // 8 * 3 if case["axes"] == 3 else half // 2
    return [half - rest * (case["axes"] - 1)] + [rest] * (case["axes"] - 1)


# -------------------------------------------------------------- plain forms
def _plain_plan(s):
    page = s["case"]["page"]
    table, before, new, free, count = s["table"], s["before"], s["new"], s["free"], s["free_count"]
    n, width = table.shape
    total = s["tokens"]
    dev = table.device
    ended = new < 0
    old_pages = torch.div(before + page - 1, page, rounding_mode="floor")
    # pages of ended requests go back on the list, in the order of requests and pages
    back = torch.where(ended, old_pages, torch.zeros_like(old_pages))
    back_end = torch.cumsum(back, 0)
    col = torch.arange(width, device=dev)
    where = count + (back_end - back).unsqueeze(1) + col
    give = col < back.unsqueeze(1)
    spill = torch.cat([free, free.new_zeros(1)])
    spill[torch.where(give, where, torch.full_like(where, free.numel())).long()] = table
    free.copy_(spill[:-1])
    have = count + back_end[-1]
    # a request is admitted when the step has room for its tokens and its pages
    want = new.clamp(min=0)
    after = before + want
    pages = torch.div(after + page - 1, page, rounding_mode="floor")
    fits = ~ended & (torch.cumsum(want, 0) <= total) & (pages <= width)
    need = torch.where(fits, pages - old_pages, torch.zeros_like(pages))
    need_end = torch.cumsum(need, 0)
    fits &= (need == 0) | (need_end <= have)
    need = torch.where(fits, need, torch.zeros_like(need))
    start = need_end - need
    take = (col >= old_pages.unsqueeze(1)) & (col < (old_pages + need).unsqueeze(1))
    pop = have - 1 - (start.unsqueeze(1) + col - old_pages.unsqueeze(1))
    table.copy_(torch.where(take, free[pop.clamp(0, free.numel() - 1).long()], table))
    got = torch.where(fits, want, torch.zeros_like(want))
    cu = torch.cat([got.new_zeros(1), torch.cumsum(got, 0)]).int()
    tok = torch.arange(total, device=dev)
    req = torch.searchsorted(cu, tok.int(), right=True) - 1
    live = tok < cu[-1]
    req = torch.where(live, req, torch.zeros_like(req))
    pos = torch.where(live, before[req] + tok - cu[req], torch.zeros_like(tok))
    slot = table[req, torch.div(pos, page, rounding_mode="floor")].long() * page + pos % page
    return {"block_table": table, "free_blocks": free, "free_count": (have - need.sum()).int(),
            "seq_lens": torch.where(ended, torch.zeros_like(before), before + got).int(), "cu_tokens": cu,
            "slots": torch.where(live, slot, torch.full_like(slot, -1)),
            "token_seq": torch.where(live, req, torch.full_like(req, -1)).int(), "positions": pos.int(),
            "refused": (~fits & (new > 0))}


def _turn(x, cos, sin, interleaved):
    rot = cos.shape[-1] * 2
    xf = x.float()
    if interleaved:
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, xf[..., rot:]], -1)


def _plain_rope(s):
    c = s["case"]
    pos = s["positions"] if s["positions"].dim() == 2 else s["positions"].unsqueeze(0)
    half = c["rot"] // 2
    cols, at = [], 0
    for a, w in enumerate(s["sections"]):
        rows = s["cos_sin"][pos[a].long()]
        cols.append((rows[:, at:at + w], rows[:, half + at:half + at + w]))
        at += w
    cos = torch.cat([x for x, _ in cols], 1).unsqueeze(1)
    sin = torch.cat([x for _, x in cols], 1).unsqueeze(1)
    q = _turn(s["q"], cos, sin, c["interleaved"]).to(s["q"].dtype)
    k = _turn(s["k"], cos, sin, c["interleaved"]).to(s["k"].dtype)
    live = (s["slots"] >= 0).nonzero().squeeze(1)
    slot = s["slots"][live]
    block, row = torch.div(slot, c["page"], rounding_mode="floor"), slot % c["page"]
    s["k_pages"][block, row] = k[live]
    s["v_pages"][block, row] = s["v"][live]
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(q, k_pages, v_pages, blocks, valid):
    """q [B, Hq, D]; blocks [B, Hkv or 1, n] physical pages; valid [B, Hkv or 1, n, page] rows that count."""
    b, hq, d = q.shape
    hkv, page = k_pages.shape[2], k_pages.shape[1]
    qf = q.float().view(b, hkv, hq // hkv, d)
    out = torch.empty(b, hq, d, dtype=torch.float32, device=q.device)
    heads = torch.arange(hkv, device=q.device).view(1, hkv, 1)
    # requests in groups, so that the gathered 32-bit keys stay within a few GB
    step = max(1, int(1.5e9 / (hkv * blocks.shape[-1] * page * d * 4)))
    for i in range(0, b, step):
        blk = blocks[i:i + step].clamp(min=0).long().expand(-1, hkv, -1)
        ok = valid[i:i + step].expand(-1, hkv, -1, -1).flatten(2)
        kk = k_pages.transpose(1, 2)[blk, heads].float().flatten(2, 3)
        kk = torch.where(ok.unsqueeze(-1), kk, torch.zeros((), device=q.device))
        sc = torch.matmul(qf[i:i + step], kk.transpose(-1, -2)) * (1.0 / math.sqrt(d))
        del kk
        sc = torch.where(ok.unsqueeze(2), sc, torch.full((), -math.inf, device=q.device))
        top = sc.amax(-1, keepdim=True)
        p = torch.exp(sc - torch.where(top == -math.inf, torch.zeros_like(top), top))
        p = torch.where(ok.unsqueeze(2), p, torch.zeros_like(p))
        total = p.sum(-1, keepdim=True)
        vv = v_pages.transpose(1, 2)[blk, heads].float().flatten(2, 3)
        vv = torch.where(ok.unsqueeze(-1), vv, torch.zeros((), device=q.device))
        o = torch.matmul(p, vv) / torch.where(total == 0, torch.ones_like(total), total)
        del vv
        out[i:i + step] = o.reshape(-1, hq, d)
    return out.to(q.dtype)


def _plain_attention(s):
    page, lens = s["case"]["page"], s["lens"]
    width = s["table"].shape[1]
    rows = torch.arange(width * page, device=lens.device).view(width, page)
    valid = rows.unsqueeze(0) < lens.view(-1, 1, 1)
    return {"out": _attend(s["q"], s["k_pages"], s["v_pages"], s["table"].unsqueeze(1), valid.unsqueeze(1))}


def _bounds_of(k):
    """Pages [n, page, heads, dim] -> their bounds: codes [n, heads, 2, dim] (upper, lower) and a power-of-two
    scale [n, heads]. Non-finite keys give an infinite scale and codes of zero."""
    kf = k.float()
    hi, lo = kf.amax(1), kf.amin(1)
    most = torch.maximum(hi.abs().amax(-1), lo.abs().amax(-1))
    power = (most.view(torch.int32) & 0x7F800000).view(torch.float32)
    finite = torch.isfinite(most)
    scale = torch.where(finite, power * 0.015625, torch.full_like(power, math.inf))
    div = torch.where(finite & (power > 0), scale, torch.ones_like(scale)).unsqueeze(-1)
    live = (finite & (power > 0)).unsqueeze(-1)
    up = torch.where(live, torch.ceil(hi / div), torch.zeros_like(hi)).clamp(-127, 127)
    down = torch.where(live, torch.floor(lo / div), torch.zeros_like(lo)).clamp(-127, 127)
    return torch.stack([up, down], 2).to(torch.int8), scale


def _plain_bounds(s):
    page = s["case"]["page"]
    width = s["table"].shape[1]
    col = torch.arange(width, device=s["table"].device)
    full = (col < torch.div(s["lens"], page, rounding_mode="floor").unsqueeze(1)) & \
        (col >= torch.div(s["before"], page, rounding_mode="floor").unsqueeze(1))
    blocks = s["table"][full].long()
    hkv, d = s["k_pages"].shape[2:]
    step = max(1, (1 << 28) // (hkv * page * d))
    for i in range(0, blocks.numel(), step):
        b = blocks[i:i + step]
        s["codes"][b], s["scales"][b] = _bounds_of(s["k_pages"][b])
    return {"codes": s["codes"], "scales": s["scales"]}


def _plain_select(s, sinks=1, local=1):
    c = s["case"]
    page, top, table = c["page"], c["top"], s["table"]
    q = s["q"].float()
    b, hq, d = q.shape
    hkv = s["codes"].shape[1]
    g = hq // hkv
    qg = q.view(b, hkv, g, d)
    most = qg.abs().amax((-1, -2), keepdim=True)
    power = (most.view(torch.int32) & 0x7F800000).view(torch.float32) * 0.015625
    live = torch.isfinite(most) & (power > 0)
    q8 = torch.where(live, torch.round(qg / torch.where(live, power, torch.ones_like(power))), torch.zeros_like(qg))
    q8 = q8.clamp(-127, 127)
    blk = table.clamp(min=0).long()
    codes = s["codes"][blk].float()                                  # [B, width, Hkv, 2, D]
    up, down = codes[:, :, :, 0].transpose(1, 2), codes[:, :, :, 1].transpose(1, 2)
    # products of whole numbers below 2^14, sums below 2^24: exact in 32 bits in any order
    sc = torch.zeros(b, hkv, g, table.shape[1], device=q.device)
    for j in range(g):
        qj = q8[:, :, j].unsqueeze(2)
        sc[:, :, j] = torch.where(qj > 0, qj * up, qj * down).sum(-1)
    scale = s["scales"][blk].transpose(1, 2)
    key = sc.amax(2) * scale
    key = torch.where(torch.isfinite(scale), key, torch.full_like(key, math.inf))
    pages = torch.div(s["lens"] + page - 1, page, rounding_mode="floor").view(-1, 1, 1)
    col = torch.arange(table.shape[1], device=q.device)
    live_col = col < pages
    forced = live_col & ((col < sinks) | (col >= pages - local))
    # rank: forced pages, then by score, ties to the lowest page; pages past the end last
    key = torch.where(forced, torch.full_like(key, math.inf), key)
    tier = torch.where(forced, 0, torch.where(live_col, 1, 2)).expand_as(key)
    by_key = torch.sort(-key, dim=-1, stable=True).indices
    by_tier = torch.sort(torch.gather(tier, -1, by_key), dim=-1, stable=True).indices
    order = torch.gather(by_key, -1, by_tier)
    k = min(top, table.shape[1])
    counts = torch.clamp(pages.squeeze(-1), max=top).expand(b, hkv)
    chosen = torch.where(torch.arange(k, device=q.device) < counts.unsqueeze(-1), order[..., :k],
                         torch.full_like(order[..., :k], table.shape[1]))
    chosen = torch.sort(chosen, dim=-1).values
    out = torch.full((b, hkv, top), -1, dtype=torch.int32, device=q.device)
    out[..., :k] = torch.where(chosen < table.shape[1], chosen, torch.full_like(chosen, -1)).int()
    return out, counts.int().contiguous()


def _plain_sparse(s):
    page = s["case"]["page"]
    pages, counts = _plain_select(s)
    b = pages.shape[0]
    idx = pages.clamp(min=0).long()
    blocks = torch.gather(s["table"].unsqueeze(1).expand(-1, pages.shape[1], -1), 2, idx)
    rows = idx.unsqueeze(-1) * page + torch.arange(page, device=idx.device)
    valid = (pages >= 0).unsqueeze(-1) & (rows < s["lens"].view(b, 1, 1, 1))
    return {"out": _attend(s["q"], s["k_pages"], s["v_pages"], blocks, valid), "pages": pages, "counts": counts}


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "rope": _plain_rope, "attention": _plain_attention, "bounds": _plain_bounds,
                "sparse": _plain_sparse}[op](s)
    import zipserv_asplos26_b200 as zs
    if op == "plan":
        p = zs.plan_step(s["table"], s["before"], s["new"], s["free"], s["free_count"], page_size=s["case"]["page"],
                         max_tokens=s["tokens"])
        return {"block_table": s["table"], "free_blocks": s["free"], "free_count": p.free_count,
                "seq_lens": p.seq_lens, "cu_tokens": p.cu_tokens, "slots": p.slots, "token_seq": p.token_seq,
                "positions": p.positions, "refused": p.refused}
    if op == "rope":
        q = zs.rope_write(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["slots"], s["k_pages"],
                          s["v_pages"], sections=s["sections"], interleaved=s["case"]["interleaved"])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "attention":
        return {"out": zs.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"])}
    if op == "bounds":
        zs.page_bounds(s["k_pages"], s["table"], s["before"], s["lens"], s["codes"], s["scales"],
                       max_new=s["case"]["longest"])
        return {"codes": s["codes"], "scales": s["scales"]}
    out, pages, counts = zs.sparse_attention(s["q"], s["k_pages"], s["v_pages"], s["codes"], s["scales"], s["table"],
                                             s["lens"], top_pages=s["case"]["top"])
    return {"out": out, "pages": pages, "counts": counts}


# ------------------------------------------------------------------- exact
def _exact_plan(s):
    page = s["case"]["page"]
    table, before, new = (s[k].cpu().numpy().astype(np.int64) for k in ("table", "before", "new"))
    free, count = s["free"].cpu().numpy().astype(np.int64), int(s["free_count"].item())
    width, room = table.shape[1], s["tokens"]
    for r in range(len(new)):
        if new[r] < 0:
            p = -(-before[r] // page)
            free[count:count + p] = table[r, :p]
            count += p
    have, asked, claimed = count, 0, 0
    lens, cu, refused = before.copy(), [0], np.zeros(len(new), bool)
    slots, seqs, poss = [], [], []
    for r in range(len(new)):
        if new[r] < 0:
            lens[r] = 0
            cu.append(cu[-1])
            continue
        asked += new[r]
        old, now = -(-before[r] // page), -(-(before[r] + new[r]) // page)
        ok = asked <= room and now <= width
        if ok:
            claimed += now - old
            ok = now == old or claimed <= have
        if not ok:
            refused[r] = new[r] > 0
            cu.append(cu[-1])
            continue
        for p in range(old, now):
            count -= 1
            table[r, p] = free[count]
        lens[r] += new[r]
        cu.append(cu[-1] + new[r])
        pos = np.arange(before[r], lens[r])
        slots.append(table[r, pos // page] * page + pos % page)
        seqs.append(np.full(len(pos), r))
        poss.append(pos)
    pad = room - cu[-1]

    def joined(parts, fill):
        return np.concatenate(parts + [np.full(pad, fill)]).astype(np.int64)

    def t(x, dtype=torch.int32):
        return torch.from_numpy(np.ascontiguousarray(x)).to(dtype)

    return {"block_table": t(table), "free_blocks": t(free), "free_count": t(np.array([count])), "seq_lens": t(lens),
            "cu_tokens": t(np.array(cu)), "slots": t(joined(slots, -1), torch.int64), "token_seq": t(joined(seqs, -1)),
            "positions": t(joined(poss, 0)), "refused": t(refused, torch.bool)}


def _exact_rope(s):
    c = s["case"]
    half, n = c["rot"] // 2, c["tokens"]
    pos = s["positions"].reshape(c["axes"], n).long()
    axis = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(s["sections"])).to(pos.device)
    at = pos[axis].t()                                              # [n, half]: the position each channel turns by
    chan = torch.arange(half, device=pos.device)
    z = torch.complex(s["cos_sin"].double()[at, chan], s["cos_sin"].double()[at, half + chan]).unsqueeze(1)

    def turn(x):
        y = x.double().clone()
        lo = slice(0, c["rot"], 2) if c["interleaved"] else slice(0, half)
        hi = slice(1, c["rot"], 2) if c["interleaved"] else slice(half, c["rot"])
        w = torch.complex(y[..., lo], y[..., hi]) * z
        y[..., lo], y[..., hi] = w.real, w.imag
        return y

    k, kp, vp = turn(s["k"]), s["k_pages"].double().clone(), s["v_pages"].double().clone()
    live = s["slots"] >= 0
    slot = s["slots"][live]
    kp[slot // c["page"], slot % c["page"]] = k[live]
    vp[slot // c["page"], slot % c["page"]] = s["v"][live].double()
    return {"q": turn(s["q"]), "k_pages": kp, "v_pages": vp}


def _exact_attend(s, rows_of):
    """rows_of(request, head) -> the physical (block, row) pairs that the head attends."""
    q = s["q"].double()
    b, hq, d = q.shape
    hkv = s["k_pages"].shape[2]
    out = torch.zeros(b, hkv, hq // hkv, d, dtype=torch.float64, device=q.device)
    for r in range(b):
        for h in range(hkv):
            blk, row = rows_of(r, h)
            if blk.numel() == 0:
                continue
            k, v = s["k_pages"][blk, row, h].double(), s["v_pages"][blk, row, h].double()
            out[r, h] = torch.softmax(q[r].view(hkv, -1, d)[h] @ k.t() / math.sqrt(d), -1) @ v
    return out.view(b, hq, d)


def _exact_attention(s):
    page, lens = s["case"]["page"], s["lens"].tolist()

    def rows_of(r, h):
        i = torch.arange(lens[r], device="cuda")
        return s["table"][r].long()[i // page], i % page

    return {"out": _exact_attend(s, rows_of)}


def _exact_bounds(s):
    page = s["case"]["page"]
    codes, scales = s["codes"].clone(), s["scales"].clone()
    table = s["table"].long()
    for r, (a, z) in enumerate(zip(s["before"].tolist(), s["lens"].tolist())):
        blocks = table[r, a // page:z // page]
        for b in blocks.split(256):
            k = s["k_pages"][b].double()
            hi, lo = k.amax(1), k.amin(1)
            most = torch.maximum(hi.abs(), lo.abs()).amax(-1)
            _, e = torch.frexp(most)
            step = torch.where(most > 0, torch.pow(2.0, (e - 7).double()), torch.ones_like(most))
            codes[b, :, 0] = torch.ceil(hi / step[..., None]).clamp(-127, 127).to(torch.int8)
            codes[b, :, 1] = torch.floor(lo / step[..., None]).clamp(-127, 127).to(torch.int8)
            scales[b] = torch.where(most > 0, step, torch.zeros_like(step)).float()
    return {"codes": codes, "scales": scales}


def _exact_sparse(s):
    c = s["case"]
    page, top, hkv = c["page"], c["top"], s["codes"].shape[1]
    q = s["q"].double().cpu().numpy()
    lens, table = s["lens"].tolist(), s["table"].cpu().numpy()
    codes, scales = s["codes"].cpu().numpy(), s["scales"].cpu().numpy().astype(np.float64)
    b, hq, d = q.shape
    g = hq // hkv
    pages = np.full((b, hkv, top), -1, np.int64)
    counts = np.zeros((b, hkv), np.int64)
    for r in range(b):
        n = -(-lens[r] // page)
        blk = table[r, :n]
        for h in range(hkv):
            qg = q[r, h * g:(h + 1) * g]
            most = np.abs(qg).max()
            step = 2.0 ** (math.frexp(most)[1] - 7) if most > 0 else 1.0
            q8 = np.clip(np.round(qg / step), -127, 127)
            up, down = codes[blk, h, 0].astype(np.float64), codes[blk, h, 1].astype(np.float64)
            key = (np.maximum(q8, 0) @ up.T + np.minimum(q8, 0) @ down.T).max(0) * scales[blk, h] if n else np.zeros(0)
            key[:1] = np.inf
            key[n - 1:] = np.inf
            pick = np.sort(np.lexsort((np.arange(n), -key))[:top])
            counts[r, h] = len(pick)
            pages[r, h, :len(pick)] = pick
    t = s["table"].long()

    def rows_of(r, h):
        i = (torch.from_numpy(pages[r, h, :counts[r, h]])[:, None] * page + torch.arange(page)).flatten()
        i = i[i < lens[r]].cuda()
        return t[r][i // page], i % page

    return {"out": _exact_attend(s, rows_of), "pages": torch.from_numpy(pages).int(),
            "counts": torch.from_numpy(counts).int()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "attention": _exact_attention, "bounds": _exact_bounds,
            "sparse": _exact_sparse}[case["op"]](s)
