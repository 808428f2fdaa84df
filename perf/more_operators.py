"""Operators of a decode step over a paged KV cache held in 4 bits: what is measured.

* write      rotary positions on q and k, k and v quantised to 4 bits at their
             slots of the cache, and the written rows read back (what a step with
             prompts does)
* read       rows of the cache read back by slot
* attention  one new token per request over its pages of 4-bit keys and values
* sample     one token per row of logits from a given random number, with
             temperature, top-k, top-p and min-p

A row of `dim` channels is held in groups of `group` channels, a 4-bit code u per
channel and a bf16 scale s and centre c per group; it stands for c + s (u - 8):

    s = bf16((max - min) / 15), c = bf16(min + 8 s), u = clamp(rint((x - c) / s) + 8, 0, 15)

With `own` false, `run` computes an operator with elementary torch operations in
32 bits (sampling in 64: a sum's place among a hundred thousand borders); with
`own` true it calls the framework.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GOLDEN = 0.6180339887498949
LONGEST = 32768          # rows of the table of angles


# ------------------------------------------------------------------- cases
def listed():
    return [
        # The decode step of 32 requests: latency.
        {"name": "write-32-tokens", "op": "write", "tokens": 32, "hq": 32, "hkv": 8, "dim": 128, "rot": 128, "axes": 1,
         "page": 64, "group": 64, "dtype": "bf16", "layout": "heads", "interleaved": False},
        # A prompt with images and video: three axes, pairs side by side, half of each head turns.
        {"name": "write-4099-three-axes", "op": "write", "tokens": 4099, "hq": 24, "hkv": 4, "dim": 128, "rot": 64,
         "axes": 3, "page": 16, "group": 32, "dtype": "fp16", "layout": "tokens", "interleaved": True},
        # Prompts of a busy server's step, admitted together.
        {"name": "write-16411-tokens", "op": "write", "tokens": 16411, "hq": 32, "hkv": 8, "dim": 128, "rot": 128,
         "axes": 1, "page": 64, "group": 64, "dtype": "bf16", "layout": "heads", "interleaved": False},
        # The prefix of a chat whose prompt goes on: small heads.
        {"name": "read-2057-tokens", "op": "read", "tokens": 2057, "hkv": 4, "dim": 64, "page": 32, "group": 32,
         "dtype": "bf16", "layout": "tokens"},
        # The prefix of a long document before its next piece is attended.
        {"name": "read-65553-tokens", "op": "read", "tokens": 65553, "hkv": 8, "dim": 128, "page": 64, "group": 64,
         "dtype": "bf16", "layout": "heads"},
        # One short chat: latency.
        {"name": "attention-1x97", "op": "attention", "requests": 1, "shortest": 97, "longest": 97, "hq": 32, "hkv": 8,
         "dim": 128, "page": 64, "group": 64, "dtype": "bf16", "layout": "heads"},
        # The ordinary decode step: 32 requests of some 4000 tokens.
        {"name": "attention-32x4129", "op": "attention", "requests": 32, "shortest": 4129, "longest": 4129, "hq": 32,
         "hkv": 8, "dim": 128, "page": 64, "group": 64, "dtype": "bf16", "layout": "heads"},
        # One long document.
        {"name": "attention-1x131105", "op": "attention", "requests": 1, "shortest": 131105, "longest": 131105,
         "hq": 32, "hkv": 8, "dim": 128, "page": 64, "group": 64, "dtype": "bf16", "layout": "heads"},
        # A ragged batch, new requests and long ones, finer groups, small pages.
        {"name": "attention-61-ragged", "op": "attention", "requests": 61, "shortest": 0, "longest": 16417, "hq": 64,
         "hkv": 8, "dim": 128, "page": 16, "group": 32, "dtype": "fp16", "layout": "tokens"},
        # Three chats with the usual settings: latency.
        {"name": "sample-3x32000", "op": "sample", "rows": 3, "vocab": 32000, "dtype": "bf16", "kind": "both"},
        # A batch whose requests bring settings of their own, some of them greedy, logits from a bf16 head: many ties.
        {"name": "sample-64x128000", "op": "sample", "rows": 64, "vocab": 128000, "dtype": "bf16", "kind": "mixed"},
        # The largest: every row by its nucleus over the whole vocabulary, in fp32.
        {"name": "sample-256x131071", "op": "sample", "rows": 256, "vocab": 131071, "dtype": "fp32", "kind": "top_p"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention", "attention", "sample", "sample"])
    if op == "sample":
        vocab = _log(rng, 1000, 131071)
        rows = min(_log(rng, 1, 256), 256 * 131071 // vocab)
        return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "kind": rng.choice(["plain", "top_k", "top_p", "both", "mixed"])}
    c = {"op": op, "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
         "layout": rng.choice(["heads", "tokens"]), "dim": rng.choice([64, 128, 128]), "group": rng.choice([32, 64])}
    hkv = rng.choice([1, 2, 4, 8, 8])
    g = rng.choice([1, 2, 4, 4, 7, 8, 16])
    c["hkv"] = hkv
    if op == "write":
        c.update(tokens=_log(rng, 1, 16000), hq=min(hkv * g, 32) // hkv * hkv, axes=rng.choice([1, 2, 3]),
                 interleaved=rng.random() < 0.5)
        c["rot"] = c["dim"] if rng.random() < 0.6 else c["dim"] // 2
        return c
    if op == "read":
        c["tokens"] = _log(rng, 1, 65000)
        return c
    longest = _log(rng, 1, 65536)
    values = 0.9e9 * min(1.0, 8 / g)
    c.update(requests=max(1, min(_log(rng, 1, 128), int(values / (longest * hkv * c["dim"] * 2.0)))), hq=hkv * g,
             shortest=int(longest * rng.choice([0.0, 0.3, 1.0])), longest=longest)
    return c


def _spread(n, lo, hi):
    """n lengths from lo to hi, the same for every seed (the seed permutes them)."""
    if n == 1:
        return np.array([hi], np.int64)
    f = np.modf((np.arange(n) + 1) * GOLDEN)[0]
    out = np.floor(lo + (hi - lo) * f + 0.5).astype(np.int64)
    out[int(f.argmax())] = hi
    out[int(f.argmin())] = lo
    return out


def work(case):
    op = case["op"]
    if op == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * (4 if case["dtype"] == "fp32" else 2) + 28 * n, "flops": 4 * n * v}
    d, hkv = case["dim"], case["hkv"]
    row = hkv * (d // 2 + 4 * (d // case["group"]))            # a token's keys, or its values, in the cache
    if op == "write":
        n, hq = case["tokens"], case["hq"]
        return {"bytes": 2 * n * (2 * hq + 4 * hkv) * d + 4 * n * row + n * (8 + 4 * case["axes"] + 4 * case["rot"]),
                "flops": 3 * n * (hq + hkv) * case["rot"] + 10 * n * hkv * d}
    if op == "read":
        n = case["tokens"]
        return {"bytes": n * (2 * row + 4 * hkv * d + 8), "flops": 4 * n * hkv * d}
    lens = _spread(case["requests"], case["shortest"], case["longest"])
    t, b, hq = int(lens.sum()), case["requests"], case["hq"]
    return {"bytes": 2 * t * row + 4 * b * hq * d + 4 * b + 4 * int((-(-lens // case["page"])).sum()),
            "flops": 4 * t * hq * d}


# ------------------------------------------------------------------ inputs
def _quantise(x, group):
    """x [..., dim] in 32 bits -> codes [..., dim / 2] (channel 2i in the low half of byte i) and parameters
    [..., 2, dim / group] (scales, then centres)."""
    y = x.unflatten(-1, (-1, group))
    low, high = y.amin(-1), y.amax(-1)
    scale = ((high - low) / torch.full_like(low, 15.0)).to(torch.bfloat16)      # a quotient, not a product with 1 / 15
    centre = (low + 8.0 * scale.float()).to(torch.bfloat16)
    flat = scale.float() < 2.0 ** -126                           # nothing to tell apart
    by = torch.where(flat, torch.ones_like(low), scale.float()).unsqueeze(-1)
    code = (torch.round((y - centre.float().unsqueeze(-1)) / by) + 8.0).clamp(0.0, 15.0)
    code = torch.where(flat.unsqueeze(-1), torch.full_like(code, 8.0), code).to(torch.uint8).flatten(-2)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    scale = torch.where(flat, torch.zeros_like(scale), scale)
    centre = torch.where(flat, low.to(torch.bfloat16), centre)
    return codes, torch.stack([scale, centre], -2)


def _values(codes, params):
    """What codes and parameters stand for, in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8.0
    scale, centre = params.float().unbind(-2)
    return (centre.unsqueeze(-1) + scale.unsqueeze(-1) * code.unflatten(-1, (scale.shape[-1], -1))).flatten(-2)


def _pool(blocks, case, gen, chan):
    """A pool of quantised random rows: codes [blocks, page, heads, dim / 2] and parameters [blocks, page, heads,
    2, dim / group]; layout "heads" keeps each head's rows of a page together."""
    page, heads, dim, group = case["page"], case["hkv"], case["dim"], case["group"]
    at = (heads, page) if case["layout"] == "heads" else (page, heads)
    codes = torch.empty(blocks, *at, dim // 2, dtype=torch.uint8, device="cuda")
    params = torch.empty(blocks, *at, 2, dim // group, dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 26) // (heads * page * dim))
    for i in range(0, blocks, step):
        x = torch.randn(min(step, blocks - i), *at, dim, device="cuda", generator=gen)
        x *= chan.unsqueeze(1) if case["layout"] == "heads" else chan
        codes[i:i + step], params[i:i + step] = _quantise(x, group)
    if case["layout"] == "heads":
        return codes.transpose(1, 2), params.transpose(1, 2)
    return codes, params


def _gpu(x, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device="cuda", dtype=dtype)


def _sections(case):
    half = case["rot"] // 2
    if case["axes"] == 1:
        return [half]
    rest = half // 8 * 3 if case["axes"] == 3 else half // 2
    return [half - rest * (case["axes"] - 1)] + [rest] * (case["axes"] - 1)


def _prepare_sample(case, rng, gen):
    n, v, kind = case["rows"], case["vocab"], case["kind"]
    # a head's logits: a wide bulk, some likely tokens far above it, in every fifth row tokens that a grammar forbids
    x = torch.randn(n, v, device="cuda", generator=gen) * 2.2
    likely = torch.randint(0, v, (n, 24), device="cuda", generator=gen)
    x.scatter_(1, likely, torch.empty(n, 24, device="cuda").uniform_(5.0, 14.0, generator=gen))
    for r in range(0, n, 5):
        a = int(rng.integers(0, v // 2))
        x[r, a:a + v // 3] = -math.inf
    s = {"logits": x.to(TYPES[case["dtype"]]), "u": torch.rand(n, device="cuda", generator=gen),
         "temperature": 0.8, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if kind in ("top_k", "both"):
        s["top_k"] = 50
    if kind in ("top_p", "both"):
        s["top_p"] = 0.95
    if kind == "top_p":
        s["temperature"] = 1.0
    if kind == "mixed":                          # settings of each request's own
        s["temperature"] = _gpu(rng.choice([0.0, 0.6, 0.8, 1.0, 1.3], n), torch.float32)
        s["top_k"] = _gpu(rng.choice([0, 0, 1, 20, 50, 1000], n))
        s["top_p"] = _gpu(rng.choice([1.0, 1.0, 0.9, 0.95, 0.5], n), torch.float32)
        s["min_p"] = _gpu(rng.choice([0.0, 0.0, 0.05, 0.1], n), torch.float32)
    return s


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "sample":
        s.update(_prepare_sample(case, rng, gen))
        return s
    dtype, dim, hkv, page = TYPES[case["dtype"]], case["dim"], case["hkv"], case["page"]
    # some channels are far larger than others, as keys have them
    chan = torch.exp(torch.empty(2, hkv, dim, device="cuda").uniform_(math.log(0.3), math.log(3.0), generator=gen))
    if op == "attention":
        lens = _spread(case["requests"], case["shortest"], case["longest"])
        lens = lens[rng.permutation(len(lens))]
        pages = -(-lens // page)
        blocks = int(pages.sum()) + 5
        order = rng.permutation(blocks)
        table = np.full((len(lens), int(pages.max(initial=0)) + 2), -1, np.int32)
        ends = np.cumsum(pages)
        for i, p in enumerate(pages):
            table[i, :p] = order[ends[i] - p:ends[i]]
        s.update(table=_gpu(table), lens=_gpu(lens))
        s["q"] = torch.randn(case["requests"], case["hq"], dim, device="cuda", generator=gen).to(dtype)
        s["k_pages"], s["v_pages"] = _pool(blocks, case, gen, chan[0]), _pool(blocks, case, gen, chan[1])
        return s
    n = case["tokens"]
    i = np.arange(n)
    blocks = -(-n // page) + 3
    slots = rng.permutation(blocks)[i // page] * page + i % page
    slots[rng.random(n) < 0.002] = -1              # padding of the step
    s["slots"] = _gpu(slots, torch.int64)
    s["k_pages"], s["v_pages"] = _pool(blocks, case, gen, chan[0]), _pool(blocks, case, gen, chan[1])
    if op == "read":
        return s
    hq, rot = case["hq"], case["rot"]
    qkv = torch.randn(n, hq + 2 * hkv, dim, device="cuda", generator=gen)
    qkv[:, hq:] *= chan.flatten(0, 1)
    qkv = qkv.to(dtype)                             # one projection's output; its slices
    s["q"], s["k"], s["v"] = qkv.split([hq, hkv, hkv], 1)
    # text first, then frames of a grid: the axes are time, height and width
    start, side = int(rng.integers(0, LONGEST // 4)), 24
    pos = [start + (i if case["axes"] == 1 else i // (side * side)), start + i // side % side, start + i % side]
    s["positions"] = _gpu(pos[0] if case["axes"] == 1 else np.stack(pos[:case["axes"]]))
    ang = np.arange(LONGEST)[:, None] * 500000.0 ** (-np.arange(rot // 2) * 2.0 / rot)[None]
    s["cos_sin"] = _gpu(np.concatenate([np.cos(ang), np.sin(ang)], 1), torch.float32)
    s["sections"] = _sections(case)
    return s


# -------------------------------------------------------------- plain forms
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


def _plain_read(s):
    page, dtype = s["case"]["page"], TYPES[s["case"]["dtype"]]
    live = s["slots"] >= 0
    slot = s["slots"].clamp(min=0)
    block, row = torch.div(slot, page, rounding_mode="floor"), slot % page
    out = []
    for codes, params in (s["k_pages"], s["v_pages"]):
        x = _values(codes[block, row], params[block, row]).to(dtype)
        out.append(torch.where(live.view(-1, 1, 1), x, torch.zeros((), dtype=dtype, device=x.device)))
    return {"k": out[0], "v": out[1]}


def _plain_write(s):
    c = s["case"]
    pos = s["positions"] if s["positions"].dim() == 2 else s["positions"].unsqueeze(0)
    half, ends = c["rot"] // 2, np.cumsum(s["sections"])
    rows = [s["cos_sin"][p.long()] for p in pos]
    cos = torch.cat([x[:, e - w:e] for x, e, w in zip(rows, ends, s["sections"])], 1).unsqueeze(1)
    sin = torch.cat([x[:, half + e - w:half + e] for x, e, w in zip(rows, ends, s["sections"])], 1).unsqueeze(1)
    q = _turn(s["q"], cos, sin, c["interleaved"]).to(s["q"].dtype)
    live = (s["slots"] >= 0).nonzero().squeeze(1)
    slot = s["slots"][live]
    block, row = torch.div(slot, c["page"], rounding_mode="floor"), slot % c["page"]
    for x, (codes, params) in ((_turn(s["k"], cos, sin, c["interleaved"]), s["k_pages"]),
                               (s["v"].float(), s["v_pages"])):
        codes[block, row], params[block, row] = _quantise(x[live], c["group"])
    return {"q": q, **_plain_read(s)}


def _plain_attention(s):
    q, lens, (kc, kp), (vc, vp) = s["q"], s["lens"], s["k_pages"], s["v_pages"]
    b, hq, d = q.shape
    page, hkv, width = kc.shape[1], kc.shape[2], s["table"].shape[1]
    valid = torch.arange(width * page, device=q.device) < lens.unsqueeze(1)
    qf = q.float().view(b, hkv, hq // hkv, d)
    out = torch.empty(b, hkv, hq // hkv, d, dtype=torch.float32, device=q.device)
    # requests in groups, so that the gathered 32-bit keys stay within a few GB
    step = max(1, int(1.5e9 / (hkv * width * page * d * 4)))
    for i in range(0, b, step):
        at = s["table"][i:i + step].clamp(min=0).long()
        ok = valid[i:i + step].unsqueeze(1).unsqueeze(2)
        kk = _values(kc[at], kp[at]).flatten(1, 2).transpose(1, 2)
        sc = torch.matmul(qf[i:i + step], kk.transpose(-1, -2)) * (1.0 / math.sqrt(d))
        del kk
        sc = torch.where(ok, sc, torch.full((), -math.inf, device=q.device))
        top = sc.amax(-1, keepdim=True)
        w = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        vv = _values(vc[at], vp[at]).flatten(1, 2).transpose(1, 2)
        vv = torch.where(ok.transpose(-1, -2), vv, torch.zeros((), device=q.device))
        total = w.sum(-1, keepdim=True)
        out[i:i + step] = torch.matmul(w, vv) / torch.where(total > 0, total, torch.ones_like(total))
    return {"out": out.view(b, hq, d).to(q.dtype)}


def _plain_sample(s):
    x = s["logits"].double()
    n, v = x.shape

    def per_row(value):
        return value.double().view(-1, 1) if torch.is_tensor(value) else \
            torch.full((n, 1), float(value), dtype=torch.float64, device=x.device)

    temp, top_k, top_p, min_p = (per_row(s[name]) for name in ("temperature", "top_k", "top_p", "min_p"))
    far = (x - x.amax(-1, keepdim=True)) / torch.where(temp > 0, temp, torch.ones_like(temp))
    w, index = torch.sort(torch.exp(far), stable=True, dim=-1, descending=True)      # equal ones by index
    place = torch.arange(v, device=x.device)
    limit = torch.where(temp > 0, torch.where(top_k > 0, top_k, torch.full_like(top_k, v)), torch.ones_like(temp))
    w = torch.where(place < limit, w, torch.zeros_like(w))
    before = torch.cumsum(w, -1) - w
    keep = ((before < top_p * w.sum(-1, keepdim=True)) | (top_p >= 1)) & (w >= min_p) | (place == 0)
    w = torch.where(keep, w, torch.zeros_like(w))
    sums = torch.cumsum(torch.zeros_like(w).scatter_(1, index, w), -1)           # by index again
    return {"tokens": (sums <= s["u"].double().view(-1, 1) * sums[:, -1:]).sum(-1).clamp(max=v - 1)}


def run(state):
    s, op = state, state["case"]["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attention": _plain_attention, "sample": _plain_sample}[op](s)
    import zipserv_asplos26_b200 as zs
    if op == "sample":
        return {"tokens": zs.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                    top_p=s["top_p"], min_p=s["min_p"])}
    kp, vp = zs.Int4Pages(*s["k_pages"]), zs.Int4Pages(*s["v_pages"])
    if op == "attention":
        return {"out": zs.paged_attention_int4(s["q"], kp, vp, s["table"], s["lens"])}
    out = {}
    if op == "write":
        out["q"] = zs.rope_write_int4(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["slots"], kp, vp,
                                      sections=s["sections"], interleaved=s["case"]["interleaved"])
    out["k"], out["v"] = zs.read_int4(kp, vp, s["slots"], dtype=TYPES[s["case"]["dtype"]])
    return out


# --------------------------------------------------- the definitions, in 64 bits
def _bf16_of(x):
    """Doubles rounded to bf16's 8 bits, ties to even, as doubles."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256.0) / 256.0, e)


def _held(x, group):
    """Rows x [..., dim] of doubles as the cache holds them."""
    y = x.reshape(*x.shape[:-1], x.shape[-1] // group, group)
    low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    s = _bf16_of((high - low) / 15.0)
    c = _bf16_of(low + 8.0 * s)
    u = torch.round((y - c) / torch.where(s > 0, s, torch.ones_like(s))).clamp(-8.0, 7.0)
    return (c + s * u).reshape(x.shape)


def _rows(pool, block, row, heads=slice(None)):
    """Rows of a pool in 64 bits."""
    codes, params = pool[0][block, row][..., heads, :], pool[1][block, row][..., heads, :, :].double()
    u = torch.empty(*codes.shape[:-1], codes.shape[-1] * 2, dtype=torch.float64, device=codes.device)
    u[..., 0::2], u[..., 1::2] = (codes % 16).double(), torch.div(codes, 16, rounding_mode="floor").double()
    each = u.shape[-1] // params.shape[-1]
    return (u - 8.0) * params[..., 0, :].repeat_interleave(each, -1) + params[..., 1, :].repeat_interleave(each, -1)


def _exact_write(s):
    c = s["case"]
    half, n = c["rot"] // 2, c["tokens"]
    axis = torch.repeat_interleave(torch.arange(c["axes"]), torch.tensor(s["sections"])).cuda()
    at = s["positions"].reshape(c["axes"], n).long()[axis].t()
    chan = torch.arange(half, device="cuda")
    z = torch.complex(s["cos_sin"].double()[at, chan], s["cos_sin"].double()[at, half + chan]).unsqueeze(1)
    lo = slice(0, c["rot"], 2) if c["interleaved"] else slice(0, half)
    hi = slice(1, c["rot"], 2) if c["interleaved"] else slice(half, c["rot"])

    def turn(x):
        y = x.double().clone()
        t = torch.complex(y[..., lo], y[..., hi]) * z
        y[..., lo], y[..., hi] = t.real, t.imag
        return y

    live = (s["slots"] >= 0).view(-1, 1, 1)
    return {"q": turn(s["q"]), "k": _held(turn(s["k"]), c["group"]) * live,
            "v": _held(s["v"].double(), c["group"]) * live}


def _exact_read(s):
    page, out = s["case"]["page"], {}
    for name in ("k", "v"):
        parts = []
        for slot in s["slots"].split(1 << 14):
            at = slot.clamp(min=0)
            parts.append(_rows(s[name + "_pages"], at // page, at % page) * (slot >= 0).view(-1, 1, 1))
        out[name] = torch.cat(parts)
    return out


def _exact_attention(s):
    page, hkv = s["case"]["page"], s["case"]["hkv"]
    q = s["q"].double()
    b, hq, d = q.shape
    out = torch.zeros(b, hkv, hq // hkv, d, dtype=torch.float64, device=q.device)
    for r, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        i = torch.arange(n, device=q.device)
        block, row = s["table"][r].long()[i // page], i % page
        for h in range(hkv):
            k, v = (_rows(s[x], block, row, slice(h, h + 1)).squeeze(-2) for x in ("k_pages", "v_pages"))
            out[r, h] = torch.softmax(q[r].view(hkv, -1, d)[h] @ k.t() / math.sqrt(d), -1) @ v
    return {"out": out.view(b, hq, d)}


def _exact_sample(s):
    x, u = s["logits"].double().cpu().numpy(), s["u"].double().cpu().numpy()
    n, v = x.shape
    t, k, p, m = (s[name].double().cpu().numpy() if torch.is_tensor(s[name]) else np.full(n, float(s[name]))
                  for name in ("temperature", "top_k", "top_p", "min_p"))
    tokens = np.empty(n, np.int64)
    for r in range(n):
        if t[r] <= 0:
            tokens[r] = x[r].argmax()               # the first of the largest
            continue
        order = np.lexsort((np.arange(v), -x[r]))[:int(k[r]) if k[r] > 0 else v]
        w = np.exp((x[r, order] - x[r, order[0]]) / t[r])
        sums = np.add.accumulate(w.astype(np.longdouble))
        count = len(w) if p[r] >= 1 else int(np.searchsorted(sums, p[r] * sums[-1])) + 1     # the first sum to reach it
        count = max(1, min(count, int((w >= m[r]).sum())))
        some = order[:count]
        by_index = np.argsort(some)
        sums = np.add.accumulate(w[:count][by_index].astype(np.longdouble))
        tokens[r] = some[by_index][min(count - 1, int(np.searchsorted(sums, u[r] * sums[-1], side="right")))]
    return {"tokens": torch.from_numpy(tokens)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attention": _exact_attention,
            "sample": _exact_sample}[case["op"]](s)
