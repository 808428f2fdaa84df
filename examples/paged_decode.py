"""Decoding with compressed weights over a paged KV cache, of 16-bit pages or 4-bit ones.

A small decoder of random weights: every projection is a TCA-TBE compressed
matrix multiplied by ZipGEMM, the KV cache is a PagedKVCache. Prompts of
different lengths come in as one step (their attention in plain torch), then
every decode step is one CUDA graph replay: plan_step gives the new tokens their
slots, each layer turns q and k, writes k and v (with --bits 4 quantised) and attends,
over the whole cache or, with --top, over chosen pages, and the rows' tokens are
sampled (with --temperature 0, the largest logits' tokens). One request ends on the way
and another takes its row and its pages.

    python examples/paged_decode.py [--steps 48] [--top 4 | --bits 4] [--temperature 0.8 --top-k 50 --top-p 0.95]
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import zipserv_asplos26_b200 as zs  # noqa: E402


class Decoder:
    def __init__(self, layers=2, hidden=1024, hq=8, hkv=2, dim=128, inter=2048, vocab=512, max_pos=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(rows, cols, std=0.03):
            return (torch.randn(rows, cols, device="cuda", generator=g) * std).to(torch.bfloat16)

        self.hq, self.hkv, self.dim, self.hidden = hq, hkv, dim, hidden
        self.embed = weight(vocab, hidden, 1.0)
        self.dense = [dict(qkv=weight((hq + 2 * hkv) * dim, hidden), o=weight(hidden, hq * dim),
                           gate_up=weight(2 * inter, hidden), down=weight(hidden, inter)) for _ in range(layers)]
        self.layers = [{n: zs.compress(w) for n, w in layer.items()} for layer in self.dense]
        self.head = weight(vocab, hidden)
        self.head_c = zs.compress(self.head)
        ang = torch.arange(max_pos, device="cuda")[:, None] * \
            (10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim))[None]
        self.cos_sin = torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()

    def norm(self, x):
        xf = x.float()
        return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + 1e-6)).to(x.dtype)

    def forward(self, tokens, plan, cache, attend):
        """Logits of the step's tokens; attend(layer, q) -> attention output."""
        x = self.embed[tokens]
        n = x.shape[0]
        for i, w in enumerate(self.layers):
            qkv = zs.zipgemm(w["qkv"], self.norm(x)).view(n, -1, self.dim)
            q, k, v = qkv.split([self.hq, self.hkv, self.hkv], 1)
            q = cache.write(q, k, v, self.cos_sin, plan, i)
            x = x + zs.zipgemm(w["o"], attend(i, q, cache).reshape(n, -1))
            gate, up = zs.zipgemm(w["gate_up"], self.norm(x)).chunk(2, -1)
            x = x + zs.zipgemm(w["down"], (torch.nn.functional.silu(gate.float()) * up.float()).to(x.dtype))
        return zs.zipgemm(self.head_c, self.norm(x))


def prompt_attention(model, cache, plan):
    """Causal attention of whole prompts in plain torch, over the keys just written."""
    cu = plan.cu_tokens.tolist()

    def attend(layer, q, cache):
        out = torch.zeros_like(q)
        for r, (a, b) in enumerate(zip(cu, cu[1:])):
            if a == b:
                continue
            k, v = (x.float() for x in cache.read(plan.slots[a:b], layer))
            g = model.hq // model.hkv
            s = torch.einsum("thd,shd->hts", q[a:b].float(), k.repeat_interleave(g, 1)) * model.dim ** -0.5
            s.masked_fill_(torch.ones(b - a, b - a, device=q.device, dtype=torch.bool).triu(1), -torch.inf)
            out[a:b] = torch.einsum("hts,shd->thd", s.softmax(-1), v.repeat_interleave(g, 1)).to(q.dtype)
        return out

    return attend


def run(steps=48, top=0, prompts=(33, 120, 7), seed=0, page=16, bits=16, temperature=0.0, top_k=0, top_p=1.0):
    """Decodes `steps` tokens for each prompt. Returns the tokens of each row and
    the logits of the last step."""
    torch.manual_seed(seed)
    model = Decoder(seed=seed)
    rows = len(prompts)
    longest = max(prompts) + 2 * steps + page
    pages = -(-longest // page)
    cache = zs.PagedKVCache(rows * pages, rows, pages, model.hkv, model.dim, page, num_layers=len(model.layers), bits=bits)
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    luck = torch.Generator(device="cuda").manual_seed(seed + 2)

    def choose(logits, u):
        return zs.sample(logits, u, temperature, top_k, top_p)

    def admit(lens):
        """One step in which the rows of positive `lens` get a prompt; their first decoded tokens."""
        n = sum(max(t, 0) for t in lens)
        new = torch.tensor(lens, dtype=torch.int32, device="cuda")
        plan = cache.step(new, n)
        tokens = torch.randint(0, model.embed.shape[0], (n,), device="cuda", generator=gen)
        logits = model.forward(tokens, plan, cache, prompt_attention(model, cache, plan))
        last = (plan.cu_tokens[1:] - 1)[new > 0].long()
        return tokens, choose(logits[last], torch.rand(len(last), device="cuda", generator=luck)), \
            [r for r, t in enumerate(lens) if t > 0]

    prompt, first, _ = admit(list(prompts))
    history = [list(t) for t in (x.tolist() for x in prompt.split(list(prompts)))]
    tokens = first.clone()                                     # static input of the graph: row r's last token
    ones = torch.ones(rows, dtype=torch.int32, device="cuda")
    u = torch.zeros(rows, device="cuda")                       # the step's random numbers

    def step():
        plan = cache.step(ones, rows)
        own = cache.token_rows(plan)                           # each token attends its own row

        def decode(layer, q, cache):
            if top:
                return cache.sparse_attention(q, top, layer, rows=own)[0]
            return cache.attention(q, layer, rows=own)

        logits = model.forward(tokens, plan, cache, decode)
        return logits, choose(logits, u)

    state = [cache.seqlens, cache.free_count, cache.block_table, cache.free_blocks]
    kept = [t.clone() for t in state]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                              # warm up, then take the step back
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, k in zip(state, kept):
        t.copy_(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, chosen = step()

    for i in range(steps):
        if i == steps // 2:                                    # row 0 ends; a new prompt takes its place
            cache.step(torch.tensor([-1] + [0] * (rows - 1), dtype=torch.int32, device="cuda"), 0)
            prompt, first, _ = admit([prompts[0] + 5] + [0] * (rows - 1))
            history[0] = prompt.tolist()
            tokens[0] = first[0]
        for r, t in enumerate(tokens.tolist()):
            history[r].append(t)
        u.uniform_(generator=luck)
        graph.replay()
        tokens.copy_(chosen)
    torch.cuda.synchronize()
    if cache.check_errors():
        raise RuntimeError(f"error bits {cache.check_errors()}")
    return model, history, logits


def held(x, group=64):
    """Rows as a 4-bit cache holds them."""
    y = x.unflatten(-1, (-1, group))
    low, high = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    s = ((high - low) / 15).bfloat16().float()
    c = (low + 8 * s).bfloat16().float()
    return (c + s * ((y - c) / s).round().clamp(-8, 7)).flatten(-2)


def reference_logits(model, history, bits=16):
    """Last-token logits of each row in fp32 on the dense weights, without a cache."""
    out = []
    for tokens in history:
        x = model.embed[torch.tensor(tokens, device="cuda")].float()
        n = x.shape[0]
        cs = model.cos_sin[:n]
        cos, sin = cs[:, None, :model.dim // 2], cs[:, None, model.dim // 2:]

        def turn(t):
            a, b = t.chunk(2, -1)
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

        def norm(t):
            return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + 1e-6)

        for w in model.dense:
            qkv = (norm(x) @ w["qkv"].float().t()).view(n, -1, model.dim)
            q, k, v = qkv.split([model.hq, model.hkv, model.hkv], 1)
            g = model.hq // model.hkv
            q, k = turn(q), turn(k)
            if bits == 4:
                k, v = held(k), held(v)
            k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
            s = torch.einsum("thd,shd->hts", q, k) * model.dim ** -0.5
            s.masked_fill_(torch.ones(n, n, device="cuda", dtype=torch.bool).triu(1), -torch.inf)
            x = x + torch.einsum("hts,shd->thd", s.softmax(-1), v).reshape(n, -1) @ w["o"].float().t()
            gate, up = (norm(x) @ w["gate_up"].float().t()).chunk(2, -1)
            x = x + (torch.nn.functional.silu(gate) * up) @ w["down"].float().t()
        out.append((norm(x) @ model.head.float().t())[-1])
    return torch.stack(out)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=48)
    ap.add_argument("--top", type=int, default=0, help="pages attended per KV head (0: all)")
    ap.add_argument("--bits", type=int, default=16, choices=[4, 16], help="bits a value of the cache")
    ap.add_argument("--temperature", type=float, default=0.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    args = ap.parse_args()
    model, history, logits = run(args.steps, args.top, bits=args.bits, temperature=args.temperature, top_k=args.top_k,
                                 top_p=args.top_p)
    ref = reference_logits(model, history, args.bits)
    err = float((logits.float() - ref).norm() / ref.norm())
    print(f"{len(history)} rows, {[len(h) for h in history]} tokens; last logits against fp32 without a cache: "
          f"rel-L2 {err:.4f}{' (sparse attention is an approximation)' if args.top else ''}")


if __name__ == "__main__":
    main()
