"""A small decoder served from pins: pinned linears around the serving operators of glint_serve.h.

Prompts go through attend_prompt and into the paged 4-bit cache, later chunks of a prompt see what the
cache gives back, new tokens are read against it by kv4_attend, and token_logprobs scores what was said.
Weights are random; `python -m glint_amd.decoder` serves a few requests and prints times and scores.
"""
from __future__ import annotations

import time

import torch

from . import glint_hip as H


class PinLinear:
    """y = x W^T with W [n, k] held as a pin."""

    def __init__(self, w):
        self.n, self.k = w.shape
        self.pin = H.encode_bf16(w)

    def __call__(self, x):
        return H.htile_bf16(*self.pin, x.contiguous(), self.n, self.k)


def norm(x):
    y = x.float()
    return (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


def rotate(x, pos):
    """Rotary positions: x [T, heads, D], pos [T]."""
    half = x.shape[-1] // 2
    freq = 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float32) / half)
    angle = pos[:, None, None].float() * freq
    c, s, y = angle.cos(), angle.sin(), x.float()
    a, b = y[..., :half], y[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


class Layer:
    def __init__(self, m, gen):
        w = lambda n, k: (torch.randn((n, k), device="cuda", generator=gen) * k ** -0.5).bfloat16()
        self.qkv = PinLinear(w((m.heads + 2 * m.kv_heads) * m.head_dim, m.dim))
        self.out = PinLinear(w(m.dim, m.heads * m.head_dim))
        self.up, self.down = PinLinear(w(2 * m.ffn, m.dim)), PinLinear(w(m.dim, m.ffn))
        self.cache = H.kv4_cache(m.pages, m.kv_heads, m.head_dim)


class Decoder:
    """Requests are numbered 0 .. requests - 1; a request's tokens live in the pages of its table row."""

    def __init__(self, vocab=1000, dim=512, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=1024, pages=64, requests=8, seed=0):
        if heads % kv_heads:
            raise ValueError(f"{heads} heads over {kv_heads}")
        self.dim, self.heads, self.kv_heads, self.head_dim, self.ffn, self.pages = dim, heads, kv_heads, head_dim, ffn, pages
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.embed = torch.randn((vocab, dim), device="cuda", generator=gen).bfloat16()
        self.layers = [Layer(self, gen) for _ in range(layers)]
        self.head = PinLinear((torch.randn((vocab, dim), device="cuda", generator=gen) * dim ** -0.5).bfloat16())
        self.table = torch.full((requests, pages), -1, dtype=torch.int32, device="cuda")
        self.held = [0] * requests  # tokens in the cache
        self.own = [[] for _ in range(requests)]
        self.free = list(range(pages))

    def _pages(self, request, n):
        """Pages that n more tokens of a request need."""
        return max(0, (self.held[request] + n + H.KV_PAGE - 1) // H.KV_PAGE - len(self.own[request]))

    def _refuse(self, news):
        """Raises, before any request changes, where one of {request: tokens} does not exist or they do not all fit."""
        for r in news:
            if not 0 <= r < len(self.held):
                raise IndexError(f"request {r} of {len(self.held)}")
        want = {r: self._pages(r, len(some)) for r, some in news.items()}
        if sum(want.values()) > len(self.free):
            raise RuntimeError(f"requests {list(news)}: {list(want.values())} pages more, {len(self.free)} left")

    def _slots(self, request, n):
        """Places for n more tokens of a request, with the pages that they need; _refuse has seen that there are enough."""
        first = self.held[request]
        for _ in range(self._pages(request, n)):
            page = self.free.pop()
            self.table[request, len(self.own[request])] = page
            self.own[request].append(page)
        self.held[request] = first + n
        return [self.own[request][t // H.KV_PAGE] * H.KV_PAGE + t % H.KV_PAGE for t in range(first, first + n)]

    def drop(self, request):
        """The request is over: its pages are free."""
        self.free += self.own[request]
        self.own[request], self.held[request] = [], 0
        self.table[request] = -1

    def _run(self, tokens, pos, attend):
        x = self.embed[torch.tensor(tokens, device="cuda")]
        pos = torch.tensor(pos, device="cuda")
        for layer in self.layers:
            qkv = layer.qkv(norm(x)).unflatten(1, (-1, self.head_dim))
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            x = x + layer.out(attend(layer, rotate(q, pos), rotate(k, pos), v).flatten(1))
            gate, up = layer.up(norm(x)).chunk(2, -1)
            x = x + layer.down(torch.nn.functional.silu(gate) * up)
        return self.head(norm(x))

    def prefill(self, prompts):
        """prompts: {request: tokens}, new prompts or further chunks. Logits [all tokens, vocab], in order.
        Where the tokens do not fit, no request changes."""
        self._refuse(prompts)
        ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device="cuda")
        tokens, pos, new, seen, keys_new, keys_old, old = [], [], [], [], [], [], []
        cu_q, cu_k = [0], [0]
        for r, chunk in prompts.items():
            had = self.held[r]
            old += [self.own[r][t // H.KV_PAGE] * H.KV_PAGE + t % H.KV_PAGE for t in range(had)]
            new += self._slots(r, len(chunk))
            tokens += chunk
            pos += range(had, had + len(chunk))
            keys_old += range(cu_k[-1], cu_k[-1] + had)
            keys_new += range(cu_k[-1] + had, cu_k[-1] + had + len(chunk))
            cu_q.append(cu_q[-1] + len(chunk))
            cu_k.append(cu_k[-1] + had + len(chunk))
        longest = max(len(c) for c in prompts.values())
        cu_q, cu_k, total = ints(cu_q), ints(cu_k), cu_k[-1]
        new, old, keys_new, keys_old = (ints(v, torch.int64) for v in (new, old, keys_new, keys_old))

        def attend(layer, q, k, v):
            H.kv4_append(k, v, new, layer.cache)
            if len(old):  # what the earlier chunks left, in front of the new keys
                both = q.new_empty((2, total, self.kv_heads, self.head_dim))
                for i, (before, now) in enumerate(zip(H.kv4_gather(old, layer.cache), (k, v))):
                    both[i, keys_old], both[i, keys_new] = before, now
                k, v = both
            return H.attend_prompt(q, k, v, cu_q, cu_k, max_q=longest)

        return self._run(tokens, pos, attend)

    def step(self, news):
        """news: {request: tokens}, the next token of each (or a few drafted ones). Logits [all tokens, vocab].
        Where the tokens do not fit, no request changes."""
        self._refuse(news)
        tokens, pos, slots, cu_q = [], [], [], [0]
        for r, some in news.items():
            pos += range(self.held[r], self.held[r] + len(some))
            slots += self._slots(r, len(some))
            tokens += some
            cu_q.append(len(tokens))
        rows = list(news)
        lens = torch.tensor([self.held[r] for r in rows], dtype=torch.int32, device="cuda")
        cu = torch.tensor(cu_q, dtype=torch.int32, device="cuda")
        slots, table = torch.tensor(slots, device="cuda"), self.table[rows]

        def attend(layer, q, k, v):
            H.kv4_append(k, v, slots, layer.cache)
            return H.kv4_attend(q, layer.cache, table, lens, cu, max_q=max(len(t) for t in news.values()))

        return self._run(tokens, pos, attend)


def main():
    gen = torch.Generator().manual_seed(1)
    m = Decoder(vocab=32000, dim=2048, layers=4, heads=16, kv_heads=4, head_dim=128, ffn=4096, pages=256)
    prompts = {r: torch.randint(32000, (n,), generator=gen).tolist() for r, n in enumerate((5, 300, 77, 1200))}

    def timed(what, f):
        torch.cuda.synchronize()
        t = time.perf_counter()
        y = f()
        torch.cuda.synchronize()
        print(f"{what}: {(time.perf_counter() - t) * 1e3:.2f} ms", flush=True)
        return y

    logits = timed("prompts", lambda: m.prefill(prompts))
    ends = torch.tensor([len(p) for p in prompts.values()]).cumsum(0) - 1
    last = logits[ends.cuda()]
    said = {r: [] for r in prompts}
    for i in range(16):
        s = H.token_logprobs(last, last.argmax(-1), top=3)
        pick = s["top_index"][:, 0].tolist()
        for r, t in enumerate(pick):
            said[r].append((t, float(s["logprob"][r])))
        last = timed(f"token {i}", lambda: m.step({r: [t] for r, t in enumerate(pick)}))
    for r, t in said.items():
        print(f"request {r}: " + " ".join(f"{k}({p:.2f})" for k, p in t))


if __name__ == "__main__":
    main()
