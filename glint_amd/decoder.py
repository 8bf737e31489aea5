"""A small decoder served from pins: pinned linears around the serving operators of glint_serve.h.

Prompts go through attend_prompt and into the paged 4-bit cache, later chunks of a prompt see what the
cache gives back, new tokens are read against it by kv4_attend, and token_logprobs scores what was said.
With `rotary` (frequencies of rotate_qk), queries and keys are normed per head and turned on their way into the
cache in one launch, and later chunks attend over its pages where they lie; `window` and `sinks` bound
what a token sees, and pages that no later token sees are free again.
Weights are random; `python -m glint_amd.decoder` serves a few requests and prints times and scores.
"""
from __future__ import annotations

import contextlib
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
        if m.rotary is not None:  # a trained model's are its own
            self.q_norm, self.k_norm = torch.ones((2, m.head_dim), dtype=torch.bfloat16, device="cuda")


class Decoder:
    """Requests are numbered 0 .. requests - 1; a request's tokens live in the pages of its table row."""

    def __init__(self, vocab=1000, dim=512, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=1024, pages=64, requests=8, seed=0,
                 rotary=None, window=None, sinks=0, context=None):
        """context: tokens that a request may reach (all pages' where None; more with a window, which gives pages back)."""
        if heads % kv_heads:
            raise ValueError(f"{heads} heads over {kv_heads}")
        if window is not None and rotary is None:
            raise ValueError("a window goes with rotary frequencies")
        H._bounds(window, sinks)  # refused here, where no request has begun
        if rotary is not None:
            rot = 2 * rotary.numel()
            if rotary.dtype is not torch.float64 or rotary.dim() != 1 or not rotary.is_contiguous() or not rotary.is_cuda:
                raise ValueError(f"rotary frequencies: a contiguous float64 vector on the GPU, got {rotary.dtype} {tuple(rotary.shape)}")
            if rot % 16 or not 16 <= rot <= head_dim:
                raise ValueError(f"{rot} of {head_dim} dimensions turned: a multiple of 16")
        self.rotary, self.window, self.sinks = rotary, window, sinks
        self.dim, self.heads, self.kv_heads, self.head_dim, self.ffn, self.pages = dim, heads, kv_heads, head_dim, ffn, pages
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.embed = torch.randn((vocab, dim), device="cuda", generator=gen).bfloat16()
        self.layers = [Layer(self, gen) for _ in range(layers)]
        self.head = PinLinear((torch.randn((vocab, dim), device="cuda", generator=gen) * dim ** -0.5).bfloat16())
        places = pages if context is None else (context + H.KV_PAGE - 1) // H.KV_PAGE
        self.table = torch.full((requests, places), -1, dtype=torch.int32, device="cuda")
        self.held = [0] * requests  # tokens in the cache
        self.own = [[] for _ in range(requests)]  # pages; None: given back
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
        for r in news:
            if len(self.own[r]) + want[r] > self.table.shape[1]:
                raise RuntimeError(f"request {r}: past its {self.table.shape[1]} places for pages")

    def _slots(self, request, n):
        """Places for n more tokens of a request, with the pages that they need; _refuse has seen that there are enough."""
        first = self.held[request]
        for _ in range(self._pages(request, n)):
            page = self.free.pop()
            self.table[request, len(self.own[request])] = page
            self.own[request].append(page)
        self.held[request] = first + n
        return [self.own[request][t // H.KV_PAGE] * H.KV_PAGE + t % H.KV_PAGE for t in range(first, first + n)]

    @contextlib.contextmanager
    def _undone(self, news):
        """Requests are as they were where what is within raises: an operator may refuse what _refuse does not know of, or memory
        run out. What layers wrote belongs to tokens that nobody holds then."""
        before = {r: (self.held[r], len(self.own[r])) for r in news}
        try:
            yield
        except BaseException:
            for r, (held, pages) in reversed(before.items()):
                self.free += reversed(self.own[r][pages:])
                del self.own[r][pages:]
                self.table[r, pages:] = -1
                self.held[r] = held
            raise

    def _slide(self, requests):
        """Pages that no later token of the requests sees are free."""
        if self.window is None:
            return
        for r in requests:
            keep = (self.sinks + H.KV_PAGE - 1) // H.KV_PAGE
            for i in range(keep, max(keep, (self.held[r] - self.window + 1) // H.KV_PAGE)):
                if self.own[r][i] is not None:
                    self.free.append(self.own[r][i])
                    self.own[r][i] = None
                    self.table[r, i] = -1

    def drop(self, request):
        """The request is over: its pages are free."""
        self.free += [p for p in self.own[request] if p is not None]
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

    def _rotated(self, tokens, pos, slots, attend, keys):
        """_run with q and k normed and turned and k and v in the cache before attend(layer, q[, k, v])."""
        x = self.embed[torch.tensor(tokens, device="cuda")]
        pos = torch.tensor(pos, dtype=torch.int64, device="cuda")
        for layer in self.layers:
            q, k, v = layer.qkv(norm(x)).unflatten(1, (-1, self.head_dim)).split([self.heads, self.kv_heads, self.kv_heads], 1)
            turned = H.kv4_append_rotated(q, k, v, pos, self.rotary, slots, layer.cache, q_norm=layer.q_norm,
                                          k_norm=layer.k_norm, keys=keys)
            x = x + layer.out((attend(layer, *turned, v) if keys else attend(layer, turned)).flatten(1))
            gate, up = layer.up(norm(x)).chunk(2, -1)
            x = x + layer.down(torch.nn.functional.silu(gate) * up)
        return self.head(norm(x))

    def _prefill_rotated(self, prompts):
        rows, tokens, pos, slots, cu = list(prompts), [], [], [], [0]
        fresh = all(self.held[r] == 0 for r in rows)
        for r, chunk in prompts.items():
            pos += range(self.held[r], self.held[r] + len(chunk))
            slots += self._slots(r, len(chunk))
            tokens += chunk
            cu.append(len(tokens))
        most = max(len(c) for c in prompts.values())
        ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device="cuda")
        lens, cu, slots = ints([self.held[r] for r in rows]), ints(cu), ints(slots, torch.int64)
        table = self.table[rows][:, :max(len(self.own[r]) for r in rows)]

        def attend(layer, q, k, v):
            bounds = dict(window=self.window, sinks=self.sinks)
            if fresh:
                return H.attend_prompt(q, k, v, cu, max_q=most, **bounds)
            return H.kv4_attend_chunk(q, layer.cache, table, lens, cu, max_q=most, k=k, v=v, **bounds)

        return self._rotated(tokens, pos, slots, attend, True)

    def prefill(self, prompts):
        """prompts: {request: tokens}, new prompts or further chunks. Logits [all tokens, vocab], in order. Where the tokens
        do not fit, or are more than attention takes in a call, no request changes."""
        self._refuse(prompts)
        with self._undone(prompts):
            logits = (self._prefill if self.rotary is None else self._prefill_rotated)(prompts)
        self._slide(prompts)
        return logits

    def _prefill(self, prompts):
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
        """news: {request: tokens}, the next token of each (or a few drafted ones). Logits [all tokens, vocab]. Where the tokens
        do not fit, or are more than attention takes in a call, no request changes."""
        self._refuse(news)
        with self._undone(news):
            logits = self._step(news)
        self._slide(news)
        return logits

    def _step(self, news):
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

        most = max(len(t) for t in news.values())
        if self.rotary is not None:
            return self._rotated(tokens, pos, slots, lambda layer, q: H.kv4_attend(
                q, layer.cache, table, lens, cu, max_q=most, window=self.window, sinks=self.sinks), False)

        def attend(layer, q, k, v):
            H.kv4_append(k, v, slots, layer.cache)
            return H.kv4_attend(q, layer.cache, table, lens, cu, max_q=most)

        return self._run(tokens, pos, attend)


def main():
    gen = torch.Generator().manual_seed(1)
    m = Decoder(vocab=32000, dim=2048, layers=4, heads=16, kv_heads=4, head_dim=128, ffn=4096, pages=256,
                rotary=H.rotary_freqs(128), window=1024, sinks=4)
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
    further = timed("a further chunk", lambda: m.prefill({3: torch.randint(32000, (400,), generator=gen).tolist()}))
    last[3] = further[-1]
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
