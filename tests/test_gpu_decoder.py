"""The serving operators together: a small decoder's prompts, chunks, steps and scores against plain forms."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests.gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

SHAPE = dict(vocab=997, dim=256, layers=2, heads=6, kv_heads=2, head_dim=64, ffn=512, pages=40, requests=4)


def decoder():
    torch_cuda()
    from glint_amd.decoder import Decoder
    return Decoder(**SHAPE)


def plain(m, old, news):
    """Logits of {request: tokens} after the cached tokens {request: [(k, v) per layer]}, attention in f32 on the CPU."""
    import torch
    at = {}

    def attend(layer, q, k, v):
        i = m.layers.index(layer)
        out, at_row = torch.empty(q.shape), 0
        for r, some in news.items():
            rows = slice(at_row, at_row + len(some))
            at_row += len(some)
            ks, vs = (torch.cat([o.float().cpu(), n[rows].float().cpu()]) for o, n in zip(old[r][i], at["now"](layer, k, v)))
            had = len(ks) - len(some)
            for h in range(m.heads):
                z = q[rows, h].float().cpu() @ ks[:, h * m.kv_heads // m.heads].T * m.head_dim ** -0.5
                z += torch.full(z.shape, -torch.inf).triu(had + 1)
                out[rows, h] = z.softmax(-1) @ vs[:, h * m.kv_heads // m.heads]
        return out.to(q).to(q.dtype)

    def run(now):
        at["now"] = now
        tokens = [t for some in news.values() for t in some]
        pos = [len(old[r][0][0]) + j for r, some in news.items() for j in range(len(some))]
        return m._run(tokens, pos, attend).float()

    return run


def cached(m):
    """{request: [(k, v) per layer]} as the cache holds them."""
    import torch
    out = {}
    for r in range(len(m.held)):
        slots = torch.tensor([m.own[r][t // 64] * 64 + t % 64 for t in range(m.held[r])], dtype=torch.int64, device="cuda")
        out[r] = [H.kv4_gather(slots, layer.cache) for layer in m.layers]
    return out


def from_cache(m, news):
    """The new tokens' keys and values as the step left them in the cache."""
    import torch
    slots = torch.tensor([m.own[r][t // 64] * 64 + t % 64 for r, some in news.items()
                          for t in range(m.held[r] - len(some), m.held[r])], dtype=torch.int64, device="cuda")
    return lambda layer, k, v: H.kv4_gather(slots, layer.cache)


def close(got, want):
    """Every row within what some 20 bf16 roundings (2^-9 rms at most, independent) of the residual
    stream leave of its norm, twice: 2 * sqrt(20) * 2^-9."""
    far = (got.float() - want).norm(dim=-1) / want.norm(dim=-1)
    assert far.max() < 2 * 20 ** 0.5 * 2.0 ** -9, far.max()


def tokens(rng, n):
    return rng.integers(0, SHAPE["vocab"], n).tolist()


def test_prompts_chunks_and_steps():
    import torch
    m, rng = decoder(), np.random.default_rng(0)
    direct = lambda layer, k, v: (k, v)
    print("prompts", flush=True)
    prompts = {0: tokens(rng, 5), 2: tokens(rng, 130), 3: tokens(rng, 64)}
    run = plain(m, cached(m), prompts)
    close(m.prefill(prompts), run(direct))
    print("chunks", flush=True)
    chunks = {2: tokens(rng, 70), 1: tokens(rng, 3), 0: tokens(rng, 60)}
    run = plain(m, cached(m), chunks)
    close(m.prefill(chunks), run(direct))
    print("steps", flush=True)
    for news in ({r: tokens(rng, 1) for r in range(4)}, {0: tokens(rng, 4), 3: tokens(rng, 2), 1: tokens(rng, 4)}, {2: tokens(rng, 1)}):
        run = plain(m, cached(m), news)
        logits = m.step(news)
        close(logits, run(from_cache(m, news)))
    x = logits.float().double().cpu()
    s = H.token_logprobs(logits, logits.argmax(-1), top=4)
    assert (s["rank"] == 0).all() and torch.equal(s["top_index"][:, 0].long(), logits.argmax(-1))
    assert (s["logprob"].double().cpu() - x.log_softmax(-1).amax(-1)).abs().max() < 1e-5
    m.drop(2)
    assert len(m.free) + sum(len(o) for o in m.own) == m.pages and (m.table[2] == -1).all()


def test_too_many_tokens():
    m = decoder()
    with pytest.raises(RuntimeError, match="pages more"):
        m.prefill({0: [1] * (41 * 64)})
