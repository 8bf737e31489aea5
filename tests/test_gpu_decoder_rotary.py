"""A decoder's rotated queries and keys, chunks and bounded steps together, against plain forms."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests.gpu_util import torch_cuda
from tests.test_gpu_decoder import close, tokens

pytestmark = pytest.mark.gpu

SHAPE = dict(vocab=997, dim=256, layers=2, heads=6, kv_heads=2, head_dim=64, ffn=512, pages=24, requests=4)


def decoder(**kw):
    torch_cuda()
    from glint_amd.decoder import Decoder
    m = Decoder(**SHAPE, rotary=H.rotary_freqs(32, base=500.0), **kw)
    import torch
    gen = torch.Generator(device="cuda").manual_seed(9)
    for layer in m.layers:
        layer.q_norm, layer.k_norm = (1 + 0.3 * torch.randn((2, 64), device="cuda", generator=gen)).bfloat16()
    return m


def turned(m, x, pos, weight):
    """The first half of a head's dimensions turned, after its norm, in 64 bits."""
    import torch
    y = x.double()
    y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    angle = torch.tensor(pos, device="cuda", dtype=torch.float64)[:, None, None] * m.rotary
    a, b = y[..., :16], y[..., 16:32]
    return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), y[..., 32:]], -1).to(x.dtype)


def cached(m, r):
    """[(k, v) per layer] of a request as the cache holds them; anything where a page was given back."""
    import torch
    slots = [(m.own[r][t // 64] or 0) * 64 + t % 64 for t in range(m.held[r])]
    return [H.kv4_gather(torch.tensor(slots, dtype=torch.int64, device="cuda"), layer.cache) for layer in m.layers]


def plain(m, old, news, held=None):
    """Logits of {request: tokens} after what the cache held, attention in f32 on the CPU; held: what it holds of the
    new tokens where those are read from it."""
    import torch
    from glint_amd.decoder import norm
    pos = [len(old[r][0][0]) + j for r, some in news.items() for j in range(len(some))]
    x = m.embed[torch.tensor([t for some in news.values() for t in some], device="cuda")]
    for i, layer in enumerate(m.layers):
        q, k, v = layer.qkv(norm(x)).unflatten(1, (-1, m.head_dim)).split([m.heads, m.kv_heads, m.kv_heads], 1)
        q, k = turned(m, q, pos, layer.q_norm), turned(m, k, pos, layer.k_norm)
        out, at = torch.empty(q.shape), 0
        for r, some in news.items():
            rows = slice(at, at + len(some))
            at += len(some)
            had = len(old[r][i][0])
            now = (k[rows], v[rows]) if held is None else [y[had:] for y in held[r][i]]
            ks, vs = (torch.cat([o, n]).float().cpu() for o, n in zip(old[r][i], now))
            p, j = torch.arange(had, had + len(some))[:, None], torch.arange(len(ks))[None]
            hidden = j > p
            if m.window is not None:
                hidden |= (j <= p - m.window) & (j >= m.sinks)
            for h in range(m.heads):
                z = q[rows, h].float().cpu() @ ks[:, h * m.kv_heads // m.heads].T * m.head_dim ** -0.5
                out[rows, h] = z.masked_fill(hidden, -torch.inf).softmax(-1) @ vs[:, h * m.kv_heads // m.heads]
        x = x + layer.out(out.to(q).to(q.dtype).flatten(1))
        gate, up = layer.up(norm(x)).chunk(2, -1)
        x = x + layer.down(torch.nn.functional.silu(gate) * up)
    return m.head(norm(x)).float()


@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3), (128, 70)])
def test_prompts_chunks_and_steps(window, sinks):
    m, rng = decoder(window=window, sinks=sinks), np.random.default_rng(1)
    for news in ({0: tokens(rng, 5), 2: tokens(rng, 230), 3: tokens(rng, 64)}, {2: tokens(rng, 90), 1: tokens(rng, 3), 0: tokens(rng, 60)}):
        print("prefill", {r: len(t) for r, t in news.items()}, flush=True)
        old = {r: cached(m, r) for r in news}
        want = plain(m, old, news)
        close(m.prefill(news), want)
    for news in ({r: tokens(rng, 1) for r in range(4)}, {0: tokens(rng, 4), 3: tokens(rng, 2), 1: tokens(rng, 4)}, {2: tokens(rng, 1)}):
        print("step", {r: len(t) for r, t in news.items()}, flush=True)
        old = {r: cached(m, r) for r in news}
        slide, m._slide = m._slide, lambda rows: None  # what the step read is looked at before pages go
        logits = m.step(news)
        close(logits, plain(m, old, news, {r: cached(m, r) for r in news}))
        m._slide = slide
        m._slide(list(news))
    assert len(m.free) + sum(p is not None for o in m.own for p in o) == m.pages


def test_pages_are_given_back():
    """A request runs on past what the pool holds; its table has the pages that it still sees and no others."""
    import torch
    m, rng = decoder(window=100, sinks=65, context=4000), np.random.default_rng(2)
    for _ in range(9):
        m.prefill({1: tokens(rng, 350)})
        kept = [i for i, p in enumerate(m.own[1]) if p is not None]
        first = (m.held[1] - 100 + 1) // 64
        assert kept == [0, 1, *range(max(2, first), len(m.own[1]))]
        assert (m.table[1, :len(m.own[1])] >= 0).nonzero()[:, 0].tolist() == kept
    assert m.held[1] == 3150 > m.pages * 64
    assert torch.isfinite(m.step({1: [5]})).all()
    m.drop(1)
    assert sorted(m.free) == list(range(m.pages))
    with pytest.raises(RuntimeError, match="places"):
        for _ in range(20):
            m.prefill({1: tokens(rng, 350)})
    with pytest.raises(ValueError):
        from glint_amd.decoder import Decoder
        Decoder(**SHAPE, window=5)


def test_the_command_runs(capsys):
    torch_cuda()
    from glint_amd import decoder as D
    D.main()
    assert "request 3:" in capsys.readouterr().out
