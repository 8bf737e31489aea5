"""The serving operators at masks, strides, defaults and batches where a call once went wrong."""
import math

import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu, random_planes

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ log probabilities
def logits_of(x, f32, shift=0):
    """x [T, V] on the GPU as F32 or BF16, rows `shift` elements past a 16-B boundary, and what it holds in 64 bits."""
    t = gpu(x.astype(np.float32)) if f32 else bf16(x.astype(np.float32))
    vals = (host(t) if f32 else S.bf16_values(host(t)).reshape(x.shape)).astype(np.float64)
    if shift:
        wide = t.new_full((x.shape[0], (x.shape[1] + shift + 15) // 16 * 16), float("nan"))
        wide[:, shift:shift + x.shape[1]] = t
        t = wide[:, shift:shift + x.shape[1]]
    return t, vals


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,V,shift", [(3, 128256, 0), (1, 128251, 3), (100, 40007, 1), (6, 32003, 0), (6, 32003, 5), (300, 9001, 0), (4, 77, 2)])
def test_rank_of_a_forbidden_token(T, V, shift, f32):
    """A token at -inf among allowed and forbidden entries: every larger entry comes before it, and every equal one at a
    lower index, wherever the token lies and however the row is shared out."""
    torch_cuda()
    print(f"rank at -inf T={T} V={V} shift={shift} f32={f32}", flush=True)
    rng = np.random.default_rng(T + V)
    x = rng.normal(0, 3, (T, V))
    x[rng.random((T, V)) < 0.5] = -np.inf
    x[:, [0, 1, V // 3, V // 2, V - 2, V - 1]] = -np.inf
    x[0, : V - 1] = 1.0  # the token alone is forbidden, or
    x[-1] = -np.inf      # it and all but one are
    x[-1, 5] = 2.0
    places = [V - 1, 0, V // 2, V // 3, V - 2, 1]
    t, vals = logits_of(x, f32, shift)
    for first in range(3):
        tok = np.array([places[(i + first) % 6] for i in range(T)])
        tok[0] = V - 1
        want = [(np.count_nonzero(v > v[k]) + np.count_nonzero(v[:k] == v[k])) for v, k in zip(vals, tok)]
        r = {k: host(v) for k, v in H.token_logprobs(t, gpu(tok), top=2).items()}
        assert r["rank"].tolist() == want, first
        assert (r["logprob"] == -np.inf).all()


def score_bound(x, tok):
    """One row of finite logits, each lse' = log s from the maximum m: (x - m) - log s, entropy, and how far f32 may be off
    log s: sums of a thread's elements and of the threads, and the exponents (x - r) log2 e, r within 14 of m, of three
    roundings (2^-24 each, the constant's included)."""
    m = x.max()
    d = x - m
    e = np.exp(d)
    s = e.sum()
    mean = -(e[e > 0] * d[e > 0]).sum() / s
    off = (len(x) / 1024 + 40) * 2.0 ** -24 + (mean + 14) * 3 * 2.0 ** -24
    return m, math.log(s), mean, off


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("T,V", [(9, 500), (9, 32003), (9, 128256), (300, 2000)])
def test_scores_of_the_largest_finite_logits(T, V, f32):
    """Masks of the type's lowest value and logits as far out as the type goes: log probabilities stay those of the definition
    (-log V in a row of nothing else) and become infinite only where they pass f32's range."""
    torch_cuda()
    print(f"finite extremes T={T} V={V} f32={f32}", flush=True)
    rng = np.random.default_rng(V)
    low = float(np.finfo(np.float32).min) if f32 else -3.3895313892515355e38
    x = rng.normal(0, 3, (T, V))
    x[0] = low                                       # nothing is allowed
    x[1, rng.random(V) < 0.9] = low                  # a mask
    x[2], x[2, 3] = low, 1.5                         # one entry is allowed
    x[3] = -low                                      # the largest value everywhere
    x[4, V // 2] = -low                              # and once
    x[5] = rng.choice([2.5e38, 2.4e38, -2.5e38, 0.0], V)
    x[6, : V // 2] = -1e38                           # long stretches far below what follows
    x[7] = np.linspace(-3e38, 3e38, V)
    x[8, :] = low
    x[8, V // 4:] = -2.5e38
    tok = rng.integers(0, V, T)
    tok[1] = int(np.flatnonzero(x[1] == low)[0])
    tok[2], tok[6] = 0, 1
    top = 5
    t, vals = logits_of(x, f32)
    r = {k: host(v) for k, v in H.token_logprobs(t, gpu(tok), top=top).items()}
    for i in range(T):
        v = vals[i]
        m, log_s, mean, off = score_bound(v, tok[i])
        order = np.lexsort((np.arange(V), -v))[:top]
        assert r["rank"][i] == np.count_nonzero(v > v[tok[i]]) + np.count_nonzero(v[: tok[i]] == v[tok[i]]), i
        assert r["top_index"][i].tolist() == order.tolist(), i
        for got, at in [(r["logprob"][i], tok[i])] + list(zip(r["top_logprob"][i], order)):
            want = (v[at] - m) - log_s
            with np.errstate(over="ignore"):
                assert got == np.float32(want) or abs(float(got) - want) <= off + 2.0 ** -22 * (abs(want) + log_s), (i, at, got, want)
        assert abs(r["entropy"][i] - (log_s + mean)) <= 4 * (off + 2.0 ** -22 * (log_s + mean)), (i, r["entropy"][i], log_s + mean)


def test_ties_cost_no_more_than_their_order():
    """Two threads of every wave share its largest value: the list's floor is that value, as where the two differ, and the
    entries below it are no candidates (their search, quadratic over 1024 of them, took 2 times the call)."""
    torch = torch_cuda()
    T, V = 256, 8192  # a 16-B load of BF16 a thread
    x = torch.zeros((T, 1024, 8), device="cuda")
    x[:, 0::64, 0] = 10.0
    x[:, 1::64, 3] = 10.0
    apart = x.clone()
    apart[:, 0::64, 0] = 11.0
    tok = torch.zeros(T, dtype=torch.int64, device="cuda")
    times = {}
    rows = {"tie": x.view(T, V).bfloat16(), "apart": apart.view(T, V).bfloat16()}
    for name in ("tie", "apart"):
        r = H.token_logprobs(rows[name], tok, top=20)
        want = torch.sort(rows[name].float(), dim=1, descending=True, stable=True).indices[:, :20]
        assert torch.equal(r["top_index"].long(), want)
    for _ in range(3):
        for name, y in rows.items():
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            for _ in range(5):
                H.token_logprobs(y, tok, top=20)
            a.record()
            for _ in range(30):
                H.token_logprobs(y, tok, top=20)
            b.record()
            b.synchronize()
            times[name] = min(times.get(name, 1e9), a.elapsed_time(b) / 30)
    print({k: round(1e3 * v, 2) for k, v in times.items()}, flush=True)
    assert times["tie"] < 1.25 * times["apart"]


# ------------------------------------------------------------------ strides of single rows
@pytest.mark.parametrize("heads,T", [(8, 1), (1, 1), (1, 5)])
def test_single_rows_of_any_stride(heads, T):
    """Where there is one token, or one head, its stride means nothing, whatever it is."""
    torch = torch_cuda()
    rng = np.random.default_rng(heads)
    D, G = 128, 3
    if T == 1:  # a row of a projection whose width is odd
        buf = bf16(rng.normal(0, 1, (4, (G + 2) * heads * D + 5)).astype(np.float32))
        q, k, v = (buf[:, at * heads * D:(at + n) * heads * D].unflatten(1, (n * heads, D))[:1] for at, n in ((0, G), (G, 1), (G + 1, 1)))
    else:  # rows that follow each other; the one head's stride is odd
        q = bf16(rng.normal(0, 1, (T, G, D)).astype(np.float32))
        k, v = (torch.as_strided(bf16(rng.normal(0, 1, (T, D)).astype(np.float32)), (T, 1, D), (D, 13, 1)) for _ in range(2))
    slots = torch.arange(T, device="cuda")
    caches = []
    for same in (lambda t: t, lambda t: torch.empty(t.shape, dtype=t.dtype, device="cuda").copy_(t)):
        c = H.kv4_cache(2, heads, D)
        H.kv4_append(same(k), same(v), slots, c)
        H.kv4_append(same(k).float(), same(v).float(), slots + 64, c)
        caches.append(c)
    assert all(torch.equal(a, b) for a, b in zip(*caches))
    assert any((p != 0).any() for p in caches[0])
    cu = gpu(np.array([0, T], np.int32))
    lens = gpu(np.array([T], np.int32))
    want = H.attend_prompt(q.clone(memory_format=torch.contiguous_format), *(torch.empty(t.shape, dtype=t.dtype, device="cuda").copy_(t) for t in (k, v)), cu)
    assert torch.equal(H.attend_prompt(q, k, v, cu), want)
    if T == 1:
        table = gpu(np.array([[0, 1], [1, 0]], np.int32)).t()[:1]
        one = gpu(np.array([[0]], np.int32))
        want = H.kv4_attend(torch.empty(q.shape, dtype=q.dtype, device="cuda").copy_(q), caches[0], one, lens)
        assert torch.equal(H.kv4_attend(q, caches[0], one, lens), want)
        assert torch.equal(H.kv4_attend(q, caches[0], table[:, :1], lens), want)


# ------------------------------------------------------------------ defaults
def test_rows_of_every_sequence_by_default():
    """Where cu_q says how many rows a sequence has and max_q is left out, all of them are computed."""
    torch = torch_cuda()
    rng = np.random.default_rng(40)
    planes = tuple(gpu(p) for p in random_planes(rng, 20, 2, 128))
    nqs = np.array([3, 0, 9, 1])
    cu = gpu(np.concatenate([[0], np.cumsum(nqs)]).astype(np.int32))
    q = bf16(rng.normal(0, 1, (13, 8, 128)).astype(np.float32))
    table, lens = gpu(rng.permutation(20).astype(np.int32).reshape(4, 5)), gpu(np.array([300, 5, 64, 1], np.int32))
    want = H.kv4_attend(q, planes, table, lens, cu, max_q=9)
    out = torch.full_like(q, 7.0)
    H.kv4_attend(q, planes, table, lens, cu, out=out)
    assert torch.equal(out, want)
    assert torch.equal(H.kv4_attend(q, planes, table, lens, cu), want)
    single = H.kv4_attend(q[:4], planes, table, lens)
    assert torch.equal(single, H.kv4_attend(q[:4], planes, table, lens, max_q=1))


@pytest.mark.parametrize("packed", [False, True])
def test_more_work_than_one_list(packed):
    """Batches whose list of work, by the table's width and the rows that a sequence may have, is past one launch's bound:
    the same as their parts, for lengths of one round of pages, which nothing splits."""
    torch = torch_cuda()
    rng = np.random.default_rng(42)
    pages, heads, G, D = 30, 8, 4, 64
    planes = tuple(gpu(p) for p in random_planes(rng, pages, heads, D))
    B, wide = (1024, 1024) if packed else (1100, 131072)
    table = gpu(np.resize(rng.permutation(pages), wide).astype(np.int32))[None].expand(B, wide)
    lens = rng.integers(0, 500, B).astype(np.int32)
    nqs = rng.integers(0, 3, B) if packed else np.full(B, 2)
    starts = np.concatenate([[0], np.cumsum(nqs)]).astype(np.int32)
    wider = bf16(rng.normal(0, 1, (int(starts[-1]), (heads + 1) * G, D)).astype(np.float32))
    q = wider[:, G:]
    print(f"packed={packed} B={B} wide={wide}", flush=True)
    if packed:
        got = H.kv4_attend(q, planes, table, gpu(lens), gpu(starts))
    else:
        got = H.kv4_attend(q, planes, table, gpu(lens), max_q=2)
    for a in range(0, B, 100):
        z = min(a + 100, B)
        rows = slice(int(starts[a]), int(starts[z]))
        part = H.kv4_attend(q[rows], planes, table[a:z, :8], gpu(lens[a:z]), gpu(starts[a:z + 1] - starts[a]), max_q=2)
        assert torch.equal(got[rows], part), a


def test_many_prompts_without_a_longest():
    """512 prompts of 65536 tokens in all and no max_q: more row blocks than a launch holds, most of them empty."""
    torch = torch_cuda()
    rng = np.random.default_rng(41)
    B, heads, G, D = 512, 1, 32, 64
    cuts = np.sort(rng.choice(np.arange(1, 65536), B - 1, replace=False))
    cu = gpu(np.concatenate([[0], cuts, [65536]]).astype(np.int32))
    longest = int(np.diff(np.concatenate([[0], cuts, [65536]])).max())
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn((65536, n, D), device="cuda", generator=g).bfloat16() for n in (heads * G, heads, heads))
    want = H.attend_prompt(q, k, v, cu, max_q=longest)
    print("without max_q", flush=True)
    assert torch.equal(H.attend_prompt(q, k, v, cu), want)


def test_rows_outside_stay_without_keys():
    """Rows outside every sequence are left as they are where there is no key and no page either; those inside are zero."""
    torch = torch_cuda()
    q = torch.randn((9, 2, 64), device="cuda").bfloat16()
    cu = gpu(np.array([2, 5, 6], np.int32))
    none = q.new_empty((0, 1, 64))
    for run in (lambda out: H.attend_prompt(q, none, none, cu, gpu(np.array([0, 0, 0], np.int32)), out=out),
                lambda out: H.kv4_attend(q, H.kv4_cache(2, 1, 64), gpu(np.zeros((2, 0), np.int32)), gpu(np.array([0, 3], np.int32)),
                                         cu, max_q=3, out=out)):
        out = torch.full_like(q, 5.0)
        run(out)
        assert (out[:2] == 5).all() and (out[6:] == 5).all() and (out[2:6] == 0).all()


def test_a_workspace_is_as_large_as_its_kernels_need():
    """A stream's workspace takes some 4 MiB of the memory that cache pages want, not the matrix products' 128."""
    torch = torch_cuda()
    lib = H.serve_lib()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for s in streams:
        assert lib.glint_serve_workspace_release(s.cuda_stream) == 0
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for s in streams:
        assert lib.glint_serve_workspace_reserve(s.cuda_stream) == 0
    torch.cuda.synchronize()
    taken = free - torch.cuda.mem_get_info()[0]
    for s in streams:
        assert lib.glint_serve_workspace_release(s.cuda_stream) == 0
    print(f"{taken / 2 ** 20:.1f} MiB for {len(streams)} streams", flush=True)
    assert taken <= len(streams) * 16 << 20


# ------------------------------------------------------------------ the decoder
def test_a_refused_call_changes_nothing():
    """Where a later request does not fit, or does not exist, the requests before it keep what they had."""
    torch = torch_cuda()
    from glint_amd.decoder import Decoder
    shape = dict(vocab=97, dim=128, layers=1, heads=2, kv_heads=1, head_dim=64, ffn=128, pages=4, requests=3)
    m, twin = Decoder(**shape), Decoder(**shape)
    state = lambda d: (list(d.held), [list(o) for o in d.own], list(d.free), d.table.tolist())
    for d in (m, twin):
        d.prefill({0: list(range(60)), 1: [1, 2, 3]})
    before = state(m)
    for call, error in ((lambda: m.prefill({0: [5, 6], 2: [1] * 200}), RuntimeError), (lambda: m.step({0: [5] * 5, 1: [6] * 200}), RuntimeError),
                        (lambda: m.step({0: [5] * 70, 1: [6] * 70}), RuntimeError), (lambda: m.prefill({1: [5], 9: [5]}), IndexError),
                        (lambda: m.step({0: [5] * 10, 9: [5]}), IndexError)):
        with pytest.raises(error):
            call()
        assert state(m) == before
    assert torch.equal(m.step({0: [7], 1: [8]}), twin.step({0: [7], 1: [8]}))


# ------------------------------------------------------------------ the order of prompt work
@pytest.mark.parametrize("B,heads", [(3, 3), (5, 2), (2, 6), (13, 1), (11, 1)])
def test_groups_past_whole_rounds_of_xcds(B, heads):
    """More groups than XCDs, and a rest: 1, 2, 4, 5 and 3 of them."""
    torch = torch_cuda()
    rng = np.random.default_rng(B)
    G, D = 3, 64
    n = rng.integers(1, 300, B)
    cu = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    q, k, v = (bf16(rng.normal(0, 1, (cu[-1], c, D)).astype(np.float32)) for c in (heads * G, heads, heads))
    got = H.attend_prompt(q, k, v, gpu(cu), max_q=300)
    for b in range(B):
        part = slice(int(cu[b]), int(cu[b + 1]))
        one = gpu(np.array([0, n[b]], np.int32))
        assert torch.equal(got[part], H.attend_prompt(q[part], k[part], v[part], one)), b
