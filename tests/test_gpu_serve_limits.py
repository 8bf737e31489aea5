"""The serving operators where launches, offsets and workspaces reach their limits."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, check, gpu, random_planes

pytestmark = pytest.mark.gpu


def side_stream(torch):
    """A stream that no other test's workspace belongs to."""
    side = torch.cuda.Stream()
    assert H.serve_lib().glint_serve_workspace_release(side.cuda_stream) == 0
    side.wait_stream(torch.cuda.current_stream())
    return side


@pytest.mark.parametrize("reserved", [False, True])
def test_graphs_with_and_without_a_workspace(reserved):
    """A capture on a stream that has no workspace leaves the work whole; one on a stream that has one
    splits it. Replays among eager calls of the same stream match what the inputs then say."""
    torch = torch_cuda()
    rng = np.random.default_rng(20)
    planes = tuple(gpu(p) for p in random_planes(rng, 120, 2, 128))
    q = bf16(rng.normal(0, 1, (3, 8, 128)).astype(np.float32))
    table, lens = gpu(rng.permutation(120).astype(np.int32).reshape(3, 40)), gpu(np.array([2560, 1, 700], np.int32))
    x = bf16(rng.normal(0, 3, (4, 128256)).astype(np.float32))
    tok = gpu(np.array([0, 128255, 77, 5], np.int64))
    kb, slots = bf16(rng.normal(0, 1, (3, 2, 128)).astype(np.float32)), gpu(np.array([5, -1, 64 * 119], np.int64))
    side = side_stream(torch)
    lib = H.serve_lib()
    if reserved:
        assert lib.glint_serve_workspace_reserve(side.cuda_stream) == 0
    work = tuple(p.clone() for p in planes)
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        H.kv4_append(kb, kb, slots, work)
        k, v = H.kv4_gather(slots, work)
        out = H.kv4_attend(q, work, table, lens)
        cu = torch.arange(4, dtype=torch.int32, device="cuda")
        prompt = H.attend_prompt(q, k, v, cu, max_q=1)
        scores = H.token_logprobs(x, tok, top=20)
    for i in range(4):
        out.fill_(3.0)
        if i == 2:
            lens.copy_(lens.flip(0))
            x.copy_(x.flip(0))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            H.kv4_attend(q, planes, table, lens)  # the stream's eager calls have a workspace of their own
            H.token_logprobs(x, tok, top=20)
        torch.cuda.synchronize()
        again = tuple(p.clone() for p in planes)
        H.kv4_append(kb, kb, slots, again)
        assert all(torch.equal(a, b) for a, b in zip(work, again)), i
        want = H.kv4_attend(q, again, table, lens)
        wk, wv = H.kv4_gather(slots, again)
        assert torch.equal(k, wk) and torch.equal(v, wv) and torch.equal(prompt, H.attend_prompt(q, wk, wv, cu, max_q=1)), i
        ws = H.token_logprobs(x, tok, top=20)
        assert torch.equal(scores["rank"], ws["rank"]) and torch.equal(scores["top_index"], ws["top_index"]), i
        if reserved:
            assert torch.equal(out, want), i
            assert all(torch.equal(scores[n], ws[n]) for n in ws), i
        else:  # other partial sums: weights' f16 roundings (2^-12 of values up to 3, on both sides) fall elsewhere
            assert ((out.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 3 * 2.0 ** -11).all(), i
            for n in ("logprob", "entropy", "top_logprob"):
                assert torch.allclose(scores[n], ws[n], rtol=1e-5, atol=1e-5), (i, n)
    del graph
    torch.cuda.synchronize()
    assert lib.glint_serve_workspace_release(side.cuda_stream) == 0


@pytest.mark.parametrize("B,held", [(70, 0.8), (150, 0.5), (200, 0.02), (65, 0)])
def test_more_sequences_than_a_wave(B, held):
    """Batches past 64 sequences, most of them without a token in some, rows of their own for each."""
    torch_cuda()
    print(f"B={B}", flush=True)
    rng = np.random.default_rng(B)
    lens = np.where(rng.random(B) < held, rng.integers(1, 200, B), 0)
    nqs = rng.integers(0, 4, B)
    nqs[0] = 2
    planes = random_planes(rng, 50, 1, 64)
    table = rng.integers(0, 50, (B, 4))
    got = check(rng.normal(0, 1, (int(nqs.sum()), 2, 64)).astype(np.float32), planes, table, lens.tolist(), nqs.tolist(), 2, 64)
    starts = np.cumsum(nqs)
    for b in np.flatnonzero(lens == 0):
        assert (got[starts[b] - nqs[b]:starts[b]] == 0).all()


def test_runs_of_many_rounds():
    """More than a million tokens a sequence, from a few pages named again and again: their softmax is that of the
    pool's tokens, each counted as often as it is named."""
    torch_cuda()
    rng = np.random.default_rng(30)
    pages, wide, heads, D = 40, 20000, 8, 64
    planes = random_planes(rng, pages, heads, D)
    table = rng.integers(0, pages, (2, wide)).astype(np.int32)
    lens = [wide * 64, 700001]
    q = bf16(rng.normal(0, 1, (2, heads, D)).astype(np.float32))
    got = S.bf16_values(host(H.kv4_attend(q, tuple(gpu(p) for p in planes), gpu(table), gpu(np.array(lens, np.int32)))))
    got, qf = got.reshape(2, heads, D), S.bf16_values(host(q)).reshape(2, heads, D).astype(np.float64)
    k, v = S.held(planes, np.arange(pages * 64))
    for b in range(2):
        at = np.arange(lens[b])
        count = np.bincount(table[b][at // 64] * 64 + at % 64, minlength=pages * 64)
        for h in range(heads):
            z = k[:, h] @ qf[b, h] * D ** -0.5
            p = count * np.exp(z - z.max())
            p /= p.sum()
            size = (np.abs(k[:, h]) @ np.abs(qf[b, h])).max() * D ** -0.5
            out, mass = p @ v[:, h], p @ np.abs(v[:, h])
            far = np.abs(got[b, h] - out) - S.kv4_bound(out[None], mass[None], np.array([size]))[0]
            assert (far <= 0).all(), (b, h, float(far.max()))


def test_a_cache_past_32_bits():
    """Pages whose codes lie past 4 GiB are written, read and attended like the first ones."""
    torch = torch_cuda()
    rng = np.random.default_rng(31)
    heads, D, T = 8, 128, 150
    small, large = H.kv4_cache(4, heads, D), H.kv4_cache(140000, heads, D)
    assert large.k_hole.numel() > 1 << 32
    k, v = (bf16(rng.normal(0, 1, (T, heads, D)).astype(np.float32)) for _ in range(2))
    near, far = gpu(np.array([2, 0, 3], np.int64)), gpu(np.array([139999, 131072, 135000], np.int64))
    t = torch.arange(T, device="cuda")
    place = lambda pages: pages[t // 64] * 64 + t % 64
    for n in (T, 40):  # element by element as well
        H.kv4_append(k[:n], v[:n], place(near)[:n], small)
        H.kv4_append(k[:n], v[:n], place(far)[:n], large)
    for a, b in zip(small, large):
        assert torch.equal(a[near[:2]], b[far[:2]])
    for a, b in zip(H.kv4_gather(place(near), small), H.kv4_gather(place(far), large)):
        assert torch.equal(a, b)
    many = torch.arange(200 * 64, device="cuda") % (139990 - 131072) + 131072 * 64  # enough to go by tiles
    wide_k, wide_v = (bf16(rng.normal(0, 1, (2200, heads, D)).astype(np.float32)) for _ in range(2))
    H.kv4_append(wide_k, wide_v, many[:2200], large)
    first = H.kv4_cache(40, heads, D)
    H.kv4_append(wide_k, wide_v, torch.arange(2200, device="cuda"), first)
    for a, b in zip(H.kv4_gather(torch.arange(2200, device="cuda"), first), H.kv4_gather(many[:2200], large)):
        assert torch.equal(a, b)
    H.kv4_append(k, v, place(far), large)
    H.kv4_append(k, v, place(near), small)
    q = bf16(rng.normal(0, 1, (1, 4 * heads, D)).astype(np.float32))
    n = gpu(np.array([T], np.int32))
    assert torch.equal(H.kv4_attend(q, small, near.int()[None], n), H.kv4_attend(q, large, far.int()[None], n))


def test_rows_past_32_bits():
    """Strides that put keys, values and logits past 4 GiB."""
    torch = torch_cuda()
    rng = np.random.default_rng(32)
    T, heads, D = 150, 2, 64
    wide = torch.empty((T, 1 << 24), dtype=torch.bfloat16, device="cuda")
    kv = bf16(rng.normal(0, 1, (T, 2 * heads * D)).astype(np.float32))
    wide[:, :2 * heads * D] = kv
    k, v = wide[:, :heads * D].unflatten(1, (heads, D)), wide[:, heads * D:2 * heads * D].unflatten(1, (heads, D))
    q = bf16(rng.normal(0, 1, (T, 3 * heads, D)).astype(np.float32))
    cu = gpu(np.array([0, T], np.int32))
    assert torch.equal(H.attend_prompt(q, k, v, cu), H.attend_prompt(q, k.contiguous(), v.contiguous(), cu))
    slots = torch.arange(T, device="cuda")
    a, b = H.kv4_cache(3, heads, D), H.kv4_cache(3, heads, D)
    H.kv4_append(k, v, slots, a)
    H.kv4_append(k.contiguous(), v.contiguous(), slots, b)
    for x, y in zip(H.kv4_gather(slots, a), H.kv4_gather(slots, b)):
        assert torch.equal(x, y)
    x = bf16(rng.normal(0, 3, (T, 1000)).astype(np.float32))
    wide[:, :1000] = x
    tok = slots * 6
    want, got = H.token_logprobs(x, tok, top=5), H.token_logprobs(wide[:, :1000], tok, top=5)
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_helpers_refuse_mixed_devices_and_types():
    torch = torch_cuda()
    cache = H.kv4_cache(2, 1, 64)
    k = torch.zeros((3, 1, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    cu = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for call in (lambda: H.kv4_append(k.cpu(), k, slots, cache), lambda: H.kv4_append(k, k, slots.cpu(), cache),
                 lambda: H.kv4_append(k.half(), k.half(), slots, cache), lambda: H.kv4_append(k, k[:2], slots, cache),
                 lambda: H.kv4_append(k, k, slots[:2], cache), lambda: H.kv4_append(k, k, slots.int(), cache),
                 lambda: H.kv4_gather(slots.cpu(), cache), lambda: H.kv4_attend(k.float(), cache, cu[None], cu[1:]),
                 lambda: H.kv4_attend(k[:1], cache, slots[None], cu[1:]), lambda: H.kv4_attend(k[:1], cache, cu[None], cu),
                 lambda: H.attend_prompt(k, k, k, cu.cpu()), lambda: H.attend_prompt(k, k, k.float(), cu),
                 lambda: H.token_logprobs(k[:, 0], slots[:2]), lambda: H.token_logprobs(k[:, 0].double(), slots)):
        with pytest.raises((ValueError, TypeError)):
            call()
    assert all((p == 0).all() for p in cache)
