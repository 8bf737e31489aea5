"""Attention over a sliding window and first tokens: over the cache and over packed prompts, within the bounds of the unbounded forms."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import bounded_util as R
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu, random_planes

pytestmark = pytest.mark.gpu


def values(t):
    return S.bf16_values(host(t)).reshape(t.shape).astype(np.float64)


def paged(rng, lens, heads, D, spare=2):
    """(planes, table, pages): pages in no order, further pages in each row of the table."""
    wide = max(1, max((n + 63) // 64 for n in lens))
    pages = len(lens) * wide + spare
    planes = random_planes(rng, pages, heads, D)
    return planes, rng.permutation(pages)[:len(lens) * wide].reshape(len(lens), wide).astype(np.int32), pages


def spoil(planes, table, lens, nqs, window, sinks):
    """Infinite and NaN scales wherever no row of a sequence looks: past its end, between its sinks and its window."""
    for b, (n, nq) in enumerate(zip(lens, nqs)):
        t = np.arange(table.shape[1] * 64)
        hidden = (t >= n) | ((t >= sinks) & (t <= n - nq - window)) if window else t >= n
        for j in np.flatnonzero(hidden):
            for plane in (planes[1], planes[3]):
                plane[table[b, j // 64], :, :, j % 64] = [np.inf, np.nan, -np.inf, 3e38][j % 4]


def check_cache(lens, nqs, heads, G, D, window, sinks, seed=0, call=None, bound=R.KV4):
    rng = np.random.default_rng(seed)
    planes, table, pages = paged(rng, lens, heads, D)
    clean = [p.copy() for p in planes]
    spoil(planes, table, lens, nqs, window, sinks)
    cu = np.concatenate([[0], np.cumsum(nqs)]).astype(np.int32)
    q = bf16(rng.normal(0, 1, (cu[-1], heads * G, D)).astype(np.float32))
    cache = tuple(gpu(p) for p in planes)
    same = len(set(nqs)) == 1
    call = call or H.kv4_attend
    out = call(q, cache, gpu(table), gpu(np.array(lens, np.int32)), cu_q=None if same and call is H.kv4_attend else gpu(cu),
               max_q=max(nqs), window=window or None, sinks=sinks)
    got, qf = values(out), values(q)
    for b, (n, nq) in enumerate(zip(lens, nqs)):
        if nq == 0:
            continue
        k, v = S.held(clean, table[b][np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64) if n else np.zeros((2, 0, heads, D))
        ok = R.seen(np.arange(nq) + n - nq, n, window, sinks)
        for h in range(heads * G):
            rows = slice(cu[b], cu[b + 1])
            worst = R.far(got[rows, h], *R.attend(qf[rows, h], k[:, h // G], v[:, h // G], ok, D ** -0.5), bound)
            assert worst <= 0, (b, h, worst)
    return q, cache, table, out


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (63, 0), (64, 4), (65, 64), (200, 70), (1000, 3), (5000, 0), (100, 9000), (1 << 30, 5)])
def test_window_of_one_token(window, sinks):
    torch_cuda()
    for D, heads, G in ((64, 2, 3), (128, 3, 4)):
        print(f"window={window} sinks={sinks} D={D}", flush=True)
        check_cache([1, 64, 65, 130, 0, 1000, 777, 64 * 9 + 1], [1] * 8, heads, G, D, window, sinks, seed=window + sinks)


@pytest.mark.parametrize("window,sinks", [(1, 2), (3, 0), (70, 4), (129, 128)])
def test_window_of_drafts(window, sinks):
    """Several rows a sequence, none, more than it has tokens, more than a group's 16."""
    torch_cuda()
    for D, heads, G in ((64, 1, 5), (128, 2, 8)):
        print(f"drafts window={window} sinks={sinks} D={D}", flush=True)
        check_cache([3, 200, 65, 400, 64, 500], [5, 3, 0, 70, 1, 20], heads, G, D, window, sinks, seed=window)


def test_long_sequences_are_split():
    torch_cuda()
    check_cache([9000], [1], 2, 4, 128, 5000, 130, seed=1)
    check_cache([7001, 12], [2, 1], 1, 4, 64, 6000, 4, seed=2)
    check_cache([70 + 40 * i for i in range(70)], [1] * 70, 1, 2, 64, 90, 66, seed=3)


@pytest.mark.parametrize("sink_scale,edge_scale,rest_scale", [(1, 1, 8), (8, 1, 1), (1, 8, 1), (1 / 64, 1, 30), (30, 1 / 64, 1), (1, 1 / 30, 64)])
def test_scales_of_unlike_pages(sink_scale, edge_scale, rest_scale):
    """Pages seen in part come before whole ones whose values are larger or smaller, and a wave has several of them: 80
    sequences with the same pages."""
    torch_cuda()
    for D, heads, G, nq, window, sinks in ((128, 2, 4, 1, 2048, 4), (64, 2, 5, 3, 2000, 70), (128, 1, 3, 5, 2001, 3)):
        rng = np.random.default_rng(D + nq)
        B, n = 80, 4096 + 17
        planes, table, _ = paged(rng, [n], heads, D)
        at = table[0]
        planes[3][:] *= np.float32(rest_scale)
        planes[3][at[:(sinks + 63) // 64]] *= np.float32(sink_scale / rest_scale)
        low = (n - nq - window + 1) // 64
        planes[3][at[low:low + 1]] *= np.float32(edge_scale / rest_scale)
        q = bf16(rng.normal(0, 0.3, (nq, heads * G, D)).astype(np.float32))
        out = H.kv4_attend(q.repeat(B, 1, 1), tuple(gpu(p) for p in planes), gpu(table).repeat(B, 1), gpu(np.full(B, n, np.int32)),
                           max_q=nq, window=window, sinks=sinks)
        got, qf = values(out).reshape(B, nq, heads * G, D), values(q)
        k, v = S.held(planes, at[np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64)
        ok = R.seen(np.arange(nq) + n - nq, n, window, sinks)
        for h in range(heads * G):
            worst = R.far(got[:, :, h], *R.attend(qf[:, h], k[:, h // G], v[:, h // G], ok, D ** -0.5), R.KV4)
            assert worst <= 0, (D, nq, h, worst)


def test_dropped_pages_are_not_read():
    """Pages between sinks and window may be -1 or any other number."""
    torch = torch_cuda()
    q, cache, table, out = check_cache([1500, 700], [2, 2], 2, 4, 128, 300, 65, seed=4)
    lens = gpu(np.array([1500, 700], np.int32))
    for gone in (-1, 1 << 30, 0):
        t = table.copy()
        for b, n in enumerate((1500, 700)):
            j = np.arange(t.shape[1]) * 64
            t[b, (j >= 65) & (j + 63 <= n - 2 - 300)] = gone
        assert (t != table).any()
        assert torch.equal(H.kv4_attend(q, cache, gpu(t), lens, max_q=2, window=300, sinks=65), out), gone


def test_a_window_past_everything_is_no_window():
    torch = torch_cuda()
    rng = np.random.default_rng(5)
    planes, table, _ = paged(rng, [300, 65], 2, 64)
    cache, lens, q = tuple(gpu(p) for p in planes), gpu(np.array([300, 65], np.int32)), bf16(rng.normal(0, 1, (2, 4, 64)))
    assert torch.equal(H.kv4_attend(q, cache, gpu(table), lens, window=300), H.kv4_attend(q, cache, gpu(table), lens))
    x = bf16(rng.normal(0, 1, (3, 200, 2, 64)))
    cu = gpu(np.array([0, 130, 200], np.int32))
    assert torch.equal(H.attend_prompt(*x, cu, window=130), H.attend_prompt(*x, cu))


# ------------------------------------------------------------------ prompts
def check_prompt(nq, nk, heads, G, D, window, sinks, seed=0, odd=False):
    rng = np.random.default_rng(seed)
    cq, ck = (np.concatenate([[0], np.cumsum(n)]).astype(np.int32) for n in (nq, nk))
    q = bf16(rng.normal(0, 1, (cq[-1], heads * G, D)).astype(np.float32))
    k, v = rng.normal(0, 1, (2, ck[-1], heads, D)).astype(np.float32)
    clean = values(bf16(k)), values(bf16(v))
    if odd:  # what no row of a sequence sees
        for b in range(len(nq)):
            j = np.arange(nk[b])
            hidden = ck[b] + j[(j >= sinks) & (j <= nk[b] - nq[b] - window)]
            k[hidden], v[hidden] = np.nan, np.inf
            v[hidden[::2]] = np.nan
    got = values(H.attend_prompt(q, bf16(k), bf16(v), gpu(cq), gpu(ck), max_q=max(nq), window=window, sinks=sinks))
    qf = values(q)
    for b in range(len(nq)):
        ok = R.seen(np.arange(nq[b]) + nk[b] - nq[b], nk[b], window, sinks)
        for h in range(heads * G):
            rows, keys = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
            z = R.attend(qf[rows, h], clean[0][keys, h // G], clean[1][keys, h // G], ok, D ** -0.5)
            worst = R.far(got[rows, h], *z, R.PROMPT)
            assert worst <= 0, (b, h, worst)


@pytest.mark.parametrize("D,heads,G", [(64, 2, 3), (128, 1, 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (31, 0), (64, 64), (65, 1), (130, 100), (128, 0), (700, 4), (40, 5000), (1 << 30, 0)])
def test_prompts(D, heads, G, window, sinks):
    """Sequences of 0, 1 and more tokens, some after keys they already have, one without keys, one with more
    queries than keys; infinite and NaN keys and values where nobody looks."""
    torch_cuda()
    print(f"prompts window={window} sinks={sinks} D={D}", flush=True)
    check_prompt([5, 0, 130, 1, 64, 9, 7, 300], [5, 3, 530, 129, 64, 0, 4, 300], heads, G, D, window, sinks, seed=window, odd=True)


def test_one_long_prompt():
    torch_cuda()
    check_prompt([1500], [1700], 1, 2, 128, 257, 5, seed=2)
    check_prompt([1100], [1100], 1, 1, 64, 1, 0, seed=3)


def test_values_that_are_not_finite_stay_with_their_window():
    """An infinite value shows in the rows that see it and in no other, wherever the window begins in its tile."""
    torch = torch_cuda()
    rng = np.random.default_rng(6)
    n, D, window, sinks = 400, 64, 100, 2
    q, k, v = (bf16(rng.normal(0, 1, (n, 1, D))) for _ in range(3))
    cu = gpu(np.array([0, n], np.int32))
    clean = H.attend_prompt(q, k, v, cu, window=window, sinks=sinks)
    for j in (1, 70, 200, 390):
        spoilt = v.clone()
        spoilt[j, 0, 7] = float("inf")
        y = H.attend_prompt(q, k, spoilt, cu, window=window, sinks=sinks)
        i = torch.arange(n, device="cuda")
        sees = (i >= j) & ((i < j + window) | (j < sinks))
        assert (y[sees][:, 0, 7] == float("inf")).all()
        same = y.clone()
        same[sees, 0, 7] = clean[sees, 0, 7]
        assert torch.equal(same, clean), j
        k2 = k.clone()
        k2[j] = float("nan")
        y = H.attend_prompt(q, k2, v, cu, window=window, sinks=sinks)
        assert torch.equal(y[~sees], clean[~sees]) and y[sees].isnan().all()


def test_captured():
    """Both forms in a graph, replayed over new queries beside eager calls."""
    torch = torch_cuda()
    rng = np.random.default_rng(7)
    planes, table, _ = paged(rng, [900, 300], 2, 64)
    cache, table, lens = tuple(gpu(p) for p in planes), gpu(table), gpu(np.array([900, 300], np.int32))
    q, x = bf16(rng.normal(0, 1, (2, 4, 64))), bf16(rng.normal(0, 1, (3, 300, 2, 64)))
    cu = gpu(np.array([0, 100, 300], np.int32))
    call = lambda: (H.kv4_attend(q, cache, table, lens, window=200, sinks=3), H.attend_prompt(*x, cu, window=50, sinks=3))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(3):
        q.copy_(bf16(rng.normal(0, 1, (2, 4, 64))))
        x.copy_(bf16(rng.normal(0, 1, (3, 300, 2, 64))))
        graph.replay()
        want = call()
        # the graph's own call may run unsplit: a workspace is its stream's
        assert torch.equal(got[1], want[1]), i
        assert torch.allclose(got[0].float(), want[0].float(), atol=2.0 ** -7, rtol=2.0 ** -7), i
