"""Chunks of new tokens over the 4-bit cache on the GPU, within the bounds of the roundings that they meet."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import bounded_util as R
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu, random_planes
from tests.test_gpu_window import paged, spoil, values

pytestmark = pytest.mark.gpu


def bound(own):
    """f16 products: as kv4_attend's, whose one rounding of a value, of a weight and of a key element they share (2^-12 there, half
    of what f16's worst is; all of it here), twice for the weights, whose sum is of the rounded ones. An own key or value
    is bf16 and rounds no more in f16."""
    def far(out, mass, size):
        return 2.0 ** -8 * np.abs(out) + mass * (3 * 2.0 ** -11 + np.expm1(2 * (2.0 ** -11 + 2.0 ** -18) * size)[:, None] + 2.0 ** -16)
    return far


def many(table, rows):
    """The table with further columns and a max_q that bounds more rows: both only bounds, for which the call takes the
    kernels for many rows."""
    wide = np.full((table.shape[0], 4200), -3, np.int32)
    wide[:, :table.shape[1]] = table
    return wide, max(rows, 257)


def check(lens, nqs, heads, G, D, window=0, sinks=0, own=False, seed=0, spread=None, scale=None):
    rng = np.random.default_rng(seed)
    planes, table, pages = paged(rng, lens, heads, D)
    if spread is not None:
        for i in (1, 3):
            planes[i] = (planes[i] * 2.0 ** rng.uniform(-spread, spread, planes[i].shape)).astype(np.float32)
    clean = [p.copy() for p in planes]
    spoil(planes, table, lens, nqs, window, sinks)
    cu = np.concatenate([[0], np.cumsum(nqs)]).astype(np.int32)
    q = bf16(rng.normal(0, 1, (cu[-1], heads * G, D)).astype(np.float32))
    k, v = (bf16(rng.normal(0, 1, (cu[-1], heads, D)).astype(np.float32)) for _ in range(2))
    if own:  # what the cache holds of the new tokens is not read
        for b, (n, nq) in enumerate(zip(lens, nqs)):
            j = np.arange(max(0, n - nq), n)
            for plane in (planes[1], planes[3]):
                plane[table[b, j // 64], :, :, j % 64] = np.nan
    wide, max_q = many(table, max(nqs))
    assert H.serve_lib().glint_kv4_attend_chunk_scratch(len(lens), max_q, heads * G, heads, D, wide.shape[1], own) > 0
    out = H.kv4_attend_chunk(q, tuple(gpu(p) for p in planes), gpu(wide), gpu(np.array(lens, np.int32)), gpu(cu), max_q=max_q,
                             k=k if own else None, v=v if own else None, window=window or None, sinks=sinks, scale=scale)
    got, qf, kf, vf = values(out), values(q), values(k), values(v)
    for b, (n, nq) in enumerate(zip(lens, nqs)):
        if nq == 0:
            continue
        hk, hv = S.held(clean, table[b][np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64) if n else np.zeros((2, 0, heads, D))
        rows = slice(cu[b], cu[b + 1])
        if own and n:
            m = min(nq, n)
            hk[n - m:], hv[n - m:] = kf[rows][nq - m:], vf[rows][nq - m:]
        ok = R.seen(np.arange(nq) + n - nq, n, window, sinks)
        for h in range(heads * G):
            z = R.attend(qf[rows, h], hk[:, h // G], hv[:, h // G], ok, D ** -0.5 if scale is None else scale)
            worst = R.far(got[rows, h], *z, bound(own))
            assert worst <= 0, (b, h, worst)
    return out


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D,heads,G", [(64, 2, 3), (128, 1, 4)])
@pytest.mark.parametrize("n,nq", [(1, 1), (64, 64), (65, 3), (200, 64), (130, 130), (700, 33), (63, 62)])
def test_one_sequence(D, heads, G, n, nq, own):
    torch_cuda()
    print(f"chunk D={D} n={n} nq={nq} own={own}", flush=True)
    check([n], [nq], heads, G, D, own=own, seed=n)


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D,heads,G", [(64, 3, 1), (128, 1, 8), (128, 2, 5)])
def test_ragged_batch(D, heads, G, own):
    """Sequences without tokens, without rows, with more rows than tokens, of one row and of several blocks."""
    torch_cuda()
    print(f"ragged D={D} H={heads} G={G} own={own}", flush=True)
    check([5, 300, 330, 129, 0, 64, 4, 400], [5, 0, 130, 1, 3, 9, 7, 300], heads, G, D, own=own, seed=D + G)


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (64, 64), (65, 1), (130, 100), (257, 0), (2000, 7), (40, 5000)])
def test_windows(window, sinks, own):
    torch_cuda()
    for D, heads, G in ((64, 2, 3), (128, 1, 4)):
        print(f"chunk window={window} sinks={sinks} D={D} own={own}", flush=True)
        check([5, 700, 530, 129, 0, 64, 4], [5, 90, 130, 1, 3, 9, 7], heads, G, D, window, sinks, own=own, seed=window)
    check([200], [200], 1, 2, 64, window, sinks, own=own, seed=window + 1)


def test_a_long_context_is_split():
    """Few rows over many pages, whose parts meet, and parts of which some see nothing."""
    torch_cuda()
    check([9000], [20], 1, 4, 128, seed=1)
    check([6001], [70], 2, 2, 64, seed=2, own=True)
    check([5000, 77, 3000], [40, 30, 1], 1, 4, 64, 900, 130, seed=3)
    check([2500], [600], 1, 1, 128, seed=4)


def test_scales_of_every_size():
    """Absmax over 2^-12 .. 2^12 in one page, far from 1, and a maximum that grows page after page."""
    torch_cuda()
    check([500], [70], 1, 3, 128, spread=3, scale=0.02, seed=5)
    check([500], [70], 1, 3, 64, spread=12, scale=2.0 ** -13, seed=6)
    check([300], [40], 1, 1, 64, scale=-0.3, seed=7)
    check([300], [40], 1, 1, 128, scale=0.0, seed=8)


def test_rows_outside_stay():
    """Rows past max_q, and rows of no sequence, hold what they held."""
    torch = torch_cuda()
    rng = np.random.default_rng(9)
    planes, table, _ = paged(rng, [100, 200], 1, 64)
    cache, lens = tuple(gpu(p) for p in planes), gpu(np.array([100, 200], np.int32))
    q = bf16(rng.normal(0, 1, (60, 2, 64)))
    full = H.kv4_attend_chunk(q, cache, gpu(table), lens, gpu(np.array([3, 33, 53], np.int32)))
    out = torch.full_like(q, 7.0)
    got = H.kv4_attend_chunk(q, cache, gpu(table), lens, gpu(np.array([3, 33, 53], np.int32)), max_q=20, out=out)
    assert got is out
    assert (out[:3] == 7).all() and (out[23:33] == 7).all() and (out[53:] == 7).all()
    assert torch.equal(out[3:23], full[3:23]) and torch.equal(out[33:53], full[33:53])
    assert torch.equal(full[3:53], H.kv4_attend(q, cache, gpu(table), lens, gpu(np.array([3, 33, 53], np.int32)))[3:53])
    wide, _ = many(table, 0)
    k = bf16(rng.normal(0, 1, (60, 1, 64)))
    for own in (None, k):
        out.fill_(7.0)
        H.kv4_attend_chunk(q, cache, gpu(wide), lens, gpu(np.array([3, 33, 53], np.int32)), max_q=260, k=own, v=own, out=out)
        assert (out[:3] == 7).all() and (out[53:] == 7).all() and (out[3:53] != 7).any()
    out.fill_(7.0)
    H.kv4_attend_chunk(q, cache, gpu(table), lens, gpu(np.array([3, 33, 53], np.int32)), max_q=20, k=k, v=k, out=out)
    assert (out[:3] == 7).all() and (out[23:33] == 7).all() and (out[53:] == 7).all()
    for cu in ([-1, 5, 70], [5, 5, 4]):  # bounds that lie outside: nothing is written
        out.fill_(7.0)
        H.kv4_attend_chunk(q, cache, gpu(table), lens, gpu(np.array(cu, np.int32)), max_q=20, out=out)
        H.kv4_attend_chunk(q, cache, gpu(wide), lens, gpu(np.array(cu, np.int32)), max_q=260, out=out)
        assert (out == 7).all(), cu


def test_missing_pages_are_not_seen():
    """Pages outside the pool are as if their tokens were not there; none at all gives zeros."""
    torch = torch_cuda()
    rng = np.random.default_rng(10)
    n, nq, D = 500, 40, 64
    planes, table, pages = paged(rng, [n], 1, D)
    cache, lens, cu = tuple(gpu(p) for p in planes), gpu(np.array([n], np.int32)), gpu(np.array([0, nq], np.int32))
    q = bf16(rng.normal(0, 1, (nq, 2, D)))
    k, v = S.held(planes, table[0][np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64)
    t = table.copy()
    t[0, 1], t[0, 3], t[0, 7] = -1, pages, 1 << 30
    wide, max_q = many(t, nq)
    got = values(H.kv4_attend_chunk(q, cache, gpu(wide), lens, cu, max_q=max_q))
    there = ~np.isin(np.arange(n) // 64, (1, 3, 7))
    ok = R.seen(np.arange(nq) + n - nq, n, 0, 0) & there
    for h in range(2):
        assert R.far(got[:, h], *R.attend(values(q)[:, h], k[:, 0], v[:, 0], ok, D ** -0.5), bound(False)) <= 0
    assert (H.kv4_attend_chunk(q, cache, gpu(np.full_like(wide, -1)), lens, cu, max_q=max_q) == 0).all()
    assert (H.kv4_attend_chunk(q, cache, gpu(np.full_like(table, -1)), lens, cu, max_q=nq) == 0).all()
    assert (H.kv4_attend_chunk(q, cache, gpu(table[:, :0]), lens, cu, max_q=nq) == 0).all()


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_finite_stays_with_its_rows(D, own):
    """An infinite value scale (or value) shows as itself or NaN in the rows that see it, and nowhere else; a NaN key
    likewise in whole rows. Short enough for one part, and long enough for several."""
    torch = torch_cuda()
    for n, nq in ((200, 90), (3000, 90)):
        rng = np.random.default_rng(n)
        planes, table, _ = paged(rng, [n], 1, D)
        q = bf16(rng.normal(0, 1, (nq, 2, D)))
        lens, cu = gpu(np.array([n], np.int32)), gpu(np.array([0, nq], np.int32))
        k, v = (bf16(rng.normal(0, 1, (nq, 1, D))) for _ in range(2))
        wide, max_q = many(table, nq)
        run = lambda p, k, v: H.kv4_attend_chunk(q, tuple(gpu(x) for x in p), gpu(wide), lens, cu, max_q=max_q,
                                                 k=k if own else None, v=v if own else None)
        clean = run(planes, k, v)
        assert torch.isfinite(clean).all()
        p = torch.arange(n - nq, n, device="cuda")
        for j in (3, n - nq - 1, n - nq + 17, n - 1):
            sees = p >= j
            if own and j >= n - nq:
                v2, k2 = v.clone(), k.clone()
                v2[j - n + nq, 0, 5], k2[j - n + nq, 0, 9] = float("inf"), float("nan")
                y, z = run(planes, k, v2), run(planes, k2, v)
                dims = torch.arange(D, device="cuda") == 5
            else:
                at = (table[0, j // 64], 0, 0, j % 64)
                a, b = [x.copy() for x in planes], [x.copy() for x in planes]
                a[3][at], b[1][at] = np.inf, np.nan
                y, z = run(a, k, v), run(b, k, v)
                dims = torch.arange(D, device="cuda") < 64
            assert not torch.isfinite(y[sees][..., dims]).any(), (n, j)
            rest = y.clone()
            rest[sees.nonzero()[:, 0][:, None], :, dims.nonzero()[:, 0][None]] = clean[sees.nonzero()[:, 0][:, None], :, dims.nonzero()[:, 0][None]]
            assert torch.equal(rest, clean), (n, j)
            assert z[sees].isnan().all() and torch.equal(z[~sees], clean[~sees]), (n, j)


def test_strides_and_streams():
    torch = torch_cuda()
    rng = np.random.default_rng(12)
    planes, table, _ = paged(rng, [300, 90], 2, 64)
    cache, lens = tuple(gpu(p) for p in planes), gpu(np.array([300, 90], np.int32))
    qkv = bf16(rng.normal(0, 1, (80, 8, 64)))
    q, k, v = qkv.split([4, 2, 2], 1)
    cu = gpu(np.array([0, 30, 80], np.int32))
    want = H.kv4_attend_chunk(q.contiguous(), cache, gpu(table), lens, cu, max_q=50, k=k.contiguous(), v=v.contiguous())
    assert torch.equal(H.kv4_attend_chunk(q, cache, gpu(table), lens, cu, max_q=50, k=k, v=v), want)
    wide = torch.full((2, 9), -5, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + table.shape[1]] = gpu(table)
    assert torch.equal(H.kv4_attend_chunk(q, cache, wide[:, 2:], lens, cu, max_q=50, k=k, v=v), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = H.kv4_attend_chunk(q, cache, gpu(table), lens, cu, max_q=50, k=k, v=v, stream=side)
    side.synchronize()
    assert torch.equal(y, want)
    # without cu_q: as many rows each
    assert torch.equal(H.kv4_attend_chunk(q, cache, gpu(table), lens, max_q=40, k=k, v=v),
                       H.kv4_attend_chunk(q, cache, gpu(table), lens, gpu(np.array([0, 40, 80], np.int32)), max_q=40, k=k, v=v))


def test_captured():
    """Two graphs over the same tensors, replayed in turn over new queries beside eager calls."""
    torch = torch_cuda()
    rng = np.random.default_rng(13)
    planes, table, _ = paged(rng, [2900, 300], 2, 64)
    cache, table, lens = tuple(gpu(p) for p in planes), gpu(table), gpu(np.array([2900, 300], np.int32))
    q, k, v = (bf16(rng.normal(0, 1, (80, h, 64))) for h in (4, 2, 2))
    cu = gpu(np.array([0, 30, 80], np.int32))
    broad = gpu(many(host(table), 0)[0])
    calls = [lambda: H.kv4_attend_chunk(q, cache, broad, lens, cu, max_q=260),
             lambda: H.kv4_attend_chunk(q, cache, table, lens, cu, max_q=50, k=k, v=v, window=700, sinks=4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            c()
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    for c in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(c())
        graphs.append(g)
    for i in range(3):
        q.copy_(bf16(rng.normal(0, 1, (80, 4, 64))))
        lens -= 7
        for g in graphs:
            g.replay()
        for y, c in zip(got, calls):
            assert torch.equal(y, c()), i


@pytest.mark.parametrize("own", [False, True])
def test_many_sequences(own):
    """More sequences than a launch's list holds, most of them short, and (where the table's width bounds their tiles)
    than its scratch memory does."""
    torch_cuda()
    rng = np.random.default_rng(14)
    B = 700 if own else 130
    nqs = rng.integers(0, 4, B).tolist()
    lens = [n + int(x) for n, x in zip(nqs, rng.integers(0, 90, B))]
    check(lens, nqs, 1, 1, 64, own=own, seed=14)


def test_equal_groups():
    """Groups that come out even over the device's workgroups: whole ones, and equal parts."""
    torch_cuda()
    check([900], [300], 2, 8, 64, seed=15)
    check([1300] * 3, [200] * 3, 1, 4, 128, seed=16)


def test_heads_in_several_launches():
    """A table so wide that its scratch memory holds 3 of 4 heads."""
    torch_cuda()
    rng = np.random.default_rng(17)
    n, nq, heads, D = 300, 260, 4, 64
    planes, table, _ = paged(rng, [n], heads, D)
    wide = np.full((1, 50000), -1, np.int32)
    wide[:, :table.shape[1]] = table
    q = bf16(rng.normal(0, 1, (nq, heads, D)).astype(np.float32))
    size = H.serve_lib().glint_kv4_attend_chunk_scratch(1, nq, heads, heads, D, wide.shape[1], 0)
    assert 2 * 50000 * 256 * D < size < 4 * 50000 * 256 * D
    got = values(H.kv4_attend_chunk(q, tuple(gpu(p) for p in planes), gpu(wide), gpu(np.array([n], np.int32)), max_q=nq))
    k, v = S.held(planes, table[0][np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64)
    ok, qf = R.seen(np.arange(nq) + n - nq, n, 0, 0), values(q)
    for h in range(heads):
        worst = R.far(got[:, h], *R.attend(qf[:, h], k[:, h], v[:, h], ok, D ** -0.5), bound(False))
        assert worst <= 0, (h, worst)


def test_two_calls_at_once():
    """Calls on two streams, several in turn, each with scratch memory of its own."""
    torch = torch_cuda()
    rng = np.random.default_rng(18)
    planes, table, _ = paged(rng, [2900, 700], 2, 64)
    cache, lens = tuple(gpu(p) for p in planes), gpu(np.array([2900, 700], np.int32))
    wide, cu = gpu(many(table, 0)[0]), gpu(np.array([0, 300, 420], np.int32))
    qs = [bf16(rng.normal(0, 1, (420, 8, 64))) for _ in range(2)]
    bounds = [{}, {"window": 900, "sinks": 5}]
    want = [H.kv4_attend_chunk(q, cache, wide, lens, cu, max_q=300, **b) for q, b in zip(qs, bounds)]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[] for _ in qs]
    for _ in range(4):
        for i, s in enumerate(streams):
            got[i].append(H.kv4_attend_chunk(qs[i], cache, wide, lens, cu, max_q=300, stream=s, **bounds[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for ys, w in zip(got, want) for y in ys)
