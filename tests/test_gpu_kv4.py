"""The 4-bit key/value cache on the GPU: append and gather bit for bit, attention within its derived bound."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.gpu_util import bf16_bits, host, torch_cuda

pytestmark = pytest.mark.gpu


def gpu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def bf16(a):
    import torch
    return gpu(bf16_bits(a).view(np.int16).reshape(a.shape)).view(torch.bfloat16)


def planes_of(cache):
    return [host(t) for t in cache]


def random_planes(rng, pages, heads, D, low=0.5, high=3.0):
    p = S.empty_planes(pages, heads, D)
    for i in (0, 2):
        c = np.clip(np.round(rng.normal(7.3, 3.2, p[i].shape + (2,))), 0, 15).astype(np.uint8)
        p[i] = c[..., 0] | c[..., 1] << 4
    for i in (1, 3):
        p[i] = rng.uniform(low, high, p[i].shape).astype(np.float32)
    return p


# ------------------------------------------------------------------ append, gather
@pytest.mark.parametrize("T,heads,D,dtype", [(1, 1, 64, "bf16"), (3, 2, 128, "f32"), (65, 5, 64, "f32"), (130, 3, 128, "bf16"),
                                             (200, 8, 128, "bf16")])
def test_append_and_gather(T, heads, D, dtype):
    torch = torch_cuda()
    print(f"append T={T} H={heads} D={D} {dtype}", flush=True)
    rng = np.random.default_rng(T)
    k, v = rng.normal(0, 1, (2, T, heads, D)).astype(np.float32)
    k *= np.where(rng.random(D) < 0.1, 20, 1).astype(np.float32)
    k[0, 0, :64] = 0  # absmax 0
    v[-1, -1, 3], v[-1, -1, 7] = np.nan, -np.nan
    k[T // 2, 0, 5] = np.inf
    v[T // 2, 0, :64] = 1e-41  # subnormal
    if dtype == "bf16":
        kb, vb = bf16(k), bf16(v)
        k, v = S.bf16_values(host(kb)).reshape(k.shape), S.bf16_values(host(vb)).reshape(v.shape)
    else:
        kb, vb = gpu(k), gpu(v)
    pages = T // 64 + 3
    slots = rng.permutation(pages * 64)[:T].astype(np.int64)
    slots[T // 3] = -1 if T > 2 else slots[T // 3]
    if T > 10:
        slots[T // 4] = pages * 64  # past the pool: skipped as well
    want = S.empty_planes(pages, heads, D, fill=0x5A)
    cache = tuple(gpu(p) for p in want)
    for t in range(T):
        if 0 <= slots[t] < pages * 64:
            S.put(want, slots[t], k[t], v[t])
    H.kv4_append(kb, vb, gpu(slots), cache)
    for got, w, name in zip(planes_of(cache), want, ("k_hole", "k_absmax", "v_hole", "v_absmax")):
        assert got.tobytes() == w.tobytes(), name
    gk, gv = H.kv4_gather(gpu(slots), cache)
    ok = (slots >= 0) & (slots < pages * 64)
    with np.errstate(all="ignore"):
        for got, w in zip((gk, gv), S.held(want, np.where(ok, slots, 0))):
            w = np.where(ok[:, None, None], w, 0).astype(np.float32)
            assert np.array_equal(S.bf16_values(host(got)).reshape(w.shape), S.bf16_values(bf16_bits(w)).reshape(w.shape),
                                  equal_nan=True)


def test_append_in_a_row_fills_whole_pages():
    """A prompt's tokens in a row, starting inside a page, in an order of pages that is not theirs."""
    torch_cuda()
    rng = np.random.default_rng(5)
    T, heads, D, pages = 300, 4, 128, 7
    k, v = rng.normal(0, 1, (2, T, heads, D)).astype(np.float32)
    order = rng.permutation(pages)
    at = np.arange(T) + 37
    slots = order[at // 64] * 64 + at % 64
    want = S.empty_planes(pages, heads, D)
    cache = tuple(gpu(p) for p in want)
    for t in range(T):
        S.put(want, slots[t], k[t], v[t])
    H.kv4_append(gpu(k), gpu(v), gpu(slots), cache)
    for got, w in zip(planes_of(cache), want):
        assert got.tobytes() == w.tobytes()


@pytest.mark.parametrize("T,heads,D,dtype", [(33, 311, 64, "f32"), (64, 256, 128, "bf16"), (130, 127, 64, "bf16"), (700, 24, 128, "f32")])
def test_append_and_gather_in_tiles(T, heads, D, dtype):
    """Enough tokens of one head for the launches by tiles: runs of slots that start at every place modulo 4,
    single slots, tokens that are skipped, tiles that are not whole, special values."""
    torch_cuda()
    print(f"append T={T} H={heads} D={D} {dtype}", flush=True)
    rng = np.random.default_rng(T)
    k, v = rng.normal(0, 1, (2, T, heads, D)).astype(np.float32)
    k[0, 0, :64] = 0
    v[-1, -1, 3], v[-1, -1, 7], k[T // 2, 0, 5] = np.nan, -np.nan, np.inf
    v[T // 2, 0, :64] = 1e-41
    v[T // 2, 1] *= 1e30
    if dtype == "bf16":
        kb, vb = bf16(k), bf16(v)
        k, v = S.bf16_values(host(kb)).reshape(k.shape), S.bf16_values(host(vb)).reshape(v.shape)
    else:
        kb, vb = gpu(k), gpu(v)
    pages = T // 64 + 3
    for first in (0, 1, 3, 64, 66):
        slots = np.arange(T, dtype=np.int64) + first
        slots[T // 3:T // 3 + 9] = rng.permutation(slots[T // 3:T // 3 + 9])
        slots[T // 2], slots[T // 4] = -1, pages * 64
        want = S.empty_planes(pages, heads, D, fill=0x5A)
        cache = tuple(gpu(p) for p in want)
        ok = (slots >= 0) & (slots < pages * 64)
        S.put_all(want, slots[ok], k[ok], v[ok])
        H.kv4_append(kb, vb, gpu(slots), cache)
        for got, w, name in zip(planes_of(cache), want, ("k_hole", "k_absmax", "v_hole", "v_absmax")):
            assert got.tobytes() == w.tobytes(), (name, first)
        some = np.concatenate([slots, rng.permutation(slots)[:17], [pages * 64 - 1]])
        ok = (some >= 0) & (some < pages * 64)
        with np.errstate(all="ignore"):
            for got, w in zip(H.kv4_gather(gpu(some), cache), S.held(want, np.where(ok, some, 0))):
                w = np.where(ok[:, None, None], w, 0).astype(np.float32)
                assert np.array_equal(S.bf16_values(host(got)).reshape(w.shape),
                                      S.bf16_values(bf16_bits(w)).reshape(w.shape), equal_nan=True), first


@pytest.mark.parametrize("T", [8, 64, 5120])
def test_append_at_the_edges(T):
    """Quotients at and one float beside every edge between two codes, under an absmax of 1 (5120 tokens of
    2 heads are appended by tiles)."""
    torch_cuda()
    edges = ((S.PARENT[1:].astype(np.float64) + S.PARENT[:-1]) / 2).astype(np.float32)
    near = (edges.view(np.int32)[:, None] + np.arange(-2, 3)).astype(np.int32).view(np.float32).ravel()
    rows = np.concatenate([near, S.PARENT, [0.0, -0.0, 0.5 / 16, 1.5 / 16, -2.5 / 16]]).astype(np.float32)
    rows = np.resize(rows, T * 2 * 63).reshape(T, 2, 63)
    k = np.concatenate([rows, np.ones((T, 2, 1), np.float32)], -1)
    v = np.concatenate([-np.ones((T, 2, 1), np.float32), rows[::-1]], -1)
    want = S.empty_planes(T // 64 + 2, 2, 64)
    cache = tuple(gpu(p) for p in want)
    S.put_all(want, np.arange(T) + 3, k, v)
    H.kv4_append(gpu(k), gpu(v), gpu(np.arange(T, dtype=np.int64) + 3), cache)
    for got, w, name in zip(planes_of(cache), want, ("k_hole", "k_absmax", "v_hole", "v_absmax")):
        assert got.tobytes() == w.tobytes(), name


def test_append_takes_strided_rows():
    """k and v as slices of one projection's output, an odd offset among them, and one head for all."""
    torch = torch_cuda()
    rng = np.random.default_rng(6)
    T, heads, D = 9, 2, 64
    slots = gpu(np.arange(T, dtype=np.int64) * 5)
    qkv = bf16(rng.normal(0, 1, (T, 4 * heads * D + 3)).astype(np.float32))
    for off in (0, 2 * heads * D, 3):
        k = qkv[:, off:off + heads * D].view(T, heads, D) if off != 3 else qkv[:, 3:3 + heads * D].unflatten(1, (heads, D))
        v = qkv[:, heads * D:heads * D + D].unflatten(1, (1, D)).expand(T, heads, D)
        a, b = H.kv4_cache(1, heads, D), H.kv4_cache(1, heads, D)
        H.kv4_append(k, v, slots, a)
        H.kv4_append(k.contiguous(), v.contiguous(), slots, b)
        assert all(torch.equal(x, y) for x, y in zip(a, b)), off


# ------------------------------------------------------------------ attention
def check(q, planes, table, lens, nqs, G, D, scale=None, max_q=None, cu=True, shape=None):
    """Runs the kernel on packed rows and compares every row with the definition in 64 bits."""
    heads = planes[0].shape[1]
    scale = D ** -0.5 if scale is None else scale
    starts = np.concatenate([[0], np.cumsum(nqs)]).astype(np.int32)
    qb = bf16(q)
    q = S.bf16_values(host(qb)).reshape(q.shape).astype(np.float64)
    cache = tuple(gpu(p) for p in planes)
    got = H.kv4_attend(qb, cache, gpu(np.asarray(table, np.int32)), gpu(np.asarray(lens, np.int32)),
                       cu_q=gpu(starts) if cu else None, max_q=max_q or max(nqs), scale=scale)
    got = S.bf16_values(host(got)).reshape(q.shape).astype(np.float64)
    pages = planes[0].shape[0]
    for b, n in enumerate(lens):
        n = min(max(n, 0), len(table[b]) * 64)
        slots, pos = [], []
        for t in range(n):
            if 0 <= table[b][t // 64] < pages:
                slots.append(table[b][t // 64] * 64 + t % 64)
                pos.append(t)
        k, v = S.held(planes, slots)
        for h in range(heads * G):
            rows = slice(starts[b], starts[b + 1])
            last = [np.searchsorted(pos, n - nqs[b] + i, side="right") - 1 for i in range(nqs[b])]
            out, mass, size = S.attend(q[rows, h], k[:, h // G], v[:, h // G], last, scale)
            far = np.abs(got[rows, h] - out) - S.kv4_bound(out, mass, size)
            assert (far <= 0).all(), (b, h, float(far.max()))
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads,G", [(1, 1), (2, 4), (3, 5), (1, 16), (2, 20)])
def test_attend_single_tokens(D, heads, G):
    torch_cuda()
    lens = [0, 1, 63, 64, 65, 130, 700, 2]
    print(f"attend D={D} H={heads} G={G}", flush=True)
    rng = np.random.default_rng(D + G)
    wide = 11
    planes = random_planes(rng, 8 * wide + 2, heads, D)
    table = rng.permutation(8 * wide + 2)[:8 * wide].reshape(8, wide)
    got = check(rng.normal(0, 1, (8, heads * G, D)).astype(np.float32), planes, table, lens, [1] * 8, G, D, cu=False)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("D,G,nqs", [(64, 4, [3, 0, 5, 1]), (128, 8, [4, 4, 4, 4]), (128, 3, [7, 2, 1, 6]), (64, 1, [40, 17, 0, 33])])
def test_attend_several_tokens(D, G, nqs):
    """New tokens see each other causally; a sequence with fewer tokens than rows leaves rows empty."""
    torch_cuda()
    rng = np.random.default_rng(D + G)
    lens = [200, 64, 3, 129]
    planes = random_planes(rng, 20, 2, D)
    table = rng.permutation(20)[:16].reshape(4, 4)
    print(f"attend D={D} G={G} nq={nqs}", flush=True)
    check(rng.normal(0, 1, (sum(nqs), 2 * G, D)).astype(np.float32), planes, table, lens, nqs, G, D)


def test_attend_long_split_context():
    torch_cuda()
    rng = np.random.default_rng(9)
    planes = random_planes(rng, 160, 1, 128)
    check(rng.normal(0, 2, (1, 4, 128)).astype(np.float32), planes, rng.permutation(160)[:150].reshape(1, 150), [9555], [1], 4, 128)


def test_attend_pages_that_are_not_there():
    """Entries outside the pool are not seen, nor is what a length past the table would name."""
    torch_cuda()
    rng = np.random.default_rng(10)
    planes = random_planes(rng, 6, 2, 64)
    table = np.array([[3, -1, 2, 99], [0, 1, -7, 6], [-1, -1, -1, -1]])
    check(rng.normal(0, 1, (3, 2, 64)).astype(np.float32), planes, table, [250, 1000, 60], [1, 1, 1], 1, 64)


def test_attend_scales_of_every_size():
    """Value scales from 1e-30 to 1e30 in one sequence, growing and falling, zero ones, key scales that
    make one token win, and queries far from 1."""
    torch_cuda()
    rng = np.random.default_rng(11)
    for grow in (1, -1):
        planes = random_planes(rng, 10, 1, 128)
        planes[3][:] = (10.0 ** (grow * np.linspace(-30, 30, 10)))[:, None, None, None] * rng.uniform(0.5, 1, planes[3].shape)
        planes[3][4] = 0
        check(rng.normal(0, 1, (1, 3, 128)).astype(np.float32), planes, np.arange(10)[None], [640], [1], 3, 128)
    planes = random_planes(rng, 4, 1, 64)
    planes[1][2, 0, 0, 17] = 300.0
    for size in (1e-20, 1e-3, 30.0, 1e18):
        q = (rng.normal(0, 1, (1, 2, 64)) * size).astype(np.float32)
        check(q, planes, np.arange(4)[None], [256], [1], 2, 64, scale=0.1 / size)
    check(np.zeros((1, 2, 64), np.float32), planes, np.arange(4)[None], [256], [1], 2, 64)


def test_attend_ignores_what_it_does_not_see():
    """NaN and inf scales past a row's last position change nothing; one it sees shows."""
    torch = torch_cuda()
    rng = np.random.default_rng(12)
    planes = random_planes(rng, 3, 1, 128)
    q = bf16(rng.normal(0, 1, (3, 2, 128)).astype(np.float32))
    table, cu = gpu(np.array([[2, 0, 1]], np.int32)), gpu(np.array([0, 3], np.int32))
    run = lambda n: host(H.kv4_attend(q, tuple(gpu(p) for p in planes), table, gpu(np.array([n], np.int32)), cu_q=cu, max_q=3))
    clean = run(100)
    for plane in (1, 3):
        for value in (np.nan, np.inf):
            keep = planes[plane].copy()
            planes[plane][0, 0, :, 36:] = value  # positions 100 on
            planes[plane][1] = value
            assert np.array_equal(run(100), clean), (plane, value)
            planes[plane][0, 0, :, 35] = value  # position 99: the last row's alone
            got = run(100)
            assert np.array_equal(got[:2], clean[:2]), (plane, value)
            assert not np.isfinite(S.bf16_values(got[2])).all()
            planes[plane] = keep


def test_attend_strides_streams_and_graphs():
    torch = torch_cuda()
    rng = np.random.default_rng(13)
    B, heads, G, D = 5, 2, 4, 128
    planes = tuple(gpu(p) for p in random_planes(rng, 200, heads, D))
    wide = gpu(np.arange(200, dtype=np.int32).reshape(B, 40))
    lens = gpu(np.array([2500, 17, 0, 1300, 64], np.int32))
    qkv = bf16(rng.normal(0, 1, (B, 3 * heads * G * D + 8)).astype(np.float32))
    q = qkv[:, 8:8 + heads * G * D].unflatten(1, (heads * G, D))
    want = H.kv4_attend(q.contiguous(), planes, wide, lens)
    assert torch.equal(H.kv4_attend(q, planes, wide, lens), want)
    odd = torch.cat([q.flatten(), q.flatten()[:1]])[1:]  # one element on: rows that are not 16-B aligned
    odd = torch.as_strided(torch.cat([q.new_zeros(1), q.flatten()]), q.shape, q.contiguous().stride(), 1)
    assert torch.equal(H.kv4_attend(odd, planes, wide, lens), want)
    pad = torch.full((B, 60), -1, dtype=torch.int32, device="cuda")
    pad[:, :40] = wide
    assert torch.equal(H.kv4_attend(q, planes, pad[:, :40], lens), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = H.kv4_attend(q, planes, wide, lens, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        H.kv4_attend(q, planes, wide, lens, out=out)
    for i in range(4):
        out.fill_(7.0)
        if i == 2:
            lens.copy_(lens.flip(0))
            want = H.kv4_attend(q, planes, wide, lens)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_attend_runs_repeat():
    """The same call gives the same bits."""
    torch = torch_cuda()
    rng = np.random.default_rng(14)
    planes = tuple(gpu(p) for p in random_planes(rng, 100, 2, 64))
    q = bf16(rng.normal(0, 1, (2, 8, 64)).astype(np.float32))
    table, lens = gpu(np.arange(100, dtype=np.int32).reshape(2, 50)), gpu(np.array([3200, 1999], np.int32))
    first = H.kv4_attend(q, planes, table, lens)
    for _ in range(5):
        assert torch.equal(H.kv4_attend(q, planes, table, lens), first)
