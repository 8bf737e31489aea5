"""Rotated queries and keys on the GPU: within the bound of f32 arithmetic, and into the cache bit for bit."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import bounded_util as R
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu, planes_of

pytestmark = pytest.mark.gpu


def rows(rng, T, heads, D, dtype):
    """[T, heads, D] on the GPU and its f64 values."""
    x = (rng.normal(0, 1, (T, heads, D)) * rng.choice([1.0, 30.0, 1e-3], (T, heads, 1))).astype(np.float32)
    t = gpu(x) if dtype == "f32" else bf16(x)
    return t, values(t)


def values(t):
    import torch
    return t.double().cpu().numpy() if t.dtype != torch.bfloat16 else S.bf16_values(host(t)).reshape(t.shape).astype(np.float64)


def check(got, want, off, dtype):
    rounding = 2.0 ** -8 * np.abs(want) if dtype == "bf16" else 2.0 ** -24 * np.abs(want)
    d = np.abs(values(got) - want) - rounding - off - 2.0 ** -133
    assert (d <= 0).all(), float(d.max())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,heads,D,rot,norm,dtype", [
    (1, 1, 1, 64, 64, False, "bf16"), (8, 32, 8, 128, 128, True, "bf16"), (3, 5, 2, 128, 32, True, "f32"), (17, 7, 1, 80, 48, True, "bf16"),
    (5, 3, 3, 96, 96, False, "f32"), (2, 4, 1, 16, 16, True, "bf16"), (70, 2, 1, 256, 64, True, "f32"), (2300, 9, 3, 64, 32, True, "bf16"),
    (2100, 3, 2, 240, 240, True, "bf16")])
def test_rotate(T, Hq, heads, D, rot, norm, dtype, interleaved):
    torch_cuda()
    print(f"rotate T={T} Hq={Hq} H={heads} D={D} rot={rot} norm={norm} {dtype} interleaved={interleaved}", flush=True)
    rng = np.random.default_rng(T + D)
    (q, qf), (k, kf) = rows(rng, T, Hq, D, dtype), rows(rng, T, heads, D, dtype)
    pos = rng.integers(0, 100000, T)
    pos[0] = 0
    freqs = H.rotary_freqs(rot, base=500000.0, factor=8.0, trained=8192)
    qn = kn = None
    if norm:
        qn, kn = (gpu(rng.normal(1, 0.3, D).astype(np.float32)) for _ in range(2))
        if D == 128:
            qn, kn = qn.bfloat16(), kn.bfloat16()
    gq, gk = H.rotate_qk(q, k, gpu(pos), freqs, interleaved=interleaved, magnitude=1.2, q_norm=qn, k_norm=kn, eps=1e-5)
    fr = freqs.cpu().numpy()
    for got, x, w in ((gq, qf, qn), (gk, kf, kn)):
        want, off = R.turned(x, pos, fr, interleaved, 1.2, None if w is None else values(w), float(np.float32(1e-5)))
        check(got, want, off, dtype)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_root_is_rounded_once(D):
    """Small whole numbers, whose mean square is exact: a row of f32 holds its elements times the nearest f32 to the root's inverse."""
    torch = torch_cuda()
    rng = np.random.default_rng(D)
    x = rng.integers(-9, 10, (3000, 5, D)).astype(np.float32)
    x[:, :, 0] = 1
    x[0] = 0
    eps = np.float32(2.0 ** -12)  # exact beside a mean of up to 81 in steps of 1 / D
    one = torch.ones(D, device="cuda")
    got, _ = H.rotate_qk(gpu(x), gpu(x), gpu(np.zeros(3000, np.int64)), torch.zeros(D // 2, dtype=torch.float64, device="cuda"),
                         q_norm=one, k_norm=one, eps=float(eps))
    r = (1 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + float(eps))).astype(np.float32)
    assert np.array_equal(got.cpu().numpy(), x * r)


def test_far_and_negative_positions():
    """Angles of positions up to 2^40 and below 0, and of any frequency."""
    torch_cuda()
    rng = np.random.default_rng(2)
    pos = np.array([0, 1, -1, 2 ** 20 + 1, -(2 ** 31) - 7, 2 ** 40 + 3, 123456789, 2 ** 31 - 1])
    (q, qf), (k, kf) = rows(rng, 8, 2, 64, "f32"), rows(rng, 8, 1, 64, "f32")
    fr = np.concatenate([rng.uniform(0, 7, 16), np.geomspace(1e-9, 100, 15), [0.0]])
    for got, x in zip(H.rotate_qk(q, k, gpu(pos), gpu(fr)), (qf, kf)):
        want, off = R.turned(x, pos, fr)
        check(got, want, off, "f32")


def test_strides_in_place_and_special_values():
    torch = torch_cuda()
    rng = np.random.default_rng(3)
    qkv, _ = rows(rng, 33, 12, 128, "bf16")
    freqs, pos = H.rotary_freqs(64), torch.arange(33, device="cuda")
    q, k = qkv[:, :8], qkv[:, 8:10]
    want = H.rotate_qk(q.contiguous(), k.contiguous(), pos, freqs)
    for a, b in zip(H.rotate_qk(q, k, pos, freqs), want):
        assert torch.equal(a, b)
    odd = torch.empty(33 * 8 * 128 + 8, dtype=torch.bfloat16, device="cuda")[3:3 + 33 * 8 * 128].view(33, 8, 128).copy_(q)
    assert torch.equal(H.rotate_qk(odd, k, pos, freqs)[0], want[0])
    a, b = q.contiguous(), k.contiguous()
    ga, gb = H.rotate_qk(a, b, pos, freqs, out=(a, b))
    assert ga is a and torch.equal(a, want[0]) and torch.equal(b, want[1])
    # what is not turned keeps its bits beside NaN and infinities; a NaN spoils its own pair alone
    x = q.contiguous()
    x[0, 0, 3], x[1, 1, 70], x[2, 2, 127] = float("nan"), float("inf"), float("-inf")
    y = H.rotate_qk(x, k, pos + 1, freqs)[0]
    assert torch.equal(y[..., 64:].view(torch.int16), x[..., 64:].view(torch.int16))
    spoilt = ~torch.isfinite(y[..., :64])
    assert spoilt.nonzero().tolist() == [[0, 0, 3], [0, 0, 35]]
    empty = H.rotate_qk(q[:0], k[:0], pos[:0], freqs)
    assert empty[0].shape == (0, 8, 128) and empty[1].shape == (0, 2, 128)


@pytest.mark.parametrize("T,Hq,heads,D,rot,norm,dtype,interleaved", [
    (1, 4, 1, 64, 64, False, "bf16", False), (9, 32, 8, 128, 128, True, "bf16", False), (40, 6, 2, 128, 64, False, "f32", True),
    (33, 2, 200, 64, 32, True, "bf16", False), (2500, 4, 3, 128, 128, True, "bf16", False), (700, 9, 9, 64, 64, True, "f32", True)])
def test_append_rotated_is_rotate_then_append(T, Hq, heads, D, rot, norm, dtype, interleaved):
    """The turned queries and keys, and every byte of the cache, those of skipped and of other places too."""
    torch = torch_cuda()
    print(f"append rotated T={T} Hq={Hq} H={heads} D={D} rot={rot} norm={norm} {dtype}", flush=True)
    rng = np.random.default_rng(T)
    qkv, _ = rows(rng, T, Hq + 2 * heads, D, dtype)
    qkv[T // 2, Hq, 5], qkv[0, -1, :64] = float("inf"), 0
    qkv[T // 3, -1, 7] = float("nan")
    q, k, v = qkv.split([Hq, heads, heads], 1)
    pages = T // 64 + 3
    slots = np.arange(T, dtype=np.int64) + 5
    slots[T // 3:T // 3 + 9] = rng.permutation(slots[T // 3:T // 3 + 9])
    if T > 4:
        slots[T // 2], slots[T // 4] = -1, pages * 64
    slots = gpu(slots)
    pos, freqs = gpu(rng.integers(0, 5000, T)), H.rotary_freqs(rot)
    how = dict(interleaved=interleaved, magnitude=0.75)
    if norm:
        how["q_norm"], how["k_norm"] = (gpu(rng.normal(1, 0.3, D).astype(np.float32)) for _ in range(2))
    start = S.empty_planes(pages, heads, D, fill=0x5A)
    want, got, alone = (tuple(gpu(p) for p in start) for _ in range(3))
    wq, wk = H.rotate_qk(q, k, pos, freqs, **how)
    H.kv4_append(wk, v, slots, want)
    gq, gk = H.kv4_append_rotated(q, k, v, pos, freqs, slots, got, keys=True, **how)
    bits = torch.int16 if dtype == "bf16" else torch.int32
    assert torch.equal(gq.view(bits), wq.view(bits)) and torch.equal(gk.view(bits), wk.view(bits))
    aq = H.kv4_append_rotated(q, k, v, pos, freqs, slots, alone, **how)
    assert torch.equal(aq.view(bits), wq.view(bits))
    for a, b, w, name in zip(planes_of(got), planes_of(alone), planes_of(want), ("k_hole", "k_absmax", "v_hole", "v_absmax")):
        assert a.tobytes() == w.tobytes() and b.tobytes() == w.tobytes(), name


def test_captured_and_on_another_stream():
    torch = torch_cuda()
    rng = np.random.default_rng(8)
    qkv, _ = rows(rng, 6, 10, 64, "bf16")
    pos, slots, freqs = torch.arange(6, device="cuda"), torch.arange(6, device="cuda"), H.rotary_freqs(64)
    cache, other = H.kv4_cache(2, 2, 64), H.kv4_cache(2, 2, 64)
    call = lambda c: H.kv4_append_rotated(qkv[:, :6], qkv[:, 6:8], qkv[:, 8:], pos, freqs, slots, c)
    call(other)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(cache)
    for i in range(3):
        qkv.copy_(rows(rng, 6, 10, 64, "bf16")[0])
        pos += 3
        graph.replay()
        want = call(other)
        assert torch.equal(y, want), i
        for a, b in zip(cache, other):
            assert torch.equal(a, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    z = H.rotate_qk(qkv[:, :6], qkv[:, 6:8], pos, freqs, stream=s)
    s.synchronize()
    assert torch.equal(z[0], want)
