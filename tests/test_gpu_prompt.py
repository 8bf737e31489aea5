"""Causal attention over packed prompts on the GPU, within the bound derived from its roundings."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu

pytestmark = pytest.mark.gpu


def values(t):
    return S.bf16_values(host(t)).reshape(t.shape).astype(np.float64)


def check(nq, nk, heads, G, D, seed=0, scale=None, k_size=1.0, max_q=None):
    rng = np.random.default_rng(seed)
    cq, ck = (np.concatenate([[0], np.cumsum(n)]).astype(np.int32) for n in (nq, nk))
    q = bf16(rng.normal(0, 1, (cq[-1], heads * G, D)).astype(np.float32))
    k = bf16((rng.normal(0, 1, (ck[-1], heads, D)) * k_size).astype(np.float32))
    v = bf16(rng.normal(0, 1, (ck[-1], heads, D)).astype(np.float32))
    got = values(H.attend_prompt(q, k, v, gpu(cq), gpu(ck), max_q=max_q or max(nq), scale=scale))
    qf, kf, vf = values(q), values(k), values(v)
    sc = D ** -0.5 if scale is None else scale
    for b in range(len(nq)):
        for h in range(heads * G):
            rows, keys = slice(cq[b], cq[b + 1]), slice(ck[b], ck[b + 1])
            last = np.arange(nq[b]) + nk[b] - nq[b]
            out, mass, size = S.attend(qf[rows, h], kf[keys, h // G], vf[keys, h // G], last, sc)
            far = np.abs(got[rows, h] - out) - S.prompt_bound(out, mass, size)
            assert far.size == 0 or (far <= 0).all(), (b, h, float(far.max()))
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 31, 33, 64, 65, 127, 129, 300])
def test_one_sequence(D, n):
    torch_cuda()
    print(f"prompt D={D} n={n}", flush=True)
    check([n], [n], 2, 3, D, seed=n)


@pytest.mark.parametrize("D,heads,G", [(64, 3, 1), (128, 1, 8), (128, 2, 5)])
def test_packed_lengths(D, heads, G):
    """Sequences of 0, 1 and more tokens; some after keys they already have, one with no key at all, one with
    more queries than keys."""
    torch_cuda()
    print(f"packed D={D} H={heads} G={G}", flush=True)
    nq = [5, 0, 130, 1, 64, 9, 7, 200]
    nk = [5, 3, 330, 129, 64, 0, 4, 200]
    check(nq, nk, heads, G, D, seed=D + G)


def test_long_and_peaked():
    """A long sequence, scores so large that one key takes all, and a maximum that moves tile after tile."""
    torch_cuda()
    check([1100], [1100], 1, 2, 128, seed=3)
    check([400], [400], 1, 2, 64, seed=4, k_size=40.0)
    check([200], [500], 1, 1, 128, seed=5, scale=-0.3)


def test_max_q_may_be_larger():
    torch_cuda()
    check([33, 70], [33, 70], 1, 2, 64, seed=6, max_q=1000)


def test_strides_and_streams():
    torch = torch_cuda()
    rng = np.random.default_rng(7)
    T, heads, G, D = 150, 2, 3, 64
    qkv = bf16(rng.normal(0, 1, (T, (G + 2) * heads * D)).astype(np.float32))
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([G * heads * D, heads * D, heads * D], 1))
    cu = gpu(np.array([0, 50, 150], np.int32))
    want = H.attend_prompt(q.contiguous(), k.contiguous(), v.contiguous(), cu, max_q=100)
    assert torch.equal(H.attend_prompt(q, k, v, cu, max_q=100), want)
    assert torch.equal(H.attend_prompt(q, k, v, cu), want)
    shift = torch.cat([k.new_zeros(1), k.flatten()])[1:].view(k.shape)  # not 16-B aligned
    assert torch.equal(H.attend_prompt(q, shift, v, cu), want)
    turned = v.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    assert torch.equal(H.attend_prompt(q, k, turned, cu), want)
    one = H.attend_prompt(q, k[:, :1].expand(T, heads, D), v, cu)
    assert torch.equal(one, H.attend_prompt(q, k[:, :1].expand(T, heads, D).contiguous(), v, cu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = H.attend_prompt(q, k, v, cu, stream=side)
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("D", [64, 128])
def test_what_a_row_does_not_see(D):
    """NaN and infinities in keys and values past a row's last change nothing for it; a row that sees
    an infinite or NaN value shows it in that dimension alone."""
    torch = torch_cuda()
    rng = np.random.default_rng(9)
    n = 200
    q, k, v = (bf16(rng.normal(0, 1, (n, 2, D)).astype(np.float32)) for _ in range(3))
    cu = gpu(np.array([0, n], np.int32))
    clean = values(H.attend_prompt(q, k, v, cu))
    for at in (199, 150, 64, 63, 5):
        for value in (float("nan"), float("inf"), float("-inf")):
            v2, k2 = v.clone(), k.clone()
            v2[at, 1, 37] = value
            v2[at, 1, D - 1] = value
            got = values(H.attend_prompt(q, k, v2, cu))
            same = np.ones_like(got, bool)
            same[at:, 1, 37] = same[at:, 1, D - 1] = False
            assert np.array_equal(got[same], clean[same]), (at, value)
            assert not np.isfinite(got[~same]).any()
            if value != value:
                assert np.isnan(got[~same]).all()
            else:
                assert (got[~same] == value).all(), (at, value)
            k2[at, 0, 3] = value
            got = values(H.attend_prompt(q, k2, v, cu))
            assert np.array_equal(got[:at], clean[:at]) and np.array_equal(got[:, 1], clean[:, 1]), (at, value)


def test_rows_outside_the_sequences_stay():
    torch = torch_cuda()
    rng = np.random.default_rng(8)
    q = bf16(rng.normal(0, 1, (40, 2, 64)).astype(np.float32))
    out = torch.full_like(q, 5.0)
    H.attend_prompt(q, q[:, :1], q[:, 1:], gpu(np.array([4, 20], np.int32)), gpu(np.array([0, 16], np.int32)), out=out)
    assert (out[:4] == 5).all() and (out[20:] == 5).all() and not (out[4:20] == 5).any()
