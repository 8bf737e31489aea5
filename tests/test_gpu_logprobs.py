"""Token log probabilities on the GPU: whole numbers exactly, f32 sums within their derived bound."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu

pytestmark = pytest.mark.gpu


def check(x, tok, top, f32, stride=None):
    torch = torch_cuda()
    t = gpu(x.astype(np.float32)) if f32 else bf16(x.astype(np.float32))
    if stride:
        wide = t.new_full((x.shape[0], stride), float("nan"))
        wide[:, 1:1 + x.shape[1]] = t
        t = wide[:, 1:1 + x.shape[1]]
    vals = host(t.contiguous()) if f32 else S.bf16_values(host(t.contiguous())).reshape(x.shape)
    r = {k: host(v) for k, v in H.token_logprobs(t, gpu(np.asarray(tok, np.int64)), top=top).items()}
    for i, k in enumerate(tok):
        lse, lp, ent, rank, order, off = S.logprobs(vals[i], k, top)
        assert r["rank"][i] == rank, (i, r["rank"][i], rank)
        assert lp == r["logprob"][i] or abs(r["logprob"][i] - lp) <= off + 2.0 ** -22 * abs(lp), (i, lp, r["logprob"][i])
        assert abs(r["entropy"][i] - ent) <= 4 * off, (i, ent, r["entropy"][i], off)
        assert np.array_equal(r["top_index"][i], order), (i, r["top_index"][i], order)
        want = vals[i][order].astype(np.float64) - lse
        assert all(a == b or abs(a - b) <= off + 2.0 ** -22 * abs(b) for a, b in zip(r["top_logprob"][i], want)), i


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V,top", [(1, 1), (2, 2), (7, 5), (63, 20), (500, 20), (1025, 0), (8191, 3), (8193, 20), (32003, 5),
                                   (128256, 20), (262144, 20)])
def test_rows(V, top, f32):
    torch_cuda()
    print(f"logprobs V={V} top={top} f32={f32}", flush=True)
    rng = np.random.default_rng(V + top)
    x = rng.normal(0, 3, (5, V))
    tok = rng.integers(0, V, 5)
    tok[0], tok[1], tok[2] = 0, V - 1, x[2].argmax()
    check(x, tok, top, f32)


@pytest.mark.parametrize("f32", [False, True])
def test_ties_masks_and_peaks(f32):
    torch_cuda()
    rng = np.random.default_rng(1)
    V = 5000
    x = rng.integers(-3, 4, (8, V)).astype(np.float64)  # many equal entries
    x[1] = 2.5  # all equal
    x[2] = -np.inf
    x[2, 77] = -4.0  # one entry allowed
    x[3, rng.random(V) < 0.999] = -np.inf
    x[3, 10] = 1
    x[4, 3000] = 500.0  # the rest underflows
    x[5] = np.linspace(-1e4, 1e4, V)
    x[6] = -np.abs(x[6]) * 0.0  # -0 and 0 are equal
    x[6, ::2] = 0.0
    x[7] *= 1e-30
    check(x, [17, 4999, 77, 10, 2999, 0, 2500, 3], 20, f32)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("V,top", [(3, 2), (1001, 20), (40007, 20)])
def test_rows_at_any_offset(V, top, f32):
    """Rows that start at every place inside 16 B, in a wider tensor whose other entries are NaN."""
    torch_cuda()
    rng = np.random.default_rng(V)
    check(rng.normal(0, 2, (9, V)), rng.integers(0, V, 9), top, f32, stride=V + 2 + (V % 2))


def test_the_largest_in_one_place():
    """All of the largest entries where one thread reads them."""
    torch_cuda()
    rng = np.random.default_rng(3)
    x = rng.normal(0, 1, (2, 131072))
    x[0, 1600:1608] += 50
    x[0, 1600 + 8192:1608 + 8192] += 60
    x[0, 1600 + 16384:1608 + 16384] += 70
    x[1, -3:] += 99
    check(x, [1600, 131071], 20, False)


def test_special_rows_and_tokens():
    torch = torch_cuda()
    x = torch.randn(6, 1000, device="cuda")
    x[1, 5] = float("nan")
    x[2, 999] = float("inf")
    x[3] = float("-inf")
    tok = gpu(np.array([-1, 4, 4, 4, 1000, -100], np.int64))
    r = {k: host(v) for k, v in H.token_logprobs(x, tok, top=3).items()}
    assert r["logprob"][0] == 0 and r["logprob"][5] == 0 and r["rank"][0] == r["rank"][5] == r["rank"][4] == -1
    assert np.isnan(r["logprob"][[1, 2, 3, 4]]).all()
    assert np.isnan(r["entropy"][[1, 2, 3]]).all() and np.isfinite(r["entropy"][[0, 4, 5]]).all()
    assert (r["top_index"][3] == [0, 1, 2]).all() and r["top_index"][2][0] == 999 and 5 not in r["top_index"][1]
    assert np.isfinite(r["top_logprob"][[0, 4, 5]]).all() and np.isnan(r["top_logprob"][[1, 2, 3]]).all()


def test_scores_on_another_stream():
    torch = torch_cuda()
    x = torch.randn(4, 3000, device="cuda").to(torch.bfloat16)
    tok = torch.arange(4, device="cuda")
    want = H.token_logprobs(x, tok, top=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = H.token_logprobs(x, tok, top=4, stream=side)
    side.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
