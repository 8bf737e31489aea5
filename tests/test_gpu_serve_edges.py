"""The serving operators at masks, strides, defaults and batches where a call once went wrong."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.gpu_util import host, torch_cuda
from tests.test_gpu_kv4 import bf16, gpu

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
