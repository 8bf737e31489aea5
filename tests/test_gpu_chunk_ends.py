"""Chunks over the 4-bit cache at the ends of what positions may be."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import bounded_util as R
from tests import serve_util as S
from tests.gpu_util import torch_cuda
from tests.test_gpu_kv4 import bf16, gpu
from tests.test_gpu_kv4_chunk import bound
from tests.test_gpu_window import paged, values

pytestmark = pytest.mark.gpu


def far_chunk(length, window, sinks, D, nq=100, heads=2, G=2):
    """The newest nq tokens of a sequence that says `length`, with keys of their own, after two pages of its first
    tokens; rows behind the last are NaN, which whoever read them would show."""
    rng = np.random.default_rng(D)
    planes, table, _ = paged(rng, [128], heads, D)
    q = bf16(rng.normal(0, 1, (nq, heads * G, D)))
    behind = [bf16(np.concatenate([rng.normal(0, 1, (nq, heads, D)), np.full((80, heads, D), np.nan)])) for _ in range(2)]
    k, v = (x[:nq] for x in behind)
    got = values(H.kv4_attend_chunk(q, tuple(gpu(p) for p in planes), gpu(table), gpu(np.array([length], np.int32)), max_q=nq,
                                    k=k, v=v, window=window, sinks=sinks))
    hk, hv = S.held(planes, table[0][np.arange(128) // 64].astype(np.int64) * 64 + np.arange(128) % 64)
    ks, vs = np.concatenate([hk, values(k)]), np.concatenate([hv, values(v)])
    i, j = np.arange(nq)[:, None], np.arange(nq)[None]
    own = (j <= i) & ((j > i - window) if window else True)
    ok = np.concatenate([np.broadcast_to(np.arange(128) < (sinks if window else 128), (nq, 128)), own], 1)
    for h in range(heads * G):
        worst = R.far(got[:, h], *R.attend(values(q)[:, h], ks[:, h // G], vs[:, h // G], ok, D ** -0.5), bound(True))
        assert worst <= 0, (h, worst)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 30, 2 ** 31 - 64, 2 ** 31 - 65, 2 ** 30 + 5])
def test_a_window_at_the_last_positions(length, D):
    torch_cuda()
    print(f"length={length} D={D}", flush=True)
    far_chunk(length, 70, 5, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 30 + 100, 2 ** 30 + 5])
def test_without_a_window_every_position_is_seen(length, D):
    torch_cuda()
    print(f"length={length} D={D}", flush=True)
    far_chunk(length, None, 0, D)
