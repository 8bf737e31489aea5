"""Chunks over the 4-bit cache: which rows are written, and what they hold, where max_q is less than a sequence's rows."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import bounded_util as R
from tests import serve_util as S
from tests.gpu_util import torch_cuda
from tests.test_gpu_kv4 import bf16, gpu
from tests.test_gpu_kv4_chunk import bound, many
from tests.test_gpu_window import paged, values

pytestmark = pytest.mark.gpu

LENS, CU, G = [100, 300, 20], [3, 33, 153, 193], 16


@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("D,max_q", [(64, 200), (64, 120), (64, 20), (64, 13), (128, 20), (128, 63)])
def test_every_kept_row(D, max_q, window, sinks, own):
    """Rows past max_q, before the first sequence and behind the last stay; each of the others is what its positions give, a
    sequence of fewer tokens than rows among them."""
    torch = torch_cuda()
    print(f"D={D} max_q={max_q} window={window} own={own}", flush=True)
    rng = np.random.default_rng(max_q + D)
    planes, table, _ = paged(rng, LENS, 1, D)
    wide, _ = many(table, 0)
    assert H.serve_lib().glint_kv4_attend_chunk_scratch(3, max_q, G, 1, D, wide.shape[1], own) > 0
    q = bf16(rng.normal(0, 1, (200, G, D)))
    k, v = (bf16(rng.normal(0, 1, (200, 1, D))) for _ in range(2))
    out = torch.full_like(q, 7.0)
    H.kv4_attend_chunk(q, tuple(gpu(p) for p in planes), gpu(wide), gpu(np.array(LENS, np.int32)), gpu(np.array(CU, np.int32)),
                       max_q=max_q, k=k if own else None, v=v if own else None, window=window or None, sinks=sinks, out=out)
    got, qf, kf, vf = values(out), values(q), values(k), values(v)
    kept = np.zeros(200, bool)
    for b, n in enumerate(LENS):
        nq = CU[b + 1] - CU[b]
        rows = np.arange(CU[b], CU[b] + min(nq, max_q))
        kept[rows] = True
        hk, hv = S.held(planes, table[b][np.arange(n) // 64].astype(np.int64) * 64 + np.arange(n) % 64)
        if own:
            m = min(nq, n)
            hk[n - m:], hv[n - m:] = kf[CU[b + 1] - m:CU[b + 1]], vf[CU[b + 1] - m:CU[b + 1]]
        ok = R.seen(np.arange(len(rows)) + n - nq, n, window, sinks)
        for h in range(G):
            worst = R.far(got[rows, h], *R.attend(qf[rows, h], hk[:, 0], hv[:, 0], ok, D ** -0.5), bound(own))
            assert worst <= 0, (b, h, worst)
    assert (got[~kept] == 7).all()
