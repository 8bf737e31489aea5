"""f32 rows of rotate_qk bit for bit: the order in which a row's squares are summed, and one rounding for each step."""
import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests.gpu_util import torch_cuda
from tests.test_gpu_kv4 import gpu

pytestmark = pytest.mark.gpu

f32 = np.float32


def square_sum(x):
    """Eight neighbours, by pairs where a row has 64 dimensions and by fours in turn from 128 on; then the eights by pairs."""
    q = (x * x).reshape(*x.shape[:-1], -1, 8)
    q = [q[..., i] for i in range(8)]
    if x.shape[-1] == 64:
        s = ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]))
    else:
        s = (((q[0] + q[1]) + q[2]) + q[3]) + (((q[4] + q[5]) + q[6]) + q[7])
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    return s


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 32), (128, 128), (128, 48), (256, 256)])
def test_rows_bit_for_bit(D, rot, interleaved):
    """Ordinary rows under norms; angles of 0, so that the turn's products and sums are exact, at any position."""
    torch = torch_cuda()
    rng = np.random.default_rng(D + rot)
    T = 500
    x = (rng.normal(0, 1, (T, 5, D)) * rng.choice([1.0, 30.0, 1e-3], (T, 5, 1))).astype(f32)
    w = rng.normal(1, 0.3, D).astype(f32)
    y, _ = H.rotate_qk(gpu(x), gpu(x), gpu(rng.integers(0, 1 << 20, T)), torch.zeros(rot // 2, dtype=torch.float64, device="cuda"),
                       interleaved=interleaved, q_norm=gpu(w), k_norm=gpu(w), eps=1e-5)
    m = square_sum(x) * f32(1 / D) + f32(1e-5)
    r = (1 / np.sqrt(m.astype(np.float64))).astype(f32)
    assert np.array_equal(y.cpu().numpy(), x * r * w)


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_turn_rounds_each_product(interleaved):
    """A row is turned as (a c) - (b s), (b c) + (a s), no product fused: rows of one position and its cosines, which the row
    (1, 0) gives."""
    torch = torch_cuda()
    rng = np.random.default_rng(5)
    T, D = 300, 128
    a, b = (np.arange(0, D, 2), np.arange(1, D, 2)) if interleaved else (np.arange(64), np.arange(64, D))
    x = rng.normal(0, 1, (T, 3, D)).astype(f32)
    x[:, 0, a], x[:, 0, b] = 1, 0
    y, _ = H.rotate_qk(gpu(x), gpu(x), gpu(rng.integers(0, 1 << 20, T)), H.rotary_freqs(D), interleaved=interleaved, magnitude=1.25)
    y = y.cpu().numpy()
    c, s = y[:, :1, a], y[:, :1, b]
    assert np.array_equal(y[:, 1:, a], x[:, 1:, a] * c - x[:, 1:, b] * s)
    assert np.array_equal(y[:, 1:, b], x[:, 1:, b] * c + x[:, 1:, a] * s)
