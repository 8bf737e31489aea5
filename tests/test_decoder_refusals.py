"""What a Decoder's constructor refuses, before it asks for any memory."""
import pytest

from glint_amd import glint_hip as H

torch = pytest.importorskip("torch")


def vector(n, dtype=torch.float64):
    return torch.ones(n, dtype=dtype)


@pytest.mark.parametrize("how", [
    dict(sinks=4), dict(window=5), dict(window=0, rotary=vector(16)), dict(window=-3, rotary=vector(16)),
    dict(window=(1 << 30) + 1, rotary=vector(16)), dict(window=5, sinks=-1, rotary=vector(16)), dict(sinks=4, rotary=vector(16)),
    dict(rotary=vector(16)), dict(rotary=vector(16, torch.float32)), dict(rotary=vector(32).view(2, 16)), dict(heads=3, kv_heads=2)])
def test_refused(how):
    from glint_amd.decoder import Decoder
    with pytest.raises(ValueError):
        Decoder(**how)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 4, 12, 40])
def test_frequencies_for_other_widths(n):
    from tests.gpu_util import torch_cuda
    torch_cuda()
    from glint_amd.decoder import Decoder
    with pytest.raises(ValueError, match="turned"):
        Decoder(rotary=torch.ones(n, dtype=torch.float64, device="cuda"), head_dim=64)
    assert Decoder(rotary=H.rotary_freqs(64), head_dim=64, layers=1).rotary.numel() == 32
