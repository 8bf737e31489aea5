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


def state(m):
    return list(m.held), [list(o) for o in m.own], list(m.free), m.table.clone()


@pytest.mark.gpu
@pytest.mark.parametrize("rotary,window", [(False, None), (True, None), (True, 100)])
def test_a_refused_call_changes_no_request(rotary, window):
    """A chunk of more rows a key head than the attention over chunks takes, a step of more than the single tokens' does, and an
    operator that fails in a later layer: pages, lengths and what follows are as if they had not been."""
    from tests.gpu_util import torch_cuda
    torch_cuda()
    from glint_amd import decoder as D
    how = dict(vocab=50, dim=64, layers=2, heads=128, kv_heads=1, head_dim=64, ffn=64, pages=150, requests=3,
               rotary=H.rotary_freqs(64) if rotary else None, window=window)
    m, other = D.Decoder(**how), D.Decoder(**how)
    first = {0: [1, 2, 3] * 30, 2: [4] * 7}
    assert torch.equal(m.prefill(first), other.prefill(first))
    was = state(m)
    calls = [lambda: m.step({2: [6] * 8200, 1: [1]})] + ([lambda: m.prefill({0: [5] * 2049, 1: [7] * 70})] if rotary else [])
    silu, left = torch.nn.functional.silu, [1]

    def fails(x):
        left[0] -= 1
        if left[0] < 0:
            raise RuntimeError("no memory")
        return silu(x)

    for call in calls + [lambda: m.prefill({0: [5] * 200, 1: [7] * 70}), lambda: m.step({0: [5], 2: [6] * 64})]:
        if call not in calls:
            left[0], torch.nn.functional.silu = 1, fails
        try:
            with pytest.raises((RuntimeError, ValueError)):
                call()
        finally:
            torch.nn.functional.silu = silu
        now = state(m)
        assert now[:3] == was[:3] and torch.equal(now[3], was[3])
    for news in ({0: [5] * 30, 1: [8]}, {2: [3] * 70}):
        assert torch.equal(m.prefill(news), other.prefill(news))
    assert torch.equal(m.step({0: [1], 2: [2]}), other.step({0: [1], 2: [2]}))
