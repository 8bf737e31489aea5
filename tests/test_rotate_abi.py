"""Rotated rows and bounded attention on the CPU: argument codes, refusals, frequencies."""
import ctypes
import math

import pytest

from glint_amd import glint_hip as H

P = ctypes.c_void_p(64)  # aligned and not NULL; nothing reads it


def rotate(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, elt=0, pos=P, freqs=P, T=4, Hq=8, H=2, D=128, rot=128, inter=0, mag=1.0,
             qn=None, kn=None, ne=0, eps=1e-6, qo=P, ko=P, stream=None)
    a.update(kw)
    return lib.glint_rotate_qk(*a.values())


def append(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, elt=0, pos=P, freqs=P, slots=P, T=4, Hq=8, H=2,
             D=128, rot=128, inter=0, mag=1.0, qn=None, kn=None, ne=0, eps=1e-6, qo=P, ko=None, kh_=P, ka=P, vh_=P, va=P, pages=2,
             stream=None)
    a.update(kw)
    return lib.glint_kv4_append_rotated(*a.values())


def attend(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, Tq=2, kh=P, ka=P, vh=P, va=P, pages=2, table=P, ts=4, wide=4, lens=P, cu=None, B=2,
             max_q=1, Hq=8, H=2, D=128, scale=1.0, window=5, sinks=0, out=P, stream=None)
    a.update(kw)
    return lib.glint_kv4_attend_window(*a.values())


def prompt(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, cq=P, ck=P, Tq=4, Tk=4, B=1, max_q=4, Hq=8,
             H=2, D=128, scale=1.0, window=5, sinks=0, out=P, stream=None)
    a.update(kw)
    return lib.glint_attend_prompt_window(*a.values())


def chunk(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, Tq=600, kh=P, ka=P, vh=P, va=P, pages=2, table=P, ts=4, wide=4000, lens=P, cu=None, B=2, max_q=300, Hq=8,
             H=2, D=128, k=None, kt=256, kh_=128, v=None, vt=256, vh_=128, scale=1.0, window=0, sinks=0, out=P, scratch=P,
             size=1 << 40, stream=None)
    a.update(kw)
    return lib.glint_kv4_attend_chunk(*a.values())


ODD = ctypes.c_void_p(72)
TURN = [("q", None, -1), ("k", None, -1), ("pos", None, -1), ("freqs", None, -1), ("qo", None, -1), ("elt", 2, -2), ("T", -1, -2),
        ("T", 1 << 40, -2), ("Hq", 0, -2), ("H", 0, -2), ("rot", 8, -2), ("rot", 144, -2), ("rot", 0, -2), ("qt", 1028, -2),
        ("kh", 129, -2), ("q", ODD, -2), ("qo", ODD, -2), ("qn", ODD, -2), ("ko", ODD, -2)]


@pytest.mark.parametrize("call,bad", [
    (rotate, TURN + [("ko", None, -1), ("D", 264, -2), ("D", 100, -2), ("D", 272, -2)]),
    (append, TURN + [("v", None, -1), ("slots", None, -1), ("va", None, -1), ("D", 96, -2), ("D", 256, -2), ("pages", 0, -2),
                     ("v", ODD, -2), ("vt", 132, -2), ("kh_", ODD, -2)]),
    (attend, [("q", None, -1), ("window", -1, -2), ("window", (1 << 30) + 1, -2), ("sinks", -1, -2), ("D", 96, -2)]),
    (chunk, [("q", None, -1), ("k", P, -1), ("v", P, -1), ("D", 96, -2), ("H", 3, -2), ("Tq", 601, -2), ("out", ODD, -2),
             ("scratch", ODD, -2), ("size", 1000, -2), ("window", -1, -2), ("sinks", -1, -2), ("max_q", (1 << 18) + 1, -2), ("max_q", 0, -2),
             ("wide", 0, -2), ("pages", 0, -2), ("qh", 129, -2)]),
    (prompt, [("q", None, -1), ("window", -1, -2), ("window", (1 << 30) + 1, -2), ("sinks", -1, -2), ("D", 96, -2)]),
])
def test_refusals(call, bad):
    lib = H.serve_lib()
    for name, value, code in bad:
        assert call(lib, **{name: value}) == code, (name, value)
    if call is chunk:
        assert chunk(lib, scratch=None, size=0) == -1
        for name, value in (("kt", 120), ("vh_", 129), ("k", ODD), ("vt", (1 << 24) + 8)):
            assert chunk(lib, **{"k": P, "v": P, name: value}) == -2, name
    if call is rotate:
        assert rotate(lib, qn=P, ne=5) == -2


def test_empty_calls_do_nothing():
    lib = H.serve_lib()
    assert rotate(lib, T=0) == 0 and append(lib, T=0) == 0
    assert chunk(lib, B=0, Tq=0) == 0
    assert attend(lib, B=0, Tq=0) == 0 and prompt(lib, Tq=0) == 0


def test_scratch():
    """Parts, sums, and tiles: 4 * 64 * D bytes for each page and for each 64 own keys of a sequence and head."""
    size = H.serve_lib().glint_kv4_attend_chunk_scratch
    assert size(0, 4, 8, 2, 128, 4, 0) == 0
    small, wide = size(1, 64, 8, 2, 128, 4, 1), size(1, 64, 8, 2, 128, 1004, 1)
    assert 0 < 2 * 4 * 4 * 64 * 128 < small and wide - small > 1000 * 2 * 4 * 64 * 128
    assert size(1, 64, 8, 2, 128, 4, 0) == 0 and size(1, 1 << 12, 8, 2, 128, 4, 0) == 0  # few rows; few products
    assert size(64, 512, 32, 8, 64, 1 << 16, 0) < 3 << 30  # cut into launches
    for bad in ((1, 4, 8, 3, 128, 4), (1, 4, 8, 2, 96, 4), (1, 0, 8, 2, 128, 4), (1, 4, 8, 2, 128, 1 << 25), (1, 1 << 16, 8, 2, 128, 1 << 24)):
        assert size(*bad, 0) == -2, bad


def test_helpers_refuse():
    torch = pytest.importorskip("torch")
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    pos, fr = torch.zeros(2, dtype=torch.int64), H.rotary_freqs(64, device="cpu")
    cache = H.kv4_cache(1, 4, 64, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        H.rotate_qk(q, q, pos, fr)
    with pytest.raises(ValueError, match="GPU"):
        H.kv4_append_rotated(q, q, q, pos, fr, pos, cache)
    with pytest.raises(ValueError, match="GPU"):
        H.kv4_attend_chunk(q, cache, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    for window, sinks in ((0, 0), (-1, 0), (1 << 31, 0), (4, -1), (None, 4)):
        with pytest.raises(ValueError):
            H.kv4_attend(q, cache, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), window=window, sinks=sinks)
        with pytest.raises(ValueError):
            H.attend_prompt(q, q, q, torch.zeros(2, dtype=torch.int32), window=window, sinks=sinks)


@pytest.mark.parametrize("change,error", [
    (dict(q=(2, 4, 60)), ValueError), (dict(k=(3, 4, 64)), ValueError), (dict(k=(2, 4, 128)), ValueError),
    (dict(freqs=24 // 2 + 1), ValueError), (dict(freqs=64), ValueError), (dict(freqs=0), ValueError), (dict(pos=3), ValueError),
    (dict(norm=32), ValueError), (dict(dtype="float16"), TypeError)])
def test_shapes_are_refused(change, error):
    """What both helpers check before the library is called."""
    torch = pytest.importorskip("torch")
    dt = getattr(torch, change.get("dtype", "bfloat16"))
    q, k = (torch.zeros(change.get(n, (2, 4, 64)), dtype=dt) for n in ("q", "k"))
    if "q" in change:
        k = torch.zeros(change["q"], dtype=dt)
    pos = torch.zeros(change.get("pos", 2), dtype=torch.int64)
    fr = torch.zeros(change.get("freqs", 32), dtype=torch.float64)
    norm = torch.ones(change["norm"]) if "norm" in change else None
    with pytest.raises(error):
        H._turn_args(q, k, pos, fr, norm, None)


def test_frequencies():
    pytest.importorskip("torch")
    f = H.rotary_freqs(64, base=500.0, device="cpu").tolist()
    assert f == pytest.approx([500.0 ** (-2 * i / 64) for i in range(32)], rel=1e-14)
    assert H.rotary_freqs(64, base=500.0, factor=4.0, device="cpu").tolist() == pytest.approx([x / 4 for x in f], rel=1e-14)
    mixed = H.rotary_freqs(64, base=500.0, factor=4.0, trained=100, slow=1.0, fast=4.0, device="cpu").tolist()
    for x, y in zip(f, mixed):
        turns = 100 * x / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1) / 3))
        assert y == pytest.approx(x * keep + x / 4 * (1 - keep), rel=1e-13)
    assert mixed[0] == f[0] and mixed[-1] == f[-1] / 4
    for bad in (0, 8, 40):
        with pytest.raises(ValueError):
            H.rotary_freqs(bad, device="cpu")
    with pytest.raises(ValueError):
        H.rotary_freqs(64, trained=100, slow=4.0, fast=4.0, device="cpu")
