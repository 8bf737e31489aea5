"""libglint_serve.so on the CPU: exports, argument codes, the code rule's edges, and the helpers' refusals."""
import ctypes
import re

import numpy as np
import pytest

from glint_amd import glint_hip as H
from tests import serve_util as S
from tests.test_abi import ROOT, declared_functions, exported

P = ctypes.c_void_p(64)  # aligned and not NULL; nothing reads it


def test_exports_are_the_header():
    declared = set(declared_functions("glint_serve.h"))
    assert declared == set(H.SERVE_SYMBOLS) == exported(H.LIB_DIR / "libglint_serve.so")


def _edges():
    text = (ROOT / "glint_amd" / "csrc" / "kv4.h").read_text()
    body = re.search(r"#define KV4_EDGES[\s\\]*\{(.*?)\}", text, re.S).group(1).replace("\\", " ")
    return np.array([float.fromhex(x.strip().rstrip("f")) for x in body.split(",")], np.float32)


def test_code_edges_are_the_first_minimum():
    """On both sides of each edge, at every parent, and over a sweep, counting edges below v gives the
    first minimum of |v - PARENT|."""
    e = _edges()
    assert len(e) == 15 and (np.diff(e) > 0).all()
    near = np.concatenate([(e.view(np.int32)[:, None] + np.arange(-64, 65)).astype(np.int32).view(np.float32).ravel(),
                           S.PARENT, np.linspace(-1, 1, 200001, dtype=np.float32), np.float32([0.0, -0.0])])
    want = np.abs(near[:, None] - S.PARENT).argmin(1)
    assert ((near[:, None] > e).sum(1) == want).all()


def append(lib, **kw):
    a = dict(k=P, v=P, elt=0, kst=1024, ksh=128, vst=1024, vsh=128, slots=P, T=4, H=8, D=128, kh=P, ka=P, vh=P, va=P,
             pages=2, stream=None)
    a.update(kw)
    return lib.glint_kv4_append(*a.values())


def attend(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, Tq=2, kh=P, ka=P, vh=P, va=P, pages=2, table=P, ts=4, wide=4, lens=P, cu=None, B=2,
             max_q=1, Hq=8, H=2, D=128, scale=1.0, out=P, stream=None)
    a.update(kw)
    return lib.glint_kv4_attend(*a.values())


def prompt(lib, **kw):
    a = dict(q=P, qt=1024, qh=128, k=P, kt=256, kh=128, v=P, vt=256, vh=128, cq=P, ck=P, Tq=4, Tk=4, B=1, max_q=4, Hq=8,
             H=2, D=128, scale=1.0, out=P, stream=None)
    a.update(kw)
    return lib.glint_attend_prompt(*a.values())


def scores(lib, **kw):
    a = dict(x=P, elt=0, stride=100, tok=P, T=2, V=100, top=5, lp=P, ent=P, rank=P, tlp=P, ti=P, stream=None)
    a.update(kw)
    return lib.glint_token_logprobs(*a.values())


@pytest.mark.parametrize("call,bad", [
    (append, [("k", None, -1), ("slots", None, -1), ("va", None, -1), ("D", 96, -2), ("elt", 2, -2), ("kst", 1022, -2),
              ("vsh", 129, -2), ("k", ctypes.c_void_p(68), -2), ("H", 0, -2), ("T", -1, -2), ("pages", 0, -2),
              ("T", 1 << 41, -2)]),
    (attend, [("q", None, -1), ("lens", None, -1), ("out", None, -1), ("D", 256, -2), ("H", 3, -2), ("Tq", 3, -2),
              ("qt", 1020, -2), ("q", ctypes.c_void_p(72), -2), ("wide", 0, -2), ("max_q", 0, -2), ("B", -1, -2), ("wide", (1 << 24) + 1, -2),
              ("pages", 0, -2)]),
    (prompt, [("v", None, -1), ("cq", None, -1), ("out", None, -1), ("D", 80, -2), ("H", 3, -2), ("kt", 252, -2),
              ("v", ctypes.c_void_p(72), -2), ("B", -1, -2), ("max_q", -1, -2), ("Tk", -1, -2)]),
    (scores, [("x", None, -1), ("lp", None, -1), ("tlp", None, -1), ("elt", 3, -2), ("V", 0, -2), ("top", 21, -2),
              ("top", -1, -2), ("V", 4, -2), ("V", 262145, -2), ("T", 1 << 22, -2), ("x", ctypes.c_void_p(65), -2)]),
])
def test_refusals(call, bad):
    lib = H.serve_lib()
    for name, value, code in bad:
        assert call(lib, **{name: value}) == code, (name, value)


def test_empty_calls_do_nothing():
    lib = H.serve_lib()
    assert append(lib, T=0) == 0
    assert attend(lib, B=0, Tq=0) == 0
    assert prompt(lib, B=0) == 0 and prompt(lib, Tq=0) == 0 and prompt(lib, max_q=0) == 0
    assert scores(lib, T=0) == 0
    assert lib.glint_kv4_gather(P, 0, 8, 128, P, P, P, P, 2, P, P, None) == 0
    assert lib.glint_kv4_gather(P, 1, 8, 128, P, P, P, P, 2, None, P, None) == -1
    assert lib.glint_kv4_gather(P, 1, 8, 100, P, P, P, P, 2, P, P, None) == -2


def test_helpers_refuse():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError):
        H.kv4_cache(4, 2, 96, device="cpu")
    c = H.kv4_cache(4, 2, 64, device="cpu")
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):  # not on the GPU
        H.kv4_append(k, k, torch.zeros(3, dtype=torch.int64), c)
    with pytest.raises(ValueError):
        H.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        H.token_logprobs(torch.zeros(2, 10, dtype=torch.float16), torch.zeros(2, dtype=torch.int64))
