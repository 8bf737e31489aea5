"""ctypes bindings to the GLINT C ABI (libglint_encode.so, libp7_kernels.so, libglint_serve.so).

Two layers:

* ``EncodeLib`` / ``P7Lib`` / ``ServeLib``: the raw C entry points with their argtypes, as a caller of
  the reference's ``glint_cuda.py`` would bind them (the host-pointer ABI takes bytes);
* tensor helpers (``encode_bf16`` ... ``token_logprobs``) that pass torch device tensors
  and torch's current stream straight to the device entry points. torch is only the
  allocator and stream here; every result is computed by the HIP kernels.

A missing library raises RuntimeError: there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import os
from pathlib import Path
from typing import NamedTuple, Optional, Tuple

PKG = Path(__file__).resolve().parent
LIB_DIR = PKG / "lib"

_c = ctypes
VP, I64, I32 = _c.c_void_p, _c.c_int64, _c.c_int


def encode_lib_path() -> Optional[Path]:
    """$GLINT_ENCODE_SO, else glint_amd/lib/libglint_encode.so (reference glint_cuda.py:9-18)."""
    env = os.environ.get("GLINT_ENCODE_SO")
    if env:
        p = Path(env)
        return p if p.is_file() else None
    p = LIB_DIR / "libglint_encode.so"
    return p if p.is_file() else None


def p7_lib_path() -> Optional[Path]:
    env = os.environ.get("GLINT_P7_SO")
    if env:
        p = Path(env)
        return p if p.is_file() else None
    p = LIB_DIR / "libp7_kernels.so"
    return p if p.is_file() else None


def serve_lib_path() -> Optional[Path]:
    env = os.environ.get("GLINT_SERVE_SO")
    if env:
        p = Path(env)
        return p if p.is_file() else None
    p = LIB_DIR / "libglint_serve.so"
    return p if p.is_file() else None


_ENCODE_SIGS = {
    "glint_encode_n_absmax": ([I64, I32], I32),
    "glint_encode_n_packed": ([I64], I32),
    "glint_encode_bf16_host": ([VP, I64, I32, VP, VP, VP], I32),
    "glint_encode_f32_host": ([VP, I64, I32, VP, VP, VP], I32),
    "glint_expand_packed_to_f32_host": ([VP, VP, VP, I64, I32, VP], I32),
    "glint_expand_packed_to_bf16_host": ([VP, VP, VP, I64, I32, VP], I32),
    "glint_expand_packed_to_f32_device": ([VP, VP, VP, I64, I32, VP, VP], I32),
    "glint_expand_packed_to_bf16_device": ([VP, VP, VP, I64, I32, VP, VP], I32),
    "glint_encode_bf16_device": ([VP, I64, I32, VP, VP, VP, VP], I32),
    "glint_encode_f32_device": ([VP, I64, I32, VP, VP, VP, VP], I32),
    "launch_glint_htile_s3_f32_stream": ([VP, VP, VP, VP, VP, I32, I32, I32, I32, VP], I32),
    "launch_glint_htile_s3_f32": ([VP, VP, VP, VP, VP, I32, I32, I32, I32], I32),
    "launch_glint_htile_bf16_stream": ([VP, VP, VP, VP, VP, I32, I32, I32, I32, VP], I32),
    "glint_htile_workspace_reserve": ([VP], I32),
    "glint_htile_workspace_release": ([VP], I32),
    "launch_glint_htile_bf16_stream_noalloc": ([VP, VP, VP, VP, VP, I32, I32, I32, I32, VP], I32),
    "glint_kmajor_pack": ([VP, VP, VP, I32, I32, VP, VP, VP, VP], I32),
    "glint_gemv_km_fold": ([VP, VP, VP, VP, I32, I32, I32, VP, VP], I32),
    "glint_select_topk": ([VP, I32, I32, VP, VP, VP], I32),
    "glint_select_topk_ex": ([VP, I32, I32, I32, I32, VP, VP, VP, I32, VP], I32),
    "glint_apply_corr_km": ([VP, VP, VP, VP, VP, VP, VP, I32, I32, I32, VP, VP], I32),
}


class Int8MmaLinear(_c.Structure):
    """include/int8_mma_gemm.h Int8MmaLinear, passed by value."""
    _fields_ = [("q", VP), ("scale", VP), ("n_out", I32), ("k_in", I32)]


class Int8PinLinear(_c.Structure):
    """include/int8_tile_gemm.h Int8PinLinear, passed by value (same layout as Int8MmaLinear)."""
    _fields_ = [("q", VP), ("scale", VP), ("n_out", I32), ("k_in", I32)]


class GlintStreamerStats(ctypes.Structure):
    """include/glint_plug_streamer.h GlintStreamerStats."""
    _fields_ = [("total_h2d_bytes", ctypes.c_uint64), ("total_stall_ms", ctypes.c_double),
                ("per_layer_stall_ms", ctypes.c_double * 64), ("n_layers", ctypes.c_int)]


_P7_SIGS = {
    "p7_abi_version": ([], _c.c_char_p),
    "p7_abi_selftest": ([_c.c_char_p, _c.c_size_t], I32),
    "int8_mma_gemm": ([VP, Int8MmaLinear, VP, I32, VP, VP, VP], I32),
    "int8_mma_gemm_plug": ([VP, Int8MmaLinear, VP, VP, VP, I32, VP, VP, VP, VP], I32),
    "int8_mma_gemm_plug_fused": ([VP, Int8MmaLinear, VP, VP, VP, I32, VP, VP, VP], I32),
    "int8_mma_gemm_resolve": ([VP, Int8MmaLinear, VP, VP, VP, I32, VP, VP, VP, VP, VP, VP], I32),
    "p7_int8_gemm_flat": ([VP, VP, VP, I32, I32, VP, I32, VP, VP, VP], I32),
    "p7_int8_gemm_plug_flat": ([VP, VP, VP, VP, VP, I32, I32, VP, I32, VP, VP, VP], I32),
    "int8_tile_gemm_bf16": ([VP, Int8PinLinear, VP, I32, VP], I32),
    "int8_tile_gemm_workspace_release": ([VP], I32),
    "glint_int8_gemm_i32": ([VP, VP, VP, I32, I32, I32, VP], I32),
    "glint_int8_gemm_scaled_bf16": ([VP, VP, VP, VP, VP, I32, I32, I32, VP], I32),
    "glint_plug_streamer_create": ([_c.POINTER(VP), I32, _c.POINTER(_c.c_uint64), VP, VP], I32),
    "glint_plug_streamer_destroy": ([VP], None),
    "glint_plug_streamer_set_host_data": ([VP, I32, VP, _c.c_uint64], I32),
    "glint_plug_streamer_start": ([VP], I32),
    "glint_plug_streamer_acquire": ([VP, I32, _c.POINTER(VP)], I32),
    "glint_plug_streamer_release": ([VP, I32], I32),
    "glint_plug_streamer_get_stats": ([VP, _c.POINTER(GlintStreamerStats)], I32),
    "glint_plug_streamer_reset_stats": ([VP], None),
}

_SERVE_SIGS = {
    "glint_kv4_append": ([VP, VP, I32, I64, I64, I64, I64, VP, I64, I32, I32, VP, VP, VP, VP, I64, VP], I32),
    "glint_kv4_gather": ([VP, I64, I32, I32, VP, VP, VP, VP, I64, VP, VP, VP], I32),
    "glint_kv4_attend": ([VP, I64, I64, I64, VP, VP, VP, VP, I64, VP, I64, I32, VP, VP, I32, I32, I32, I32, I32,
                          _c.c_float, VP, VP], I32),
    "glint_kv4_attend_window": ([VP, I64, I64, I64, VP, VP, VP, VP, I64, VP, I64, I32, VP, VP, I32, I32, I32, I32, I32,
                                 _c.c_float, I32, I32, VP, VP], I32),
    "glint_kv4_attend_chunk_scratch": ([I32, I32, I32, I32, I32, I32, I32], I64),
    "glint_kv4_attend_chunk": ([VP, I64, I64, I64, VP, VP, VP, VP, I64, VP, I64, I32, VP, VP, I32, I32, I32, I32, I32, VP, I64,
                                I64, VP, I64, I64, _c.c_float, I32, I32, VP, VP, I64, VP], I32),
    "glint_serve_workspace_reserve": ([VP], I32),
    "glint_serve_workspace_release": ([VP], I32),
    "glint_attend_prompt": ([VP, I64, I64, VP, I64, I64, VP, I64, I64, VP, VP, I64, I64, I32, I32, I32, I32, I32,
                             _c.c_float, VP, VP], I32),
    "glint_attend_prompt_window": ([VP, I64, I64, VP, I64, I64, VP, I64, I64, VP, VP, I64, I64, I32, I32, I32, I32, I32,
                                    _c.c_float, I32, I32, VP, VP], I32),
    "glint_rotate_qk": ([VP, I64, I64, VP, I64, I64, I32, VP, VP, I64, I32, I32, I32, I32, I32, _c.c_double, VP, VP, I32,
                         _c.c_float, VP, VP, VP], I32),
    "glint_kv4_append_rotated": ([VP, I64, I64, VP, I64, I64, VP, I64, I64, I32, VP, VP, VP, I64, I32, I32, I32, I32, I32,
                                  _c.c_double, VP, VP, I32, _c.c_float, VP, VP, VP, VP, VP, VP, I64, VP], I32),
    "glint_token_logprobs": ([VP, I32, I64, VP, I64, I64, I32, VP, VP, VP, VP, VP, VP], I32),
}

ENCODE_SYMBOLS = tuple(_ENCODE_SIGS)
P7_SYMBOLS = tuple(_P7_SIGS)
SERVE_SYMBOLS = tuple(_SERVE_SIGS)


def _bind(path: Path, sigs: dict) -> ctypes.CDLL:
    # One HIP runtime per process: torch's wheel ships its own libamdhip64.so.7. If torch
    # is importable, load it first so our library binds to that already-loaded runtime
    # (same SONAME) instead of pulling in a second copy from /opt/rocm.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(str(path))
    for name, (args, res) in sigs.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = res
    return lib


_ENC: Optional[ctypes.CDLL] = None
_P7: Optional[ctypes.CDLL] = None
_SERVE: Optional[ctypes.CDLL] = None


def encode_lib() -> ctypes.CDLL:
    global _ENC
    if _ENC is None:
        p = encode_lib_path()
        if p is None:
            raise RuntimeError("libglint_encode.so not built: run `python -m glint_amd.build`")
        _ENC = _bind(p, _ENCODE_SIGS)
    return _ENC


_PROBE: Optional[ctypes.CDLL] = None


def probe_lib() -> ctypes.CDLL:
    """glint_amd/lib/libglint_probe.so: bench.py's HBM read ceiling (not part of the ABI)."""
    global _PROBE
    if _PROBE is None:
        p = LIB_DIR / "libglint_probe.so"
        if not p.is_file():
            raise RuntimeError("libglint_probe.so not built: run `python -m glint_amd.build`")
        _PROBE = _bind(p, {"glint_probe_read": ([VP, I64, VP, I32, VP], I32)})
    return _PROBE


def p7_lib() -> ctypes.CDLL:
    global _P7
    if _P7 is None:
        p = p7_lib_path()
        if p is None:
            raise RuntimeError("libp7_kernels.so not built: run `python -m glint_amd.build`")
        _P7 = _bind(p, _P7_SIGS)
    return _P7


def serve_lib() -> ctypes.CDLL:
    global _SERVE
    if _SERVE is None:
        p = serve_lib_path()
        if p is None:
            raise RuntimeError("libglint_serve.so not built: run `python -m glint_amd.build`")
        _SERVE = _bind(p, _SERVE_SIGS)
    return _SERVE


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} rc={rc}")


# ------------------------------------------------------------ tensor helpers (device)
# A decode launch lasts 5 to 12 us on the device, so what a helper does before it counts: the
# pointers go to ctypes as ints (argtypes convert them), the current stream's handle is read
# without building a Stream object, and outputs come from new_empty / empty_like. Host time of
# a call on one box: htile_bf16 10.3 -> 6.5 us, encode_f32 16.6 -> 8.5, seven
# decode linears 76 -> 52, a K-major step 28 -> 17.
_TORCH = None


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch
        _TORCH = torch
    return _TORCH


def _stream(stream=None) -> ctypes.c_void_p:
    torch = _torch()
    s = torch.cuda.current_stream() if stream is None else stream
    return VP(s.cuda_stream)


def _sh(stream) -> int:
    """The stream's handle (of the current stream of the current device for None)."""
    if stream is not None:
        return stream.cuda_stream
    torch = _TORCH or _torch()
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _p(t) -> ctypes.c_void_p:
    return VP(t.data_ptr())


def _as_u16(t):
    torch = _torch()
    if t.dtype == torch.bfloat16:
        return t.view(torch.int16)
    if t.dtype in (torch.int16, torch.uint16):
        return t
    raise TypeError(f"expected bf16 bits, got {t.dtype}")


def _check_u16(t) -> None:
    """t holds BF16 bits (_as_u16 without the view: only its data pointer is used)."""
    torch = _TORCH or _torch()
    d = t.dtype
    if d is not torch.bfloat16 and d is not torch.int16 and d is not torch.uint16:
        raise TypeError(f"expected bf16 bits, got {d}")


def _pin_out(w, n: int, blocksize: int):
    torch = _TORCH or _torch()
    hole = w.new_empty((n + 1) // 2, dtype=torch.uint8)
    return hole, torch.empty_like(hole), w.new_empty((n + blocksize - 1) // blocksize, dtype=torch.float32)


def encode_bf16(w, blocksize: int = 64, out=None, stream=None):
    """GPU encode of a BF16 device tensor -> (hole u8, plug u8, absmax f32) device tensors."""
    _check_u16(w)
    w = w.contiguous()
    n = w.numel()
    hole, plug, am = _pin_out(w, n, blocksize) if out is None else out
    _check(encode_lib().glint_encode_bf16_device(w.data_ptr(), n, blocksize, hole.data_ptr(), plug.data_ptr(),
                                                 am.data_ptr(), _sh(stream)), "glint_encode_bf16_device")
    return hole, plug, am


def encode_f32(w, blocksize: int = 64, stream=None):
    torch = _torch()
    w = w.contiguous()
    assert w.dtype == torch.float32
    n = w.numel()
    hole, plug, am = _pin_out(w, n, blocksize)
    _check(encode_lib().glint_encode_f32_device(w.data_ptr(), n, blocksize, hole.data_ptr(), plug.data_ptr(),
                                                am.data_ptr(), _sh(stream)), "glint_encode_f32_device")
    return hole, plug, am


def expand_f32(hole, plug, absmax, n: int, blocksize: int = 64, out=None, stream=None):
    out = hole.new_empty(n, dtype=_torch().float32) if out is None else out
    _check(encode_lib().glint_expand_packed_to_f32_device(hole.data_ptr(), plug.data_ptr(), absmax.data_ptr(), n,
                                                          blocksize, out.data_ptr(), _sh(stream)),
           "glint_expand_packed_to_f32_device")
    return out


def expand_bf16(hole, plug, absmax, n: int, blocksize: int = 64, out=None, stream=None):
    out = hole.new_empty(n, dtype=_torch().bfloat16) if out is None else out
    _check(encode_lib().glint_expand_packed_to_bf16_device(hole.data_ptr(), plug.data_ptr(), absmax.data_ptr(), n,
                                                           blocksize, out.data_ptr(), _sh(stream)),
           "glint_expand_packed_to_bf16_device")
    return out


def htile_f32(hole, plug, absmax, x, N: int, K: int, blocksize: int = 64, out=None, stream=None):
    """y[M, N] f32 = x[M, K] (bf16) @ W^T via launch_glint_htile_s3_f32_stream."""
    _check_u16(x)
    M = x.numel() // K
    y = x.new_empty((M, N), dtype=_TORCH.float32) if out is None else out
    _check(encode_lib().launch_glint_htile_s3_f32_stream(hole.data_ptr(), plug.data_ptr(), absmax.data_ptr(),
                                                         x.data_ptr(), y.data_ptr(), M, N, K, blocksize, _sh(stream)),
           "launch_glint_htile_s3_f32_stream")
    return y


def htile_bf16(hole, plug, absmax, x, N: int, K: int, blocksize: int = 64, out=None, stream=None):
    """y[M, N] bf16 (f32 accumulation) via launch_glint_htile_bf16_stream."""
    _check_u16(x)
    M = x.numel() // K
    y = x.new_empty((M, N), dtype=_TORCH.bfloat16) if out is None else out
    _check(encode_lib().launch_glint_htile_bf16_stream(hole.data_ptr(), plug.data_ptr(), absmax.data_ptr(),
                                                       x.data_ptr(), y.data_ptr(), M, N, K, blocksize, _sh(stream)),
           "launch_glint_htile_bf16_stream")
    return y


# ------------------------------------------------------- K-major decode path (glint_select.h)
def kmajor_pack(hole, plug, absmax, N: int, K: int, stream=None):
    """Row-major pin planes -> (hole_k, plug_k, scales_k) device tensors."""
    torch = _torch()
    hk = hole.new_empty(K * N // 2, dtype=torch.uint8)
    pk = torch.empty_like(hk)
    sk = hole.new_empty(N * K // 64, dtype=torch.float32)
    _check(encode_lib().glint_kmajor_pack(hole.data_ptr(), plug.data_ptr(), absmax.data_ptr(), N, K, hk.data_ptr(),
                                          pk.data_ptr(), sk.data_ptr(), _sh(stream)), "glint_kmajor_pack")
    return hk, pk, sk


def gemv_km_fold(hole_k, scales_k, x, N: int, K: int, ksg: int = 1, y=None, part=None, stream=None):
    """Parent-only GEMV over the K-major hole: x bf16 [K] -> y f32 [N]."""
    _check_u16(x)
    y = hole_k.new_empty(N, dtype=_TORCH.float32) if y is None else y
    if ksg > 1 and part is None:
        part = hole_k.new_empty(ksg * N, dtype=_TORCH.float32)
    _check(encode_lib().glint_gemv_km_fold(hole_k.data_ptr(), scales_k.data_ptr(), x.data_ptr(), y.data_ptr(), N, K,
                                           ksg, part.data_ptr() if part is not None else None, _sh(stream)),
           "glint_gemv_km_fold")
    return y


def select_topk(x, nsel: int, idx=None, cnt=None, stream=None, tkey: int = 0, nfloor: int = 0, cnt_log=None,
                slot: int = 0):
    """Kept channels of x (ascending) and their count, both on the device (the rank rule,
    and the price / relational / floor rules when tkey or nfloor is given)."""
    _check_u16(x)
    K = x.numel()
    idx = x.new_empty(K, dtype=_TORCH.int32) if idx is None else idx
    cnt = x.new_empty(1, dtype=_TORCH.int32) if cnt is None else cnt
    if tkey == 0 and nfloor == 0 and cnt_log is None:
        _check(encode_lib().glint_select_topk(x.data_ptr(), K, nsel, idx.data_ptr(), cnt.data_ptr(), _sh(stream)),
               "glint_select_topk")
    else:
        _check(encode_lib().glint_select_topk_ex(x.data_ptr(), K, nsel, tkey, nfloor, idx.data_ptr(), cnt.data_ptr(),
                                                 cnt_log.data_ptr() if cnt_log is not None else None, slot,
                                                 _sh(stream)), "glint_select_topk_ex")
    return idx, cnt


def apply_corr_km(hole_k, plug_k, scales_k, x, idx, cnt, y, N: int, K: int, ks: int = 1, part=None, stream=None):
    """y += the plug correction over the selected channels (in place)."""
    _check_u16(x)
    if ks > 1 and part is None:
        part = y.new_empty(ks * N, dtype=_TORCH.float32)
    _check(encode_lib().glint_apply_corr_km(hole_k.data_ptr(), plug_k.data_ptr(), scales_k.data_ptr(), x.data_ptr(),
                                            idx.data_ptr(), cnt.data_ptr(), y.data_ptr(), N, K, ks,
                                            part.data_ptr() if part is not None else None, _sh(stream)),
           "glint_apply_corr_km")
    return y


def _quant_out(x, m: int, k_in: int, xq=None, sx=None):
    """The activation scratch of m rows: int8 values and one f32 per 64 of them."""
    xq = x.new_empty(m * k_in, dtype=_TORCH.int8) if xq is None else xq
    sx = x.new_empty(m * (k_in // 64), dtype=_TORCH.float32) if sx is None else sx
    return xq, sx


def int8_mma_gemm(x, q, scale, n_out: int, k_in: int, xq=None, sx=None, stream=None):
    """The attach ABI's W8A8 GEMM: x bf16 [m, k_in] -> y f32 [m, n_out] (also returns xq, sx)."""
    _check_u16(x)
    m = x.numel() // k_in
    y = x.new_empty((m, n_out), dtype=_TORCH.float32)
    xq, sx = _quant_out(x, m, k_in, xq, sx)
    lin = Int8MmaLinear(q.data_ptr(), scale.data_ptr(), n_out, k_in)
    _check(p7_lib().int8_mma_gemm(x.data_ptr(), lin, y.data_ptr(), m, xq.data_ptr(), sx.data_ptr(), _sh(stream)),
           "int8_mma_gemm")
    return y, xq, sx


def int8_tile_gemm(x, q, scale, n_out: int, k_in: int, m: Optional[int] = None, y=None, stream=None):
    """W8A16 over an INT8 pin linear: x bf16 [m, k_in] -> y f32 [m, n_out] (int8_tile_gemm_bf16).
    x, q and scale may be views at any offset; the call takes their data pointers as they are."""
    _check_u16(x)
    m = x.numel() // k_in if m is None else m
    if y is None:
        y = x.new_empty((m, n_out), dtype=_TORCH.float32)
    lin = Int8PinLinear(q.data_ptr(), scale.data_ptr(), n_out, k_in)
    _check(p7_lib().int8_tile_gemm_bf16(x.data_ptr(), lin, y.data_ptr(), m, _sh(stream)), "int8_tile_gemm_bf16")
    return y


def int8_mma_gemm_plug(x, q, scale, plug_q4, plug_scale, n_out: int, k_in: int, fused: bool = False, stream=None):
    """The late-plug forms: two passes through int8 scratch (int8_mma_gemm_plug) or one fused
    kernel (int8_mma_gemm_plug_fused). Returns y f32 [m, n_out]."""
    _check_u16(x)
    m = x.numel() // k_in
    y = x.new_empty((m, n_out), dtype=_TORCH.float32)
    xq, sx = _quant_out(x, m, k_in)
    lin = Int8MmaLinear(q.data_ptr(), scale.data_ptr(), n_out, k_in)
    lib = p7_lib()
    if fused:
        _check(lib.int8_mma_gemm_plug_fused(x.data_ptr(), lin, plug_q4.data_ptr(), plug_scale.data_ptr(), y.data_ptr(),
                                            m, xq.data_ptr(), sx.data_ptr(), _sh(stream)), "int8_mma_gemm_plug_fused")
    else:
        pi8 = x.new_empty(n_out * k_in, dtype=_TORCH.int8)
        _check(lib.int8_mma_gemm_plug(x.data_ptr(), lin, plug_q4.data_ptr(), plug_scale.data_ptr(), y.data_ptr(), m,
                                      xq.data_ptr(), sx.data_ptr(), pi8.data_ptr(), _sh(stream)), "int8_mma_gemm_plug")
    return y


def int8_mma_gemm_resolve(x, q, scale, n_out: int, k_in: int, plug_q4=None, plug_scale=None, stream=None):
    """int8_mma_gemm_resolve: base (+ plug) plus the re-quantized activation residual.
    Returns (y, xq, sx, rq, sr)."""
    _check_u16(x)
    torch = _torch()
    m = x.numel() // k_in
    y = x.new_empty((m, n_out), dtype=torch.float32)
    xq, sx = _quant_out(x, m, k_in)
    rq = torch.empty_like(xq)
    sr = torch.empty_like(sx)
    pi8 = x.new_empty(n_out * k_in, dtype=torch.int8) if plug_q4 is not None else None
    lin = Int8MmaLinear(q.data_ptr(), scale.data_ptr(), n_out, k_in)
    opt = lambda t: t.data_ptr() if t is not None else None
    _check(p7_lib().int8_mma_gemm_resolve(x.data_ptr(), lin, opt(plug_q4), opt(plug_scale), y.data_ptr(), m,
                                          xq.data_ptr(), sx.data_ptr(), rq.data_ptr(), sr.data_ptr(), opt(pi8),
                                          _sh(stream)), "int8_mma_gemm_resolve")
    return y, xq, sx, rq, sr


class PlugStreamer:
    """The 2-slot plug ring (include/glint_plug_streamer.h) over raw device pointers.
    Methods return the C return codes unchanged."""

    def __init__(self, layer_bytes, copy_stream, compute_stream):
        self.lib = p7_lib()
        self.h = VP()
        n = len(layer_bytes)
        arr = (ctypes.c_uint64 * n)(*layer_bytes)
        rc = self.lib.glint_plug_streamer_create(ctypes.byref(self.h), n, arr, VP(copy_stream.cuda_stream),
                                                 VP(compute_stream.cuda_stream))
        if rc != 0:
            raise RuntimeError(f"glint_plug_streamer_create rc={rc}")

    def set_host_data(self, layer: int, data: bytes) -> int:
        buf = ctypes.create_string_buffer(bytes(data), len(data))
        return self.lib.glint_plug_streamer_set_host_data(self.h, layer, buf, len(data))

    def start(self) -> int:
        return self.lib.glint_plug_streamer_start(self.h)

    def acquire(self, layer: int):
        p = VP()
        rc = self.lib.glint_plug_streamer_acquire(self.h, layer, ctypes.byref(p))
        return rc, p.value

    def release(self, layer: int) -> int:
        return self.lib.glint_plug_streamer_release(self.h, layer)

    def stats(self) -> GlintStreamerStats:
        st = GlintStreamerStats()
        _check(self.lib.glint_plug_streamer_get_stats(self.h, ctypes.byref(st)), "glint_plug_streamer_get_stats")
        return st

    def close(self) -> None:
        if self.h:
            self.lib.glint_plug_streamer_destroy(self.h)
            self.h = VP()


def p7_selftest():
    """p7_abi_selftest: (rc, message)."""
    msg = ctypes.create_string_buffer(512)
    rc = p7_lib().p7_abi_selftest(msg, 512)
    return rc, msg.value.decode()


def int8_gemm_i32(A, B, stream=None):
    M, K = A.shape
    N = B.shape[0]
    C = A.new_empty((M, N), dtype=_torch().int32)
    _check(p7_lib().glint_int8_gemm_i32(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, _sh(stream)),
           "glint_int8_gemm_i32")
    return C


def int8_gemm_scaled_bf16(A, B, sa, sb, out=None, stream=None):
    M, K = A.shape
    N = B.shape[0]
    out = A.new_empty((M, N), dtype=_torch().bfloat16) if out is None else out
    _check(p7_lib().glint_int8_gemm_scaled_bf16(A.data_ptr(), B.data_ptr(), sa.data_ptr(), sb.data_ptr(),
                                                out.data_ptr(), M, N, K, _sh(stream)), "glint_int8_gemm_scaled_bf16")
    return out


# ------------------------------------------------- between the linears (glint_serve.h)
# Every helper here takes stream= (default: the current stream).
KV_PAGE = 64

# With a stream given, a helper's whole call (its outputs, scratch and copies too) belongs to it.


def _refuse_devices(*tensors) -> None:
    raise ValueError(f"tensors on {', '.join(str(t.device) for t in tensors)}: all must be on the GPU")


class Kv4Cache(NamedTuple):
    """The 4-bit key/value cache's planes (glint_serve.h); any four tensors in this order do."""
    k_hole: "object"    # u8 [pages, H, 64, D / 2]
    k_absmax: "object"  # f32 [pages, H, D / 64, 64]
    v_hole: "object"    # u8 [pages, H, D / 2, 64]
    v_absmax: "object"  # f32 [pages, H, D / 64, 64]


def kv4_cache(pages: int, heads: int, dim: int, device="cuda") -> Kv4Cache:
    """An empty cache of pages of 64 tokens (every element zero)."""
    torch = _torch()
    if dim not in (64, 128):
        raise ValueError(f"head dimension {dim}: 64 or 128")
    scales = lambda: torch.zeros((pages, heads, dim // 64, KV_PAGE), dtype=torch.float32, device=device)
    return Kv4Cache(torch.zeros((pages, heads, KV_PAGE, dim // 2), dtype=torch.uint8, device=device), scales(),
                    torch.zeros((pages, heads, dim // 2, KV_PAGE), dtype=torch.uint8, device=device), scales())


def _planes(cache):
    """(pages, H, D, the four data pointers) of a cache whose planes agree."""
    kh, ka, vh, va = cache
    if not (kh.is_cuda and ka.is_cuda and vh.is_cuda and va.is_cuda):
        _refuse_devices(kh, ka, vh, va)
    torch = _TORCH or _torch()
    pages, heads, page, half = kh.shape
    scales = (pages, heads, half // 32, page)
    if page != KV_PAGE or half not in (32, 64) or vh.shape != (pages, heads, half, page) or ka.shape != scales or \
            va.shape != scales:
        raise ValueError(f"cache planes {tuple(kh.shape)}, {tuple(ka.shape)}, {tuple(vh.shape)}, {tuple(va.shape)}")
    if not (kh.dtype is torch.uint8 and vh.dtype is torch.uint8 and ka.dtype is torch.float32 and
            va.dtype is torch.float32):
        raise TypeError("cache planes are uint8 holes and float32 absmax")
    if not (kh.is_contiguous() and ka.is_contiguous() and vh.is_contiguous() and va.is_contiguous()):
        raise ValueError("cache planes are contiguous")
    return pages, heads, 2 * half, kh.data_ptr(), ka.data_ptr(), vh.data_ptr(), va.data_ptr()


def _rows(t, align: int, low: int = 0, high: int = 1 << 62):
    """A [tokens, heads, D] tensor whose rows the kernels can load, its tokens' and its heads' stride: itself, or a
    contiguous one where D is strided, an address or stride is no multiple of `align` elements or the tokens' stride
    lies outside low .. high. A contiguous tensor's strides are counted, not asked for: torch leaves any number on a
    dimension of one."""
    st, sh, sd = t.stride()
    if sd != 1 or st % align or sh % align or t.data_ptr() % (align * t.element_size()) or not low <= st <= high:
        t = t.contiguous()
        if t.data_ptr() % (align * t.element_size()):
            t = t.clone()
        _, heads, dim = t.shape
        st, sh = heads * dim, dim
    return t, st, sh


def _kv_elt(t) -> int:
    torch = _TORCH or _torch()
    if t.dtype is torch.bfloat16:
        return 0
    if t.dtype is torch.float32:
        return 1
    raise TypeError(f"expected bfloat16 or float32, got {t.dtype}")


def _ints(t, dtype, n: int, what: str):
    """t's data pointer, for a contiguous vector of n."""
    if t.dtype is not dtype or t.dim() != 1 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} vector of {n}, got {t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


def kv4_append(k, v, slots, cache, stream=None) -> None:
    """Encode keys and values [T, H, D] (bf16 or f32) into the cache at slots [T] (int64: page * 64
    + place; negative ones are skipped)."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return kv4_append(k, v, slots, cache)
    torch = _TORCH or _torch()
    pages, heads, dim, *planes = _planes(cache)
    T = k.shape[0]
    if k.shape != (T, heads, dim) or v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError(f"k {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}, cache of {heads} heads of {dim}")
    elt = _kv_elt(k)
    if not (k.is_cuda and v.is_cuda and slots.is_cuda):
        _refuse_devices(k, v, slots)
    k, kt, kh = _rows(k, 4)
    v, vt, vh = _rows(v, 4)
    at = _ints(slots, torch.int64, T, "slots")
    if T == 0:
        return
    _check(serve_lib().glint_kv4_append(k.data_ptr(), v.data_ptr(), elt, kt, kh, vt, vh, at, T, heads, dim, *planes,
                                        pages, _sh(None)), "glint_kv4_append")


def kv4_gather(slots, cache, out=None, stream=None):
    """The cache's tokens at slots [T] (int64) as bf16 (k, v), each [T, H, D]; zeros for negative slots."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return kv4_gather(slots, cache, out)
    torch = _TORCH or _torch()
    pages, heads, dim, *planes = _planes(cache)
    T = slots.numel()
    if not slots.is_cuda:
        _refuse_devices(slots)
    at = _ints(slots, torch.int64, T, "slots")
    if out is None:
        k = slots.new_empty((T, heads, dim), dtype=torch.bfloat16)
        v = torch.empty_like(k)
    else:
        k, v = out
        if any(t.shape != (T, heads, dim) or t.dtype is not torch.bfloat16 or not t.is_contiguous() or not t.is_cuda
               for t in (k, v)):
            raise ValueError(f"out: two contiguous bfloat16 tensors of {(T, heads, dim)} on the GPU")
    if T:
        _check(serve_lib().glint_kv4_gather(at, T, heads, dim, *planes, pages, k.data_ptr(), v.data_ptr(), _sh(None)),
               "glint_kv4_gather")
    return k, v


def _bounds(window: Optional[int], sinks: int):
    """window and sinks as the C entry points take them."""
    if window is None:
        if sinks:
            raise ValueError(f"{sinks} sinks without a window")
        return 0, 0
    if not 1 <= window <= 1 << 30 or sinks < 0:
        raise ValueError(f"window {window}, sinks {sinks}: a window of 1 .. 2^30, sinks of 0 or more")
    return window, min(sinks, (1 << 31) - 1)


def kv4_attend(q, cache, page_table, lens, cu_q=None, max_q: Optional[int] = None, scale: Optional[float] = None, out=None,
               stream=None, *, window: Optional[int] = None, sinks: int = 0):
    """Attention of the newest tokens over the cache: q bf16 [rows, Hq, D] -> bf16 [rows, Hq, D].

    page_table int32 [B, max_pages] and lens int32 [B] (tokens in the cache, the new ones
    included) say what each sequence sees; its rows are cu_q[b] .. cu_q[b + 1] (int32, at most
    max_q each: all rows where None), or max_q each (1 where None) where cu_q is None. A row sees
    the positions up to its own; with a window, the last `window` of them and the first `sinks`
    positions, and pages that no row sees may have left the table. Rows past max_q, or of no sequence,
    are not written: they hold what `out` held, anything where it is None."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return kv4_attend(q, cache, page_table, lens, cu_q, max_q, scale, out, window=window, sinks=sinks)
    window, sinks = _bounds(window, sinks)
    torch = _TORCH or _torch()
    pages, heads, dim, *planes = _planes(cache)
    rows, hq, d = q.shape
    B, wide = page_table.shape
    if not (q.is_cuda and page_table.is_cuda and lens.is_cuda and (cu_q is None or cu_q.is_cuda)):
        _refuse_devices(q, page_table, lens, lens if cu_q is None else cu_q)
    if d != dim or hq % heads:
        raise ValueError(f"q {tuple(q.shape)}, cache of {heads} heads of {dim}")
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"expected bfloat16, got {q.dtype}")
    if max_q is None:
        max_q = max(rows, 1) if cu_q is not None else 1
    if max_q < 1 or (cu_q is None and rows != B * max_q):
        raise ValueError(f"{rows} query rows, {B} sequences of {max_q}")
    if page_table.dtype is not torch.int32 or (page_table.stride(1) != 1 and wide > 1):
        raise ValueError("page_table: int32 with adjacent columns")
    q, qt, qh = _rows(q, 8)
    n = _ints(lens, torch.int32, B, "lens")
    cu = None if cu_q is None else _ints(cu_q, torch.int32, B + 1, "cu_q")
    out = _attend_out(out, q, rows, hq, dim)
    if rows == 0 or B == 0:
        return out
    if wide == 0:  # nobody has a page
        page_table, wide = page_table.new_full((B, 1), -1), 1
    _check(serve_lib().glint_kv4_attend_window(q.data_ptr(), qt, qh, rows, *planes, pages, page_table.data_ptr(),
                                               page_table.stride(0), wide, n, cu, B, max_q, hq, heads, dim,
                                               dim ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
                                               _sh(None)), "glint_kv4_attend")
    return out


def kv4_attend_chunk(q, cache, page_table, lens, cu_q=None, max_q: Optional[int] = None, scale: Optional[float] = None,
                     out=None, stream=None, *, k=None, v=None, window: Optional[int] = None, sinks: int = 0):
    """kv4_attend for many new tokens a sequence: arguments, masks and result as there.

    k, v bf16 [rows, H, D], both or neither: the new tokens' own keys and values, seen in place of what the
    cache holds of them (which may then be nothing). max_q times the query heads of a key head: at most 2^18. out overlaps
    no input."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return kv4_attend_chunk(q, cache, page_table, lens, cu_q, max_q, scale, out, k=k, v=v, window=window, sinks=sinks)
    torch = _TORCH or _torch()
    window, sinks = _bounds(window, sinks)
    _here(q, page_table, lens, cu_q, k, v, out, *cache)
    pages, heads, dim, *planes = _planes(cache)
    rows, hq, d = q.shape
    B, wide = page_table.shape
    if d != dim or hq % heads:
        raise ValueError(f"q {tuple(q.shape)}, cache of {heads} heads of {dim}")
    if (k is None) != (v is None):
        raise ValueError("k and v: both or neither")
    if k is not None and not k.shape == v.shape == (rows, heads, dim):
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}: both {(rows, heads, dim)}")
    if any(t is not None and t.dtype is not torch.bfloat16 for t in (q, k, v)):
        raise TypeError(f"expected bfloat16, got {', '.join(str(t.dtype) for t in (q, k, v) if t is not None)}")
    if max_q is None:
        max_q = max(rows, 1) if cu_q is not None else 1
    if max_q < 1 or (cu_q is None and rows != B * max_q):
        raise ValueError(f"{rows} query rows, {B} sequences of {max_q}")
    if page_table.dtype is not torch.int32 or (page_table.stride(1) != 1 and wide > 1):
        raise ValueError("page_table: int32 with adjacent columns")
    n = _ints(lens, torch.int32, B, "lens")
    cu = None if cu_q is None else _ints(cu_q, torch.int32, B + 1, "cu_q")
    q, qt, qh = _rows(q, 8)
    kt = kh = vt = vh = 0
    if k is not None:
        k, kt, kh = _rows(k, 8, dim, 1 << 24)
        v, vt, vh = _rows(v, 8, dim, 1 << 24)
    if out is not None and out.data_ptr() % 16:
        raise ValueError("out: 16-B aligned")
    out = _attend_out(out, q, rows, hq, dim)
    if rows == 0 or B == 0:
        return out
    if wide == 0:  # nobody has a page
        page_table, wide = page_table.new_full((B, 1), -1), 1
    size = serve_lib().glint_kv4_attend_chunk_scratch(B, max_q, hq, heads, dim, wide, k is not None)
    if size < 0:
        raise ValueError(f"{max_q} new tokens a sequence, {hq} heads over {heads}, {wide} pages: more than a launch can hold")
    scratch = q.new_empty(size, dtype=torch.uint8) if size else None
    _check(serve_lib().glint_kv4_attend_chunk(
        q.data_ptr(), qt, qh, rows, *planes, pages, page_table.data_ptr(), page_table.stride(0), wide, n, cu, B, max_q, hq,
        heads, dim, None if k is None else k.data_ptr(), kt, kh, None if v is None else v.data_ptr(), vt, vh,
        dim ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
        scratch.data_ptr() if size else None, size, _sh(None)),
        "glint_kv4_attend_chunk")
    return out


def _attend_out(out, q, rows: int, hq: int, dim: int):
    if out is None:
        return q.new_empty((rows, hq, dim))
    if out.shape != (rows, hq, dim) or out.dtype is not q.dtype or not out.is_contiguous() or not out.is_cuda:
        raise ValueError(f"out: a contiguous bfloat16 tensor of {(rows, hq, dim)} on the GPU")
    return out


def attend_prompt(q, k, v, cu_q, cu_k=None, max_q: Optional[int] = None, scale: Optional[float] = None, out=None,
                  stream=None, *, window: Optional[int] = None, sinks: int = 0):
    """Causal attention over packed sequences: q bf16 [Tq, Hq, D], k and v bf16 [Tk, H, D] -> bf16 [Tq, Hq, D].

    cu_q, cu_k int32 [B + 1]: where each sequence's queries and keys start (cu_k is cu_q where
    None); a sequence's last query sees its last key. With a window a query sees the last `window`
    keys up to its own and its sequence's first `sinks`. max_q: no sequence has more queries (Tq where None). Queries past max_q, or of no sequence, are not written: they hold what `out`
    held, anything where it is None."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return attend_prompt(q, k, v, cu_q, cu_k, max_q, scale, out, window=window, sinks=sinks)
    window, sinks = _bounds(window, sinks)
    torch = _TORCH or _torch()
    Tq, hq, dim = q.shape
    Tk, heads, _ = k.shape
    if not (q.is_cuda and k.is_cuda and v.is_cuda and cu_q.is_cuda and (cu_k is None or cu_k.is_cuda)):
        _refuse_devices(q, k, v, cu_q, cu_q if cu_k is None else cu_k)
    if k.shape != v.shape or k.shape[2] != dim or heads == 0 or hq % heads:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    if any(t.dtype is not torch.bfloat16 for t in (q, k, v)):
        raise TypeError(f"expected bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    B = cu_q.numel() - 1
    cq = _ints(cu_q, torch.int32, B + 1, "cu_q")
    ck = cq if cu_k is None else _ints(cu_k, torch.int32, B + 1, "cu_k")
    q, qt, qh = _rows(q, 8)
    k, kt, kh = _rows(k, 8, dim, 1 << 24)
    v, vt, vh = _rows(v, 8, dim, 1 << 24)
    out = _attend_out(out, q, Tq, hq, dim)
    if Tq == 0 or B <= 0:
        return out
    if Tk == 0:  # an address for the kernel, which reads no key
        k, v = q, q
    _check(serve_lib().glint_attend_prompt_window(q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, cq, ck,
                                                  Tq, Tk, B, Tq if max_q is None else max_q, hq, heads, dim,
                                                  dim ** -0.5 if scale is None else scale, window, sinks, out.data_ptr(),
                                                  _sh(None)), "glint_attend_prompt")
    return out


def rotary_freqs(rot: int, base: float = 10000.0, factor: float = 1.0, trained: Optional[int] = None, slow: float = 1.0,
                 fast: float = 4.0, device="cuda"):
    """Frequencies for rotate_qk, float64 [rot / 2] in radians a position: base^(-2 i / rot), divided by
    `factor`; with `trained` (a context length) only those that turn less than `slow` times in it, while those
    that turn `fast` times or more stay and the ones between are mixed. Any others do as well."""
    torch = _torch()
    if rot < 16 or rot % 16:
        raise ValueError(f"{rot} turned dimensions: a multiple of 16")
    f = base ** (torch.arange(rot // 2, dtype=torch.float64) * (-2.0 / rot))
    keep = torch.zeros_like(f)
    if trained is not None:
        if not fast > slow:
            raise ValueError(f"turns from {slow} to {fast}")
        keep = ((trained * f / 6.283185307179586 - slow) / (fast - slow)).clamp(0, 1)
    return (f * keep + f / factor * (1 - keep)).to(device)


def _here(*tensors) -> None:
    """Refuses tensors that are not on the current device; None among them is no tensor."""
    at = (_TORCH or _torch())._C._cuda_getDevice() if tensors[0].is_cuda else -2
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"a tensor on {t.device}: all must be on the current GPU")


def _turn_args(q, k, pos, freqs, q_norm, k_norm):
    """What rotate_qk and kv4_append_rotated have in common: (elt, T, Hq, H, D, rot, pos, freqs, the norms' pointers and type)."""
    torch = _TORCH or _torch()
    T, hq, dim = q.shape
    kT, heads, kdim = k.shape if k.dim() == 3 else (-1, 0, 0)
    if kT != T or kdim != dim or k.dtype is not q.dtype:
        raise ValueError(f"q {tuple(q.shape)} {q.dtype}, k {tuple(k.shape)} {k.dtype}")
    elt, rot = _kv_elt(q), 2 * freqs.numel()
    if dim & 15 or not 16 <= dim <= 256 or rot & 15 or not 16 <= rot <= dim:
        raise ValueError(f"head dimension {dim}, {rot} of it turned: multiples of 16, at most 256")
    at, fr = _ints(pos, torch.int64, T, "pos"), _ints(freqs, torch.float64, rot // 2, "freqs")
    qn = kn = None
    norm_elt = 0
    if q_norm is not None:
        qn, norm_elt = _norm(q_norm, dim)
    if k_norm is not None:
        kn, norm_elt = _norm(k_norm, dim)
        if q_norm is not None and q_norm.dtype is not k_norm.dtype:
            raise TypeError(f"norms of {q_norm.dtype} and {k_norm.dtype}")
    return elt, T, hq, heads, dim, rot, at, fr, qn, kn, norm_elt


def _norm(w, dim: int):
    at = w.data_ptr()
    if w.dim() != 1 or w.numel() != dim or not w.is_contiguous() or at & 15:
        raise ValueError(f"a norm: a contiguous, 16-B aligned vector of {dim}, got {tuple(w.shape)}")
    return at, _kv_elt(w)


def _turn_out(out, like, shape):
    if out is None:
        return like.new_empty(shape)
    if out.shape != shape or out.dtype is not like.dtype or not out.is_contiguous() or out.data_ptr() % 16 or \
            out.device != like.device:
        raise ValueError(f"out: a contiguous, 16-B aligned {like.dtype} tensor of {shape} beside q and k")
    return out


def rotate_qk(q, k, pos, freqs, *, interleaved: bool = False, magnitude: float = 1.0, q_norm=None, k_norm=None,
              eps: float = 1e-6, out=None, stream=None):
    """Queries [T, Hq, D] and keys [T, H, D] (bf16 or f32), normed per head and turned to positions pos [T]
    (int64): (q, k) of the same types and shapes.

    freqs float64 [rot / 2] (rotary_freqs, or any): the first rot dimensions turn, pair i by the angle
    pos * freqs[i], pairs being (i, i + rot / 2), or (2 i, 2 i + 1) where interleaved; turned dimensions are
    multiplied by `magnitude`. q_norm, k_norm [D] (bf16 or f32): each row is first divided by the root of its mean
    square (plus eps) and multiplied by them; None: as it is. out: (q, k) to write, which may be the inputs
    where those are contiguous."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return rotate_qk(q, k, pos, freqs, interleaved=interleaved, magnitude=magnitude, q_norm=q_norm, k_norm=k_norm,
                             eps=eps, out=out)
    _here(q, k, pos, freqs, q_norm, k_norm)
    elt, T, hq, heads, dim, rot, at, fr, qn, kn, ne = _turn_args(q, k, pos, freqs, q_norm, k_norm)
    q_out, k_out = (None, None) if out is None else out
    q_out, k_out = _turn_out(q_out, q, (T, hq, dim)), _turn_out(k_out, k, (T, heads, dim))
    if T == 0:
        return q_out, k_out
    q, qt, qh = _rows(q, 4 if elt else 8)
    k, kt, kh = _rows(k, 4 if elt else 8)
    _check(serve_lib().glint_rotate_qk(q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, elt, at, fr, T, hq, heads, dim, rot,
                                       interleaved, magnitude, qn, kn, ne, eps, q_out.data_ptr(), k_out.data_ptr(),
                                       _sh(None)), "glint_rotate_qk")
    return q_out, k_out


def kv4_append_rotated(q, k, v, pos, freqs, slots, cache, *, interleaved: bool = False, magnitude: float = 1.0, q_norm=None,
                       k_norm=None, eps: float = 1e-6, keys: bool = False, out=None, stream=None):
    """rotate_qk and kv4_append in one launch: the turned keys, and the values [T, H, D], go into the cache at slots
    [T] (int64; negative ones are skipped). The turned queries, or (queries, keys) with keys=True; out: the
    tensor, or both, to write."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return kv4_append_rotated(q, k, v, pos, freqs, slots, cache, interleaved=interleaved, magnitude=magnitude,
                                      q_norm=q_norm, k_norm=k_norm, eps=eps, keys=keys, out=out)
    torch = _TORCH or _torch()
    _here(q, k, v, pos, freqs, slots, q_norm, k_norm, *cache)
    pages, cache_heads, cache_dim, *planes = _planes(cache)
    elt, T, hq, heads, dim, rot, at, fr, qn, kn, ne = _turn_args(q, k, pos, freqs, q_norm, k_norm)
    if heads != cache_heads or dim != cache_dim or v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)} {v.dtype}, cache of {cache_heads} heads of {cache_dim}")
    sl = _ints(slots, torch.int64, T, "slots")
    q_out, k_out = out if keys and out is not None else (out, None)
    q_out = _turn_out(q_out, q, (T, hq, dim))
    k_out = _turn_out(k_out, k, (T, heads, dim)) if keys else None
    if T:
        q, qt, qh = _rows(q, 4 if elt else 8)
        k, kt, kh = _rows(k, 4 if elt else 8)
        v, vt, vh = _rows(v, 4 if elt else 8)
        _check(serve_lib().glint_kv4_append_rotated(
            q.data_ptr(), qt, qh, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, elt, at, fr, sl, T, hq, heads, dim, rot,
            interleaved, magnitude, qn, kn, ne, eps, q_out.data_ptr(), k_out.data_ptr() if keys else None, *planes, pages,
            _sh(None)), "glint_kv4_append_rotated")
    return (q_out, k_out) if keys else q_out


def token_logprobs(logits, tokens, top: int = 0, stream=None) -> dict:
    """Scores of tokens [T] (int64) under logits [T, V] (bf16 or f32): f32 "logprob" and "entropy"
    [T], int32 "rank" [T] (entries ahead of the token; 0 where it is the likeliest), and the
    `top` likeliest entries, "top_logprob" f32 and "top_index" int32 [T, top], equal ones by
    index. A negative token gives logprob 0 and rank -1."""
    if stream is not None:
        with _torch().cuda.stream(stream):
            return token_logprobs(logits, tokens, top)
    torch = _TORCH or _torch()
    T, V = logits.shape
    elt = _kv_elt(logits)
    if not (logits.is_cuda and tokens.is_cuda):
        _refuse_devices(logits, tokens)
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    at = _ints(tokens, torch.int64, T, "tokens")
    logprob = logits.new_empty(T, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    rank = logits.new_empty(T, dtype=torch.int32)
    top_logprob = logits.new_empty((T, top), dtype=torch.float32)
    top_index = logits.new_empty((T, top), dtype=torch.int32)
    if T:
        _check(serve_lib().glint_token_logprobs(logits.data_ptr(), elt, logits.stride(0), at, T, V, top,
                                                logprob.data_ptr(), entropy.data_ptr(), rank.data_ptr(),
                                                top_logprob.data_ptr(), top_index.data_ptr(), _sh(None)),
               "glint_token_logprobs")
    return {"logprob": logprob, "entropy": entropy, "rank": rank, "top_logprob": top_logprob, "top_index": top_index}


# ------------------------------------------------------------- host-pointer wrappers
def encode_bf16_host(raw_bf16: bytes, n: int, blocksize: int = 64) -> Tuple[bytes, bytes, bytes]:
    """Same contract as the reference's glint_cuda.encode_bf16_cuda (glint_cuda.py:52-65)."""
    lib = encode_lib()
    n_am = lib.glint_encode_n_absmax(n, blocksize)
    n_pk = lib.glint_encode_n_packed(n)
    hole = (_c.c_uint8 * n_pk)()
    plug = (_c.c_uint8 * n_pk)()
    am = (_c.c_float * n_am)()
    buf = (_c.c_uint16 * n).from_buffer_copy(raw_bf16[: n * 2])
    rc = lib.glint_encode_bf16_host(_c.byref(buf), n, blocksize, hole, plug, am)
    if rc != 0:
        raise RuntimeError(f"glint_encode_bf16_host rc={rc}")
    return bytes(hole), bytes(plug), bytes(_c.string_at(_c.addressof(am), n_am * 4))


def expand_host(hole: bytes, plug: bytes, absmax_f32: bytes, n: int, blocksize: int = 64) -> bytes:
    """Same contract as the reference's glint_cuda.expand_cuda (glint_cuda.py:66-78)."""
    lib = encode_lib()
    out = (_c.c_float * n)()
    h = _c.create_string_buffer(bytes(hole), len(hole))
    p = _c.create_string_buffer(bytes(plug), len(plug))
    a = _c.create_string_buffer(bytes(absmax_f32), len(absmax_f32))
    rc = lib.glint_expand_packed_to_f32_host(h, p, a, n, blocksize, out)
    if rc != 0:
        raise RuntimeError(f"glint_expand_packed_to_f32_host rc={rc}")
    return bytes(_c.string_at(_c.addressof(out), n * 4))


def expand_bf16_host(hole: bytes, plug: bytes, absmax_f32: bytes, n: int, blocksize: int = 64) -> bytes:
    lib = encode_lib()
    out = (_c.c_uint16 * n)()
    h = _c.create_string_buffer(bytes(hole), len(hole))
    p = _c.create_string_buffer(bytes(plug), len(plug))
    a = _c.create_string_buffer(bytes(absmax_f32), len(absmax_f32))
    rc = lib.glint_expand_packed_to_bf16_host(h, p, a, n, blocksize, out)
    if rc != 0:
        raise RuntimeError(f"glint_expand_packed_to_bf16_host rc={rc}")
    return bytes(_c.string_at(_c.addressof(out), n * 2))
