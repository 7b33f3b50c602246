"""Kernel-level building blocks over torch CUDA tensors (thin ctypes wrappers).

Each function checks shapes/dtypes/devices, allocates its outputs with torch
and calls the matching ``libtj.so`` entry point on the current stream.  These
are the same kernels ``tj_forward`` chains; they are exposed for tests,
profiling and callers composing their own pipelines.

The training and 8-bit operators (from ``Act8`` on) are the exception: the
forward does not call them, a caller that trains or runs 8-bit products does.
Their row masks are bool tensors with one element per row (``MaskInfo.mask``
serves); masked rows are not read, leave zeros in row-shaped outputs and
nothing in sums.  Gradients are returned, not accumulated into anything.
"""

from __future__ import annotations

import ctypes
import threading
from typing import NamedTuple, Optional

import torch

from . import _lib


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _need_cuda(*ts):
    for t in ts:
        if t is not None and (t.device.type != "cuda" or not t.is_contiguous()):
            raise ValueError("techjam_b200.ops needs contiguous CUDA tensors")


class MaskInfo(NamedTuple):
    lengths: torch.Tensor     # int32 [B]
    general: torch.Tensor     # uint8 [B]
    tile_list: torch.Tensor   # int32 [n_tiles]
    n_live: torch.Tensor      # int32 [1]
    tile_live: torch.Tensor   # uint8 [n_tiles]
    mask: Optional[torch.Tensor]
    batch: int
    seq_len: int


def prepare_mask(mask: Optional[torch.Tensor], batch: int, seq_len: int, device=None) -> MaskInfo:
    """Per-sample valid lengths, non-prefix flags and the live 128-row tile list."""
    if mask is not None:
        _need_cuda(mask)
        if mask.dtype != torch.bool or mask.shape != (batch, seq_len):
            raise ValueError("mask must be bool [B, N]")
        device = mask.device
    device = torch.device(device or "cuda")
    n_tiles = (batch * seq_len + 127) // 128
    lengths = torch.empty(batch, dtype=torch.int32, device=device)
    general = torch.empty(batch, dtype=torch.uint8, device=device)
    tile_list = torch.zeros(max(n_tiles, 1), dtype=torch.int32, device=device)
    n_live = torch.zeros(1, dtype=torch.int32, device=device)
    tile_live = torch.zeros(max(n_tiles, 1), dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        _lib.call("tj_prepare_mask", _ptr(mask), batch, seq_len, lengths.data_ptr(), general.data_ptr(),
                  tile_list.data_ptr(), n_live.data_ptr(), tile_live.data_ptr(), _stream(lengths))
    return MaskInfo(lengths, general, tile_list, n_live, tile_live, mask, batch, seq_len)


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, info: MaskInfo, eps: float = 1e-5,
              out_fp16: bool = True) -> torch.Tensor:
    """LayerNorm of x [B*N, d] (fp32); invalid rows are written as zeros."""
    _need_cuda(x, weight, bias)
    rows, d = x.shape
    if rows != info.batch * info.seq_len:
        raise ValueError("x rows must equal B*N")
    out = torch.zeros(rows, d, dtype=torch.float16 if out_fp16 else torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.call("tj_layernorm", x.data_ptr(), weight.data_ptr(), bias.data_ptr(), info.batch, info.seq_len, d,
                  float(eps), out.data_ptr(), int(out_fp16), info.lengths.data_ptr(), _ptr(info.mask),
                  info.tile_live.data_ptr(), _stream(x))
    return out


def gemm(a: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, info: MaskInfo, epilogue: int,
         resid: Optional[torch.Tensor] = None, heads: int = 0, err: Optional[torch.Tensor] = None):
    """tcgen05 GEMM ``a @ w.T + bias`` (fp16 operands, fp32 accumulate) with a fused epilogue.

    Returns fp16 [M, N] (GELU/plain), fp32 [M, N] (residual) or a (q, k, v)
    tuple of fp16 [B, H, N, hd] (QKV scatter).
    """
    _need_cuda(a, w, bias, resid)
    if a.dtype != torch.float16 or w.dtype != torch.float16 or bias.dtype != torch.float32:
        raise ValueError("a, w must be fp16 and bias fp32")
    m, k = a.shape
    n = w.shape[0]
    if w.shape[1] != k or bias.shape != (n,) or m != info.batch * info.seq_len:
        raise ValueError("shape mismatch")
    err = err if err is not None else torch.zeros(1, dtype=torch.int32, device=a.device)
    out = q = kk = v = None
    if epilogue == _lib.EPI_QKV:
        d = n // 3
        hd = d // heads
        q, kk, v = (torch.zeros(info.batch, heads, info.seq_len, hd, dtype=torch.float16, device=a.device)
                    for _ in range(3))
    elif epilogue == _lib.EPI_RESID:
        out = torch.empty(m, n, dtype=torch.float32, device=a.device)
        if resid is None:
            raise ValueError("residual epilogue needs resid")
    else:
        out = torch.empty(m, n, dtype=torch.float16, device=a.device)
    with torch.cuda.device(a.device):
        _lib.call("tj_gemm_f16", a.data_ptr(), w.data_ptr(), bias.data_ptr(), info.batch, info.seq_len, n, k,
                  epilogue, _ptr(out), _ptr(resid), _ptr(q), _ptr(kk), _ptr(v), heads, info.tile_list.data_ptr(),
                  info.n_live.data_ptr(), info.lengths.data_ptr(), _ptr(info.mask), err.data_ptr(), _stream(a))
    return (q, kk, v) if epilogue == _lib.EPI_QKV else out


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, info: MaskInfo, causal: bool,
              err: Optional[torch.Tensor] = None, sched: Optional[torch.Tensor] = None,
              dynamic: bool = True) -> torch.Tensor:
    """Flash attention over fp16 [B, H, N, hd]; returns the fp16 context [B*N, H*hd].

    ``sched``: two zeroed int32 words for the dynamic work scheduler (made
    here when not given); ``dynamic=False`` uses the static item assignment.
    """
    _need_cuda(q, k, v)
    b, h, n, hd = q.shape
    if q.dtype != torch.float16 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must be fp16 [B, H, N, hd]")
    err = err if err is not None else torch.zeros(1, dtype=torch.int32, device=q.device)
    if dynamic and sched is None:
        sched = torch.zeros(2, dtype=torch.int32, device=q.device)
    ctx = torch.zeros(b * n, h * hd, dtype=torch.float16, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("tj_attention_f16", q.data_ptr(), k.data_ptr(), v.data_ptr(), ctx.data_ptr(), b, h, n, hd,
                  int(causal), info.lengths.data_ptr(), _ptr(info.mask), info.general.data_ptr(), err.data_ptr(),
                  _ptr(sched) if dynamic else None, _stream(q))
    return ctx


class PolyStatus(NamedTuple):
    admit: bool
    c0: float
    c1: float
    c2: float
    sigma: float
    max_abs: float


def poly_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, exact_prefix: int = 4096,
                   err: Optional[torch.Tensor] = None):
    """Guarded polynomial causal attention (head_dim 64, no padding).

    Returns (ctx fp16 [B*N, H*64], PolyStatus).  Queries below ``exact_prefix``
    -- or all of them if the device-side guard rejects the route -- come from
    the exact flash kernel.
    """
    _need_cuda(q, k, v)
    b, h, n, hd = q.shape
    if hd != 64 or q.dtype != torch.float16 or k.shape != q.shape or v.shape != q.shape:
        raise ValueError("q, k, v must be fp16 [B, H, N, 64]")
    nbytes = ctypes.c_size_t()
    _lib.call("tj_poly_workspace_bytes", b, h, n, exact_prefix, ctypes.byref(nbytes))
    ws = torch.zeros(int(nbytes.value), dtype=torch.uint8, device=q.device)
    err = err if err is not None else torch.zeros(1, dtype=torch.int32, device=q.device)
    lengths = torch.full((b,), n, dtype=torch.int32, device=q.device)
    ctx = torch.zeros(b * n, h * hd, dtype=torch.float16, device=q.device)
    with torch.cuda.device(q.device):
        _lib.call("tj_poly_attention_f16", q.data_ptr(), k.data_ptr(), v.data_ptr(), ctx.data_ptr(),
                  lengths.data_ptr(), b, h, n, exact_prefix, ws.data_ptr(), ws.numel(), err.data_ptr(), _stream(q))
    head = ws[:24].cpu()
    admit = int(head[:4].view(torch.int32).item())
    c0, c1, c2, sigma, max_abs = (float(v) for v in head[4:24].view(torch.float32))
    return ctx, PolyStatus(bool(admit), c0, c1, c2, sigma, max_abs)


# ---------------------------------------------------------------- training and 8-bit activations

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_F32 = (torch.float32,)
_MAX = 0x7fffff00  # sizes that the entries take as int


class Act8(NamedTuple):
    """An activation [rows, cols] in 8 bits: e4m3 codes and a power-of-two
    scale for each row and run of 128 columns (value = code * scale)."""
    codes: torch.Tensor   # float8_e4m3fn [rows, cols]
    scales: torch.Tensor  # float8_e8m0fnu [rows, ceil(cols / 128)]
    dtype: torch.dtype    # the type the values came from, and restore8's default


class Weight8(NamedTuple):
    """A weight [n, k] in 8 bits: e4m3 codes and a scale per 128 x 128 block."""
    codes: torch.Tensor   # float8_e4m3fn [n, k]
    scales: torch.Tensor  # float8_e8m0fnu [ceil(n / 128), ceil(k / 128)]


class LayerNormOut(NamedTuple):
    y: object             # tensor [rows, d], or Act8
    mean: torch.Tensor    # fp32 [rows]
    rstd: torch.Tensor    # fp32 [rows]
    x8: Optional[Act8]    # 8-bit copy of the input, when asked for


# what a torch that lacks them needs only for the operators below (e8m0: from 2.7 on)
_E4M3, _E8M0 = getattr(torch, "float8_e4m3fn", None), getattr(torch, "float8_e8m0fnu", None)
# the handle and the index alone: the public forms build objects on each call
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_entries: dict = {}


def _need_8_bits():
    if _E4M3 is None or _E8M0 is None:
        raise RuntimeError(f"8-bit tensors need torch.float8_e4m3fn and torch.float8_e8m0fnu, which torch "
                           f"{torch.__version__} lacks")


def _run(index: int, name: str, *args) -> None:
    """Call an entry point on the current stream of CUDA device ``index``."""
    entry = _entries.get(name)
    if entry is None:
        entry = _entries[name] = getattr(_lib.load(), name)
    if _current_device() == index:
        status = entry(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            status = entry(*args, _stream_of(index))
    if status:
        _lib.check(status)


def _matrix(t: torch.Tensor, what: str, dtypes, shape=None, index: Optional[int] = None) -> int:
    """Check an operand ([rows, cols], or the given shape) and return its CUDA device's index."""
    at = t.get_device()
    if (at >= 0 and t.is_contiguous() and t.dtype in dtypes and (index is None or at == index)
            and (t.shape == shape if shape is not None else t.dim() == 2 and 0 < t.shape[1] < _MAX)):
        return at
    if at < 0 or not t.is_contiguous():
        raise ValueError(f"{what}: techjam_b200.ops needs contiguous CUDA tensors")
    if t.dtype not in dtypes:
        raise ValueError(f"{what}: dtype {t.dtype}, need one of {', '.join(map(str, dtypes))}")
    if index is not None and at != index:
        raise ValueError(f"{what}: on {t.device}, need cuda:{index}")
    if t.dim() == 2 and shape is None:
        raise ValueError(f"{what}: {t.shape[1]} columns")
    raise ValueError(f"{what}: shape {tuple(t.shape)}, need {'[rows, cols]' if shape is None else tuple(shape)}")


def _row_mask(mask: Optional[torch.Tensor], rows: int, index: int):
    if mask is None:
        return None
    if (mask.get_device() != index or not mask.is_contiguous() or mask.dtype != torch.bool or mask.numel() != rows):
        raise ValueError(f"mask must be a contiguous bool tensor with one element per row ({rows}) on cuda:{index}")
    return mask.data_ptr()


def _blocks(n: int) -> int:
    return (n + 127) // 128


def _check_act(a: Act8, what: str, index: Optional[int] = None):
    """Check an 8-bit activation; (device index, rows, cols)."""
    _need_8_bits()
    if not isinstance(a, Act8):
        raise ValueError(f"{what} must be an Act8")
    index = _matrix(a.codes, what, (_E4M3,), None, index)
    rows, cols = a.codes.shape
    _matrix(a.scales, what, (_E8M0,), (rows, _blocks(cols)), index)
    return index, rows, cols


def _new_act(rows: int, cols: int, device, dtype) -> Act8:
    _need_8_bits()
    return Act8(torch.empty(rows, cols, dtype=_E4M3, device=device),
                torch.empty(rows, _blocks(cols), dtype=_E8M0, device=device), dtype)


_err_words: dict = {}


def _err_word(index: int) -> torch.Tensor:
    """The device's error word of the operators that wait inside a kernel
    (one per device, kept; first used outside a stream capture)."""
    word = _err_words.get(index)
    if word is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("call this operator once on the device before capturing it")
        word = torch.zeros(1, dtype=torch.int32, device=torch.device("cuda", index))
        torch.cuda.current_stream(index).synchronize()
        word = _err_words.setdefault(index, word)
    return word


def _err_ptr(err: Optional[torch.Tensor], index: int) -> int:
    if err is None:
        return _err_word(index).data_ptr()
    _matrix(err, "err", (torch.int32,), (1,), index)
    return err.data_ptr()


_err_lock = threading.Lock()
_err_log: dict = {}            # device index: every site read from its word so far
_err_seen = threading.local()  # per thread and device: how much of the log it has been told


def device_error(device=None) -> int:
    """Read (synchronously) the error word that gemm8, gemm8_gelu and
    linear_wgrad share on a device: 0, or the site of the first bounded wait
    that expired since this thread's last call (the results of the call that
    waited are void, later ones are not affected).  Reading clears the word for
    the kernels to come, not for other threads: each is told."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    with _err_lock:
        word = _err_word(device.index)
        torch.cuda.synchronize(device)
        code = int(word.item())
        log = _err_log.setdefault(device.index, [])
        if code:
            log.append(code)
            word.zero_()
            torch.cuda.synchronize(device)  # zero before a call on any other stream can set it again
        seen = _err_seen.__dict__.setdefault("count", {})
        new = log[seen.get(device.index, 0):]
        seen[device.index] = len(log)
    return new[0] if new else 0


def checkpoint8(x: torch.Tensor, mask: Optional[torch.Tensor] = None) -> Act8:
    """x [rows, cols] (fp32, fp16 or bf16) into 8 bits.  A block's codes depend
    on its values alone; infinities and NaN become NaN."""
    index = _matrix(x, "x", _DTYPES)
    rows, cols = x.shape
    mptr = _row_mask(mask, rows, index)
    out = _new_act(rows, cols, x.device, x.dtype)
    _run(index, "tj_act8_pack", x.data_ptr(), _DTYPES[x.dtype], rows, cols, mptr, out.codes.data_ptr(),
         out.scales.data_ptr())
    return out


def restore8(a: Act8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values of an 8-bit activation: exact in fp32 and bf16 within their
    normal range, rounded in fp16; beyond a type's range its largest value."""
    index, rows, cols = _check_act(a, "a")
    dtype = a.dtype if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError(f"dtype {dtype}, need one of {', '.join(map(str, _DTYPES))}")
    out = torch.empty(rows, cols, dtype=dtype, device=a.codes.device)
    _run(index, "tj_act8_unpack", a.codes.data_ptr(), a.scales.data_ptr(), rows, cols, out.data_ptr(), _DTYPES[dtype])
    return out


def pack_weight8(w: torch.Tensor, transpose: bool = False) -> Weight8:
    """A weight [n, k] (fp32, fp16 or bf16) into 8 bits, or its transpose (for
    the product that takes a gradient back through the layer)."""
    _need_8_bits()
    index = _matrix(w, "w", _DTYPES)
    n, k = w.shape
    if not 0 < n < _MAX:
        raise ValueError(f"w: {n} rows")
    r, c = (k, n) if transpose else (n, k)
    out = Weight8(torch.empty(r, c, dtype=_E4M3, device=w.device),
                  torch.empty(_blocks(r), _blocks(c), dtype=_E8M0, device=w.device))
    _run(index, "tj_weight8_pack", w.data_ptr(), _DTYPES[w.dtype], n, k, int(transpose), out.codes.data_ptr(),
         out.scales.data_ptr())
    return out


def layernorm_train(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, mask: Optional[torch.Tensor] = None,
                    eps: float = 1e-5, out_dtype: torch.dtype = torch.float16,
                    checkpoint: bool = False) -> LayerNormOut:
    """LayerNorm of x [rows, d] (fp32, fp16 or bf16; d <= 4096) that keeps mean
    and 1/std for ``layernorm_backward``.  ``out_dtype`` torch.float8_e4m3fn
    gives y as an Act8; ``checkpoint`` also returns an 8-bit copy of x."""
    index = _matrix(x, "x", _DTYPES)
    rows, d = x.shape
    _matrix(weight, "weight", _F32, (d,), index)
    _matrix(bias, "bias", _F32, (d,), index)
    mptr = _row_mask(mask, rows, index)
    dev = x.device
    if out_dtype == _E4M3 and out_dtype is not None:
        y = _new_act(rows, d, dev, x.dtype)
        yp, ys, yd = y.codes.data_ptr(), y.scales.data_ptr(), _lib.E4M3
    elif out_dtype in _DTYPES:
        y = torch.empty(rows, d, dtype=out_dtype, device=dev)
        yp, ys, yd = y.data_ptr(), None, _DTYPES[out_dtype]
    else:
        raise ValueError(f"out_dtype {out_dtype} not supported")
    mean = torch.empty(rows, dtype=torch.float32, device=dev)
    rstd = torch.empty(rows, dtype=torch.float32, device=dev)
    x8 = _new_act(rows, d, dev, x.dtype) if checkpoint else None
    _run(index, "tj_layernorm_train", x.data_ptr(), _DTYPES[x.dtype], weight.data_ptr(), bias.data_ptr(), rows, d, eps,
         mptr, yp, yd, ys, mean.data_ptr(), rstd.data_ptr(), x8.codes.data_ptr() if checkpoint else None,
         x8.scales.data_ptr() if checkpoint else None)
    return LayerNormOut(y, mean, rstd, x8)


_workspace_sizes: dict = {}


def _workspace(name: str, device: torch.device, *sizes: int):
    """A fresh workspace from torch's allocator (so that calls on different
    streams, or captured into different graphs, never share one), its address
    and size; only the size that a shape needs is kept."""
    key = (name, device.index, sizes)
    n = _workspace_sizes.get(key)
    if n is None:
        nbytes = ctypes.c_size_t()
        with torch.cuda.device(device):
            _lib.call(name, *sizes, ctypes.byref(nbytes))
        if len(_workspace_sizes) >= 4096:
            _workspace_sizes.clear()
        n = _workspace_sizes[key] = int(nbytes.value)
    if n == 0:
        return None, None, 0
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), n


def layernorm_backward(dy: torch.Tensor, x, weight: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       mask: Optional[torch.Tensor] = None, resid_grad: Optional[torch.Tensor] = None):
    """Gradients (dx, dweight, dbias) of LayerNorm for dy [rows, d] (fp32, fp16
    or bf16).  x: the input or its 8-bit copy; dx has its type.  ``resid_grad``
    (x's type) is the gradient of the branch around the norm, added to dx."""
    index = _matrix(dy, "dy", _DTYPES)
    rows, d = shape = dy.shape
    if isinstance(x, Act8):
        if _check_act(x, "x", index)[1:] != shape:
            raise ValueError(f"x: shape {tuple(x.codes.shape)}, need {tuple(shape)}")
        if x.dtype not in _DTYPES:
            raise ValueError(f"x: dtype {x.dtype} not supported")
        xp, xs = x.codes.data_ptr(), x.scales.data_ptr()
    else:
        _matrix(x, "x", _DTYPES, shape, index)
        xp, xs = x.data_ptr(), None
    _matrix(weight, "weight", _F32, (d,), index)
    _matrix(mean, "mean", _F32, (rows,), index)
    _matrix(rstd, "rstd", _F32, (rows,), index)
    rp = None
    if resid_grad is not None:
        _matrix(resid_grad, "resid_grad", (x.dtype,), shape, index)
        rp = resid_grad.data_ptr()
    mptr = _row_mask(mask, rows, index)
    dev = dy.device
    dx = torch.empty(rows, d, dtype=x.dtype, device=dev)
    dweight = torch.empty(d, dtype=torch.float32, device=dev)
    dbias = torch.empty(d, dtype=torch.float32, device=dev)
    _ws, wp, wn = _workspace("tj_layernorm_backward_workspace_bytes", dev, rows, d)
    _run(index, "tj_layernorm_backward", dy.data_ptr(), _DTYPES[dy.dtype], xp, xs, weight.data_ptr(), mean.data_ptr(),
         rstd.data_ptr(), rows, d, mptr, rp, dx.data_ptr(), _DTYPES[x.dtype], dweight.data_ptr(), dbias.data_ptr(), wp,
         wn)
    return dx, dweight, dbias


def gelu_backward(dy: torch.Tensor, h, mask: Optional[torch.Tensor] = None, pack: bool = False):
    """dh = dy * gelu'(h) (exact GELU) for dy [rows, cols] (fp32, fp16 or
    bf16); h: the input of the GELU in dy's type, or its 8-bit copy.  ``pack``
    returns (dh, Act8 of dh) in one pass."""
    index = _matrix(dy, "dy", _DTYPES)
    rows, cols = shape = dy.shape
    if isinstance(h, Act8):
        if _check_act(h, "h", index)[1:] != shape:
            raise ValueError(f"h: shape {tuple(h.codes.shape)}, need {tuple(shape)}")
        hp, hs = h.codes.data_ptr(), h.scales.data_ptr()
    else:
        _matrix(h, "h", (dy.dtype,), shape, index)
        hp, hs = h.data_ptr(), None
    mptr = _row_mask(mask, rows, index)
    dh = torch.empty_like(dy)
    dh8 = _new_act(rows, cols, dy.device, dy.dtype) if pack else None
    _run(index, "tj_gelu_backward", dy.data_ptr(), _DTYPES[dy.dtype], hp, hs, rows, cols, mptr, dh.data_ptr(),
         dh8.codes.data_ptr() if pack else None, dh8.scales.data_ptr() if pack else None)
    return (dh, dh8) if pack else dh


def _check_product(a: Act8, w: Weight8, bias, what: str, step: int):
    index, m, k = _check_act(a, "a")
    if not isinstance(w, Weight8):
        raise ValueError("w must be a Weight8")
    _matrix(w.codes, "w", (_E4M3,), None, index)
    n, wk = w.codes.shape
    if wk != k:
        raise ValueError(f"w: shape {(n, wk)}, need [n, {k}]")
    if m > _MAX or n > _MAX:
        raise ValueError(f"{what}: {m} x {n} x {k} is too large")
    if n == 0 or n % step or k % 16:
        raise ValueError(f"{what} needs n % {step} == 0 and k % 16 == 0, got n {n}, k {k}")
    _matrix(w.scales, "w", (_E8M0,), (_blocks(n), _blocks(k)), index)
    if bias is None:
        return index, m, n, k, None
    _matrix(bias, "bias", _F32, (n,), index)
    return index, m, n, k, bias.data_ptr()


def gemm8(a: Act8, w: Weight8, bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
          resid: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float16,
          err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ w.T [+ bias] [+ resid] on 8-bit operands with FP32 sums; ``resid``
    (fp32 [m, n]) needs out_dtype torch.float32.  n % 8 == 0, k % 16 == 0.
    ``err``: the error word to use instead of the device's own."""
    index, m, n, k, bp = _check_product(a, w, bias, "gemm8", 8)
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype {out_dtype} not supported")
    rp = None
    if resid is not None:
        if out_dtype != torch.float32:
            raise ValueError("resid needs out_dtype torch.float32")
        _matrix(resid, "resid", _F32, (m, n), index)
        rp = resid.data_ptr()
    mptr = _row_mask(mask, m, index)
    ep = _err_ptr(err, index)
    out = torch.empty(m, n, dtype=out_dtype, device=a.codes.device)
    _run(index, "tj_gemm8", a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), bp, m, n, k,
         mptr, rp, out.data_ptr(), _DTYPES[out_dtype], ep)
    return out


def gemm8_gelu(a: Act8, w: Weight8, bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
               err: Optional[torch.Tensor] = None):
    """(gelu(h), h) in 8 bits for h = a @ w.T [+ bias]: the FFN-in layer, whose
    output feeds the next product and whose h serves ``gelu_backward``.
    n % 16 == 0, k % 16 == 0."""
    index, m, n, k, bp = _check_product(a, w, bias, "gemm8_gelu", 16)
    dev = a.codes.device
    mptr = _row_mask(mask, m, index)
    ep = _err_ptr(err, index)
    g, h = _new_act(m, n, dev, a.dtype), _new_act(m, n, dev, a.dtype)
    _run(index, "tj_gemm8_gelu", a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), bp, m,
         n, k, mptr, g.codes.data_ptr(), g.scales.data_ptr(), h.codes.data_ptr(), h.scales.data_ptr(), ep)
    return g, h


def linear_wgrad(dy: torch.Tensor, x: Act8, mask: Optional[torch.Tensor] = None,
                 err: Optional[torch.Tensor] = None):
    """Gradients (dweight [n, k], dbias [n], fp32) of a linear layer for dy
    [rows, n] (fp16 or bf16) and the 8-bit copy of its input [rows, k].  x
    enters the product in dy's type: exact in bf16, as ``restore8`` in fp16.
    n % 8 == 0, k % 16 == 0.  Takes a workspace of 2 * rows * k bytes and more."""
    index = _matrix(dy, "dy", (torch.float16, torch.bfloat16))
    rows, n = dy.shape
    _, xrows, k = _check_act(x, "x", index)
    if xrows != rows:
        raise ValueError(f"x: {xrows} rows, need {rows}")
    if n % 8 or k % 16:
        raise ValueError(f"linear_wgrad needs n % 8 == 0 and k % 16 == 0, got n {n}, k {k}")
    mptr = _row_mask(mask, rows, index)
    ep = _err_ptr(err, index)
    dev = dy.device
    dw = torch.empty(n, k, dtype=torch.float32, device=dev)
    db = torch.empty(n, dtype=torch.float32, device=dev)
    _ws, wp, wn = _workspace("tj_wgrad8_workspace_bytes", dev, rows, n, k)
    _run(index, "tj_wgrad8", dy.data_ptr(), _DTYPES[dy.dtype], x.codes.data_ptr(), x.scales.data_ptr(), rows, n, k, mptr,
         dw.data_ptr(), db.data_ptr(), wp, wn, ep)
    return dw, db
