"""Rows held in 8 bits: the format, the product with 8-bit weights, the weight gradient from 8-bit rows.

A row x is kept as whole numbers q in [-127, 127] and one float32 scale = max|x| / 127 (include/mpnn_amd.h has the
definition to the bit).  The reference keeps everything in float32 (models/layers.py:104,140); here the same Linear
calls can answer from 8-bit weights (``linear_int8``) or train while their inputs wait for the backward in 8 bits
(``dense.project`` / ``dense.update`` with ``checkpoint="int8"``).
"""
from __future__ import annotations

import torch

from . import _lib

MAX_WIDTH = 8192


class Rows8:
    """A matrix [N, K] whose rows are held in 8 bits: ``values`` int8 [N, K] and ``scale`` float32 [N].

    The rows of ``values`` start on 16-byte boundaries and whole 16-byte pieces of them can be read; what lies behind
    column K does not count.  A matrix that is laid out otherwise is copied once, here."""

    __slots__ = ("values", "scale")

    def __init__(self, values: torch.Tensor, scale: torch.Tensor):
        if values.dim() != 2 or values.dtype != torch.int8 or not 1 <= values.size(1) <= MAX_WIDTH:
            raise ValueError(f"values must be int8 [N, K] with 1 <= K <= {MAX_WIDTH}, got {values.dtype} {tuple(values.shape)}")
        if scale.dtype != torch.float32 or scale.shape != (values.size(0),) or scale.device != values.device:
            raise ValueError(f"scale must be float32 [{values.size(0)}] on {values.device}, got {scale.dtype} "
                             f"{tuple(scale.shape)} on {scale.device}")
        self.values = values if _in_place(values) else _padded(values)
        self.scale = scale.contiguous()

    @property
    def shape(self):
        return self.values.shape

    @property
    def device(self):
        return self.values.device

    @property
    def pitch(self) -> int:
        """Bytes from row to row."""
        return self.values.stride(0) if self.values.size(0) > 1 else _pitch(self.values.size(1))

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values the rows stand for: a whole number times the scale in float32, rounded once, then to ``dtype``."""
        return (self.values.float() * self.scale.unsqueeze(1)).to(dtype)


_MAX_PITCH = 1 << 21     # bytes (8-bit rows) or elements (their partners in gemm_tn8) from row to row


def _pitch(k: int) -> int:
    return (k + 15) // 16 * 16


def _in_place(v: torch.Tensor) -> bool:
    n, k = v.shape
    if v.data_ptr() % 16 or (k > 1 and v.stride(1) != 1) or (n > 1 and (v.stride(0) % 16 or not _pitch(k) <= v.stride(0) <= _MAX_PITCH)):
        return False
    # the last row's 16-byte pieces must lie inside the storage
    end = v.storage_offset() + (max(n, 1) - 1) * v.stride(0) + _pitch(k)
    return n == 0 or end <= v.untyped_storage().nbytes()


def _padded(v: torch.Tensor) -> torch.Tensor:
    store = torch.zeros((v.size(0), _pitch(v.size(1))), dtype=torch.int8, device=v.device)
    out = store[:, :v.size(1)]
    out.copy_(v)
    return out


def rows8_of(values: torch.Tensor, scale: torch.Tensor) -> Rows8:
    """Rows8 of parts that this module laid out itself (nothing is checked or copied)."""
    r = Rows8.__new__(Rows8)
    r.values, r.scale = values, scale
    return r


def rows8_again(values: torch.Tensor, scale: torch.Tensor) -> Rows8:
    """Rows8 of what an autograd node saved: a hook on saved tensors may have brought it back in another layout."""
    return rows8_of(values if _in_place(values) else _padded(values), scale.contiguous())


def _new(n: int, k: int, device) -> Rows8:
    return rows8_of(torch.empty((n, _pitch(k)), dtype=torch.int8, device=device)[:, :k],
                    torch.empty(n, dtype=torch.float32, device=device))


def _check_rows(name: str, x: torch.Tensor) -> None:
    _lib.require_device(x, name)
    _lib.dtype_code(x.dtype)
    if x.dim() != 2 or not 1 <= x.size(1) <= MAX_WIDTH:
        raise ValueError(f"{name} must have shape [N, K] with 1 <= K <= {MAX_WIDTH}, got {tuple(x.shape)}")


def quantize_rows(x: torch.Tensor) -> Rows8:
    """The rows of ``x`` (float32 or bfloat16 [N, K], any row stride) in 8 bits.  No gradient passes through."""
    return (_marked_quantize if torch.compiler.is_compiling() else _checked_quantize)(x)


def _checked_quantize(x: torch.Tensor) -> Rows8:
    _check_rows("x", x)
    return to_rows8(_lib.rows_in_place(x.detach()))


_marked_quantize = torch.compiler.disable(_checked_quantize)


def to_rows8(x: torch.Tensor) -> Rows8:
    """quantize_rows of a checked matrix whose rows lie in place."""
    n, k = x.shape
    r = _new(n, k, x.device)
    _lib.check(_lib.load().mpnn_quantize_rows(_lib.ptr(x), _lib.leading(x), _lib.dtype_code(x.dtype), n, k,
                                              _lib.ptr(r.values), r.pitch, _lib.ptr(r.scale), _lib.stream_handle(x.device)),
               "mpnn_quantize_rows")
    return r


def linear_int8(x, weight: Rows8, bias: torch.Tensor | None = None, relu: bool = False,
                dtype: torch.dtype | None = None) -> torch.Tensor:
    """``act(x @ weight^T + bias)`` on 8-bit rows with exact integer sums: x [N, K] as ``Rows8``, or in float32 / bfloat16
    (taken to 8 bits on the way, one scale per row); ``weight`` [M, K] one scale per output channel, made once with
    ``quantize_rows(w)``.  The result is ``dtype`` (x's own by default, float32 for ``Rows8``); ``bias`` [M] of that dtype.
    For answering only: operands that want a gradient are refused where gradients are recorded."""
    return (_marked_linear if torch.compiler.is_compiling() else _linear_int8)(x, weight, bias, relu, dtype)


def _linear_int8(x, weight, bias, relu, dtype):
    held = isinstance(x, Rows8)
    if not isinstance(weight, Rows8):
        raise TypeError(f"weight must be Rows8 (quantize_rows(w)), got {type(weight).__name__}")
    if torch.is_grad_enabled() and ((x.scale if held else x).requires_grad or weight.scale.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        raise RuntimeError("linear_int8 has no gradient: call it under torch.no_grad() (or with detached operands), or train "
                           'with dense.project(..., checkpoint="int8")')
    if held:
        _lib.require_device(x.values, "x")
    else:
        _check_rows("x", x)
        x = _lib.rows_in_place(x)
    n, k = x.shape
    m = weight.shape[0]
    if weight.shape[1] != k or m < 1:
        raise ValueError(f"weight must have shape [M, {k}], got {tuple(weight.shape)}")
    if dtype is None:
        dtype = torch.float32 if held else x.dtype
    code = _lib.dtype_code(dtype)
    if bias is not None and (bias.shape != (m,) or bias.dtype != dtype):
        raise ValueError(f"bias must be {dtype} [{m}], got {bias.dtype} {tuple(bias.shape)}")
    if weight.device != x.device or (bias is not None and bias.device != x.device):
        raise _lib.MpnnError(f"x, weight and bias must be on one device, got {x.device}, {weight.device}")
    bias = None if bias is None else bias.detach().contiguous()
    lib = _lib.load()
    y = torch.empty((n, m), dtype=dtype, device=x.device)
    if held:
        kind, ptr, ld, scale, space = _lib.MPNN_I8, _lib.ptr(x.values), x.pitch, _lib.ptr(x.scale), None
    else:
        kind, ptr, ld, scale = _lib.dtype_code(x.dtype), _lib.ptr(x), _lib.leading(x), None
        need = lib.mpnn_linear_int8_workspace_bytes(n, k, m, kind)
        space = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _lib.check(lib.mpnn_linear_int8(ptr, ld, kind, scale, _lib.ptr(weight.values), weight.pitch, _lib.ptr(weight.scale),
                                    _lib.ptr(bias), _lib.ptr(y), m, code, n, k, m, 1 if relu else 0, _lib.ptr(space),
                                    _lib.stream_handle(x.device)), "mpnn_linear_int8")
    return y


_marked_linear = torch.compiler.disable(_linear_int8)


def kept_linear(x: torch.Tensor, w: torch.Tensor, x2: torch.Tensor | None = None, relu: bool = False):
    """act(x @ w[:, :K]^T [+ x2 @ w[:, K:]^T]) with the inputs' 8-bit rows and the relu's bits from the same pass:
    (y, rows of x, rows of x2 or None, bits or None).  None where the shapes or layouts do not fit the kernel.  In float32
    y is gemm_nt's to the bit."""
    lib = _lib.load()
    code = _lib.dtype_code(x.dtype)
    n, k = x.shape
    m, k2 = w.size(0), (x2.size(1) if x2 is not None else 0)
    if not lib.mpnn_kept_linear_fits(k, k2, m, code):
        return None
    unit = 8 if code == _lib.MPNN_BF16 else 4      # elements of 16 bytes
    for t in (x, w, x2):
        if t is not None and (t.stride(1) != 1 or t.stride(0) % unit or t.data_ptr() % 16
                              or (t.size(0) > 1 and t.stride(0) < t.size(1))):
            return None
    r, r2 = _new(n, k, x.device), (_new(n, k2, x.device) if x2 is not None else None)
    y = torch.empty((n, m), dtype=x.dtype, device=x.device)
    bits = torch.empty((n, (m + 31) // 32), dtype=torch.int32, device=x.device) if relu else None
    q2, ld2, s2 = (_lib.ptr(r2.values), r2.pitch, _lib.ptr(r2.scale)) if r2 is not None else (None, 0, None)
    _lib.check(lib.mpnn_kept_linear(_lib.ptr(x), _lib.leading(x), k, _lib.ptr(r.values), r.pitch, _lib.ptr(r.scale),
                                    _lib.ptr(x2), _lib.leading(x2), k2, q2, ld2, s2, _lib.ptr(w), _lib.leading(w),
                                    _lib.ptr(y), m, _lib.ptr(bits), n, m, 1 if relu else 0, code,
                                    _lib.stream_handle(x.device)), "mpnn_kept_linear")
    return y, r, r2, bits


def gemm_nn(g: torch.Tensor, w: torch.Tensor):
    """g @ w for w [K, M] as it lies, None where the widths or layouts do not fit the kernel.  In float32 it is
    gemm_nt(g, w^T) to the bit."""
    lib = _lib.load()
    code = _lib.dtype_code(g.dtype)
    (n, k), m = g.shape, w.size(1)
    # float32 wider than 128: the pieces fill the registers (1 M x 256 -> 64: 295 us, by the transpose 287; 1 M x 128 -> 128: 238 and 278)
    if code == _lib.MPNN_F32 and k > 128:
        return None
    if not lib.mpnn_kept_linear_fits(k, 0, m, code):
        return None
    ldg, ldw = _lib.leading(g), _lib.leading(w)
    if (g.stride(1) != 1 or w.stride(1) != 1 or ldg % (8 if code == _lib.MPNN_BF16 else 4) or g.data_ptr() % 16
            or (n > 1 and g.stride(0) < k) or (k > 1 and w.stride(0) < m)):
        return None
    y = torch.empty((n, m), dtype=g.dtype, device=g.device)
    _lib.check(lib.mpnn_gemm_nn(_lib.ptr(g), ldg, _lib.ptr(w), ldw, _lib.ptr(y), m, n, k, m, code,
                                _lib.stream_handle(g.device)), "mpnn_gemm_nn")
    return y


def relu_bits(y: torch.Tensor) -> torch.Tensor:
    """One bit per entry of a relu's output [N, M]: int32 [N, ceil(M / 32)], set where the relu is open."""
    n, m = y.shape
    bits = torch.empty((n, (m + 31) // 32), dtype=torch.int32, device=y.device)
    _lib.check(_lib.load().mpnn_relu_bits(_lib.ptr(y), _lib.leading(y), _lib.dtype_code(y.dtype), n, m, _lib.ptr(bits),
                                          _lib.stream_handle(y.device)), "mpnn_relu_bits")
    return bits


def open_entries(g: torch.Tensor, bits: torch.Tensor) -> torch.Tensor:
    """g [N, M] where the relu that left ``bits`` (relu_bits) is open, zeros elsewhere."""
    g = _lib.rows_in_place(g)
    n, m = g.shape
    out = torch.empty((n, m), dtype=g.dtype, device=g.device)
    _lib.check(_lib.load().mpnn_open_entries(_lib.ptr(g), _lib.leading(g), _lib.dtype_code(g.dtype), _lib.ptr(bits), _lib.ptr(out), m, n, m,
                                             _lib.stream_handle(g.device)), "mpnn_open_entries")
    return out


def gemm_tn8(g: torch.Tensor, x: Rows8, x2: Rows8 | None = None, bits=None, g_out=None) -> torch.Tensor:
    """(g * open)^T @ [x | x2] -> [M, K (+ K2)] in g's dtype, x and x2 the values their 8-bit rows stand for; ``bits``
    (relu_bits) tell which entries of g are open, ``g_out`` ([N, M], contiguous) receives g * open."""
    lib = _lib.load()
    g = _lib.rows_in_place(g)
    if _lib.leading(g) > _MAX_PITCH or (g.dtype == torch.bfloat16 and (g.data_ptr() % 4 or _lib.leading(g) % 2)):
        g = g.clone(memory_format=torch.contiguous_format)
    n, m = g.shape
    code = _lib.dtype_code(g.dtype)
    k, k2 = x.shape[1], (x2.shape[1] if x2 is not None else 0)
    out = torch.empty((m, k + k2), dtype=g.dtype, device=g.device)
    scratch = torch.empty(lib.mpnn_gemm_tn8_scratch_floats(n, m, k, k2, code), dtype=torch.float32, device=g.device)
    q2, ld2, s2 = (_lib.ptr(x2.values), x2.pitch, _lib.ptr(x2.scale)) if x2 is not None else (None, 0, None)
    _lib.check(lib.mpnn_gemm_tn8(_lib.ptr(g), _lib.leading(g), code, _lib.ptr(bits), _lib.ptr(x.values), x.pitch,
                                 _lib.ptr(x.scale), k, q2, ld2, s2, k2, _lib.ptr(out), k + k2, _lib.ptr(scratch),
                                 _lib.ptr(g_out), _lib.leading(g_out), n, m, _lib.stream_handle(g.device)), "mpnn_gemm_tn8")
    return out
