"""The quantised output head and what is read off it, over the C ABI (section 4 of ``include/dsx_moe.h``).

MXFP4 rows (``Mxfp4Quantize``, ``Mxfp4Dequantize``), their product (``Mxfp4Matmul``) and the log probabilities of given tokens
with entropy and top alternatives (``TokenLogprobs``, what a teacher-forced fidelity check reads, tests/v41_golden_gate.rs of the
reference).  A head of a decode step::

    w = Mxfp4Rows(codes, scales)                       # as a checkpoint stores it, or Mxfp4Quantize.launch(weight)
    x = Mxfp4Quantize.launch(hidden, n_terms=3)        # three terms: about 1.6e-3 relative error of the activations
    logits = Mxfp4Matmul.launch(x, w, torch.float32)
    logprobs, entropy, ids, alternatives = TokenLogprobs.launch(logits, tokens, n_alt=5)

torch is used only for device memory and the current stream; tensors live on the current device.
"""
from __future__ import annotations

import ctypes as C

import torch

from .moe import DsxError, lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_P, _I, _L, _F = C.c_void_p, C.c_int, C.c_int64, C.c_float
_SIGNATURES = {
    "dsx_mxfp4_quantize": [_P, _I, _L, _L, _L, _I, _P, _P, _P],
    "dsx_mxfp4_dequantize": [_P, _P, _L, _L, _I, _P, _I, _L, _P],
    "dsx_mxfp4_matmul": [_P, _P, _I, _L, _P, _P, _L, _L, _P, _I, _L, _P],
    "dsx_token_logprobs": [_P, _I, _L, _L, _L, _F, _P, _I, _P, _P, _I, _P, _P, _P],
    "dsx_mxfp4_matmul_tiling": [_I, _L, _L, _L, C.POINTER(C.c_int32)],
    "dsx_mxfp4_matmul_pin": [_I, _I, _I],
    "dsx_mxfp4_matmul_set_polls": [C.c_uint32],
    "dsx_head_check": [_P, C.POINTER(C.c_uint32)],
}
_functions = {}


def _call(name, *args):
    """One C call: plain integers for pointers and sizes (a call of this file is a few microseconds of host time; wrapping
    every argument by hand costs as much again)."""
    fn = _functions.get(name)
    if fn is None:
        fn = getattr(lib(), name)
        fn.argtypes = _SIGNATURES[name]
        _functions[name] = fn
    rc = fn(*args)
    if rc != 0:
        raise DsxError(rc, lib().dsx_last_error().decode())


def _here(*tensors) -> int:
    """All on the current device, whose current stream (returned) the kernels run on."""
    device = torch.cuda.current_device() if tensors[0].is_cuda else None
    for t in tensors:
        assert t.get_device() == device, f"tensor on {t.device}, not on the current GPU"   # the CPU's is -1
    return torch._C._cuda_getCurrentRawStream(device)


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows of a 2-D tensor whose columns are contiguous."""
    assert t.dim() == 2, "a matrix of rows"
    rows, cols = t.shape
    row_stride, col_stride = t.stride()
    assert cols <= 1 or col_stride == 1, "rows must have contiguous columns"
    if rows <= 1:
        return cols
    assert row_stride >= cols, "rows must not overlap"
    return row_stride


class Mxfp4Rows:
    """Rows as sums of MXFP4 terms: uint8 ``codes`` [terms, rows, K / 2] (element 2i in the low nibble) and E8M0 ``scales``
    [terms, rows, K / 32]; two-dimensional tensors are one term (a stored matrix)."""
    __slots__ = ("n_terms", "rows", "k", "codes_at", "scales_at", "_buffer", "_codes", "_scales", "_given")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8 and codes.is_contiguous() and scales.is_contiguous()
        shape = codes.shape
        assert len(shape) in (2, 3) and shape[:-1] == scales.shape[:-1] and shape[-1] == 16 * scales.shape[-1], "codes [.., K / 2] and scales [.., K / 32]"
        assert codes.get_device() == scales.get_device()
        self.n_terms, self.rows, self.k = shape[0] if len(shape) == 3 else 1, shape[-2], 2 * shape[-1]
        self._buffer, self._codes, self._scales, self._given = codes, codes, scales, True
        self.codes_at, self.scales_at = codes.data_ptr(), scales.data_ptr()

    @classmethod
    def _empty(cls, n_terms: int, rows: int, k: int, device) -> "Mxfp4Rows":
        """Room for the quantiser's result: one allocation, the tensors made when they are asked for."""
        assert n_terms >= 1 and k % 32 == 0, f"{n_terms} terms of rows of {k} columns (a multiple of 32)"
        q = cls.__new__(cls)
        n = n_terms * rows * k
        q.n_terms, q.rows, q.k, q._codes, q._scales, q._given = n_terms, rows, k, None, None, False
        q._buffer = torch.empty(n // 2 + n // 32, dtype=torch.uint8, device=device)
        q.codes_at = q._buffer.data_ptr()
        q.scales_at = q.codes_at + n // 2
        return q

    def _follow(self):
        """Given tensors are asked where they lie at every call: their owner may have put other memory, of the same form, under them."""
        codes, scales = self._codes, self._scales
        if codes.data_ptr() != self.codes_at or scales.data_ptr() != self.scales_at:
            now = Mxfp4Rows(codes, scales)
            assert (now.n_terms, now.rows, now.k) == (self.n_terms, self.rows, self.k), "codes and scales have changed shape"
            self.codes_at, self.scales_at = now.codes_at, now.scales_at

    @property
    def device(self) -> torch.device:
        return self._buffer.device

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            row = self.k // 2
            self._codes = self._buffer.as_strided((self.n_terms, self.rows, row), (self.rows * row, row, 1), 0)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            row = self.k // 32
            self._scales = self._buffer.as_strided((self.n_terms, self.rows, row), (self.rows * row, row, 1), self.n_terms * self.rows * self.k // 2)
        return self._scales


class Mxfp4Quantize:
    """Rows of f32 / bf16 / f16 -> sums of 1 to 3 MXFP4 terms, each of what the earlier ones leave over (the FP4
    fake-quantiser of scripts/v41_oracle/kernel.py:129-147, applied to the residuals).  Any row stride."""

    @staticmethod
    def launch(x: torch.Tensor, n_terms: int = 1) -> Mxfp4Rows:
        assert x.dtype in DTYPES, f"rows of {x.dtype}"
        stride = _row_stride(x)
        stream = _here(x)
        rows, k = x.shape
        q = Mxfp4Rows._empty(n_terms, rows, k, x.device)
        _call("dsx_mxfp4_quantize", x.data_ptr(), DTYPES[x.dtype], rows, k, stride, n_terms, q.codes_at, q.scales_at, stream)
        return q


class Mxfp4Dequantize:
    """The values MXFP4 rows stand for (terms added in f32, rounded once)."""

    @staticmethod
    def launch(q: Mxfp4Rows, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
        if out is None:
            out = torch.empty(q.rows, q.k, dtype=dtype, device=q.device)
        assert out.shape == (q.rows, q.k) and out.dtype == dtype and dtype in DTYPES
        if q._given:
            q._follow()
        _call("dsx_mxfp4_dequantize", q.codes_at, q.scales_at, q.rows, q.k, q.n_terms, out.data_ptr(), DTYPES[dtype], _row_stride(out),
              _here(q._buffer, out))
        return out


class Mxfp4Matmul:
    """out[m, n] = a[m, :] . w[n, :] over MXFP4 rows: ``a`` with 1 to 3 terms (activations), ``w`` with one (a stored matrix)."""

    @staticmethod
    def launch(a: Mxfp4Rows, w: Mxfp4Rows, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
        assert w.n_terms == 1, "a weight has one term"
        assert a.k == w.k, f"rows of {a.k} and of {w.k} columns"
        if out is None:
            out = torch.empty(a.rows, w.rows, dtype=dtype, device=a.device)
        assert out.shape == (a.rows, w.rows) and out.dtype == dtype and dtype in DTYPES
        if a._given:
            a._follow()
        if w._given:
            w._follow()
        _call("dsx_mxfp4_matmul", a.codes_at, a.scales_at, a.n_terms, a.rows, w.codes_at, w.scales_at, w.rows, a.k, out.data_ptr(), DTYPES[dtype],
              _row_stride(out), _here(a._buffer, w._buffer, out))
        return out

    @staticmethod
    def tiling(n_terms: int, m: int, n: int, k: int) -> dict:
        """How a product of these sizes is cut up on the current device (for tests and tuning)."""
        values = (C.c_int32 * 8)()
        _call("dsx_mxfp4_matmul_tiling", n_terms, m, n, k, values)
        return dict(zip(("pair", "tokens", "splits", "tiles", "at_once", "stages", "scale_bufs", "slots"), values))

    @staticmethod
    def pin(pair: int = -1, tokens: int = 0, splits: int = 0):
        """Fixes parts of the tiling for this process's products until the next call (no arguments: all chosen again)."""
        _call("dsx_mxfp4_matmul_pin", pair, tokens, splits)

    @staticmethod
    def set_polls(polls: int = 0):
        """How often a wait inside the product is tried before it gives up (0: the default)."""
        _call("dsx_mxfp4_matmul_set_polls", polls)


def check() -> int:
    """The product's device-side error word on the current device (0 = clean).  Clears it; synchronises the stream."""
    w = C.c_uint32()
    try:
        _call("dsx_head_check", torch.cuda.current_stream().cuda_stream, C.byref(w))
    except DsxError as e:
        if e.code != -3:   # DSX_ERR_DEVICE only says that the word is non-zero
            raise
    return w.value


class TokenLogprobs:
    """Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits, in one pass over them."""

    @staticmethod
    def launch(logits: torch.Tensor, tokens: torch.Tensor | None = None, n_alt: int = 0, inv_temperature: float = 1.0):
        """logits [T, V] f32 / bf16 / f16 (any row stride), tokens int32 [T] or [T, n] -> (logprobs f32 like tokens or None,
        entropy f32 [T], ids int32 [T, n_alt], their log probabilities f32 [T, n_alt]).  -inf logits are masked; see
        ``dsx_token_logprobs`` for rows with nothing left and rows that hold a NaN."""
        assert logits.dtype in DTYPES, f"logits of {logits.dtype}"
        stride = _row_stride(logits)
        T, V = logits.shape
        dev = logits.device
        given, logprobs, tokens_at, logprobs_at = 0, None, None, None
        if tokens is not None:
            assert tokens.dtype == torch.int32 and tokens.is_contiguous() and tokens.dim() in (1, 2) and tokens.shape[0] == T, "int32 tokens [T] or [T, n]"
            stream = _here(logits, tokens)
            given = 1 if tokens.dim() == 1 else tokens.shape[1]
            logprobs = torch.empty_like(tokens, dtype=torch.float32)
            tokens_at, logprobs_at = tokens.data_ptr(), logprobs.data_ptr()
        else:
            stream = _here(logits)
        entropy = torch.empty(T, dtype=torch.float32, device=dev)
        ids = torch.empty(T, n_alt, dtype=torch.int32, device=dev)
        alternatives = torch.empty_like(ids, dtype=torch.float32)
        _call("dsx_token_logprobs", logits.data_ptr(), DTYPES[logits.dtype], T, V, stride, inv_temperature, tokens_at, given, logprobs_at,
              entropy.data_ptr(), n_alt, ids.data_ptr(), alternatives.data_ptr(), stream)
        return logprobs, entropy, ids, alternatives
