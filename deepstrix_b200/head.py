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
from dataclasses import dataclass

import torch

from .moe import _check, _dptr, _stream, lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _here(*tensors):
    """All on the current device (kernels run on its current stream)."""
    for t in tensors:
        assert t.is_cuda, "tensors must be on the GPU"
        assert t.device.index == torch.cuda.current_device(), f"tensor on {t.device}, current device is cuda:{torch.cuda.current_device()}"


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows of a 2-D tensor whose columns are contiguous."""
    assert t.dim() == 2 and (t.shape[1] <= 1 or t.stride(1) == 1), "rows must have contiguous columns"
    stride = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    assert stride >= t.shape[1], "rows must not overlap"
    return stride


@dataclass
class Mxfp4Rows:
    """Rows as sums of MXFP4 terms: uint8 codes [terms, rows, K / 2] (element 2i in the low nibble) and E8M0 scales
    [terms, rows, K / 32]; two-dimensional tensors are one term (a stored matrix)."""
    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self):
        c, s = self.codes, self.scales
        assert c.dtype == torch.uint8 and s.dtype == torch.uint8 and c.is_contiguous() and s.is_contiguous()
        assert c.dim() in (2, 3) and c.shape[:-1] == s.shape[:-1] and c.shape[-1] == 16 * s.shape[-1], "codes [.., K / 2] and scales [.., K / 32]"
        assert c.device == s.device

    @property
    def n_terms(self) -> int:
        return self.codes.shape[0] if self.codes.dim() == 3 else 1

    @property
    def rows(self) -> int:
        return self.codes.shape[-2]

    @property
    def k(self) -> int:
        return self.codes.shape[-1] * 2


class Mxfp4Quantize:
    """Rows of f32 / bf16 / f16 -> sums of 1 to 3 MXFP4 terms, each of what the earlier ones leave over (the FP4
    fake-quantiser of scripts/v41_oracle/kernel.py:129-147, applied to the residuals).  Any row stride."""

    @staticmethod
    def launch(x: torch.Tensor, n_terms: int = 1) -> Mxfp4Rows:
        assert x.dtype in DTYPES
        stride = _row_stride(x)
        _here(x)
        rows, k = x.shape
        codes = torch.empty((n_terms, rows, k // 2), dtype=torch.uint8, device=x.device)
        scales = torch.empty((n_terms, rows, k // 32), dtype=torch.uint8, device=x.device)
        _check(lib().dsx_mxfp4_quantize(_dptr(x), DTYPES[x.dtype], C.c_int64(rows), C.c_int64(k), C.c_int64(stride), n_terms, _dptr(codes), _dptr(scales),
                                        _stream()))
        return Mxfp4Rows(codes, scales)


class Mxfp4Dequantize:
    """The values MXFP4 rows stand for (terms added in f32, rounded once)."""

    @staticmethod
    def launch(q: Mxfp4Rows, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
        _here(q.codes)
        if out is None:
            out = torch.empty((q.rows, q.k), dtype=dtype, device=q.codes.device)
        assert out.shape == (q.rows, q.k) and out.dtype == dtype
        _here(out)
        _check(lib().dsx_mxfp4_dequantize(_dptr(q.codes), _dptr(q.scales), C.c_int64(q.rows), C.c_int64(q.k), q.n_terms, _dptr(out), DTYPES[dtype],
                                          C.c_int64(_row_stride(out)), _stream()))
        return out


class Mxfp4Matmul:
    """out[m, n] = a[m, :] . w[n, :] over MXFP4 rows: ``a`` with 1 to 3 terms (activations), ``w`` with one (a stored matrix)."""

    @staticmethod
    def launch(a: Mxfp4Rows, w: Mxfp4Rows, dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
        assert w.n_terms == 1 and a.k == w.k
        _here(a.codes, w.codes)
        if out is None:
            out = torch.empty((a.rows, w.rows), dtype=dtype, device=a.codes.device)
        assert out.shape == (a.rows, w.rows) and out.dtype == dtype
        _here(out)
        _check(lib().dsx_mxfp4_matmul(_dptr(a.codes), _dptr(a.scales), a.n_terms, C.c_int64(a.rows), _dptr(w.codes), _dptr(w.scales), C.c_int64(w.rows),
                                      C.c_int64(a.k), _dptr(out), DTYPES[dtype], C.c_int64(_row_stride(out)), _stream()))
        return out


def check() -> int:
    """The product's device-side error word on the current device (0 = clean).  Clears it; synchronises the stream."""
    w = C.c_uint32()
    rc = lib().dsx_head_check(_stream(), C.byref(w))
    if rc != -3:   # DSX_ERR_DEVICE only says that the word is non-zero
        _check(rc)
    return w.value


class TokenLogprobs:
    """Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits, in one pass over them."""

    @staticmethod
    def launch(logits: torch.Tensor, tokens: torch.Tensor | None = None, n_alt: int = 0, inv_temperature: float = 1.0):
        """logits [T, V] f32 / bf16 / f16 (any row stride), tokens int32 [T] or [T, n] -> (logprobs f32 like tokens or None,
        entropy f32 [T], ids int32 [T, n_alt], their log probabilities f32 [T, n_alt]).  -inf logits are masked; see
        ``dsx_token_logprobs`` for rows with nothing left and rows that hold a NaN."""
        assert logits.dtype in DTYPES
        stride = _row_stride(logits)
        _here(logits)
        T, V = logits.shape
        dev = logits.device
        given, logprobs = 0, None
        if tokens is not None:
            assert tokens.dtype == torch.int32 and tokens.is_contiguous() and tokens.dim() in (1, 2) and tokens.shape[0] == T
            _here(tokens)
            given = 1 if tokens.dim() == 1 else tokens.shape[1]
            logprobs = torch.empty(tokens.shape, dtype=torch.float32, device=dev)
        entropy = torch.empty((T,), dtype=torch.float32, device=dev)
        ids = torch.empty((T, n_alt), dtype=torch.int32, device=dev)
        alternatives = torch.empty((T, n_alt), dtype=torch.float32, device=dev)
        _check(lib().dsx_token_logprobs(_dptr(logits), DTYPES[logits.dtype], C.c_int64(T), C.c_int64(V), C.c_int64(stride), C.c_float(inv_temperature),
                                        _dptr(tokens), given, _dptr(logprobs), _dptr(entropy), n_alt, _dptr(ids), _dptr(alternatives), _stream()))
        return logprobs, entropy, ids, alternatives
