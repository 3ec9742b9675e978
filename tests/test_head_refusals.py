"""What the quantised head's entry points refuse (no GPU: arguments are checked before anything is launched)."""
import ctypes as C

import pytest
import torch

from deepstrix_b200 import head

P = C.c_void_p(1 << 20)          # stands for a device pointer: aligned, never read, since every call below is refused
N = C.c_void_p(0)
ODD = C.c_void_p((1 << 20) + 1)
F32, BF16, F16 = 0, 1, 2
L = C.c_int64


def _refused(moe, name, *args):
    rc = getattr(moe.lib(), name)(*args)
    assert rc == -1, (name, rc)
    return moe.lib().dsx_last_error().decode()


def test_quantize_and_dequantize_refusals(moe):
    def q(x=P, dt=BF16, rows=4, k=64, stride=64, terms=1, codes=P, scales=P):
        return _refused(moe, "dsx_mxfp4_quantize", x, dt, L(rows), L(k), L(stride), terms, codes, scales, N)

    def d(codes=P, scales=P, rows=4, k=64, terms=1, out=P, dt=BF16, stride=64):
        return _refused(moe, "dsx_mxfp4_dequantize", codes, scales, L(rows), L(k), terms, out, dt, L(stride), N)
    for f in (q, d):
        assert "element type" in f(dt=3)
        assert "multiple of 32" in f(k=48) and "multiple of 32" in f(k=0) and "multiple of 32" in f(rows=-1)
        assert "terms" in f(terms=0) and "terms" in f(terms=4)
        assert "stride" in f(stride=63)
        assert "null" in f(codes=N) and "null" in f(scales=N)
        assert "aligned" in f(codes=ODD)
    assert "aligned" in q(x=ODD) and "aligned" in d(out=ODD)
    assert "null" in q(x=N) and "null" in d(out=N)


def test_matmul_refusals(moe):
    def f(a=P, sa=P, terms=1, m=4, w=P, sw=P, n=8, k=64, out=P, dt=F32, stride=8):
        return _refused(moe, "dsx_mxfp4_matmul", a, sa, terms, L(m), w, sw, L(n), L(k), out, dt, L(stride), N)
    assert "element type" in f(dt=-1)
    assert "multiple of 32" in f(k=16) and "multiple of 32" in f(m=-1) and "multiple of 32" in f(n=-1) and "multiple of 32" in f(m=1 << 22)
    assert "terms" in f(terms=0) and "terms" in f(terms=4)
    for name in ("a", "sa", "w", "sw", "out"):
        assert "null" in f(**{name: N})
    assert "stride" in f(stride=7)
    assert "aligned" in f(a=ODD) and "aligned" in f(w=ODD) and "aligned" in f(out=ODD)


def test_logprobs_refusals(moe):
    def f(x=P, dt=F32, t=2, v=100, stride=100, temp=1.0, tok=P, given=1, lp=P, ent=P, alt=1, ids=P, alp=P):
        return _refused(moe, "dsx_token_logprobs", x, dt, L(t), L(v), L(stride), C.c_float(temp), tok, given, lp, ent, alt, ids, alp, N)
    assert "element type" in f(dt=5)
    assert "logits" in f(v=0) and "logits" in f(t=-1) and "logits" in f(v=1 << 31)
    assert "alternatives" in f(alt=33) and "alternatives" in f(alt=-1) and "given" in f(given=-1) and "given" in f(given=1025)
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert "temperature" in f(temp=bad)
    assert "stride" in f(stride=99)
    for name in ("x", "tok", "lp", "ids", "alp"):
        assert "null" in f(**{name: N})
    assert "aligned" in f(x=ODD)


def test_refused_sizes_and_alignments(moe):
    """Sizes whose products would pass 64 bits, rows longer than a wait is meant to last, arrays that are not aligned to their elements."""
    assert "values" in _refused(moe, "dsx_mxfp4_quantize", P, F32, L(1 << 58), L(64), L(64), 1, P, P, N)
    assert "values" in _refused(moe, "dsx_mxfp4_dequantize", P, P, L(1 << 58), L(64), 1, P, F32, L(64), N)
    assert "2^24" in _refused(moe, "dsx_mxfp4_matmul", P, P, 1, L(1), P, P, L(8), L((1 << 24) + 32), P, F32, L(8), N)
    arrays = [P, P, P, P, P]
    for i in range(5):
        tok, lp, ent, ids, alp = arrays[:i] + [ODD] + arrays[i + 1:]
        assert "aligned" in _refused(moe, "dsx_token_logprobs", P, F32, L(2), L(100), L(100), C.c_float(1.0), tok, 1, lp, ent, 1, ids, alp, N)


def test_nothing_to_do_is_not_an_error(moe):
    lib = moe.lib()
    assert lib.dsx_mxfp4_quantize(N, BF16, L(0), L(64), L(64), 1, N, N, N) == 0
    assert lib.dsx_mxfp4_dequantize(N, N, L(0), L(64), 1, N, F32, L(64), N) == 0
    assert lib.dsx_mxfp4_matmul(N, N, 1, L(0), N, N, L(8), L(64), N, F32, L(8), N) == 0
    assert lib.dsx_mxfp4_matmul(N, N, 1, L(8), N, N, L(0), L(64), N, F32, L(0), N) == 0
    assert lib.dsx_token_logprobs(N, F32, L(0), L(8), L(8), C.c_float(1), N, 1, N, N, 1, N, N, N) == 0


def test_python_checks(moe):
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    q = head.Mxfp4Rows(u8(2, 5, 32), u8(2, 5, 2))
    assert (q.n_terms, q.rows, q.k) == (2, 5, 64)
    assert head.Mxfp4Rows(u8(5, 32), u8(5, 2)).n_terms == 1
    for codes, scales in ((u8(5, 32), u8(5, 3)), (u8(5, 32), u8(4, 2)), (u8(5, 64)[:, ::2], u8(5, 2)), (u8(32), u8(2)),
                          (torch.zeros((5, 32)), u8(5, 2)), (u8(2, 5, 32), u8(5, 2))):
        with pytest.raises(AssertionError):
            head.Mxfp4Rows(codes, scales)
    for bad in (torch.zeros((4, 64)), torch.zeros((4, 64), dtype=torch.float64)):      # not on the device / no such type
        with pytest.raises(AssertionError):
            head.Mxfp4Quantize.launch(bad)
        with pytest.raises(AssertionError):
            head.TokenLogprobs.launch(bad)
    with pytest.raises(AssertionError):
        head.Mxfp4Quantize.launch(torch.zeros((64, 4)).T)                              # columns not contiguous
    with pytest.raises(AssertionError):
        head.Mxfp4Matmul.launch(head.Mxfp4Rows(u8(5, 32), u8(5, 2)), head.Mxfp4Rows(u8(2, 5, 32), u8(2, 5, 2)))   # a weight of two terms


def test_tiling_and_pin_refusals(moe):
    lib = moe.lib()
    out = (C.c_int32 * 8)()

    def tiling(terms=1, m=4, n=8, k=64, to=out):
        return _refused(moe, "dsx_mxfp4_matmul_tiling", terms, L(m), L(n), L(k), to)
    assert "multiple of 32" in tiling(k=48) and "multiple of 32" in tiling(m=-1) and "terms" in tiling(terms=4)
    assert "null" in tiling(to=None) and "nothing" in tiling(m=0) and "nothing" in tiling(n=0)
    for pin in ((-2, 0, 0), (2, 0, 0), (0, -16, 0), (0, 8, 0), (0, 224, 0), (0, 0, -1), (0, 0, 3), (0, 0, 16)):
        assert "pin" in _refused(moe, "dsx_mxfp4_matmul_pin", *pin)
    assert lib.dsx_mxfp4_matmul_pin(1, 208, 1) == 0 and lib.dsx_mxfp4_matmul_pin(-1, 0, 0) == 0


def test_rows_follow_their_tensors(moe, monkeypatch):
    """The memory of a given tensor may be exchanged under it (weights loaded anew): the next call takes what lies there then, if it has
    the same form."""
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    calls = []
    monkeypatch.setattr(head, "_call", lambda name, *args: calls.append(args))
    monkeypatch.setattr(head, "_here", lambda *tensors: 0)
    codes, scales, other = u8(5, 32), u8(5, 2), head.Mxfp4Rows(u8(3, 32), u8(3, 2))
    q = head.Mxfp4Rows(codes, scales)

    def addresses():
        head.Mxfp4Dequantize.launch(q)
        head.Mxfp4Matmul.launch(q, other)
        head.Mxfp4Matmul.launch(other, q)
        return {calls[-3][:2], calls[-2][:2], calls[-1][4:6]}
    assert addresses() == {(codes.data_ptr(), scales.data_ptr())}
    codes.data, new_scales = u8(5, 32) + 1, u8(5, 2)
    scales.set_(new_scales)
    assert addresses() == {(codes.data_ptr(), new_scales.data_ptr())} and q.codes[0, 0] == 1
    codes.data = u8(6, 32)
    with pytest.raises(AssertionError):
        addresses()
    scales.data = u8(6, 2)
    with pytest.raises(AssertionError, match="changed shape"):
        addresses()
    codes.data, scales.data = u8(5, 32), u8(5, 2)
    assert addresses() == {(codes.data_ptr(), scales.data_ptr())}
