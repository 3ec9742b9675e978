"""The quantised head's operators against plain 64-bit restatements: MXFP4 rows (bit for bit against the CPU oracle), their product
(exact where every sum is representable, else within a derived bound), token log probabilities."""
import ctypes as C
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}     # a rounding is off by at most this, relatively
TINY = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}       # half the smallest subnormal


def _dtype(torch, name):
    return getattr(torch, name)


def _values64(codes, scales):
    """f64 values of MXFP4 rows [.., K / 2], [.., K / 32]."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    v = np.stack([E2M1[codes & 15], E2M1[codes >> 4]], -1).reshape(codes.shape[:-1] + (-1,))
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, -1)


def _oracle_rows(oracle, x, terms):
    """(codes [terms, rows, K / 2], scales [terms, rows, K / 32], sum of the terms [rows, K]) of the CPU oracle."""
    rows, k = x.shape
    codes, scales, total = oracle.act_terms_mxfp4(x, terms)
    return codes.reshape(terms, rows, k // 2), scales.reshape(terms, rows, k // 32), total.reshape(rows, k)


# ------------------------------------------------------------------ quantise
def _hard_rows(rng, rows, k):
    """Normal rows, with blocks at every border of the scale rule and of E2M1's rounding."""
    x = rng.standard_normal((rows, k)).astype(np.float32)
    flat = x.reshape(-1, 32)
    n = len(flat)
    hard = [np.zeros(32), np.full(32, -0.0), np.array([6.0] + [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0] * 3 + [0] * 4),
            np.full(32, 6.0 * 2.0 ** -20), np.full(32, 1.5), np.full(32, np.nextafter(np.float32(1.5), np.float32(2))), np.full(32, -3.0e4),
            np.array([2.0 ** -14] * 16 + [2.0 ** -20] * 16), np.full(32, 2.0 ** -24), np.array([1e4, 1e-4] * 16)]
    for i, h in enumerate(hard):
        flat[(i * 7 + 3) % n] = h
    return x


@pytest.mark.parametrize("terms", [1, 2, 3])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,k,pad,offset", [(1, 32, 0, 0), (3, 96, 0, 0), (257, 2304, 0, 0), (64, 4096, 8, 0), (9, 160, 3, 1), (1, 4096, 5, 3), (33, 32, 32, 0)])
def test_quantize_bitexact(torch_cuda, moe, oracle, rows, k, pad, offset, dtype, terms):
    """Codes and scale bytes of every term against the CPU oracle; padded rows, and rows off the 16-byte boundary (offset, odd pad)."""
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(rows * k + terms)
    wide = torch.zeros(rows * (k + pad) + offset, dtype=_dtype(torch, dtype), device="cuda")
    x = wide[offset:].view(rows, k + pad)[:, :k]
    x.copy_(torch.from_numpy(_hard_rows(rng, rows, k)))
    got = head.Mxfp4Quantize.launch(x, terms)
    codes, scales, total = _oracle_rows(oracle, x.float().cpu().numpy(), terms)
    assert np.array_equal(got.scales.cpu().numpy(), scales)
    assert np.array_equal(got.codes.cpu().numpy(), codes)
    back = head.Mxfp4Dequantize.launch(got, torch.float32).cpu().numpy()
    assert np.array_equal(back, total)


def test_quantize_f32_extremes_and_written_set(torch_cuda, moe, oracle):
    """Largest and smallest f32 magnitudes, subnormals; bytes around the outputs stay as they are."""
    torch = torch_cuda
    x = np.zeros((4, 64), np.float32)
    x[0] = np.finfo(np.float32).max
    x[1, :32] = 2.0 ** -149
    x[1, 32:] = 2.0 ** -126
    x[2, 5] = -np.finfo(np.float32).max
    x[2, 6] = 1.0
    x[3, 40] = 2.0 ** -127
    want_c, want_s, _ = _oracle_rows(oracle, x, 2)
    # the largest magnitude rounds to 4 * 2^126 = 2^128, which the oracle's f32 residual cannot hold (it becomes infinite); a power of two
    # smaller the same codes come out with smaller scale bytes, and the kernel's fused residual is exact at both
    small_c, small_s, _ = _oracle_rows(oracle, x * np.float32(2.0 ** -20), 2)
    for r, b in ((0, 0), (0, 1), (2, 0)):
        want_c[:, r, 16 * b:16 * b + 16], want_s[:, r, b] = small_c[:, r, 16 * b:16 * b + 16], small_s[:, r, b] + 20
    codes = torch.full((16 + 2 * 4 * 32 + 16,), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((3 + 2 * 4 * 2 + 3,), 0xEE, dtype=torch.uint8, device="cuda")
    dx = torch.from_numpy(x).cuda()
    moe._check(moe.lib().dsx_mxfp4_quantize(C.c_void_p(dx.data_ptr()), 0, C.c_int64(4), C.c_int64(64), C.c_int64(64), 2, C.c_void_p(codes.data_ptr() + 16),
                                            C.c_void_p(scales.data_ptr() + 3), moe._stream()))
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(c[16:-16].reshape(2, 4, 32), want_c) and (c[:16] == 0xEE).all() and (c[-16:] == 0xEE).all()
    assert np.array_equal(s[3:-3].reshape(2, 4, 2), want_s) and (s[:3] == 0xEE).all() and (s[-3:] == 0xEE).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_quantize_non_finite_blocks(torch_cuda, moe, dtype):
    """A block with a NaN or an infinity is NaN as a whole, its neighbours are untouched."""
    torch = torch_cuda
    from deepstrix_b200 import head
    x = torch.ones((3, 96), dtype=_dtype(torch, dtype), device="cuda")
    x[0, 40], x[1, 0], x[2, 95] = math.nan, math.inf, -math.inf
    q = head.Mxfp4Quantize.launch(x, 3)
    s = q.scales.cpu().numpy()
    bad = np.zeros((3, 3), bool)
    bad[0, 1] = bad[1, 0] = bad[2, 2] = True
    assert (s[0] == 255).tolist() == bad.tolist() and not (s[1:] == 255).any()
    v = head.Mxfp4Dequantize.launch(q, x.dtype).float().cpu().numpy().reshape(3, 3, 32)
    assert np.isnan(v[bad]).all() and (v[~bad] == 1.0).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_dequantize_every_scale_byte_and_strides(torch_cuda, moe, dtype):
    """Every E8M0 byte, one rounding to the type, rows of a wider buffer; columns past the row stay as they are."""
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(5)
    codes = rng.integers(0, 256, (256, 32)).astype(np.uint8)
    scales = np.stack([np.arange(256), np.arange(256)[::-1]], 1).astype(np.uint8)
    q = head.Mxfp4Rows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda())
    # one rounding: from the exact f64 value to f32 (exact here, or an f32 overflow) and to the type
    want = torch.from_numpy(_values64(codes, scales)).to(torch.float32).to(_dtype(torch, dtype))
    for pad in (0, 8, 3):
        wide = torch.full((256, 64 + pad), 7.0, dtype=_dtype(torch, dtype), device="cuda")
        head.Mxfp4Dequantize.launch(q, wide.dtype, out=wide[:, :64])
        got = wide.cpu()
        assert torch.equal(torch.nan_to_num(got[:, :64].float(), nan=12345.0), torch.nan_to_num(want.float(), nan=12345.0)) and bool((got[:, 64:] == 7).all())


# ------------------------------------------------------------------- product
def _rows(torch, rng, rows, k, terms, lo, hi):
    from deepstrix_b200 import head
    codes = rng.integers(0, 256, (terms, rows, k // 2)).astype(np.uint8)
    scales = rng.integers(lo, hi, (terms, rows, k // 32)).astype(np.uint8)
    return head.Mxfp4Rows(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda()), _values64(codes, scales)


SHAPES = [(1, 1, 32), (1, 128, 256), (2, 130, 96), (5, 1000, 2304), (8, 64, 8192), (16, 257, 544), (17, 4096, 4096), (33, 384, 1024), (64, 1024, 2048),
          (65, 127, 800), (96, 129, 128), (100, 5119, 320), (129, 33, 64), (200, 640, 1056), (209, 256, 512), (255, 511, 2336), (500, 700, 160), (1030, 300, 288), (1500, 2100, 288), (3000, 300, 1056), (2049, 1025, 96), (4100, 4100, 256)]


@pytest.mark.parametrize("terms", [1, 2, 3])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul_exact_sums(torch_cuda, moe, m, n, k, terms):
    """Scales of 2^-1 .. 2^1: values are multiples of 1/4 of at most 12, products multiples of 1/16 of at most 144, and every partial sum of
    these random rows stays far below 2^24 sixteenths -- so any f32 accumulation gives the exact sum, and one wrong or missing block shows."""
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(m * 7 + n + k + terms)
    a, av = _rows(torch, rng, m, k, terms, 126, 129)
    w, wv = _rows(torch, rng, n, k, 1, 126, 129)
    want = av.sum(0) @ wv[0].T
    assert np.abs(want).max() * 16 < 2 ** 22
    got = head.Mxfp4Matmul.launch(a, w, torch.float32).cpu().numpy()
    bad = np.argwhere(got != want.astype(np.float32))
    assert len(bad) == 0, (len(bad), bad[:4], bad[-4:])
    for dt in (torch.bfloat16, torch.float16):        # one rounding of the exact sum
        got = head.Mxfp4Matmul.launch(a, w, dt).cpu()
        assert torch.equal(got, torch.from_numpy(want).to(torch.float32).to(dt))


@pytest.mark.parametrize("m,n,k,terms", [(1, 2048, 4096, 3), (8, 1000, 4096, 1), (64, 512, 8192, 3), (300, 300, 4096, 2), (777, 640, 2336, 3)])
def test_matmul_wide_scales(torch_cuda, moe, m, n, k, terms):
    """Scales over 16 binades.  Products are exact; each of the K * terms additions is off by at most 2^-23 of the partial sum, which
    sum |a w| bounds: |error| <= K * terms * 2^-23 * sum |a w|, plus the result's rounding.  And as a whole: the same steps taken as
    independent give sqrt(K * terms) in place of K * terms for the norm, with a factor of 4 for their spread."""
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(m + n)
    a, av = _rows(torch, rng, m, k, terms, 116, 132)
    w, wv = _rows(torch, rng, n, k, 1, 112, 128)
    want = av.sum(0) @ wv[0].T
    mass = np.abs(av).sum(0) @ np.abs(wv[0]).T
    for name in ("float32", "bfloat16"):
        got = head.Mxfp4Matmul.launch(a, w, _dtype(torch, name)).double().cpu().numpy()
        bound = k * terms * 2.0 ** -23 * mass + HALF_STEP[name] * (np.abs(want) + k * terms * 2.0 ** -23 * mass) + TINY[name]
        assert (np.abs(got - want) <= bound).all()
        if name == "float32":
            assert np.linalg.norm(got - want) <= 4 * math.sqrt(k * terms) * 2.0 ** -23 * np.linalg.norm(mass)


def test_matmul_nan_scales_stay_in_their_rows(torch_cuda, moe):
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(3)
    for m, n, k in ((3, 200, 544), (300, 300, 544)):
        a, av = _rows(torch, rng, m, k, 2, 126, 129)
        w, wv = _rows(torch, rng, n, k, 1, 126, 129)
        a.scales[1, 1, 3] = 255
        w.scales[0, 150, 16] = 255
        got = head.Mxfp4Matmul.launch(a, w, torch.float32).cpu().numpy()
        want = (av.sum(0) @ wv[0].T).astype(np.float32)
        nan = np.zeros((m, n), bool)
        nan[1, :] = nan[:, 150] = True
        assert np.isnan(got[nan]).all() and np.array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("m,n,k", [(3, 130, 96), (70, 1000, 544), (300, 257, 288)])
def test_matmul_row_stride_and_written_set(torch_cuda, moe, m, n, k):
    """The result as columns of a wider buffer with more rows than the product has: nothing else is written; scales at odd addresses."""
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(n)
    a, av = _rows(torch, rng, m, k, 3, 126, 129)
    w, wv = _rows(torch, rng, n, k, 1, 126, 129)
    buf = torch.zeros(w.scales.numel() + 1, dtype=torch.uint8, device="cuda")
    buf[1:] = w.scales.flatten()
    w = head.Mxfp4Rows(w.codes, buf[1:].view(w.scales.shape))
    want = torch.from_numpy(av.sum(0) @ wv[0].T)
    for dt in (torch.float32, torch.bfloat16):
        for pad in (5, 8):
            wide = torch.full((m + 40, n + pad), 7.0, dtype=dt, device="cuda")
            head.Mxfp4Matmul.launch(a, w, dt, out=wide[:m, :n])
            got = wide.cpu()
            assert torch.equal(got[:m, :n], want.to(torch.float32).to(dt))
            assert bool((got[m:] == 7).all()) and bool((got[:m, n:] == 7).all())


def test_offsets_past_32_bits(torch_cuda, moe):
    """Rows more than 2^31 elements into their buffers, for every operator that takes a row stride."""
    torch = torch_cuda
    from deepstrix_b200 import head
    stride = (1 << 28) + 8
    buf = torch.zeros(9 * stride + 4096, dtype=torch.bfloat16, device="cuda")
    rows = buf.as_strided((10, 4096), (stride, 1))
    rng = np.random.default_rng(1)
    x = torch.from_numpy(rng.standard_normal((10, 4096)).astype(np.float32)).cuda().to(torch.bfloat16)
    rows.copy_(x)
    q, want = head.Mxfp4Quantize.launch(rows, 2), head.Mxfp4Quantize.launch(x, 2)
    assert torch.equal(q.codes, want.codes) and torch.equal(q.scales, want.scales)
    tok = torch.arange(10, dtype=torch.int32, device="cuda")
    for p, r in zip(head.TokenLogprobs.launch(rows, tok, 4), head.TokenLogprobs.launch(x, tok, 4)):
        assert torch.equal(p, r)
    w = head.Mxfp4Quantize.launch(x[:7, :].contiguous())
    y = head.Mxfp4Matmul.launch(q, w, torch.bfloat16)
    out = buf.as_strided((10, 7), (stride, 1))
    head.Mxfp4Matmul.launch(want, w, torch.bfloat16, out=out)
    assert torch.equal(out, y)
    back = buf.as_strided((10, 4096), (stride, 1))
    head.Mxfp4Dequantize.launch(want, torch.bfloat16, out=back)
    assert torch.equal(back, head.Mxfp4Dequantize.launch(want, torch.bfloat16))


# -------------------------------------------------------------- log probabilities
def _logprobs64(x, tokens, n_alt, scale):
    """x f64 [T, V]: the definition, with the same conventions for masked and non-finite rows."""
    T, V = x.shape
    lp, ent = np.full(tokens.shape, -np.inf), np.zeros(T)
    ids, alp = np.full((T, n_alt), -1, np.int32), np.full((T, n_alt), -np.inf)
    for t in range(T):
        row = x[t]
        ok = (tokens[t] >= 0) & (tokens[t] < V)
        if np.isnan(row).any() or (row == np.inf).any():
            ent[t], alp[t] = np.nan, np.nan
            lp[t][ok] = np.nan
            continue
        if not np.isfinite(row).any():
            continue
        z = row * scale
        m = z.max()
        log_p = z - m - math.log(np.exp(z - m).sum())
        p = np.exp(log_p)
        ent[t] = -(p[p > 0] * log_p[p > 0]).sum()
        lp[t][ok] = log_p[tokens[t][ok]]
        order = np.argsort(-(row + 0.0), kind="stable")[:n_alt]
        order = order[np.isfinite(row[order])]
        ids[t, :len(order)], alp[t, :len(order)] = order, log_p[order]
    return lp, ent, ids, alp


def _near(got, want, V):
    """z - m and its product with the scale are each off by 2^-24 relatively, ln s likewise; s is off by the exponentials' 2^-21 (their
    argument's rounding weighs d * 2^-23, and d exp(d) is below 1) and by the additions, at most V / 256 + 64 in a row at 2^-24 each."""
    want = want.astype(np.float32).astype(np.float64)    # what lies below -3.4e38 (the lowest value next to a large one) is -inf in f32
    tol = 2.0 ** -20 + (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -21 * np.abs(np.where(np.isfinite(want), want, 0))
    ok = (got == want) | (np.isnan(got) & np.isnan(want)) | (np.abs(got - np.where(np.isfinite(want), want, np.inf)) <= tol)
    assert ok.all(), (got[~ok][:4], want[~ok][:4])


def _check_logprobs(torch, x, tokens, n_alt, scale=1.0):
    from deepstrix_b200 import head
    lp, ent, ids, alp = head.TokenLogprobs.launch(x, torch.from_numpy(tokens).cuda(), n_alt, scale)
    w_lp, w_ent, w_ids, w_alp = _logprobs64(x.double().cpu().numpy(), tokens, n_alt, float(np.float32(scale)))
    assert np.array_equal(ids.cpu().numpy(), w_ids)
    V = x.shape[1]
    _near(lp.double().cpu().numpy(), w_lp, V)
    # the entropy's weighted sum adds the same errors, weighted with d of at most ln V or so where it matters
    got, e_tol = ent.double().cpu().numpy(), (2.0 ** -20 + (V / 256 + 64) * 2.0 ** -24) * (2 + math.log(V + 1))
    assert ((np.abs(got - w_ent) <= e_tol) | (np.isnan(got) & np.isnan(w_ent))).all(), (got, w_ent)
    _near(alp.double().cpu().numpy(), w_alp, V)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("T,V,pad,n_alt,scale", [(1, 1, 0, 3, 1.0), (1, 2, 0, 1, 1.0), (3, 31, 2, 32, 0.5), (5, 256, 0, 0, 1.0), (1, 32000, 0, 20, 1.0),
                                                 (2, 131072, 0, 32, 1.4), (7, 50021, 3, 8, 0.8), (150, 4099, 1, 5, 1.0), (700, 1000, 0, 20, 1.0), (40, 65536, 8, 5, 1.0)])
def test_logprobs_shapes(torch_cuda, moe, T, V, pad, n_alt, scale, dtype):
    torch = torch_cuda
    rng = np.random.default_rng(T + V)
    wide = torch.from_numpy((rng.standard_normal((T, V + pad)) * 3).astype(np.float32)).cuda().to(_dtype(torch, dtype))
    tokens = rng.integers(0, V, (T, 3)).astype(np.int32)
    tokens[0] = [0, V - 1, V]            # the last one is outside
    tokens[-1, 2] = -1
    _check_logprobs(torch, wide[:, :V], tokens, n_alt, scale)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("V", [37, 4096, 70001])
def test_logprobs_hard_rows(torch_cuda, moe, V, dtype):
    """Masks (-inf), a single survivor, nothing left, the type's lowest value, NaN and +inf anywhere, ties, sorted rows, one huge logit."""
    torch = torch_cuda
    rng = np.random.default_rng(V)
    lowest = float(torch.finfo(_dtype(torch, dtype)).min)
    x = np.zeros((18, V), np.float32)
    x[0] = rng.standard_normal(V)
    x[0][rng.random(V) < 0.9] = -np.inf
    x[1] = -np.inf
    x[1, V // 2] = -5.0                   # one survivor
    x[2] = -np.inf                        # nothing left
    x[3] = lowest                         # a uniform row
    x[4] = rng.standard_normal(V)
    x[4][rng.random(V) < 0.5] = lowest
    x[5] = rng.standard_normal(V); x[5, V - 1] = np.nan
    x[6] = rng.standard_normal(V); x[6, 0] = np.inf
    x[7] = -np.inf; x[7, V // 3] = np.nan
    x[8] = 0.0                            # all equal: the lowest ids
    x[9] = rng.integers(0, 3, V)          # many ties
    x[10] = np.linspace(-40, 40, V)       # ascending
    x[11] = np.linspace(40, -40, V)       # descending
    x[12] = rng.standard_normal(V); x[12, 5] = 3.0e4
    x[13] = rng.standard_normal(V) - 3.0e4
    x[14] = 0.0; x[14, ::2] = -0.0        # signed zeros tie
    x[15] = lowest; x[15, 7] = -lowest    # the widest difference
    x[16] = -np.inf; x[16, -3:] = [1.0, 2.0, 1.0]
    x[17] = np.where(np.arange(V) % 2 == 0, np.linspace(0, 8, V), -np.inf)
    dx = torch.from_numpy(x).cuda().to(_dtype(torch, dtype))
    tokens = np.stack([np.full(18, 5), np.full(18, V // 2), np.full(18, V - 1), np.full(18, 1 << 30)], 1).astype(np.int32)
    for n_alt in (1, 20, 32):
        _check_logprobs(torch, dx, tokens, n_alt)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("V", [3, 700, 5003])
def test_logprobs_many_short_rows(torch_cuda, moe, V, dtype):
    """Enough rows for the small blocks; among them equal rows, sorted rows, masked rows, each starting at another address modulo 16."""
    torch = torch_cuda
    rng = np.random.default_rng(V)
    T = 1300
    wide = rng.standard_normal((T, V + 1)).astype(np.float32)
    x = wide[:, :V]
    x[0] = 0.0
    x[1] = np.linspace(-9, 9, V)
    x[2] = np.linspace(9, -9, V)
    x[3] = -np.inf
    x[4, ::2] = -np.inf
    x[5, V // 2] = np.nan
    x[6] = rng.integers(0, 2, V)
    x[7] = float(torch.finfo(_dtype(torch, dtype)).min)
    x[8] = np.where(np.arange(V) % 7 == 0, 2.0, 1.0)
    x[1200:1209] = x[:9]
    dx = torch.from_numpy(wide).cuda().to(_dtype(torch, dtype))[:, :V]
    _check_logprobs(torch, dx, rng.integers(-1, V + 1, (T, 2)).astype(np.int32), 20)


@pytest.mark.parametrize("T,V,given,n_alt", [(2, 40000, 1024, 16), (1300, 900, 70, 17), (64, 2048, 65, 32), (9, 300, 64, 16), (160, 20011, 63, 17)])
def test_logprobs_many_given_tokens(torch_cuda, moe, T, V, given, n_alt):
    """More given tokens than are fetched ahead, the same token more than once, tokens outside; both counts of threshold groups."""
    torch = torch_cuda
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((T, V)) * 4).astype(np.float32)
    x[0, rng.random(V) < 0.5] = -np.inf
    x[1, 3] = np.nan
    tokens = rng.integers(-2, V + 2, (T, given)).astype(np.int32)
    tokens[:, given // 2:given // 2 + 3] = tokens[:, :3]
    _check_logprobs(torch, torch.from_numpy(x).cuda(), tokens, n_alt, 0.9)


def test_logprobs_without_tokens_or_alternatives(torch_cuda, moe):
    torch = torch_cuda
    from deepstrix_b200 import head
    x = torch.randn((4, 1000), device="cuda")
    lp, ent, ids, alp = head.TokenLogprobs.launch(x)
    assert lp is None and ids.shape == (4, 0) and alp.shape == (4, 0)
    p = torch.softmax(x.double(), -1)
    assert float((ent.double() + (p * p.log()).sum(-1)).abs().max()) < 1e-5
    one = torch.tensor([3, 0, 999, 5], dtype=torch.int32, device="cuda")
    lp, *_ = head.TokenLogprobs.launch(x, one)
    assert lp.shape == (4,) and float((lp.double() - torch.log_softmax(x.double(), -1).gather(1, one[:, None].long())[:, 0]).abs().max()) < 1e-5
    assert head.TokenLogprobs.launch(x[:0], one[:0], 2)[2].shape == (0, 2)


# ------------------------------------------------------------------ together
def test_expert_store_from_float_weights(torch_cuda, moe, oracle):
    """RoutedExpertWeights.load_float: f32 weights quantised on the GPU hold the bytes the CPU quantiser gives."""
    torch = torch_cuda
    from deepstrix_b200.config import FMT_MXFP4
    rng = np.random.default_rng(9)
    st = moe.RoutedExpertWeights(FMT_MXFP4, 3, 512, 256)
    gate, down = rng.standard_normal((3, 256, 512)).astype(np.float32), rng.standard_normal((512, 256)).astype(np.float32)
    st.load_float(moe.MAT_GATE, torch.from_numpy(gate).cuda())
    st.load_float(moe.MAT_UP, torch.from_numpy(gate[::-1].copy()).cuda())
    st.load_float(moe.MAT_DOWN, torch.from_numpy(down).cuda(), slot=1)
    for slot, which, w in ((0, moe.MAT_GATE, gate[0]), (2, moe.MAT_GATE, gate[2]), (2, moe.MAT_UP, gate[0]), (1, moe.MAT_DOWN, down)):
        q, s = st.unpack(slot, which)
        want_q, want_s, _ = _oracle_rows(oracle, w, 1)
        assert np.array_equal(q.cpu().numpy(), want_q[0]) and np.array_equal(s.cpu().numpy(), want_s[0])
    st.close()


@pytest.mark.parametrize("T", [2, 40])
def test_router_weights_dequantised_right_before_the_layer(torch_cuda, moe, T):
    """The layer's router may copy its weights before the kernel ahead of it has ended: what the dequantiser writes is complete all the same."""
    torch = torch_cuda
    from deepstrix_b200 import head, synth
    from deepstrix_b200.config import MoeConfig, RouterConfig
    cfg = MoeConfig(hidden=512, ffn=256, shared_ffn=256,
                    router=RouterConfig(n_expert=32, n_used=4, n_group=1, topk_group=1, score_fn=1, route_scale=2.5))
    w = synth.make_layer(cfg, 4)
    routers = [head.Mxfp4Quantize.launch(torch.from_numpy(w["router_w"]).cuda().roll(i, 0), 3) for i in range(2)]
    buffer = torch.empty((32, 512), dtype=torch.float32, device="cuda")
    store = moe.RoutedExpertWeights.from_host(cfg.fmt, cfg.hidden, cfg.ffn, w["gate"], w["up"], w["down"])
    shared = moe.RoutedExpertWeights.from_host(cfg.fmt, cfg.hidden, cfg.shared_ffn, w["shared_gate"], w["shared_up"], w["shared_down"])
    layer = moe.MoeLayer(cfg, store, shared, buffer, torch.from_numpy(w["router_bias"]).cuda(), max_tokens=T)
    x = torch.from_numpy(synth.make_tokens(cfg, 4, T).view(np.int16)).cuda().view(torch.bfloat16)
    want = []
    for q in routers:
        head.Mxfp4Dequantize.launch(q, torch.float32, out=buffer)
        torch.cuda.synchronize()
        want.append(layer.forward(x))
        torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    got = []
    for i in range(40):
        head.Mxfp4Dequantize.launch(routers[i % 2], torch.float32, out=buffer)
        got.append(layer.forward(x))
    assert all(torch.equal(g, want[i % 2]) for i, g in enumerate(got)) and layer.check() == 0


def _head_inputs(torch, T, H, V, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((T, H), generator=g, device="cuda"), torch.rand((H,), generator=g, device="cuda") + 0.5,
            torch.randn((V, H), generator=g, device="cuda") / math.sqrt(H), torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32))


def _head_step(torch, moe, x, norm, w, tokens, dtype):
    from deepstrix_b200 import head
    _, rows = moe.RmsNorm.launch_weighted_batched(x, norm)
    logits = head.Mxfp4Matmul.launch(head.Mxfp4Quantize.launch(rows, 3), w, dtype)
    return (rows, logits) + head.TokenLogprobs.launch(logits, tokens, 4)


@pytest.mark.parametrize("T", [1, 9, 200])
def test_norm_head_logprobs_together(torch_cuda, moe, T):
    """Norm -> three-term rows -> product with a quantised head -> log probabilities, against f64 from the norm's own rows."""
    torch = torch_cuda
    from deepstrix_b200 import head
    x, norm, weight, tokens = _head_inputs(torch, T, 2048, 5003, T)
    w = head.Mxfp4Quantize.launch(weight)
    rows, logits, lp, ent, ids, alp = _head_step(torch, moe, x, norm, w, tokens, torch.float32)
    w64 = torch.from_numpy(_values64(w.codes[0].cpu().numpy(), w.scales[0].cpu().numpy())).cuda()
    exact = rows.double() @ w64.T
    # what three terms drop, x minus their sum, is measured; Cauchy-Schwarz turns its norm into a bound on the logits
    rest = rows.double() - head.Mxfp4Dequantize.launch(head.Mxfp4Quantize.launch(rows, 3), torch.float32).double()
    slack = rest.norm(dim=1, keepdim=True) * w64.norm(dim=1)[None] + 3 * 2048 * 2.0 ** -23 * (rows.double().abs() @ w64.abs().T) * 1.1
    assert bool(((logits.double() - exact).abs() <= slack).all())
    ref = torch.log_softmax(logits.double(), -1)
    assert float((lp.double() - ref.gather(1, tokens[:, None].long())[:, 0]).abs().max()) < 2e-5
    top = logits.double().topk(4, -1)
    assert torch.equal(torch.gather(logits.double(), 1, ids.long()), top.values)


@pytest.mark.parametrize("T", [3, 150])
def test_captured_head_replays_on_new_inputs(torch_cuda, moe, T):
    """The whole step captured into a graph, replayed twice on other inputs in the same buffers; two graphs at once on two streams."""
    torch = torch_cuda
    from deepstrix_b200 import head
    graphs, states = [], []
    for s in range(2):
        x, norm, weight, tokens = _head_inputs(torch, T, 1024, 3001, s)
        w = head.Mxfp4Quantize.launch(weight)
        _head_step(torch, moe, x, norm, w, tokens, torch.float32)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _head_step(torch, moe, x, norm, w, tokens, torch.float32)
        graphs.append(g)
        states.append((x, norm, w, tokens, out))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed in (11, 12):
        for s in range(2):
            states[s][0].copy_(_head_inputs(torch, T, 1024, 3001, seed + 10 * s)[0])
        torch.cuda.synchronize()
        for s in range(2):
            with torch.cuda.stream(streams[s]):
                graphs[s].replay()
        torch.cuda.synchronize()
        for x, norm, w, tokens, out in states:
            for got, want in zip(out, _head_step(torch, moe, x, norm, w, tokens, torch.float32)):
                assert torch.equal(got, want)


@pytest.fixture(autouse=True)
def _no_wait_ran_out(torch_cuda, moe):
    yield
    from deepstrix_b200 import head
    assert head.check() == 0


def test_same_bits_on_every_call_and_stream(torch_cuda, moe):
    """No sum depends on the order in which blocks finish: repeated calls, on two streams at once, give the same bits."""
    torch = torch_cuda
    from deepstrix_b200 import head
    for T, H, V in ((1, 4096, 2048), (6, 8192, 300), (260, 544, 700)):
        x, norm, weight, tokens = _head_inputs(torch, T, H, V, 5)
        w = head.Mxfp4Quantize.launch(weight)
        want = _head_step(torch, moe, x, norm, w, tokens, torch.float32)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for i in range(12):
            with torch.cuda.stream(streams[i % 2]):
                outs.append(_head_step(torch, moe, x, norm, w, tokens, torch.float32))
        torch.cuda.synchronize()
        for out in outs:
            for p, r in zip(out, want):
                assert torch.equal(p, r)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("T,V", [(6, 701), (6, 9001), (6, 131077), (1200, 4099)])
def test_logprobs_long_candidate_lists(torch_cuda, moe, T, V, dtype):
    """Rows of which far more logits reach the threshold than a block lists, so that warps keep their best in a second pass: few survivors of a
    mask by the type's lowest value, steps that rise and fall in plateaus of uneven width, few levels, candidates on some lanes only."""
    torch = torch_cuda
    rng = np.random.default_rng(V)
    lowest = float(torch.finfo(_dtype(torch, dtype)).min)
    i = np.arange(V)
    wide = np.zeros((T, V + 1), np.float32)      # V + 1: rows start at different addresses modulo 16
    x = wide[:, :V]
    x[0] = lowest
    x[0, rng.choice(V, 3, replace=False)] = [1.0, 2.0, 1.0]
    x[1] = np.cumsum(rng.random(V) < 1 / 37) * 0.125 - 40      # rises, plateaus of 1 to a few hundred
    x[2] = -x[1] - 80
    x[3] = rng.integers(0, 3, V)
    x[4] = np.where(i // 8 % 5 == 0, np.minimum(i, 4000) * 0.0078125, lowest)   # rises on one chunk of five or so, then level
    x[5] = np.where(rng.random(V) < 0.3, 0.0, -0.0)
    x[6:] = x[np.arange(T - 6) % 6]
    dx = torch.from_numpy(wide).cuda().to(_dtype(torch, dtype))[:, :V]
    tokens = rng.integers(0, V, (T, 1)).astype(np.int32)
    for n_alt in (1, 20, 32):
        _check_logprobs(torch, dx, tokens, n_alt)


@pytest.mark.parametrize("m,n,k,terms", [(4100, 4100, 1024, 1), (4100, 4100, 1536, 2), (4100, 4100, 1024, 3), (2100, 5003, 1056, 1), (2050, 2100, 1536, 3)])
def test_matmul_pairs_of_ctas_exact_sums(torch_cuda, moe, m, n, k, terms):
    """Products large enough for pairs of CTAs, several tiles a pair, scales by TMA and by loaders; exact for the same reason as above.  Twice
    on two streams at once: each CTA of a pair reads what the other one's copies brought."""
    torch = torch_cuda
    from deepstrix_b200 import head
    rng = np.random.default_rng(m + n + k + terms)
    a, av = _rows(torch, rng, m, k, terms, 126, 129)
    w, wv = _rows(torch, rng, n, k, 1, 126, 129)
    want = torch.from_numpy(av.sum(0)).cuda() @ torch.from_numpy(wv[0]).cuda().T      # f64: exact
    assert float(want.abs().max()) * 16 < 2 ** 22
    want = want.float()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            got.append(head.Mxfp4Matmul.launch(a, w, torch.float32))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g, want)
    assert torch.equal(head.Mxfp4Matmul.launch(a, w, torch.bfloat16), want.to(torch.bfloat16))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_expert_store_refuses_weights_that_are_not_finite(torch_cuda, moe, value):
    """load_float with one bad weight is refused and leaves the store as it was; its neighbours in the type's range are taken."""
    torch = torch_cuda
    from deepstrix_b200.config import FMT_MXFP4
    st = moe.RoutedExpertWeights(FMT_MXFP4, 2, 512, 256)
    w = torch.randn((2, 256, 512), generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    w[0, 3, 3] = torch.finfo(torch.float32).max
    st.load_float(moe.MAT_GATE, w)
    before = [t.clone() for slot in range(2) for t in st.unpack(slot, moe.MAT_GATE)]
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        bad = torch.randn((2, 256, 512), device="cuda").to(dtype)
        bad[1, 255, 511] = value
        with pytest.raises(AssertionError, match="infinite or NaN"):
            st.load_float(moe.MAT_GATE, bad)
        with pytest.raises(AssertionError, match="infinite or NaN"):
            st.load_float(moe.MAT_GATE, bad[1], slot=1)
    after = [t for slot in range(2) for t in st.unpack(slot, moe.MAT_GATE)]
    assert all(torch.equal(a, b) for a, b in zip(before, after))
    st.close()
