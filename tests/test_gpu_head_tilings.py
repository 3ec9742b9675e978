"""Every form of the MXFP4 product, pinned, so that what is tested does not depend on which one the model of its time chooses: pairs of CTAs
and single ones, one to three terms, scales by TMA and by loaders, rings that wrap over several tiles, columns split over clusters."""
import ctypes as C
import itertools
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

E2M1 = [0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6]


@pytest.fixture(autouse=True)
def _unpinned_and_clean(torch_cuda, moe):
    from deepstrix_b200 import head
    yield
    head.Mxfp4Matmul.pin()
    head.Mxfp4Matmul.set_polls()
    assert head.check() == 0


def _rows(torch, g, terms, rows, k, shift=0):
    """Random MXFP4 rows with scales of 2^-1 .. 2^1 (sums of products are exact in f32, see test_matmul_exact_sums), their f64 values summed over
    the terms; the scale bytes start `shift` bytes off a 16-byte boundary."""
    from deepstrix_b200 import head
    codes = torch.randint(0, 256, (terms, rows, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    buf = torch.randint(126, 129, (terms * rows * (k // 32) + shift,), generator=g, device="cuda", dtype=torch.uint8)
    scales = buf[shift:].view(terms, rows, k // 32)
    table = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    total = torch.zeros((rows, k), dtype=torch.float64, device="cuda")
    for t in range(terms):
        v = torch.stack([table[(codes[t] & 15).long()], table[(codes[t] >> 4).long()]], -1).view(rows, k // 32, 32)
        total += (v * torch.exp2(scales[t].double() - 127)[..., None]).view(rows, k)
    return head.Mxfp4Rows(codes, scales), total


def _check_product(torch, a, av, w, wv, dtype):
    """Exact, in place in a wider buffer, nothing else written, the same bits again; then with one NaN scale on either side."""
    from deepstrix_b200 import head
    m, n = av.shape[0], wv.shape[0]
    exact = av @ wv.T
    assert float(exact.abs().max()) * 16 < 2 ** 22
    want = exact.float().to(dtype)
    wide = torch.full((m + 9, n + 6), 7.0, dtype=dtype, device="cuda")
    head.Mxfp4Matmul.launch(a, w, dtype, out=wide[:m, :n])
    assert torch.equal(wide[:m, :n], want) and bool((wide[m:] == 7).all()) and bool((wide[:m, n:] == 7).all())
    assert torch.equal(head.Mxfp4Matmul.launch(a, w, dtype), want)
    term, row, col = a.n_terms - 1, m - 2, n // 2
    kept = a.scales[term, row, -1].item(), w.scales[0, col, 0].item()
    a.scales[term, row, -1], w.scales[0, col, 0] = 255, 255
    got = head.Mxfp4Matmul.launch(a, w, dtype)
    a.scales[term, row, -1], w.scales[0, col, 0] = kept
    assert bool(got[row].isnan().all()) and bool(got[:, col].isnan().all())
    rest = torch.ones((m, n), dtype=torch.bool, device="cuda")
    rest[row], rest[:, col] = False, False
    assert torch.equal(got[rest], want[rest])


PAIRS = [(1, t) for t in (16, 48, 112, 128, 144, 208)] + [(2, t) for t in (16, 80, 128)] + [(3, t) for t in (16, 96, 112, 128)]
SINGLES = [(1, t) for t in (16, 32, 80, 112, 128, 160, 208)] + [(2, t) for t in (16, 64, 96)] + [(3, t) for t in (16, 32, 48, 64)]
FORMS = [(1,) + f for f in PAIRS] + [(0,) + f for f in SINGLES]


@pytest.mark.parametrize("pair,terms,tokens", FORMS)
def test_pinned_tiles(torch_cuda, moe, pair, terms, tokens):
    """Four tiles and more for some CTAs (rings of stages, buffers and slots wrap over tiles), ragged at both ends.  K: two and five steps of
    scales by TMA, an odd and an even number of stages by loaders, one short stage, scales at odd addresses."""
    torch = torch_cuda
    from deepstrix_b200 import head
    g = torch.Generator(device="cuda").manual_seed(tokens * 8 + terms * 2 + pair)
    head.Mxfp4Matmul.pin(pair, tokens, 1)
    m, rows_w = 4 * tokens - 5, 256 if pair else 128
    at_once = head.Mxfp4Matmul.tiling(terms, m, 4096, 1024)["at_once"]
    n_tiles = -(-(3 * at_once + 2) // 4)
    for k, odd, shift, dtype in ((1024, 0, 0, torch.float32), (2560, 1, 0, torch.bfloat16), (1056, 0, 0, torch.bfloat16), (1312, 1, 3, torch.float32),
                                 (160, 0, 0, torch.float16)):
        n = n_tiles * rows_w - 2 - odd
        t = head.Mxfp4Matmul.tiling(terms, m, n, k)
        assert (t["pair"], t["tokens"], t["splits"]) == (pair, tokens, 1) and t["tiles"] > 3 * t["at_once"]
        a, av = _rows(torch, g, terms, m, k, shift)
        w, wv = _rows(torch, g, 1, n, k, shift)
        _check_product(torch, a, av, w, wv, dtype)


@pytest.mark.parametrize("terms,tokens", SINGLES)
@pytest.mark.parametrize("splits", [2, 4, 8])
def test_pinned_splits(torch_cuda, moe, terms, tokens, splits):
    """Columns of a tile shared by a cluster: even and uneven shares, shares that begin inside a buffer of scales."""
    torch = torch_cuda
    from deepstrix_b200 import head
    g = torch.Generator(device="cuda").manual_seed(tokens * 8 + terms * 2 + splits)
    head.Mxfp4Matmul.pin(0, tokens, splits)
    for m, n, k, dtype in ((2 * tokens - 3, 301, 256 * splits, torch.float32), (tokens, 130, 4608, torch.bfloat16), (tokens + 1, 257, 2336, torch.float32)):
        assert head.Mxfp4Matmul.tiling(terms, m, n, k)["splits"] == splits
        a, av = _rows(torch, g, terms, m, k)
        w, wv = _rows(torch, g, 1, n, k)
        _check_product(torch, a, av, w, wv, dtype)


def test_forms_cover_the_rings(torch_cuda, moe):
    """The pinned forms include what differs in their synchronisation: two and four buffers of scales, two, three and four slots."""
    from deepstrix_b200 import head
    seen = set()
    for pair, terms, tokens in FORMS:
        head.Mxfp4Matmul.pin(pair, tokens, 1)
        t = head.Mxfp4Matmul.tiling(terms, 1000, 4096, 1024)
        seen.add((pair, t["scale_bufs"], t["slots"]))
    assert {(1, 4, 2), (1, 2, 4), (1, 4, 4), (0, 2, 2), (0, 2, 3), (0, 2, 4), (0, 4, 4)} <= seen, seen


def test_pinned_forms_agree_and_a_pin_is_taken_back(torch_cuda, moe):
    """Forms of the same product give the same exact sums; what cannot be done as pinned is refused and writes nothing."""
    torch = torch_cuda
    from deepstrix_b200 import head
    g = torch.Generator(device="cuda").manual_seed(1)
    a, av = _rows(torch, g, 3, 300, 1536)
    w, wv = _rows(torch, g, 1, 700, 1536)
    chosen = head.Mxfp4Matmul.tiling(3, 300, 700, 1536)
    want = (av @ wv.T).float()
    for pair, tokens in itertools.product((0, 1), (16, 48, 64, 96, 128)):
        head.Mxfp4Matmul.pin(pair, tokens)
        if pair or tokens * 3 <= 208:
            assert torch.equal(head.Mxfp4Matmul.launch(a, w, torch.float32), want)
            continue
        out = torch.full((300, 700), 7.0, device="cuda")
        with pytest.raises(moe.DsxError, match="pinned"):
            head.Mxfp4Matmul.launch(a, w, torch.float32, out=out)
        assert bool((out == 7).all())
    head.Mxfp4Matmul.pin()
    assert head.Mxfp4Matmul.tiling(3, 300, 700, 1536) == chosen


def test_chosen_forms(torch_cuda, moe):
    """What the model chooses on a whole B200 where the difference is large: clusters for one small matrix, single CTAs for a few tokens on a large one,
    pairs for prompts."""
    torch = torch_cuda
    from deepstrix_b200 import head
    if torch.cuda.get_device_properties(0).multi_processor_count < 140:
        pytest.skip("a partition of a device")
    tiling = head.Mxfp4Matmul.tiling
    assert tiling(3, 1, 1024, 2048)["splits"] > 1 and tiling(3, 1, 1024, 2048)["pair"] == 0
    assert (tiling(3, 8, 131072, 4096)["pair"], tiling(3, 8, 131072, 4096)["splits"]) == (0, 1)
    for terms in (1, 2, 3):
        assert tiling(terms, 8192, 8192, 4096)["pair"] == 1


@pytest.mark.parametrize("pin,terms,m,n,k", [((0, 16, 2), 3, 30, 300, 65536), ((0, 16, 1), 1, 100, 40000, 16384), ((0, 208, 1), 1, 500, 3000, 16416),
                                             ((1, 128, 1), 3, 1000, 20000, 16384), ((1, 208, 1), 1, 1000, 20000, 16416), ((1, 16, 1), 2, 100, 20000, 16384)])
def test_a_wait_that_runs_out_is_reported(torch_cuda, moe, pin, terms, m, n, k):
    """With waits of one poll (a few us, where a tile takes 20 and more) the product gives up, says so once, and returns: the call after it is right."""
    torch = torch_cuda
    from deepstrix_b200 import head
    g = torch.Generator(device="cuda").manual_seed(k + terms)

    def rows(t, r):
        return head.Mxfp4Rows(torch.randint(0, 256, (t, r, k // 2), generator=g, device="cuda", dtype=torch.uint8),
                              torch.randint(120, 125, (t, r, k // 32), generator=g, device="cuda", dtype=torch.uint8))
    a, w = rows(terms, m), rows(1, n)
    head.Mxfp4Matmul.pin(*pin)
    want = head.Mxfp4Matmul.launch(a, w, torch.float32)
    assert head.check() == 0
    wide = torch.full((m + 3, n + 5), 7.0, device="cuda")
    for polls in (1, 2):
        head.Mxfp4Matmul.set_polls(polls)
        head.Mxfp4Matmul.launch(a, w, torch.float32, out=wide[:m, :n])
        head.Mxfp4Matmul.launch(a, w, torch.float32, out=wide[:m, :n])
        head.Mxfp4Matmul.set_polls()
        got = head.Mxfp4Matmul.launch(a, w, torch.float32)
        assert head.check() == 1 and head.check() == 0
        assert torch.equal(got, want)
        assert bool((wide[m:] == 7).all()) and bool((wide[:, n:] == 7).all())
    word = C.c_uint32()
    head.Mxfp4Matmul.set_polls(1)
    head.Mxfp4Matmul.launch(a, w, torch.float32)
    head.Mxfp4Matmul.set_polls()
    assert moe.lib().dsx_head_check(moe._stream(), C.byref(word)) == -3 and word.value == 1


FIRST_CALLS = """
import sys, threading
sys.path.insert(0, sys.argv[1])
import torch
from deepstrix_b200 import head
def rows(t, r, k):
    return head.Mxfp4Rows(torch.randint(0, 256, (t, r, k // 2), device="cuda", dtype=torch.uint8),
                          torch.randint(126, 129, (t, r, k // 32), device="cuda", dtype=torch.uint8))
sizes = [(1, 300, 2048, 3), (40, 700, 544, 2), (2000, 3000, 1024, 3), (300, 300, 1024, 1)] * 4
work = [(rows(t, m, k), rows(1, n, k)) for m, n, k, t in sizes]
torch.cuda.synchronize()
got, start = [None] * len(work), threading.Barrier(len(work))
def call(i):
    with torch.cuda.stream(torch.cuda.Stream()):
        start.wait()
        got[i] = [head.Mxfp4Matmul.launch(*work[i], torch.float32) for _ in range(3)]
threads = [threading.Thread(target=call, args=(i,)) for i in range(len(work))]
[t.start() for t in threads]
[t.join() for t in threads]
torch.cuda.synchronize()
for (a, w), results in zip(work, got):
    want = head.Mxfp4Matmul.launch(a, w, torch.float32)
    assert all(torch.equal(r, want) for r in results)
assert head.check() == 0
print("same")
"""


def test_first_calls_of_a_process_from_many_threads(torch_cuda, moe):
    """What the product looks up once a device is looked up by sixteen threads at once: each gets the results that a single thread does."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for _ in range(2):
        out = subprocess.run([sys.executable, "-c", FIRST_CALLS, root], capture_output=True, text=True, timeout=300)
        assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr[-2000:]


@pytest.mark.parametrize("fmt", ["mxfp4", "q8_0"])
@pytest.mark.parametrize("T", [300, 2500])
def test_product_beside_the_layer(torch_cuda, moe, fmt, T):
    """Products of every kind of block on one stream, the layer's tensor-core kernels on another: they share SMs and tensor memory, and both
    write the bits that they write alone."""
    import numpy as np

    from deepstrix_b200 import head, synth
    from deepstrix_b200.config import FMT_MXFP4, FMT_Q8_0, MoeConfig, RouterConfig
    torch = torch_cuda
    cfg = MoeConfig(hidden=1024, ffn=512, shared_ffn=512, fmt=FMT_MXFP4 if fmt == "mxfp4" else FMT_Q8_0,
                    router=RouterConfig(n_expert=32, n_used=4, n_group=1, topk_group=1, score_fn=1, route_scale=2.5))
    layer = moe.build_layer_from_host(cfg, synth.make_layer(cfg, 5), max_tokens=T)
    x = torch.from_numpy(synth.make_tokens(cfg, 5, T).view(np.int16)).cuda().view(torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(T)
    work = [(pin, _rows(torch, g, terms, m, k)[0], _rows(torch, g, 1, n, k)[0])
            for pin, terms, m, n, k in (((0, 16, 1), 3, 16, 40000, 1024), ((0, 16, 8), 3, 1, 1024, 2048), ((1, 208, 1), 1, 900, 9000, 1024),
                                        ((0, 208, 1), 1, 400, 9000, 1056), ((1, 128, 1), 3, 500, 5000, 1056))]

    def products(times):
        results = []
        for pin, a, w in work * times:
            head.Mxfp4Matmul.pin(*pin)
            results.append(head.Mxfp4Matmul.launch(a, w, torch.float32))
        head.Mxfp4Matmul.pin()
        return results
    want_layer, want = layer.forward(x), products(1)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(6):
        with torch.cuda.stream(one):
            got = products(3)
        with torch.cuda.stream(two):
            got_layer = [layer.forward(x) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(r, want[i % len(want)]) for i, r in enumerate(got))
        assert all(torch.equal(r.view(torch.int16), want_layer.view(torch.int16)) for r in got_layer)
    assert layer.check() == 0
