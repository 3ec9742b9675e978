"""Cases, plain forms and 64-bit definitions of the quantised head's operators: MXFP4 rows (quantise, dequantise), their product,
and the log probabilities of given tokens with entropy and top alternatives.

`own` chooses between the plain torch form of an operator and the library's kernels; inputs, cases and the counted work are the same."""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
LARGEST_FLOP = 2 * 8192 * 8192 * 4096
LARGEST_QUANT = 65536 * 2048
LARGEST_ROWS = 4096 * 131072


def listed():
    return [
        # activations of a full decode batch on their way into an accurate (three-term) product
        {"name": "quantise_decode_b64", "op": "quantise", "rows": 64, "k": 4096, "pad": 0, "terms": 3, "dtype": "bf16"},
        # a ragged batch of f16 rows that are a slice of a wider buffer
        {"name": "quantise_ragged", "op": "quantise", "rows": 1237, "k": 2304, "pad": 96, "terms": 2, "dtype": "f16"},
        # the activations of a whole prompt, one term
        {"name": "quantise_prefill", "op": "quantise", "rows": 8192, "k": 4096, "pad": 0, "terms": 1, "dtype": "bf16"},
        # 32 experts' worth of down projections in f32 on their way into an expert store
        {"name": "quantise_weights", "op": "quantise", "rows": 65536, "k": 2048, "pad": 0, "terms": 1, "dtype": "f32"},
        # a projection of the small configuration, one token: launch latency
        {"name": "linear_one_token", "op": "linear", "m": 1, "n": 1024, "k": 2048, "terms": 3, "dtype": "bf16", "out": "bf16"},
        # the output head of a decode batch: the weights' bytes
        {"name": "linear_head_b8", "op": "linear", "m": 8, "n": 131072, "k": 4096, "terms": 3, "dtype": "bf16", "out": "f32"},
        # odd sizes, a few hundred tokens, accurate activations
        {"name": "linear_ragged", "op": "linear", "m": 777, "n": 5119, "k": 2336, "terms": 3, "dtype": "f16", "out": "f16"},
        # both operands quantised, a whole prompt: the tensor cores
        {"name": "product_prefill", "op": "product", "m": 8192, "n": 8192, "k": 4096, "terms": 1, "dtype": "bf16", "out": "bf16"},
        # one row of logits: latency
        {"name": "logprobs_one_row", "op": "logprobs", "t": 1, "v": 32000, "pad": 0, "given": 1, "alts": 5, "temp": 1.0, "masked": 0.0, "dtype": "f32"},
        # a decode batch with a vocabulary mask
        {"name": "logprobs_decode_b64", "op": "logprobs", "t": 64, "v": 131072, "pad": 0, "given": 1, "alts": 20, "temp": 0.7, "masked": 0.5, "dtype": "f32"},
        # odd vocabulary, a slice of wider rows, several given tokens each
        {"name": "logprobs_ragged", "op": "logprobs", "t": 333, "v": 50021, "pad": 3, "given": 4, "alts": 8, "temp": 1.3, "masked": 0.1, "dtype": "f16"},
        # teacher-forced scoring of a whole prompt
        {"name": "logprobs_prompt", "op": "logprobs", "t": 4096, "v": 131072, "pad": 0, "given": 1, "alts": 5, "temp": 1.0, "masked": 0.0, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantise", "linear", "product", "logprobs"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "quantise":
        k = 32 * _log_int(rng, 1, 256)
        terms = rng.choice([1, 2, 3])
        rows = _log_int(rng, 1, min(65536, LARGEST_QUANT // (2 * k * terms)))
        return {"op": op, "rows": rows, "k": k, "pad": rng.choice([0, 0, 8, 96]), "terms": terms, "dtype": dtype}
    if op in ("linear", "product"):
        terms = rng.choice([1, 2, 3])
        k = 32 * _log_int(rng, 1, 256)
        n = _log_int(rng, 1, 32768)
        m = _log_int(rng, 1, max(1, min(8192, LARGEST_FLOP // (2 * n * k * terms))))
        return {"op": op, "m": m, "n": n, "k": k, "terms": terms, "dtype": dtype, "out": rng.choice(["f32", "bf16", "f16"])}
    v = _log_int(rng, 2, 131072)
    t = _log_int(rng, 1, max(1, min(4096, LARGEST_ROWS // (2 * v))))
    return {"op": op, "t": t, "v": v, "pad": rng.choice([0, 0, 1, 8]), "given": rng.choice([1, 1, 4]), "alts": rng.choice([0, 1, 5, 20, 32]),
            "temp": rng.choice([1.0, 0.7, 1.3]), "masked": rng.choice([0.0, 0.1, 0.9]), "dtype": dtype}


def _normed_rows(g, rows, k, dtype):
    """Rows as a norm leaves them: unit scale, a few channels an order of magnitude above the rest."""
    x = torch.randn((rows, k), generator=g, device=DEV)
    x *= torch.where(torch.rand((k,), generator=g, device=DEV) < 0.01, 12.0, 1.0)
    return x.to(dtype)


def _stored_weight(g, n, k):
    """An MXFP4 matrix as a checkpoint holds it: packed E2M1 codes (element 2i in the low nibble) and E8M0 bytes."""
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(116, 123, (n, k // 32), generator=g, device=DEV, dtype=torch.uint8)
    return codes, scales


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    op = case["op"]
    if op == "quantise":
        wide = _normed_rows(g, case["rows"], case["k"] + case["pad"], DTYPES[case["dtype"]])
        return {"case": case, "x": wide[:, :case["k"]]}
    if op in ("linear", "product"):
        x = _normed_rows(g, case["m"], case["k"], DTYPES[case["dtype"]])
        w = _stored_weight(g, case["n"], case["k"])
        state = {"case": case, "w_codes": w[0], "w_scales": w[1]}
        if op == "linear":
            return {**state, "x": x}
        values, exponents = _terms(x.float(), case["terms"])
        return {**state, "a_codes": _pack(values, exponents), "a_scales": exponents}
    t, v = case["t"], case["v"]
    wide = torch.randn((t, v + case["pad"]), generator=g, device=DEV) * 2.5
    logits = wide[:, :v]
    if case["masked"]:
        logits.masked_fill_(torch.rand((t, v), generator=g, device=DEV) < case["masked"], -math.inf)
    tokens = torch.randint(0, v, (t, case["given"]), generator=g, device=DEV, dtype=torch.int32)
    dtype = DTYPES[case["dtype"]]
    return {"case": case, "logits": logits if dtype == torch.float32 else wide.to(dtype)[:, :v], "tokens": tokens}


# ------------------------------------------------------------------ plain forms
def _term(x):
    """One MXFP4 term of f32 rows: the values (f32, exact) and the E8M0 bytes."""
    b = x.reshape(x.shape[0], -1, 32)
    bits = b.abs().amax(-1).view(torch.int32)
    e = ((bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x400000).int()).clamp(1, 253)
    s = (e << 23).view(torch.float32)[..., None]
    v = b / s
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step * s, v).reshape(x.shape), e.to(torch.uint8)


def _terms(x, n):
    """n terms, each of what the earlier ones leave over: values [n, R, K], bytes [n, R, K / 32]."""
    v, e = _term(x)
    if n == 1:
        return v[None], e[None]
    rest, more = _terms(x - v, n - 1)
    return torch.cat([v[None], rest]), torch.cat([e[None], more])


def _pack(values, exponents):
    s = (exponents.to(torch.int32) << 23).view(torch.float32)
    v = values.reshape(*exponents.shape, 32) / s[..., None]
    mag = torch.bucketize(v.abs(), torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=v.device))
    code = (mag + 8 * torch.signbit(v)).to(torch.uint8).reshape(values.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(codes, scales):
    """f32 values of packed codes [..., K / 2] with E8M0 bytes [..., K / 32]."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    v = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).reshape(*scales.shape, 32)
    return (v * (scales.to(torch.int32) << 23).view(torch.float32)[..., None]).reshape(*codes.shape[:-1], -1)


def _plain_logprobs(logits, tokens, n_alt, scale):
    x = logits.float() + 0.0
    z = x * scale
    top = z.amax(-1, keepdim=True)
    none = torch.isinf(top)
    d = z - torch.where(none, 0.0, top)
    w = torch.exp(d)
    s = w.sum(-1, keepdim=True)
    log_s = torch.where(none, 0.0, s.log())
    weighted = torch.where(w > 0, w * d, 0.0).sum(-1, keepdim=True) / torch.where(none, 1.0, s)
    logp = d.gather(1, tokens.long()) - log_s
    n = min(n_alt, x.shape[1])
    bits = x.view(torch.int32).long()
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) + torch.arange(x.shape[1] - 1, -1, -1, device=x.device)
    ids = x.shape[1] - 1 - (key.topk(n, -1).values & 0xFFFFFFFF)
    alt = d.gather(1, ids) - log_s
    ids = torch.where(torch.isinf(x.gather(1, ids)), -1, ids).int()
    more = (x.shape[0], n_alt - n)
    return {"logprobs": logp, "entropy": (log_s - weighted)[:, 0],
            "ids": torch.cat([ids, ids.new_full(more, -1)], 1), "alternatives": torch.cat([alt, alt.new_full(more, -math.inf)], 1)}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "quantise":
        values, exponents = _terms(state["x"].float(), case["terms"])
        return {"values": values.sum(0).to(state["x"].dtype), "exponents": exponents}
    if case["op"] == "logprobs":
        return _plain_logprobs(state["logits"], state["tokens"], case["alts"], 1.0 / case["temp"])
    a = _terms(state["x"].float(), case["terms"])[0] if case["op"] == "linear" else _values(state["a_codes"], state["a_scales"])
    return {"out": (a.sum(0) @ _values(state["w_codes"], state["w_scales"]).T).to(DTYPES[case["out"]])}


def _run_own(case, state):
    from deepstrix_b200 import head
    if case["op"] == "quantise":
        q = head.Mxfp4Quantize.launch(state["x"], case["terms"])
        return {"values": head.Mxfp4Dequantize.launch(q, state["x"].dtype), "exponents": q.scales}
    if case["op"] == "logprobs":
        logprobs, entropy, ids, alternatives = head.TokenLogprobs.launch(state["logits"], state["tokens"], case["alts"], 1.0 / case["temp"])
        return {"logprobs": logprobs, "entropy": entropy, "ids": ids, "alternatives": alternatives}
    a = head.Mxfp4Quantize.launch(state["x"], case["terms"]) if case["op"] == "linear" else head.Mxfp4Rows(state["a_codes"], state["a_scales"])
    return {"out": head.Mxfp4Matmul.launch(a, head.Mxfp4Rows(state["w_codes"], state["w_scales"]), DTYPES[case["out"]])}


def work(case):
    if case["op"] == "quantise":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * SIZE[case["dtype"]] + case["terms"] * 17 / 32), "flops": 4.0 * n * case["terms"]}
    if case["op"] == "logprobs":
        t = case["t"]
        return {"bytes": t * (case["v"] * SIZE[case["dtype"]] + 4 * (2 * case["given"] + 1 + 2 * case["alts"])), "flops": 6.0 * t * case["v"]}
    m, n, k = case["m"], case["n"], case["k"]
    a = m * k * (SIZE[case["dtype"]] if case["op"] == "linear" else case["terms"] * 17 / 32)
    return {"bytes": a + n * k * 17 / 32 + m * n * SIZE[case["out"]], "flops": 2.0 * m * n * k}


# ------------------------------------------------------ definitions in 64 bits
def _exact_terms(x, n):
    """Sum of n terms by the definition: scale 2^ceil(log2(amax / 6)), nearest E2M1 value (ties to the even code)."""
    b = x.reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(amax / 6)   # in [0.5, 1): the power of two itself where it is 0.5 (a logarithm would have to be exact there)
    s = torch.ldexp(torch.ones_like(amax), (exponent - (mantissa == 0.5).int()).clamp(-126, 126))
    a = b.abs() / s
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)).long()
    v = torch.sign(b) * s * torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)[code]
    v = v.reshape(x.shape)
    return v if n == 1 else v + _exact_terms(x - v, n - 1)


def _exact_values(codes, scales):
    nib = torch.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).long()
    mag, sign = nib & 7, 1 - 2 * (nib >> 3)
    v = torch.where(mag < 2, mag * 0.5, (2.0 + (mag & 1)) * torch.exp2(((mag >> 1) - 2).double()))
    return sign * v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "quantise":
        return {"values": _exact_terms(state["x"].double(), case["terms"]), "exponents": None}
    if case["op"] in ("linear", "product"):
        a = _exact_terms(state["x"].double(), case["terms"]) if case["op"] == "linear" else _exact_values(state["a_codes"], state["a_scales"]).sum(0)
        return {"out": a @ _exact_values(state["w_codes"], state["w_scales"]).T}
    z = state["logits"].double() / case["temp"]
    log_z = torch.logsumexp(z, -1, keepdim=True)
    empty = torch.isinf(log_z)
    logp = torch.where(empty, -math.inf, z - log_z)
    p = logp.exp()
    entropy = -torch.where(p > 0, p * logp, 0.0).sum(-1)
    alternatives = torch.full((case["t"], case["alts"]), -math.inf, dtype=torch.float64, device=z.device)
    n = min(case["alts"], case["v"])
    alternatives[:, :n] = logp.topk(n, -1).values
    return {"logprobs": logp.gather(1, state["tokens"].long()), "entropy": entropy, "ids": None, "alternatives": alternatives}
