"""Measured cases of the operators for large language models: the quantisation of activations token by token, the
int8 product with a scale for each token and each channel, and the products grouped by expert with both of their
gradients.

`run` computes a case in its plain form, elementary torch operations in 32 bits (64 where a sum of integers needs
them), or, with `own` set, by the calls a user makes of rocmlir_amd.  `exact` computes it from the definition in 64
bits.  Nothing here says how far results may be off."""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4, "i8": 1}


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token's activations in front of an int8 layer: all latency
        {"name": "quantize_one_token", "op": "quantize", "t": "bf16", "m": 1, "k": 4096},
        # a long prompt's activations
        {"name": "quantize_prompt", "op": "quantize", "t": "f16", "m": 24576, "k": 4096},
        # decoding one sequence through a square int8 layer: the weights' bytes count
        {"name": "int8_one_token", "op": "gemm", "t": "bf16", "m": 1, "n": 4096, "k": 4096, "bias": False},
        # decoding an odd batch through a wide layer with a bias
        {"name": "int8_batch_of_37", "op": "gemm", "t": "f16", "m": 37, "n": 10240, "k": 1280, "bias": True},
        # a prompt of ragged length, rows that are no whole 16-byte pieces
        {"name": "int8_ragged_prompt", "op": "gemm", "t": "bf16", "m": 1001, "n": 2307, "k": 1283, "bias": False},
        # a prompt through a square layer: the matrix cores count
        {"name": "int8_prompt", "op": "gemm", "t": "f16", "m": 4096, "n": 4096, "k": 4096, "bias": False},
        # decoding 32 sequences, two experts each out of 64, int8 experts
        {"name": "experts_int8_decode", "op": "grouped_i8", "t": "bf16", "e": 64, "m": 64, "n": 2048, "k": 4096,
         "tail": 0, "skew": 0.5},
        # a prompt of ragged length over many 16-bit experts, rows behind the last expert that stay as they were
        {"name": "experts_ragged_prompt", "op": "grouped", "t": "f16", "e": 60, "m": 5003, "n": 1410, "k": 2048,
         "tail": 37, "skew": 0.8},
        # a training step's tokens over eight experts: forward
        {"name": "experts_training_forward", "op": "grouped", "t": "bf16", "e": 8, "m": 16384, "n": 4096, "k": 2048,
         "tail": 0, "skew": 0.3},
        # the same step: gradients of the tokens and of the experts' weights
        {"name": "experts_training_backward", "op": "grouped_bwd", "t": "bf16", "e": 8, "m": 16384, "n": 4096,
         "k": 2048, "tail": 0, "skew": 0.3},
        # many small experts, some without a token: gradients
        {"name": "experts_sparse_backward", "op": "grouped_bwd", "t": "f16", "e": 64, "m": 1000, "n": 768, "k": 1024,
         "tail": 24, "skew": 1.2},
        # a small mixture held in 32 bits: gradients
        {"name": "experts_small_f32_backward", "op": "grouped_bwd", "t": "f32", "e": 4, "m": 250, "n": 330, "k": 512,
         "tail": 0, "skew": 0.3},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly spread over its logarithm."""
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["quantize", "gemm", "gemm", "grouped_i8", "grouped", "grouped", "grouped_bwd", "grouped_bwd"])
    # a layer's width: mostly a multiple of 64, as layers are, else any number
    def width(lo, hi):
        w = _spread(rng, lo, hi)
        return max(lo, w // 64 * 64) if rng.random() < 0.7 and w >= 64 else w
    if op == "quantize":
        return {"op": op, "t": rng.choice(["f16", "bf16", "f32"]), "m": _spread(rng, 1, 12000), "k": width(17, 8192)}
    if op == "gemm":
        m = rng.choice([_spread(rng, 1, 64), _spread(rng, 1, 4096)])
        return {"op": op, "t": rng.choice(["f16", "bf16", "f32"]), "m": m, "n": width(33, 8192), "k": width(48, 4096),
                "bias": rng.random() < 0.3}
    t = rng.choice(["bf16", "f16"]) if op == "grouped_i8" or rng.random() < 0.85 else "f32"
    heavy = 2 if t == "f32" else 1     # f32 costs sixteen times the matrix time of 16 bits
    case = {"op": op, "t": t, "e": _spread(rng, 1, 96),
            "m": rng.choice([_spread(rng, 1, 128), _spread(rng, 1, 6000 // heavy)]),
            "n": width(40, 2816 // heavy), "k": width(40, 2560 // heavy), "tail": rng.choice([0, 0, 1, 29]),
            "skew": rng.choice([0.0, 0.5, 1.0, 2.0])}
    while case["e"] * case["n"] * case["k"] > 160_000_000:
        case["e"] = max(1, case["e"] // 2)
    return case


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _shares(case):
    """How often the router chooses each expert: falling with the expert's rank as rank^-skew."""
    p = np.arange(1, case["e"] + 1, dtype=np.float64) ** -case["skew"]
    return p / p.sum()


def _offsets(case, seed):
    """First row of every expert, and the end of the last one: `m` rows spread by the router, `tail` rows behind."""
    r = np.random.default_rng(seed)
    counts = r.permutation(r.multinomial(case["m"], _shares(case)))
    return torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()


def _activations(g, rows, cols, dtype):
    """Activations: rows of different size, a few channels that stand out."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    x *= torch.rand((rows, 1), generator=g, device="cuda") * 2.0 + 0.1
    x *= 1.0 + 12.0 * (torch.rand((1, cols), generator=g, device="cuda") < 0.01)
    return x.to(dtype)


def _int8(g, *shape):
    """What quantised normal values look like."""
    return (torch.randn(shape, generator=g, device="cuda") * 32.0).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    g, t, op = _generator(seed), _DTYPES[case["t"]], case["op"]
    s = dict(case)
    if op == "quantize":
        s["x"] = _activations(g, case["m"], case["k"], t)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    if op == "gemm":
        s["x"], s["w"] = _int8(g, m, k), _int8(g, n, k)
        s["token_scale"] = torch.rand(m, generator=g, device="cuda") * 0.05 + 0.002
        s["scale"] = torch.rand(n, generator=g, device="cuda") * 0.0008 + 0.0001
        s["b"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        return s
    e, rows = case["e"], m + case["tail"]
    s["offsets"] = _offsets(case, seed)
    if op == "grouped_i8":
        s["x"], s["w"] = _int8(g, rows, k), _int8(g, e, n, k)
        s["token_scale"] = torch.rand(rows, generator=g, device="cuda") * 0.05 + 0.002
        s["scale"] = torch.rand((e, n), generator=g, device="cuda") * 0.0008 + 0.0001
        s["out"] = torch.zeros((rows, n), dtype=t, device="cuda")
        return s
    s["w"] = (torch.randn((e, n, k), generator=g, device="cuda") * k ** -0.5).to(t)
    s["x"] = torch.randn((rows, k), generator=g, device="cuda").to(t)
    if op == "grouped":
        s["out"] = torch.zeros((rows, n), dtype=t, device="cuda")
    else:
        s["dout"] = torch.randn((rows, n), generator=g, device="cuda").to(t)
        s["dx"] = torch.zeros((rows, k), dtype=t, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    import rocmlir_amd as rock
    op = s["op"]
    if op == "quantize":
        return rock.quantize_tokens(s["x"])
    if op == "gemm":
        return rock.gemm(s["x"], s["w"], transB=True, out_dtype=s["t"], scale=s["scale"], token_scale=s["token_scale"],
                         bias=s["b"])
    if op == "grouped_i8":
        return rock.grouped_gemm(s["x"], s["w"], s["offsets"], transB=True, out_dtype=s["t"], scale=s["scale"],
                                 token_scale=s["token_scale"], out=s["out"])
    if op == "grouped":
        return rock.grouped_gemm(s["x"], s["w"], s["offsets"], transB=True, out=s["out"])
    dx = rock.grouped_gemm_bwd_data(s["dout"], s["w"], s["offsets"], transB=True, out=s["dx"])
    dw = rock.grouped_gemm_bwd_weight(s["x"], s["dout"], s["offsets"], transB=True)
    return dx, dw


def _plain(s):
    op, t = s["op"], _DTYPES[s["t"]]
    if op == "quantize":
        # a quotient next to a half is decided in 64 bits
        x = s["x"].double()
        top = x.abs().amax(dim=1)
        q = torch.round(x * 127.0 / torch.where(top > 0, top, 1.0)[:, None])
        return q.to(torch.int8), top.float() / 127.0
    if op == "gemm":
        v = (s["x"].double() @ s["w"].double().t()).float() * s["scale"] * s["token_scale"][:, None]
        if s["b"] is not None:
            v = v + s["b"]
        return v.to(t)
    ends = s["offsets"].tolist()
    spans = [(e, a, b) for e, (a, b) in enumerate(zip(ends[:-1], ends[1:])) if b > a]
    if op == "grouped_i8":
        for e, a, b in spans:
            v = (s["x"][a:b].double() @ s["w"][e].double().t()).float() * s["scale"][e]
            s["out"][a:b] = (v * s["token_scale"][a:b, None]).to(t)
        return s["out"]
    if op == "grouped":
        for e, a, b in spans:
            s["out"][a:b] = (s["x"][a:b].float() @ s["w"][e].float().t()).to(t)
        return s["out"]
    dw = torch.zeros_like(s["w"])
    for e, a, b in spans:
        dout = s["dout"][a:b].float()
        s["dx"][a:b] = (dout @ s["w"][e].float()).to(t)
        dw[e] = (dout.t() @ s["x"][a:b].float()).to(t)
    return s["dx"], dw


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, f64 = case["op"], torch.float64
    if op == "quantize":
        x = s["x"].to(f64)
        top = torch.linalg.vector_norm(x, float("inf"), dim=1)
        unit = top.clone()
        unit[top == 0] = 1.0
        return torch.round((127.0 * x) / unit.unsqueeze(1)).to(torch.int8), top / 127.0
    if op == "gemm":
        v = torch.mm(s["x"].to(f64), s["w"].to(f64).T)
        v *= torch.outer(s["token_scale"].to(f64), s["scale"].to(f64))
        return v if s["b"] is None else v + s["b"].to(f64)
    # the expert of every row: rows behind the last expert have none
    rows = s["x"].shape[0]
    expert = torch.bucketize(torch.arange(rows, device="cuda", dtype=torch.int32), s["offsets"], right=True) - 1
    if op == "grouped_bwd":
        dx, dw = torch.zeros(s["x"].shape, dtype=f64, device="cuda"), torch.zeros(s["w"].shape, dtype=f64, device="cuda")
    else:
        out = torch.zeros((rows, case["n"]), dtype=f64, device="cuda")
    for e in range(case["e"]):
        mine = (expert == e).nonzero().flatten()
        if mine.numel() == 0:
            continue
        x, w = s["x"][mine].to(f64), s["w"][e].to(f64)
        if op == "grouped_bwd":
            d = s["dout"][mine].to(f64)
            dx[mine] = torch.mm(d, w)
            dw[e] = torch.mm(d.T, x)
            continue
        v = torch.mm(x, w.T)
        if op == "grouped_i8":
            v *= torch.outer(s["token_scale"][mine].to(f64), s["scale"][e].to(f64))
        out[mine] = v
    return (dx, dw) if op == "grouped_bwd" else out


# ---------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------
def work(case):
    op, b, m, k = case["op"], _BYTES[case["t"]], case["m"], case["k"]
    if op == "quantize":
        return {"bytes": m * k * (b + 1) + 4 * m, "flops": 3 * m * k}
    n = case["n"]
    if op == "gemm":
        return {"bytes": m * k + n * k + m * n * b + 4 * (m + n * (2 if case["bias"] else 1)), "flops": 2 * m * n * k}
    # the weights of the experts that are chosen at all (their expected number), and every row that is some expert's
    e = float(np.sum(1.0 - (1.0 - _shares(case)) ** m))
    if op == "grouped_i8":
        return {"bytes": int(m * k + e * n * (k + 4) + m * n * b + 4 * m), "flops": 2 * m * n * k}
    if op == "grouped":
        return {"bytes": int((m * k + e * n * k + m * n) * b), "flops": 2 * m * n * k}
    # both gradients: dout read once for both, x and the chosen weights read, dx and every expert's gradient written
    return {"bytes": int((m * n + 2 * m * k + e * n * k + case["e"] * n * k) * b), "flops": 4 * m * n * k}
