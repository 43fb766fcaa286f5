"""The FP8 linear path with a scale for each block of 128, as measurable cases.

Weights are e4m3 codes [out][in] with one f32 scale per 128 x 128 tile, activations e4m3 codes [token][in] with one f32 scale
per token and 128 elements.  Five operators make up the path of a dense layer:

  quant    activations -> codes and scales
  norm     residual add + RMSNorm + the same quantizer, the step in front of a layer's products
  load     bf16 weights -> codes and scales;  back: codes and scales -> f32
  gemm     y = x . W^T
  gate_up  h = silu(x . Wg^T) * (x . Wu^T), left as codes and scales for the down projection

Weights and activations are seeded draws of the distributions trained models show: weights N(0, 0.02), activations N(0, 1) with
some channels ten times as strong, residual streams N(0, 2).
"""
import math

import torch

own = False

B = 128
TOP = 448.0                       # the largest e4m3 value
TINY = 2.0 ** -126                # the smallest scale
EPS = 1e-6
MAX_ELEMS = 5120 * 17408          # the largest plane of the ranges
MAX_FLOPS = 2 * 4096 * 5120 * 17408


def listed():
    return [
        # one token enters the projections of a layer
        {"name": "quantize, 1 token", "op": "quant", "t": "f32", "k": 5120, "m": 1},
        # a ragged prompt's wide activations, written by a kernel that leaves bf16
        {"name": "quantize bf16, 1000 tokens", "op": "quant", "t": "bf16", "k": 17408, "m": 1000},
        # a handful of sequences decoding: the step between two halves of a layer
        {"name": "add + norm, 7 tokens", "op": "norm", "k": 5120, "m": 7},
        # the same for a prompt
        {"name": "add + norm, 4096 tokens", "op": "norm", "k": 5120, "m": 4096},
        # a gate projection when a model is loaded from bf16
        {"name": "weights into blocks", "op": "load", "k": 5120, "n": 17408},
        # a plane read back, of a pruned, odd width
        {"name": "blocks into f32", "op": "back", "k": 5120, "n": 5003},
        # the smallest product of a decode step: a key or value projection of a grouped-query attention
        {"name": "kv projection, 1 token", "op": "gemm", "t": "f32", "k": 5120, "n": 1024, "m": 1},
        # a pruned down projection under a few sequences
        {"name": "down projection, 7 tokens", "op": "gemm", "t": "f32", "k": 17408, "n": 5003, "m": 7},
        # a prompt through a wide projection
        {"name": "wide projection, 4096 tokens", "op": "gemm", "t": "bf16", "k": 5120, "n": 17408, "m": 4096},
        # the feed-forward block's front under one sequence
        {"name": "gate and up, 1 token", "op": "gate_up", "k": 5120, "n": 17408, "m": 1},
        # a batch of sequences through a small model's, whose rows end inside a block
        {"name": "gate and up, 60 tokens", "op": "gate_up", "k": 2880, "n": 2880, "m": 60},
        # a prompt
        {"name": "gate and up, 2000 tokens", "op": "gate_up", "k": 5120, "n": 17408, "m": 2000},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(lo, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["quant", "norm", "load", "back"] + ["gemm"] * 5 + ["gate_up"] * 4)
    k = _log(rng, 512, 17408, rng.choice([16, 64, 128, 128]))
    if op == "quant":
        return {"op": op, "t": rng.choice(["f32", "bf16"]), "k": k, "m": _log(rng, 1, 8192 if k < 8192 else 2048)}
    if op == "norm":
        k = min(k, 8192)
        return {"op": op, "k": k, "m": _log(rng, 1, 4096)}
    n = _log(rng, 512, min(17408, MAX_ELEMS // k), rng.choice([16, 64, 128]) if op == "gate_up" else rng.choice([1, 8, 64, 128]))
    if op in ("load", "back"):
        return {"op": op, "k": k, "n": n}
    cap = MAX_FLOPS // ((4 if op == "gate_up" else 2) * k * n)
    m = min(cap, _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 1, 8192))
    case = {"op": op, "k": k, "n": n, "m": m}
    if op == "gemm":
        case["t"] = rng.choice(["f32", "bf16"])
    return case


# ---------------------------------------------------------------- inputs
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _normal(gen, std, *shape):
    return torch.randn(*shape, device="cuda", generator=gen) * std


def _activations(gen, m, k):
    x = _normal(gen, 1.0, m, k)
    x[:, torch.randperm(k, device="cuda", generator=gen)[: max(1, k // 64)]] *= 10.0
    return x


def _groups(v, rows):
    """f32 [n][k] -> [n / rows][rows][k / B][B], zero-padded to whole groups."""
    n, k = v.shape
    v = torch.nn.functional.pad(v, (0, -k % B, 0, -n % rows))
    return v.view(v.shape[0] // rows, rows, v.shape[1] // B, B)


def _quantized(v, rows):
    """Codes (float8 [n][k]) and scales (f32 [ceil(n / rows)][ceil(k / B)]) of f32 v, a scale for `rows` rows of B elements."""
    n, k = v.shape
    v = _groups(v, rows)
    s = (v.abs().amax(dim=(1, 3)) / v.new_full((), TOP)).clamp_min(TINY)
    q = (v * (1.0 / s)[:, None, :, None]).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return q.reshape(q.shape[0] * rows, -1)[:n, :k].contiguous(), s


def _values(q, s, rows):
    """f32 values of codes and scales."""
    n, k = q.shape
    v = _groups(q.float(), rows) * s[:, None, :, None]
    return v.reshape(v.shape[0] * rows, -1)[:n, :k]


def _codes(m, k):
    return torch.empty(m, k, dtype=torch.float8_e4m3fn, device="cuda")


def _scales(m, k):
    return torch.empty(m, -(-k // B), device="cuda")


def prepare(case, seed):
    op, k = case["op"], case["k"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if op in ("load", "back"):
        w = _normal(gen, 0.02, case["n"], k)
        if op == "load":
            s |= {"w": w.to(torch.bfloat16), "q": _codes(case["n"], k), "scale": _scales(-(-case["n"] // B), k)}
        else:
            s["q"], s["scale"] = _quantized(w, B)
            s["y"] = torch.empty(case["n"], k, device="cuda")
        return s
    m = case["m"]
    if op == "quant":
        s |= {"x": _activations(gen, m, k).to(_TYPES[case["t"]]), "q": _codes(m, k), "scale": _scales(m, k)}
    elif op == "norm":
        s |= {"x": _normal(gen, 2.0, m, k), "proj": _normal(gen, 0.5, m, k), "w": 1.0 + _normal(gen, 0.1, k),
              "xn": torch.empty(m, k, device="cuda"), "q": _codes(m, k), "scale": _scales(m, k)}
    else:
        s["xq"], s["xs"] = _quantized(_activations(gen, m, k), 1)
        s["wq"], s["ws"] = _quantized(_normal(gen, 0.02, case["n"], k), B)
        if op == "gate_up":
            s["uq"], s["us"] = _quantized(_normal(gen, 0.02, case["n"], k), B)
            s["q"], s["scale"] = _codes(m, case["n"]), _scales(m, case["n"])
        else:
            s["y"] = torch.empty(m, case["n"], dtype=_TYPES[case["t"]], device="cuda")
    return s


# ---------------------------------------------------------------- the calls
_PACK = None


def _call():
    """The pack's launch call, loaded once per process as a host program does."""
    global _PACK
    if _PACK is None:
        from paddock_b200 import KernelPack
        _PACK = KernelPack.load()
    return _PACK.call


def _run_own(s):
    case, call = s["case"], _call()
    op, k, stream = case["op"], case["k"], torch.cuda.current_stream().cuda_stream
    if op == "quant":
        name = "pdk_quantize_e4m3_blk" if case["t"] == "f32" else "pdk_quantize_e4m3_blk_bf16"
        call(name, s["x"], s["q"], s["scale"], k, case["m"], stream=stream)
        return s["q"], s["scale"]
    if op == "norm":
        call("pdk_add_rmsnorm_quant_e4m3_blk", s["x"], s["proj"], s["w"], s["xn"], s["q"], s["scale"], k, EPS, case["m"], stream=stream)
        return s["x"], s["xn"], s["q"], s["scale"]
    if op == "load":
        call("pdk_bf16_to_f8blk", s["w"], s["q"], s["scale"], k, case["n"], stream=stream)
        return s["q"], s["scale"]
    if op == "back":
        call("pdk_f8blk_dequant", s["q"], s["scale"], s["y"], k, case["n"], stream=stream)
        return s["y"]
    if op == "gemm":
        name = "pdk_f8blk_gemm" if case["t"] == "f32" else "pdk_f8blk_gemm_bf16"
        call(name, s["wq"], s["ws"], s["xq"], s["xs"], s["y"], k, case["n"], case["m"], stream=stream)
        return s["y"]
    call("pdk_f8blk_gate_up", s["wq"], s["ws"], s["uq"], s["us"], s["xq"], s["xs"], s["q"], s["scale"], k, case["n"], case["m"],
         stream=stream)
    return s["q"], s["scale"]


def _run_plain(s):
    op = s["case"]["op"]
    if op == "quant":
        return _quantized(s["x"].float(), 1)
    if op == "norm":
        x = s["x"].add_(s["proj"])
        inv = 1.0 / torch.sqrt((x * x).mean(dim=1, keepdim=True) + EPS)
        xn = x * inv * s["w"]
        return (x, xn, *_quantized(xn, 1))
    if op == "load":
        return _quantized(s["w"].float(), B)
    if op == "back":
        return _values(s["q"], s["scale"], B)
    x = _values(s["xq"], s["xs"], 1)
    y = x @ _values(s["wq"], s["ws"], B).T
    if op == "gemm":
        return y.to(s["y"].dtype)
    u = x @ _values(s["uq"], s["us"], B).T
    return _quantized(y / (1.0 + torch.exp(-y)) * u, 1)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------- the definition in 64 bits
def _nearest_e4m3(v):
    """Nearest e4m3 value (ties to the even code) of f64 v, saturating: steps of 2^(e - 3) within [2^e, 2^(e + 1)), e >= -6."""
    _, ex = torch.frexp(v)
    step = torch.pow(2.0, (ex.double() - 1.0).clamp_min(-6.0) - 3.0)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _blocks_of(size):
    return torch.arange(size, device="cuda") // B


def _exact_scales(v, rows):
    n, k = v.shape
    row_of = torch.arange(n, device="cuda") // rows
    s = torch.zeros(-(-n // rows), k, dtype=torch.float64, device="cuda").index_reduce_(0, row_of, v.abs(), "amax") if rows > 1 else v.abs()
    s = torch.stack([c.amax(dim=1) for c in s.split(B, dim=1)], dim=1)
    return (s / TOP).clamp_min(TINY), row_of


def _exact_codes(v, rows):
    s, row_of = _exact_scales(v, rows)
    return _nearest_e4m3(v / s[row_of][:, _blocks_of(v.shape[1])]), s


def _exact_values(q, s, rows):
    n, k = q.shape
    return q.double() * s.double()[torch.arange(n, device="cuda") // rows][:, _blocks_of(k)]


def exact(case, seed):
    op, s = case["op"], prepare(case, seed)
    if op == "quant":
        return _exact_codes(s["x"].double(), 1)
    if op == "load":
        return _exact_codes(s["w"].double(), B)
    if op == "back":
        return _exact_values(s["q"], s["scale"], B)
    if op == "norm":
        x = s["x"].double() + s["proj"].double()
        xn = x / (x.square().mean(dim=1, keepdim=True) + EPS).sqrt() * s["w"].double()
        return (x, xn, *_exact_codes(xn, 1))
    x = _exact_values(s["xq"], s["xs"], 1)
    y = torch.mm(x, _exact_values(s["wq"], s["ws"], B).t())
    if op == "gemm":
        return y
    return _exact_codes(y * torch.sigmoid(y) * torch.mm(x, _exact_values(s["uq"], s["us"], B).t()), 1)


# ---------------------------------------------------------------- what a pass cannot do without
def _plane(rows, k, per_rows):
    """Bytes of codes and scales."""
    return rows * k + 4 * -(-rows // per_rows) * -(-k // B)


def work(case):
    op, k = case["op"], case["k"]
    if op == "load":
        return {"bytes": 2 * k * case["n"] + _plane(case["n"], k, B), "flops": 0}
    if op == "back":
        return {"bytes": _plane(case["n"], k, B) + 4 * k * case["n"], "flops": 0}
    m = case["m"]
    if op == "quant":
        return {"bytes": (4 if case["t"] == "f32" else 2) * m * k + _plane(m, k, 1), "flops": 0}
    if op == "norm":       # x and proj in, x and the normed row out
        return {"bytes": 16 * m * k + 4 * k + _plane(m, k, 1), "flops": 0}
    n = case["n"]
    if op == "gemm":
        return {"bytes": _plane(n, k, B) + _plane(m, k, 1) + (4 if case["t"] == "f32" else 2) * m * n, "flops": 2.0 * m * n * k}
    return {"bytes": 2 * _plane(n, k, B) + _plane(m, k, 1) + _plane(m, n, 1), "flops": 4.0 * m * n * k}
