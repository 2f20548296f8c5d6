"""The operators of a decoder layer in 8-bit floating point whose speed is tracked: what lies between the cache's attention and the next layer.

  norm     root-mean-square norm of the residual's sum, in 8 bits with a scale for each 128 of a row, or in 16 bits     (ops.add_rms_norm)
  quant    the 8-bit form of a 16-bit tensor: activations, a scale for each 128 of a row; weights, for 128 x 128        (ops.fp8_quantize)
  linear   product of two such matrices, fp32 sums, one rounding to 16 bits                                             (ops.fp8_linear)
  gated    both projections of a gated feed-forward, silu(gate) * up, one rounding                                      (ops.fp8_gated)

Where `own` is true `run` makes those calls; otherwise it computes the same in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn
DEV = "cuda"
EPS = 1e-6
TOP, LEAST = 448.0, 2.0 ** -100           # e4m3's largest; what a block's largest value counts as at least


def listed():
    return [
        # one user's decode step: launch latency
        {"name": "norm-1x4096", "kind": "norm", "rows": 1, "width": 4096, "residual": True, "fp8": True, "dtype": "bf16"},
        # the final norm of a batch's last tokens, 16 bits for the vocabulary's product
        {"name": "norm-77x5120-16bit", "kind": "norm", "rows": 77, "width": 5120, "residual": True, "fp8": False, "dtype": "f16"},
        # a batch of prompts, 4 x 2048 tokens
        {"name": "norm-8192x4096", "kind": "norm", "rows": 8192, "width": 4096, "residual": True, "fp8": True, "dtype": "bf16"},
        # attention output of a batch of prompts on its way to the output projection
        {"name": "quant-8192x4096", "kind": "quant", "rows": 8192, "width": 4096, "block": 1, "dtype": "bf16"},
        # a weight at load, the smallest decoder's width, ragged blocks
        {"name": "quant-weight-4848x912", "kind": "quant", "rows": 4848, "width": 912, "block": 128, "dtype": "f16"},
        # one user's down projection: the weights' bytes
        {"name": "linear-1x12288-4096", "kind": "linear", "rows": 1, "width": 12288, "out": 4096, "bias": False, "dtype": "bf16"},
        # a batch of 48 sequences' queries, keys and values
        {"name": "linear-48x4096-6144", "kind": "linear", "rows": 48, "width": 4096, "out": 6144, "bias": False, "dtype": "bf16"},
        # an odd prompt through a small decoder's queries, keys and values with bias
        {"name": "linear-333x896-2304", "kind": "linear", "rows": 333, "width": 896, "out": 2304, "bias": True, "dtype": "f16"},
        # prompts through the down projection
        {"name": "linear-4096x12288-4096", "kind": "linear", "rows": 4096, "width": 12288, "out": 4096, "bias": False, "dtype": "bf16"},
        # one user's decode step: gate and up weights
        {"name": "gated-1x4096-12288", "kind": "gated", "rows": 1, "width": 4096, "out": 12288, "dtype": "bf16"},
        # a follow-up prompt of odd length, small decoder
        {"name": "gated-203x896-4864", "kind": "gated", "rows": 203, "width": 896, "out": 4864, "dtype": "f16"},
        # prompts, 2 x 2048 tokens
        {"name": "gated-4096x4096-12288", "kind": "gated", "rows": 4096, "width": 4096, "out": 12288, "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "quant", "linear", "linear", "gated", "gated"))
    dtype = rng.choice(("f16", "bf16"))
    width = 16 * _log(rng, 8, 1024)
    if kind == "norm":
        return {"kind": kind, "rows": _log(rng, 1, min(16384, 8192 * 4096 // width)), "width": width, "residual": rng.random() < 0.7,
                "fp8": rng.random() < 0.7, "dtype": dtype}
    if kind == "quant":
        return {"kind": kind, "rows": _log(rng, 1, min(32768, 8192 * 4096 // width)), "width": width, "block": rng.choice((1, 1, 128)), "dtype": dtype}
    products = 4096 * 4096 * 12288 // width        # of rows and outputs that the largest listed case has at this width
    if kind == "linear":
        out = _log(rng, 64, 16384)
        return {"kind": kind, "rows": _log(rng, 1, min(8192, products // out)), "width": width, "out": out, "bias": rng.random() < 0.3, "dtype": dtype}
    out = 16 * _log(rng, 8, 1024)
    return {"kind": kind, "rows": _log(rng, 1, min(8192, products // out)), "width": width, "out": out, "dtype": dtype}


# ---------------------------------------------------------------- inputs

def _blocks(y, block):
    """y [rows, width] in its blocks, filled up with zeroes: [rows / block, block, width / 128, 128]."""
    rows, width = y.shape
    y = torch.nn.functional.pad(y, (0, -width % 128, 0, -rows % block))
    return y.view(-1, block, y.size(1) // 128, 128)


def _eight(y, block):
    """The 8-bit form of y (32 bits): codes and scales.  (Scales lie block of 128 by block of 128, as the norm leaves them.)"""
    b = _blocks(y, block)
    scale = b.abs().amax(dim=(1, 3)).clamp_min(LEAST) / TOP
    codes = (b / scale[:, None, :, None]).reshape(-1, b.size(2) * 128)[:y.size(0), :y.size(1)].to(F8)
    return {"codes": codes.contiguous(), "scale": scale.t().contiguous().t()}


def _activations(case, gen):
    """What a trained model's layers pass on: normal values, a few channels several times larger."""
    x = torch.randn(case["rows"], case["width"], generator=gen, device=DEV)
    channel = torch.exp(0.3 * torch.randn(case["width"], generator=gen, device=DEV))
    loud = torch.randint(0, case["width"], (max(1, case["width"] // 512),), generator=gen, device=DEV)
    channel[loud] *= 12.0
    return x * channel


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind in ("norm", "quant"):
        x = _activations(case, gen)
        s["x"] = (0.02 * x if kind == "quant" and case["block"] > 1 else x).to(dt)
        if kind == "norm":
            s["residual"] = (3.0 * _activations(case, gen)).to(dt) if case["residual"] else None
            s["weight"] = (1.0 + 0.2 * torch.randn(case["width"], generator=gen, device=DEV)).to(dt)
        return s
    s["x"] = _eight(_activations(case, gen), 1)
    rows = case["out"] * (2 if kind == "gated" else 1)
    # weights as they come from training, at the size that keeps the products about one
    w = torch.randn(rows, case["width"], generator=gen, device=DEV) * torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device=DEV))
    s["w"] = _eight(w.mul_(case["width"] ** -0.5), 128)
    if kind == "linear":
        s["bias"] = (0.5 * torch.randn(rows, generator=gen, device=DEV)).to(dt) if case["bias"] else None
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


def _own_norm(s):
    from packkv_amd import ops
    return ops.add_rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], fp8=s["case"]["fp8"])


def _own_quant(s):
    from packkv_amd import ops
    return ops.fp8_quantize(s["x"], block=s["case"]["block"])


def _own_linear(s):
    from packkv_amd import ops
    return ops.fp8_linear(s["x"], s["w"], bias=s["bias"], dtype=DTYPES[s["case"]["dtype"]])


def _own_gated(s):
    from packkv_amd import ops
    return ops.fp8_gated(s["x"], s["w"], dtype=DTYPES[s["case"]["dtype"]])


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    y = _eight(y, 1) if s["case"]["fp8"] else y.to(s["x"].dtype)
    return y if s["residual"] is None else (y, h.to(s["x"].dtype))


def _plain_quant(s):
    return _eight(s["x"].float(), s["case"]["block"])


def _values(e, block):
    """What the 8-bit form `e` stands for, in 32 bits."""
    c = e["codes"]
    scale = e["scale"].repeat_interleave(block, 0)[:c.size(0)].repeat_interleave(128, 1)[:, :c.size(1)]
    return c.float() * scale


def _plain_linear(s):
    y = torch.matmul(_values(s["x"], 1), _values(s["w"], 128).t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DTYPES[s["case"]["dtype"]])


def _plain_gated(s):
    y = torch.matmul(_values(s["x"], 1), _values(s["w"], 128).t())
    gate, up = y[:, :s["case"]["out"]], y[:, s["case"]["out"]:]
    return (gate / (1.0 + torch.exp(-gate)) * up).to(DTYPES[s["case"]["dtype"]])


_own = {"norm": _own_norm, "quant": _own_quant, "linear": _own_linear, "gated": _own_gated}
_plain = {"norm": _plain_norm, "quant": _plain_quant, "linear": _plain_linear, "gated": _plain_gated}


def work(case):
    kind, M, K = case["kind"], case["rows"], case["width"]
    cols = -(-K // 128)
    if kind == "norm":
        return {"bytes": M * K * (2 + (4 if case["residual"] else 0) + (1 if case["fp8"] else 2)) + (4 * M * cols if case["fp8"] else 0) + 2 * K, "flops": 8 * M * K}
    if kind == "quant":
        return {"bytes": 3 * M * K + 4 * cols * -(-M // case["block"]), "flops": 3 * M * K}
    N = case["out"] * (2 if kind == "gated" else 1)
    return {"bytes": M * K + N * K + 4 * cols * (M + -(-N // 128)) + 2 * M * case["out"] + (2 * N if case.get("bias") else 0), "flops": 2 * M * N * K}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_eight(y, block):
    """Scales, and the quotients that the codes are nearest to (the codes themselves have 4 bits)."""
    rows, width = y.shape
    at = torch.arange(width, device=DEV) // 128
    top = torch.zeros(-(-rows // block), int(at[-1]) + 1, dtype=torch.float64, device=DEV)
    row = torch.arange(rows, device=DEV) // block
    most = torch.zeros(rows, top.size(1), dtype=torch.float64, device=DEV).scatter_reduce_(1, at.expand(rows, width), y.abs(), "amax")
    top.scatter_reduce_(0, row[:, None].expand_as(most), most, "amax")
    scale = torch.clamp(top, min=LEAST) / TOP
    return {"codes": y / scale[row][:, at], "scale": scale}


def _exact_product(s, columns):
    """Sums block of 128 by block of 128, each product's scales applied to its sum."""
    x, w = s["x"], s["w"]
    M, K = x["codes"].shape
    row = columns // 128
    y = torch.zeros(M, columns.numel(), dtype=torch.float64, device=DEV)
    wc = w["codes"].view(torch.uint8)[columns].view(F8)
    for j in range(-(-K // 128)):
        part = slice(128 * j, min(K, 128 * j + 128))
        dot = x["codes"][:, part].double() @ wc[:, part].double().t().contiguous()
        y += dot * (x["scale"][:, j].double()[:, None] * w["scale"][row, j].double()[None])
    return y


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_eight(s["x"].double(), case["block"])
    if kind == "norm":
        h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        size = torch.linalg.vector_norm(h, dim=-1, keepdim=True)
        y = h / torch.sqrt(size ** 2 / case["width"] + EPS) * s["weight"].double()
        y = _exact_eight(y, 1) if case["fp8"] else y
        return y if s["residual"] is None else (y, h)
    n = torch.arange(case["out"], device=DEV)
    y = _exact_product(s, n)
    if kind == "linear":
        return y if s["bias"] is None else y + s["bias"].double()
    return y * torch.sigmoid(y) * _exact_product(s, n + case["out"])
