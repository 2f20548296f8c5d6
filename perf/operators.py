"""The operators around the compressed cache whose speed is tracked: what a program that generates with it calls for each step and prompt.

  rotary   norms of queries and keys for each head with the position rotation, one or several position axes   (ops.norm_rotary)
  step     the same for a step's few tokens, keys and values written into the cache's 16-bit window            (ops.window_append_rotary)
  sample   a token for each row of logits, with its log-probability, from given uniform numbers: temperature,
           top-k, top-p, min-p                                                                                 (ops.sample)
  chunk    causal attention of several new tokens over an encoded cache and its window                         (ops.attn_chunk)

Where `own` is true `run` makes those calls; otherwise it computes the same in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
DEV = "cuda"
D = 128
BITS = {0.2: 3, 0.1: 4, 0.05: 5}          # code width by relative quantisation step
# stored bits per value by code width, keys with outlier channels and normal values
K_BITS = {3: 1.6, 4: 2.8, 5: 3.8}
V_BITS = {3: 2.7, 4: 3.5, 5: 4.5}
CAP = 320                                 # rows of a layer's window: 64 + 192 + 64
OUTLIERS = (3, 40, 77, 120)


def listed():
    return [
        # a follow-up prompt of eight tokens far into a conversation, no head norms: launch latency
        {"name": "rotary-1x8-far", "kind": "rotary", "batch": 1, "q_heads": 32, "kv_heads": 32, "tokens": 8, "far": 1000000, "norm": False,
         "axes": 1, "interleaved": False, "dtype": "f16"},
        # a batch of prompts through a layer of the default decoder shape
        {"name": "rotary-4x2048", "kind": "rotary", "batch": 4, "q_heads": 32, "kv_heads": 8, "tokens": 2048, "far": 0, "norm": True,
         "axes": 1, "interleaved": False, "dtype": "bf16"},
        # prompts of odd length with images: time, height and width positions
        {"name": "rotary-2x1031-3axes", "kind": "rotary", "batch": 2, "q_heads": 16, "kv_heads": 4, "tokens": 1031, "far": 5000, "norm": True,
         "axes": 3, "interleaved": True, "dtype": "f16"},
        # one user's decode step
        {"name": "step-1", "kind": "step", "batch": 1, "q_heads": 32, "kv_heads": 8, "tokens": 1, "far": 8192, "norm": True, "axes": 1,
         "interleaved": False, "dtype": "bf16"},
        # a full batch's step with three position axes
        {"name": "step-64-3axes", "kind": "step", "batch": 64, "q_heads": 32, "kv_heads": 8, "tokens": 1, "far": 32768, "norm": True, "axes": 3,
         "interleaved": False, "dtype": "f16"},
        # one user's next token, usual filters
        {"name": "sample-1x151936", "kind": "sample", "rows": 1, "vocab": 151936, "k": 50, "p": 0.9, "min_p": 0.0, "t": 0.8, "mixed": False,
         "allowed": 1.0, "dtype": "f32"},
        # a batch under a grammar that leaves a tenth of the vocabulary
        {"name": "sample-32x32003-masked", "kind": "sample", "rows": 32, "vocab": 32003, "k": 0, "p": 1.0, "min_p": 0.05, "t": 1.2, "mixed": False,
         "allowed": 0.1, "dtype": "f16"},
        # a large batch, every request with filters of its own
        {"name": "sample-256x151936-mixed", "kind": "sample", "rows": 256, "vocab": 151936, "k": 0, "p": 0.95, "min_p": 0.0, "t": 1.0, "mixed": True,
         "allowed": 1.0, "dtype": "bf16"},
        # a short odd conversation's follow-up of a few tokens, most of it in the window
        {"name": "chunk-1x3-896", "kind": "chunk", "batch": 1, "q_heads": 32, "kv_heads": 8, "new": 3, "tokens": 896, "window": 201, "rel": 0.1,
         "padded": False, "dtype": "bf16"},
        # drafted tokens of a batch, verified over 16384 tokens each
        {"name": "chunk-8x4-16k", "kind": "chunk", "batch": 8, "q_heads": 32, "kv_heads": 8, "new": 4, "tokens": 16384, "window": 150, "rel": 0.1,
         "padded": False, "dtype": "f16"},
        # left-padded follow-up prompts of odd length, five query heads to a KV head, tighter codes
        {"name": "chunk-2x333-4k-padded", "kind": "chunk", "batch": 2, "q_heads": 40, "kv_heads": 8, "new": 333, "tokens": 4096, "window": 77,
         "rel": 0.05, "padded": True, "dtype": "bf16"},
        # a long document's next 1024 tokens over 32768 before them
        {"name": "chunk-1x1024-32k", "kind": "chunk", "batch": 1, "q_heads": 32, "kv_heads": 8, "new": 1024, "tokens": 32768, "window": 192,
         "rel": 0.1, "padded": False, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("rotary", "step", "sample", "chunk", "chunk"))
    dtype = rng.choice(("f16", "bf16"))
    hq, hkv = rng.choice(((32, 8), (32, 8), (32, 32), (16, 4), (40, 8), (14, 2)))
    if kind in ("rotary", "step"):
        batch = _log(rng, 1, 8 if kind == "rotary" else 64)
        most = 4 * 2048 * 40 // (batch * (hq + hkv))
        tokens = _log(rng, 1, min(4096, most)) if kind == "rotary" else rng.choice((1, 1, rng.randint(2, 8)))
        return {"kind": kind, "batch": batch, "q_heads": hq, "kv_heads": hkv, "tokens": tokens, "far": rng.choice((0, 32768, 1000000)),
                "norm": rng.random() < 0.7, "axes": rng.choice((1, 1, 3)), "interleaved": rng.random() < 0.5, "dtype": dtype}
    if kind == "sample":
        rows = _log(rng, 1, 256)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 1000, 151936), "k": rng.choice((0, 0, 1, 20, 50, rng.randint(2, 900))),
                "p": rng.choice((1.0, 0.5, 0.9, 0.95)), "min_p": rng.choice((0.0, 0.0, 0.02, 0.1)), "t": rng.choice((0.3, 0.7, 1.0, 1.5)),
                "mixed": rng.random() < 0.3, "allowed": rng.choice((1.0, 1.0, 0.1, 0.001)), "dtype": rng.choice(("f16", "bf16", "f32"))}
    batch = min(_log(rng, 1, 8), 64 // hkv)
    tokens = max(128, _log(rng, 128, min(32768, 8 * 8 * 16384 // (batch * hkv))) // 128 * 128)
    new = _log(rng, 2, max(2, min(1024, tokens, 32 * 1024 * 32768 // (batch * hq * tokens))))
    return {"kind": "chunk", "batch": batch, "q_heads": hq, "kv_heads": hkv, "new": new, "tokens": tokens, "window": rng.choice((0, rng.randint(1, 255))),
            "rel": rng.choice((0.1, 0.1, 0.05, 0.2)), "padded": rng.random() < 0.3, "dtype": dtype}


# ---------------------------------------------------------------- inputs

def _sections(case):
    if case["axes"] == 1:
        return None
    return (24, 20, 20) if case["interleaved"] else (16, 24, 24)


def _rotary_inputs(case, gen):
    """The projection's output [B, n, heads, 128], as the decoder has it: queries, keys and values are views into it."""
    B, n, hq, hkv = case["batch"], case["tokens"], case["q_heads"], case["kv_heads"]
    dt = DTYPES[case["dtype"]]
    qkv = (torch.randn(B, n, hq + 2 * hkv, D, generator=gen, device=DEV) * 1.5).to(dt)
    s = {"case": case, "q": qkv[:, :, :hq].transpose(1, 2), "k": qkv[:, :, hq:hq + hkv].transpose(1, 2), "v": qkv[:, :, hq + hkv:].transpose(1, 2)}
    start = torch.randint(0, case["far"] + 1, (B, 1), generator=gen, device=DEV)
    pos = start + torch.arange(n, device=DEV)
    if case["axes"] == 3:          # patches of a picture: the axes part ways
        jit = torch.randint(0, 64, (2, B, n), generator=gen, device=DEV)
        pos = torch.stack((pos, pos + jit[0], pos + jit[1]))
    s["positions"] = pos
    s["inv_freq"] = 1.0 / (1.0e6 ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float32) / D))
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"] = (1.0 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(dt)
        s["k_norm"] = (1.0 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(dt)
    if case["kind"] == "step":
        s["k_win"] = torch.randn(B, hkv, CAP, D, generator=gen, device=DEV).to(dt)
        s["v_win"] = torch.randn(B, hkv, CAP, D, generator=gen, device=DEV).to(dt)
        s["row"] = int(torch.randint(64, CAP - 64 - n, (1,), generator=gen, device=DEV))
    return s


def _sample_inputs(case, gen):
    R, V = case["rows"], case["vocab"]
    x = torch.randn(R, V, generator=gen, device=DEV) * 2.0
    likely = torch.randint(0, V, (R, 24), generator=gen, device=DEV)         # the few tokens that a trained model puts forward
    x.scatter_add_(1, likely, -4.0 * torch.log(torch.rand(R, 24, generator=gen, device=DEV) + 1e-3))
    if case["allowed"] < 1.0:
        ok = torch.rand(R, V, generator=gen, device=DEV) < case["allowed"]
        ok.scatter_(1, torch.randint(0, V, (R, 1), generator=gen, device=DEV), True)
        x.masked_fill_(~ok, float("-inf"))
    s = {"case": case, "logits": x.to(DTYPES[case["dtype"]]), "u": torch.rand(R, generator=gen, device=DEV), "t": case["t"], "k": case["k"],
         "p": case["p"], "min_p": case["min_p"]}
    if case["mixed"]:
        pick = torch.rand(4, R, generator=gen, device=DEV)
        s["t"] = 0.2 + 1.3 * pick[0]
        s["k"] = torch.where(pick[1] < 0.5, torch.zeros_like(pick[1]), 1 + 100 * pick[1]).to(torch.int32)
        s["p"] = torch.where(pick[2] < 0.3, torch.ones_like(pick[2]), 0.3 + 0.69 * pick[2])
        s["min_p"] = torch.where(pick[3] < 0.6, torch.zeros_like(pick[3]), 0.1 * pick[3])
    return s


def _quantised(B, H, T, rel, dt, keys, gen):
    """Codes [T, B * H * 128] and the parameters [B, T] of a layer's keys or values: one scale and zero for each token."""
    codes = torch.empty(T, B * H * D, dtype=torch.uint8, device=DEV)
    scale, zero = torch.empty(B, T, dtype=dt, device=DEV), torch.empty(B, T, dtype=dt, device=DEV)
    step = max(128, (1 << 25) // (B * H * D))
    for a in range(0, T, step):
        b = min(T, a + step)
        x = torch.randn(b - a, B, H, D, generator=gen, device=DEV)
        if keys:
            x[..., list(OUTLIERS)] *= 10.0
        lo, hi = x.amin(dim=(2, 3)), x.amax(dim=(2, 3))
        sc = ((hi - lo) * rel).to(dt)
        ze = torch.round(lo / sc.float()).to(dt)
        c = torch.round(x / sc.float()[:, :, None, None]) - ze.float()[:, :, None, None]
        codes[a:b] = c.clamp_(0, (1 << BITS[rel]) - 1).to(torch.uint8).view(b - a, -1)
        scale[:, a:b], zero[:, a:b] = sc.t(), ze.t()
    return codes, scale, zero


def _chunk_inputs(case, gen):
    B, hq, hkv, n, T, W = (case[f] for f in ("batch", "q_heads", "kv_heads", "new", "tokens", "window"))
    dt = DTYPES[case["dtype"]]
    s = {"case": case, "q": torch.randn(B, n, hq, D, generator=gen, device=DEV).to(dt).transpose(1, 2)}
    for side in ("k", "v"):
        s[side + "_codes"], s[side + "_scale"], s[side + "_zero"] = _quantised(B, hkv, T, case["rel"], dt, side == "k", gen)
        s[side + "_win"] = torch.randn(B, hkv, CAP, D, generator=gen, device=DEV).to(dt) if W else None
    s["starts"] = None
    if case["padded"]:
        s["starts"] = torch.randint(0, (T + W - n) // 2 + 2, (B,), generator=gen, device=DEV).to(torch.int32)
    return s


def _encoded(s):
    """The cache such a program keeps: streams in the place of the codes."""
    from packkv_amd import ops
    case, bits = s["case"], BITS[s["case"]["rel"]]
    for side, is_k, ctx, hid in (("k", True, 64, 128), ("v", False, 128, 64)):
        codes = s.pop(side + "_codes")
        blocks = (codes.size(0) // ctx) * (codes.size(1) // hid)
        stream = torch.empty(blocks * ops.block_bound(is_k, ctx, hid, bits) + 16, dtype=torch.uint8, device=DEV)
        info = torch.empty(blocks, 2, dtype=torch.uint32, device=DEV)
        size = (ops.k_encode if is_k else ops.v_encode)(codes, stream, info, bits=bits)
        s[side] = {"stream": stream[:size + 16].clone(), "info": info, "scale": s.pop(side + "_scale"), "zero": s.pop(side + "_zero"), "size": size,
                   "bits": bits, "tokens": case["tokens"], "heads": case["kv_heads"]}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] == "chunk":
        _encoded(s)
    return s


def _inputs(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return {"rotary": _rotary_inputs, "step": _rotary_inputs, "sample": _sample_inputs, "chunk": _chunk_inputs}[case["kind"]](case, gen)


# ---------------------------------------------------------------- one pass

def run(state):
    return (_own if own else _plain)[state["case"]["kind"]](state)


def _own_rotary(s):
    from packkv_amd import ops
    return ops.norm_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], s["q_norm"], s["k_norm"], sections=_sections(s["case"]),
                           interleaved=s["case"]["interleaved"])


def _own_step(s):
    from packkv_amd import ops
    q = ops.window_append_rotary(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["k_win"], s["v_win"], s["row"], s["q_norm"], s["k_norm"],
                                 sections=_sections(s["case"]), interleaved=s["case"]["interleaved"])
    return q, s["k_win"], s["v_win"]


def _own_sample(s):
    from packkv_amd import ops
    return ops.sample(s["logits"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["min_p"], want_logprob=True)


def _own_chunk(s):
    from packkv_amd import ops
    w = s["case"]["window"]
    return ops.attn_chunk(s["q"], s["k"], s["v"], s["k_win"], s["v_win"], win_len=w or None, starts=s["starts"])


def _axis_of(case):
    """The position axis of each of the 64 frequencies."""
    if case["axes"] == 1:
        return [0] * (D // 2)
    sec = _sections(case)
    if not case["interleaved"]:
        return [a for a, w in enumerate(sec) for _ in range(w)]
    axis = [0] * (D // 2)
    for a in (1, 2):
        for j in range(sec[a]):
            axis[a + 3 * j] = a
    return axis


def _turned(x, w, cos, sin):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w.float()
    a, b = y[..., :D // 2], y[..., D // 2:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1).to(x.dtype)


def _plain_rotary(s):
    pos = s["positions"].double()
    if s["case"]["axes"] == 1:
        angle = pos[..., None] * s["inv_freq"].double()
    else:
        axis = torch.tensor(_axis_of(s["case"]), device=DEV)
        angle = pos[axis].permute(1, 2, 0) * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    return _turned(s["q"], s["q_norm"], cos, sin), _turned(s["k"], s["k_norm"], cos, sin)


def _plain_step(s):
    q, k = _plain_rotary(s)
    rows = slice(s["row"], s["row"] + k.size(2))
    s["k_win"][:, :, rows] = k
    s["v_win"][:, :, rows] = s["v"]
    return q, s["k_win"], s["v_win"]


def _column(x, R):
    return x.double()[:, None] if torch.is_tensor(x) else torch.full((R, 1), float(x), dtype=torch.float64, device=DEV)


def _plain_sample(s):
    R, V = s["logits"].shape
    x = s["logits"].double()
    t, k, p, min_p = (_column(s[f], R).float().double() for f in ("t", "k", "p", "min_p"))
    top, order = torch.sort(x, dim=1, descending=True, stable=True)
    e = torch.exp((top - top[:, :1]) / t)
    rank = torch.arange(V, device=DEV)[None]
    e = torch.where((k <= 0) | (rank < k), e, torch.zeros_like(e))
    cum = torch.cumsum(e, dim=1)
    e = torch.where((p >= 1) | (rank == 0) | (cum - e < p * cum[:, -1:]), e, torch.zeros_like(e))
    e = torch.where(e >= min_p, e, torch.zeros_like(e))
    cum = torch.cumsum(e, dim=1)
    last = (e > 0).sum(dim=1) - 1
    at = (cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(dim=1)
    at = torch.minimum(at, last)[:, None]
    logprob = torch.log(e.gather(1, at) / cum[:, -1:]).float()
    return order.gather(1, at)[:, 0], logprob[:, 0]


def _plain_chunk(s):
    case = s["case"]
    B, hq, hkv, n, T, W = (case[f] for f in ("batch", "q_heads", "kv_heads", "new", "tokens", "window"))
    G, total = hq // hkv, T + W
    out = torch.empty_like(s["q"])
    t = torch.arange(total, device=DEV)
    own_pos = torch.arange(n, device=DEV) + (total - n)
    for b in range(B):
        seen = t[None, :] <= own_pos[:, None]
        if s["starts"] is not None:
            seen = seen & (t[None, :] >= s["starts"][b])
        for h in range(hkv):
            kv = []
            for side in ("k", "v"):
                at = (b * hkv + h) * D
                x = (s[side + "_codes"][:, at:at + D].float() + s[side + "_zero"][b].float()[:, None]) * s[side + "_scale"][b].float()[:, None]
                kv.append(torch.cat((x, s[side + "_win"][b, h, :W].float())) if W else x)
            q = s["q"][b, h * G:(h + 1) * G].float().reshape(G * n, D)
            w = (torch.matmul(q, kv[0].t()) * (D ** -0.5)).view(G, n, total)
            w = w.masked_fill(~seen, float("-inf"))
            top = w.amax(-1, keepdim=True)
            w = torch.exp(w - torch.where(torch.isinf(top), torch.zeros_like(top), top))
            sums = w.sum(-1, keepdim=True)
            o = torch.matmul(w.view(G * n, total), kv[1]).view(G, n, D) / torch.where(sums > 0, sums, torch.ones_like(sums))
            out[b, h * G:(h + 1) * G] = o.to(out.dtype)
    return out


_own = {"rotary": _own_rotary, "step": _own_step, "sample": _own_sample, "chunk": _own_chunk}
_plain = {"rotary": _plain_rotary, "step": _plain_step, "sample": _plain_sample, "chunk": _plain_chunk}


def work(case):
    kind = case["kind"]
    if kind in ("rotary", "step"):
        rows = case["batch"] * case["tokens"]
        heads = case["q_heads"] + case["kv_heads"] * (2 if kind == "step" else 1)
        return {"bytes": rows * (heads * D * 2 * 2 + 8 * case["axes"]) + 64 * 4 + (2 * D * 2 if case["norm"] else 0),
                "flops": rows * (case["q_heads"] + case["kv_heads"]) * D * (7 if case["norm"] else 3)}
    if kind == "sample":
        size = case["rows"] * case["vocab"]
        return {"bytes": size * (4 if case["dtype"] == "f32" else 2) + case["rows"] * (16 + (16 if case["mixed"] else 0)), "flops": size * 12}
    B, hq, hkv, n, T, W = (case[f] for f in ("batch", "q_heads", "kv_heads", "new", "tokens", "window"))
    bits = BITS[case["rel"]]
    stored = B * T * hkv * D * (K_BITS[bits] + V_BITS[bits]) / 8 + 8 * B * T + B * hkv * W * D * 4
    seen = n * (T + W) - n * (n - 1) // 2
    if case["padded"]:                     # a quarter of the tokens is padding, on average
        seen = seen * 3 // 4
    return {"bytes": int(stored + 2 * B * hq * n * D * 2), "flops": 4 * B * hq * D * seen}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("rotary", "step"):
        return _exact_rotary(case, s)
    return _exact_sample(case, s) if case["kind"] == "sample" else _exact_chunk(case, s)


def _exact_rotary(case, s):
    pos = s["positions"].cpu().numpy().astype(np.float64)
    pos = pos[None] if case["axes"] == 1 else pos
    freq = s["inv_freq"].cpu().numpy().astype(np.float64)
    axis = np.array(_axis_of(case))
    turn = np.exp(1j * np.moveaxis(pos[axis], 0, -1) * freq)                # [B, n, 64]: one complex number turns a pair
    both = []
    for f in ("q", "k"):
        x = s[f].cpu().double().numpy()
        if s[f + "_norm"] is not None:
            x = x / np.sqrt((x ** 2).sum(-1, keepdims=True) / D + 1e-6) * s[f + "_norm"].cpu().double().numpy()
        z = (x[..., :64] + 1j * x[..., 64:]) * turn[:, None]
        both.append(torch.from_numpy(np.concatenate((z.real, z.imag), axis=-1)))
    if case["kind"] == "rotary":
        return tuple(both)
    wins = [s["k_win"].cpu().double(), s["v_win"].cpu().double()]
    for win, rows in zip(wins, (both[1], s["v"].cpu().double())):
        win[:, :, s["row"]:s["row"] + case["tokens"]] = rows
    return both[0], wins[0], wins[1]


def _exact_sample(case, s):
    if case["rows"] * case["vocab"] > 1 << 27:
        return None
    logits, u = s["logits"].cpu().double().numpy(), s["u"].cpu().double().numpy()
    par = {f: (s[f].cpu().numpy() if torch.is_tensor(s[f]) else np.full(case["rows"], s[f])) for f in ("t", "k", "p", "min_p")}
    par = {f: a.astype(np.int64) if f == "k" else a.astype(np.float32).astype(np.float64) for f, a in par.items()}
    out, logprob = np.empty(case["rows"], dtype=np.int64), np.empty(case["rows"])
    for r in range(case["rows"]):
        idx = np.nonzero(logits[r] > -np.inf)[0]
        idx = idx[np.argsort(-logits[r, idx], kind="stable")]
        if par["k"][r] > 0:
            idx = idx[:par["k"][r]]
        weight = np.exp((logits[r, idx] - logits[r, idx[0]]) / par["t"][r])
        if par["p"][r] < 1:
            before = np.concatenate(([0.0], np.cumsum(weight)[:-1]))
            idx = idx[:max(1, int((before < par["p"][r] * weight.sum()).sum()))]
        idx = idx[weight[:idx.size] >= par["min_p"][r]]
        edges = np.cumsum(weight[:idx.size])
        at = min(int(np.searchsorted(edges, u[r] * edges[-1], side="right")), idx.size - 1)
        out[r], logprob[r] = idx[at], (logits[r, idx[at]] - logits[r, idx[0]]) / par["t"][r] - math.log(edges[-1])
    return torch.from_numpy(out), torch.from_numpy(logprob)


def _exact_chunk(case, s):
    B, hq, hkv, n, T, W = (case[f] for f in ("batch", "q_heads", "kv_heads", "new", "tokens", "window"))
    G = hq // hkv
    out = torch.zeros(B, hq, n, D, dtype=torch.float64, device=DEV)
    later = torch.arange(T + W, device=DEV)[:, None] - torch.arange(T + W - n, T + W, device=DEV)[None, :]        # [tokens, queries]
    for b in range(B):
        first = 0 if s["starts"] is None else int(s["starts"][b])
        for hk in range(hkv):
            cols = slice((b * hkv + hk) * D, (b * hkv + hk + 1) * D)
            side = {}
            for f in ("k", "v"):
                x = s[f + "_codes"][:, cols].double().add_(s[f + "_zero"][b].double()[:, None]).mul_(s[f + "_scale"][b].double()[:, None])
                side[f] = x if not W else torch.cat((x, s[f + "_win"][b, hk, :W].double()))
            for g in range(G):
                score = side["k"] @ s["q"][b, hk * G + g].double().t() / math.sqrt(D)                            # [tokens, queries]
                score[later > 0] = -math.inf
                score[:first] = -math.inf
                weight = torch.softmax(score, dim=0)
                out[b, hk * G + g] = torch.nan_to_num(weight, nan=0.0).t() @ side["v"]
    return out
