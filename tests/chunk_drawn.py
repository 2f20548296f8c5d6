"""Caches of drawn codes for attn_chunk, and the call against attention in 64 bits on them (chunk_oracle)."""
import torch

import chunk_oracle as co
from packkv_amd import ops


def drawn(cuda, is_k, B, H, T, bits, dtype, g):
    """A side of drawn codes, its scales about 2 / 2^bits and zeroes down to -2^bits."""
    codes = torch.randint(0, 1 << bits, (T, B * H * 128), generator=g, device=cuda, dtype=torch.uint8)
    ctx, hid = (64, 128) if is_k else (128, 64)
    blocks = (T // ctx) * (B * H * 128 // hid)
    stream = torch.empty(blocks * ops.block_bound(is_k, ctx, hid, bits) + 16, dtype=torch.uint8, device=cuda)
    info = torch.empty(blocks, 2, dtype=torch.uint32, device=cuda)
    size = (ops.k_encode if is_k else ops.v_encode)(codes, stream, info, bits=bits)
    scale = ((0.5 + torch.rand(B, T, generator=g, device=cuda)) * 2.0 / (1 << bits)).to(dtype)
    zero = (-(1 << bits) * torch.rand(B, T, generator=g, device=cuda)).to(dtype)
    return {"stream": stream[:size].clone(), "info": info, "scale": scale, "zero": zero, "bits": bits, "size": size, "heads": H}


def check(q, k, v, kw=None, vw=None, W=0, **args):
    B, H = q.size(0), k["heads"]
    K, sizes = co.values_of(k, True, B, H, kw, W)
    V, v_sizes = co.values_of(v, False, B, H, vw, W)
    got = ops.attn_chunk(q, k, v, kw, vw, win_len=W or None, **args)
    co.check(got, q, K, V, sizes=sizes, v_sizes=v_sizes, starts=args["starts"].tolist() if "starts" in args else None)
