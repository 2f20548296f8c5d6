"""Chunk attention in 64 bits on what a cache holds, and the tolerance of the kernel that follows from its roundings."""
import torch

from packkv_amd import ops


def codes_of(side, is_k, B, H):
    """A side's codes as fp64 [B, H, T, 128], unpacked by the block decoder."""
    T, hidden = int(side.get("tokens", side["scale"].size(1))), B * H * 128
    codes = torch.empty(T, hidden, dtype=torch.uint8, device=side["stream"].device)
    blocks = (T // (64 if is_k else 128)) * (hidden // (128 if is_k else 64))
    (ops.k_decode if is_k else ops.v_decode)(side["stream"], side["info"].view(-1, 2)[:blocks].contiguous(), codes, bits=side["bits"])
    return codes.view(T, B, H, 128).permute(1, 2, 0, 3).double()


def values_of(side, is_k, B, H, win, rows):
    """(values, sum of the two terms' sizes) [B, H, T + rows, 128]: (code + zero) * scale, then the window's rows."""
    parts, sizes = [], []
    if side is not None:
        T = int(side.get("tokens", side["scale"].size(1)))
        c = codes_of(side, is_k, B, H)
        sc, ze = (side[f][:, :T].double()[:, None, :, None] for f in ("scale", "zero"))
        parts.append((c + ze) * sc)
        sizes.append((c + ze.abs()) * sc.abs())
    if rows:
        parts.append(win[:, :, :rows].double())
        sizes.append(parts[-1].abs())
    return torch.cat(parts, 2), torch.cat(sizes, 2)


def attend(q, K, V, sm=128 ** -0.5, starts=None, causal=True, sizes=None, v_sizes=None):
    """(out, tolerance) [B, Hq, n, 128] fp64.  The tolerance counts, relative to sum p |v|: the weights' rounding to fp16, 2^-11 (bf16
    window rows: two bf16 halves, less); a score's fp32 steps, 140 roundings of 2^-24 of sum |q| |k terms| * sm (128 products, scale,
    zero, exponent), which move a weight and the sum of weights; 2^-22 for exp2 and the factors.  The sums' T / 16 + 64 fp32 additions
    round what is added up, and that is sum p scale code and sum p scale zero, each by itself: relative to sum p scale (code + |zero|)
    (`v_sizes`), which stays where code + zero is 0 and the value vanishes.  And half a step of the stored type."""
    B, Hq, n, D = q.shape
    H, T = K.size(1), K.size(2)
    out, tol = torch.zeros(B, Hq, n, D, dtype=torch.float64, device=q.device), torch.zeros(B, Hq, n, D, dtype=torch.float64, device=q.device)
    half = torch.finfo(q.dtype).eps / 2
    t = torch.arange(T, device=q.device)[None]
    seen_to = torch.arange(T - n, T, device=q.device)[:, None] if causal else torch.full((n, 1), T, device=q.device)
    for b in range(B):
        ok = t <= seen_to
        if starts is not None:
            ok = ok & (t >= int(starts[b]))
        for h in range(Hq):
            x, k, v = q[b, h].double(), K[b, h // (Hq // H)], V[b, h // (Hq // H)]
            s = torch.where(ok, x @ k.t() * sm, -torch.inf)
            w = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            v = torch.where(ok.any(0)[:, None], v, 0.0)
            out[b, h] = w @ v
            size = x.abs() @ (sizes[b, h // (Hq // H)] if sizes is not None else k.abs()).t() * sm
            worst = torch.where(ok, size, 0.0).amax(-1, keepdim=True)
            rel = 2.0 ** -11 + 2 * 140 * 2.0 ** -24 * worst + 2.0 ** -22
            both = torch.where(ok.any(0)[:, None], v_sizes[b, h // (Hq // H)], 0.0) if v_sizes is not None else v.abs()
            tol[b, h] = (rel * (w @ v.abs()) + (T / 16 + 64) * 2.0 ** -24 * (w @ both)) * (1 + half) + half * out[b, h].abs() + torch.finfo(q.dtype).smallest_normal * half
    return out, tol


def check(got, q, K, V, **kw):
    want, tol = attend(q, K, V, **kw)
    err = (got.double() - want).abs()
    print("   largest error %.3e, of what is allowed %.3f" % (err.max().item(), (err / tol.clamp_min(1e-300)).max().item() if got.numel() else 0), flush=True)
    assert bool((err <= tol).all()), ((err / tol.clamp_min(1e-300)).max().item(), err.max().item())
