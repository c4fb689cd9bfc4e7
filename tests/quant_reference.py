"""Plain float64 statements of the 8-bit cache and of the attention over it, for the tests."""
import math

import torch

PAGE = 64
TOP = {"int8": 127.0, "fp8": 448.0}
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def quantize(rows, fmt):
    """float32 rows [..., hd] -> (codes, scales), in the single float32 operations that the format is defined by."""
    rows = rows.float()
    amax = rows.abs().amax(-1)
    a = torch.clamp(amax, min=2.0 ** -60)
    top = torch.full_like(a, TOP[fmt])
    fine = torch.isfinite(amax)
    y = torch.where(fine[..., None], rows * (top / a)[..., None], torch.zeros_like(rows))
    codes = torch.round(y).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)
    return codes, torch.where(fine, a / top, torch.full_like(a, math.nan))


def rotate(x, cos, sin):
    """x [T, heads, hd] float32, cos and sin [T, hd / 2]: half-split pairs, single float32 operations."""
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half], x[..., half:], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def numbers(codes, scales):
    return codes.to(torch.float64) * scales.double()[..., None]


def sequence_rows(cache, table_row, length):
    """Keys and values [length, nkv, hd] in float64 that the cache holds for a sequence."""
    pages = table_row[:-(-length // PAGE)].long()
    out = []
    for codes, scales in ((cache["k"], cache["ks"]), (cache["v"], cache["vs"])):
        c = codes.view(torch.int8)[pages].view(codes.dtype)
        n = numbers(c, scales[pages])                                  # [pages, nkv, 64, hd]
        out.append(n.transpose(1, 2).reshape(-1, n.shape[1], n.shape[3])[:length])
    return out


def attend(q, first, keys, values, scale, window=0):
    """q [n, nh, hd] float64 of tokens at positions first ..; keys, values [L, nkv, hd]: [n, nh, hd] in float64."""
    n, nh, hd = q.shape
    g = nh // keys.shape[1]
    k, v = keys.repeat_interleave(g, 1), values.repeat_interleave(g, 1)
    s = torch.einsum("nhd,lhd->hnl", q, k) * scale
    p = first + torch.arange(n, device=q.device)[:, None]
    j = torch.arange(keys.shape[0], device=q.device)[None]
    seen = j <= p
    if window:
        seen &= j > p - window
    w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
    out = torch.einsum("hnl,lhd->nhd", w, v.nan_to_num(0.0, math.inf, -math.inf))
    reached = torch.einsum("nl,lhd->nhd", seen.double(), torch.isnan(v).double()) > 0      # a value that is no number, seen
    return out.masked_fill(reached, math.nan)


def tables(n, hd, device, theta=10000.0):
    inv = theta ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    ang = torch.arange(n, dtype=torch.float64)[:, None] * inv[None]
    return torch.cos(ang).float().to(device), torch.sin(ang).float().to(device)


def make_cache(fmt, nkv, hd, lengths, device, seed, spare=2, k_size=1.0, v_spread=1.0):
    """A cache of shuffled pages whose every row (those behind a sequence's end too) is a quantised random row, and the page table."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(n, 0) // PAGE) for n in lengths]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    shape = (n_pages, nkv, PAGE, hd)
    k, ks = quantize(torch.randn(shape, generator=g) * k_size, fmt)
    v, vs = quantize(torch.randn(shape, generator=g) * torch.exp(v_spread * torch.randn(shape[:3] + (1,), generator=g)), fmt)
    return {"k": k.to(device), "ks": ks.to(device), "v": v.to(device), "vs": vs.to(device)}, table.to(device)
