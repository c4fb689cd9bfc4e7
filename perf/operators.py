"""What is timed of the quantised key/value cache: writing it, reading it back, and the attention over it.

The cache keeps a row (the `head_dim` numbers of one token and one key/value head, keys and values apart) as 8-bit codes and one
float32 scale: with A = max(|x_i|, 2^-60), scale = A / top and code_i = round(x_i * (top / A)), to whole numbers with ties to even
for "int8" (top 127) and to e4m3 for "fp8" (top 448); the row stands for code_i * scale.  A row with a number that is not finite
has the scale NaN and codes of zero.  Pages hold 64 tokens, [page][kv_head][64][head_dim], with the scales in [page][kv_head][64].

  write    the rotation of a step's queries and keys and the quantising append of its keys and values, then the rows read back
  decode   one new token a sequence: rotation, append and attention over the sequence's pages, and the new rows read back
  prompt   attention of many new tokens a sequence over pages that hold them already

Head counts are those of the Llama presets (9 query heads on 3 of 64, 15 on 5, 32 on 32) and of wider heads; drawn cases have other
head sizes, groups and windows too.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
PAGE = 64
TILE = 128                 # tokens of a tile of the prompt attention, at most
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
SMALLEST = 2.0 ** -60      # what a row's largest magnitude counts as, at least


# ----------------------------------------------------------------------------- the cases
def _case(op, fmt, dtype, nh, nkv, hd, seqs, shortest, longest, held=0, window=0, **named):
    """`shortest` .. `longest`: tokens of a sequence (decode: in the cache, with the new one; write and prompt: new ones); `held`: tokens
    that a prompt's sequence has in the cache before its new ones; `window`: keys that a token sees (0: all)."""
    return dict(named, op=op, format=fmt, dtype=dtype, heads=nh, kv_heads=nkv, head_dim=hd, seqs=seqs, shortest=shortest, longest=longest,
                held=held, window=window)


def listed():
    return [
        # a step of a few tokens that no fused kernel takes: the smallest write, a matter of latency
        _case("write", "int8", "bfloat16", 9, 3, 64, 8, 1, 3, name="write_few_int8"),
        # one long prompt of the middle model on its way into the cache
        _case("write", "fp8", "bfloat16", 15, 5, 64, 1, 2048, 2048, name="write_2048_fp8"),
        # a server's step of unequal prompts on the wide model
        _case("write", "int8", "bfloat16", 32, 32, 64, 7, 501, 1901, name="write_ragged_int8"),
        # one person's answer, a short conversation on the small model
        _case("decode", "int8", "bfloat16", 9, 3, 64, 1, 130, 130, name="decode_one_int8"),
        # a handful of requests with contexts of all lengths
        _case("decode", "fp8", "bfloat16", 15, 5, 64, 8, 130, 2040, name="decode_batch_fp8"),
        # a full server on the wide model: what the smaller cache is for
        _case("decode", "int8", "bfloat16", 32, 32, 64, 64, 700, 2300, name="decode_many_int8"),
        # one very long document
        _case("decode", "fp8", "bfloat16", 16, 4, 128, 1, 65001, 65001, name="decode_long_fp8"),
        # the 32-bit path generating for a batch
        _case("decode", "int8", "float32", 15, 5, 64, 24, 61, 701, name="decode_f32_int8"),
        # a question of a sentence
        _case("prompt", "int8", "bfloat16", 9, 3, 64, 1, 17, 17, name="prompt_short_int8"),
        # a long prompt on the wide model
        _case("prompt", "fp8", "bfloat16", 32, 32, 64, 1, 2048, 2048, name="prompt_2048_fp8"),
        # next turns of running conversations: new tokens behind those that the cache holds
        _case("prompt", "int8", "bfloat16", 16, 4, 128, 4, 65, 701, held=1501, name="prompt_turns_int8"),
        # the 32-bit path scoring a few prompts
        _case("prompt", "fp8", "float32", 9, 3, 64, 3, 61, 701, name="prompt_f32_fp8"),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(("write", "decode", "prompt"))
    fmt, dtype = rng.choice(("int8", "fp8")), rng.choice(("bfloat16", "bfloat16", "float32"))
    hd = rng.choice((32, 64, 64, 96, 128, 128, 16 * rng.randint(1, 16)))
    nkv, group = spread(1, 32), rng.choice((1, 1, 2, 3, 4, 7, 8, 12))
    window = rng.choice((0, 0, 0, spread(1, 2000)))
    if op == "write":
        seqs, longest = spread(1, 64), spread(1, 2100)
        seqs = max(1, min(seqs, 8000 // longest))
        nkv = max(1, min(nkv, 32 * 64 // hd))
        return _case(op, fmt, dtype, nkv * min(group, max(1, 4096 // (nkv * hd))), nkv, hd, seqs, rng.randint(1, longest), longest)
    if op == "decode":
        longest, seqs = spread(1, 65000), spread(1, 64)
        seqs = max(1, min(seqs, 120_000_000 // (longest * nkv * hd)))
        longest = max(1, min(longest, 120_000_000 // (seqs * nkv * hd)))
        return _case(op, fmt, dtype, nkv * group, nkv, hd, seqs, rng.randint(1, longest), longest, window=window)
    longest, held, seqs = spread(1, 2100), rng.choice((0, 0, spread(1, 4000))), spread(1, 8)
    most = (40_000_000 if dtype == "float32" else 120_000_000) * 64 // max(64, hd)
    seqs = max(1, min(seqs, most // (longest * (longest + held))))
    pairs = seqs * longest * (longest + held)
    group = max(1, min(group, most // pairs))
    nkv = max(1, min(nkv, most // (pairs * group)))
    return _case(op, fmt, dtype, nkv * group, nkv, hd, seqs, rng.randint(1, longest), longest, held=held, window=window)


def _lengths(case):
    """Tokens of every sequence: the longest first, the others spread evenly down to the shortest."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


# ----------------------------------------------------------------------------- the inputs
def _tables(n, hd):
    """Cosines and sines of the positions below n, half-split pairing, as a model keeps them: angles in float64, rounded once."""
    inv = 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=DEVICE) / hd)
    ang = torch.arange(n, dtype=torch.float64, device=DEVICE)[:, None] * inv[None]
    return torch.cos(ang).float().contiguous(), torch.sin(ang).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    dtype, lengths, held = DTYPES[case["dtype"]], _lengths(case), case["held"]
    decode = case["op"] == "decode"
    totals = [n if decode else held + n for n in lengths]           # tokens of a sequence in the cache after the step
    news = [1] * len(lengths) if decode else lengths
    first = [t - n for t, n in zip(totals, news)]
    B, T = len(news), sum(news)
    per_seq = -(-max(totals) // PAGE)
    n_pages = sum(-(-t // PAGE) for t in totals) + 1
    order = torch.randperm(n_pages, generator=g, device=DEVICE).cpu()
    table, at = torch.full((B, per_seq), -1, dtype=torch.int32), 0
    for b, t in enumerate(totals):
        k = -(-t // PAGE)
        table[b, :k] = order[at:at + k]
        at += k
    # every page holds rows (what lies behind a sequence's end is some earlier sequence's): keys whose channels differ in size as
    # those of trained models do, values whose rows differ in size
    wide = torch.exp(0.5 * torch.randn(hd, generator=g, device=DEVICE))
    kc, vc, ks, vs = [], [], [], []
    step = max(1, (1 << 25) // (nkv * PAGE * hd))
    for a in range(0, n_pages, step):
        shape = (min(step, n_pages - a), nkv, PAGE, hd)
        for codes, scales, rows in ((kc, ks, torch.randn(shape, generator=g, device=DEVICE) * wide),
                                    (vc, vs, torch.randn(shape, generator=g, device=DEVICE) * torch.exp(torch.randn(shape[:3] + (1,), generator=g, device=DEVICE)))):
            c, s = _quantised(rows, case["format"])
            codes.append(c)
            scales.append(s)
    qkv = torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device=DEVICE)
    qkv[:, nh * hd:(nh + nkv) * hd] *= wide.repeat(nkv)
    pos = torch.cat([torch.arange(p, p + n) for p, n in zip(first, news)]).to(torch.int32)
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(news)).to(torch.int32)
    tiles = [(b, sum(news[:b]) + a, min(TILE, n - a), first[b] + a) for b, n in enumerate(news) for a in range(0, n, TILE)]
    dev = lambda v: torch.as_tensor(v, dtype=torch.int32).contiguous().to(DEVICE)      # noqa: E731
    cos, sin = _tables(max(totals), hd)
    s = {"case": case, "qkv": qkv.to(dtype), "keys": torch.cat(kc), "values": torch.cat(vc), "k_scale": torch.cat(ks), "v_scale": torch.cat(vs),
         "table": table.to(DEVICE), "pos": dev(pos), "seq": dev(seq), "slot": dev(range(B)), "seq_pos": dev([t - 1 for t in totals]),
         "tiles": [dev([t[i] for t in tiles]) for i in range(4)], "cos": cos, "sin": sin, "B": B, "T": T, "most": max(totals),
         "scale": 1.0 / math.sqrt(hd), "err": torch.zeros(1, dtype=torch.int32, device=DEVICE),
         "out": torch.empty((T, nh * hd), dtype=dtype, device=DEVICE), "step_qkv": torch.empty((T, (nh + 2 * nkv) * hd), dtype=dtype, device=DEVICE),
         "row_keys": torch.empty((T, nkv, hd), dtype=torch.bfloat16, device=DEVICE),
         "row_values": torch.empty((T, nkv, hd), dtype=torch.bfloat16, device=DEVICE)}
    # where a padded query row [sequence, place] of a prompt step lies among the packed ones
    longest = max(news)
    place = torch.arange(longest, device=DEVICE)[None, :]
    s["padded"] = (torch.tensor([sum(news[:b]) for b in range(B)], device=DEVICE)[:, None] + place).clamp(max=T - 1)
    s["padded_pos"] = torch.where(place < torch.tensor(news, device=DEVICE)[:, None], torch.tensor(first, device=DEVICE)[:, None] + place, 0)
    s["packed"] = torch.tensor([b * longest + i for b, n in enumerate(news) for i in range(n)], device=DEVICE)
    return s


# ----------------------------------------------------------------------------- the plain forms
def _quantised(rows, fmt):
    """Codes (int8 or e4m3) and scales of float32 rows."""
    amax = rows.abs().amax(-1, keepdim=True)
    top = torch.full_like(amax, 127.0 if fmt == "int8" else 448.0)
    a = amax.clamp(min=SMALLEST)
    y = rows * torch.div(top, a)
    fine = torch.isfinite(amax)
    y = torch.where(fine, y, torch.zeros_like(y))
    codes = torch.round(y).clamp(-127, 127).to(torch.int8) if fmt == "int8" else y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, torch.where(fine, torch.div(a, top), torch.full_like(a, math.nan)).squeeze(-1)


def _rotated(x, cos, sin):
    """x [T, heads, hd] float32 at the rows' angles [T, hd / 2]."""
    half = x.shape[-1] // 2
    a, b, c, s = x[..., :half], x[..., half:], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _append(s, seq, pos):
    """The rotated queries [T, nh, hd] in float32; the cache gets the step's rows."""
    c = s["case"]
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"].float().view(-1, nh + 2 * nkv, hd)
    where = pos.long()
    r = _rotated(x[:, :nh + nkv], s["cos"][where], s["sin"][where])
    page, row = s["table"][seq.long(), where // PAGE].long(), where % PAGE
    for rows, codes, scales in ((r[:, nh:], s["keys"], s["k_scale"]), (x[:, nh + nkv:], s["values"], s["v_scale"])):
        q, f = _quantised(rows, c["format"])
        codes.view(torch.int8)[page, :, row] = q.view(torch.int8)
        scales[page, :, row] = f
    return r[:, :nh]


def _rows(s, seq, pos):
    where = pos.long()
    page, row = s["table"][seq.long(), where // PAGE].long(), where % PAGE
    read = lambda codes, scales: (_numbers(codes, (page, row)) * scales[page, :, row].unsqueeze(-1)).to(torch.bfloat16)     # noqa: E731
    return read(s["keys"], s["k_scale"]), read(s["values"], s["v_scale"])


def _numbers(codes, index):
    picked = codes.view(torch.int8)[index[0], :, index[1]] if isinstance(index, tuple) else codes.view(torch.int8)[index]
    return picked.view(codes.dtype).float()


def _attend(s, q, pos):
    """q [B, Q, nh, hd] float32 at positions pos [B, Q]: softmax over the keys that each sees, [B, Q, nh, hd] float32."""
    c = s["case"]
    nkv, hd = c["kv_heads"], c["head_dim"]
    table = s["table"].long().clamp(min=0)
    def laid(codes, scales):
        v = _numbers(codes, table) * scales[table].unsqueeze(-1)                 # [B, pages, nkv, 64, hd]
        return v.transpose(1, 2).reshape(v.shape[0], nkv, -1, hd)
    key = torch.arange(table.shape[1] * PAGE, device=q.device)
    seen = key <= pos[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    B, Q = pos.shape
    qg = q.view(B, Q, nkv, -1, hd).permute(0, 2, 3, 1, 4)                        # [B, nkv, group, Q, hd]
    x = torch.matmul(qg.reshape(B, nkv, -1, hd), laid(s["keys"], s["k_scale"]).transpose(-1, -2)).view(qg.shape[:4] + (-1,)) * s["scale"]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    values = laid(s["values"], s["v_scale"])
    values = torch.where((key[None] <= pos.amax(1)[:, None])[:, None, :, None], values, torch.zeros_like(values))
    o = torch.matmul(p.view(B, nkv, -1, p.shape[-1]), values).view(qg.shape) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(B, Q, -1, hd)


def run(s):
    c = s["case"]
    nh, nkv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if own:
        from edgelm_b200.csrc import ops
        cache = (s["keys"], s["values"], s["k_scale"], s["v_scale"])
        if c["op"] == "prompt":
            ops.attn_prefill_quantized(s["qkv"], s["out"], *cache, s["table"], s["slot"], *s["tiles"], s["tiles"][0].numel(), nh, nkv, hd,
                                       s["scale"], err=s["err"], window=c["window"], max_keys=s["most"])
            return s["out"]
        if c["op"] == "write":
            ops.rope_quantize_append(s["qkv"], s["pos"], s["seq"], s["slot"], s["table"], s["cos"], s["sin"], *cache, nh, nkv, hd, s["err"], q_out=s["out"])
            ops.quantized_rows(*cache, s["pos"], s["seq"], s["slot"], s["table"], s["row_keys"], s["row_values"], s["err"])
            return s["out"], s["row_keys"], s["row_values"]
        ops.attn_decode_rope_quantized(s["qkv"], s["out"], *cache, s["table"], s["slot"], s["seq_pos"], s["cos"], s["sin"], s["B"], nh, nkv, hd,
                                       s["scale"], err=s["err"], window=c["window"])
        ops.quantized_rows(*cache, s["seq_pos"], s["slot"], s["slot"], s["table"], s["row_keys"], s["row_values"], s["err"])
        return s["out"], s["row_keys"], s["row_values"]
    dtype = s["qkv"].dtype
    if c["op"] == "prompt":
        q = s["qkv"][:, :nh * hd].float().view(-1, nh, hd)
        o = _attend(s, q[s["padded"]], s["padded_pos"])
        return o.reshape(-1, nh * hd)[s["packed"]].to(dtype)
    if c["op"] == "write":
        q = _append(s, s["seq"], s["pos"])
        return (q.reshape(-1, nh * hd).to(dtype), *_rows(s, s["seq"], s["pos"]))
    q = _append(s, s["slot"], s["seq_pos"])
    o = _attend(s, q[:, None], s["seq_pos"].long()[:, None])
    return (o.reshape(-1, nh * hd).to(dtype), *_rows(s, s["slot"], s["seq_pos"]))


def _pairs(case):
    """(query, key) pairs that are scored, of one head."""
    n = 0
    for t in _lengths(case):
        lo, hi = (t - 1, t) if case["op"] == "decode" else (case["held"], case["held"] + t)
        if case["window"]:
            n += sum(min(p + 1, case["window"]) for p in range(lo, hi))
        else:
            n += (hi * (hi + 1) - lo * (lo + 1)) // 2
    return n


def work(case):
    nh, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    e = 2 if case["dtype"] == "bfloat16" else 4
    lengths = _lengths(case)
    row = 2 * nkv * (hd + 4)                    # codes and scales of a token's keys and values
    back = 2 * nkv * hd * 2                     # and those read back, as bfloat16
    if case["op"] == "write":
        T = sum(lengths)
        return {"bytes": T * ((nh + 2 * nkv) * hd * e + nh * hd * e + row + back), "flops": 6 * T * (nh + nkv) * hd // 2}
    flops = 4 * _pairs(case) * nh * hd
    if case["op"] == "decode":
        seen = sum(min(n, case["window"] or n) for n in lengths)
        return {"bytes": seen * row + len(lengths) * ((2 * nh + 2 * nkv) * hd * e + back), "flops": flops}
    seen = sum(min(case["held"] + n, (case["window"] or n + case["held"]) + n - 1) for n in lengths)
    return {"bytes": seen * row + sum(lengths) * 2 * nh * hd * e, "flops": flops}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _nearest(rows, fmt):
    """float64 rows -> the numbers that their codes and scales stand for."""
    a = np.maximum(np.abs(rows).max(-1, keepdims=True), 2.0 ** -60)
    if fmt == "int8":
        return np.rint(rows / a * 127.0) * (a / 127.0)
    y = rows / a * 448.0
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -40))), -6.0) - 3.0)
    return np.rint(y / step) * step * (a / 448.0)


def exact(case, seed):
    nh, nkv, hd, g = case["heads"], case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    if case["seqs"] * max(_lengths(case)) * nkv * hd > 400_000_000:
        return None
    s = prepare(case, seed)
    f64 = lambda t: t.double().cpu().numpy()                                     # noqa: E731
    news = [1] * case["seqs"] if case["op"] == "decode" else _lengths(case)
    last = s["seq_pos"].tolist()
    qkv = f64(s["qkv"]).reshape(-1, nh + 2 * nkv, hd)
    outs, keys, values, turned = [], [], [], []
    t0 = 0
    for b, n in enumerate(news):
        x, p = qkv[t0:t0 + n], np.arange(last[b] + 1 - n, last[b] + 1)
        t0 += n
        if case["op"] != "prompt":
            z = (x[..., :hd // 2] + 1j * x[..., hd // 2:])[:, :nh + nkv]
            ang = f64(s["cos"])[p] + 1j * f64(s["sin"])[p]                       # the tables are what the operator is given
            z = z * ang[:, None]
            r = np.concatenate([z.real, z.imag], -1)
            x = np.concatenate([r, x[:, nh + nkv:]], 1)
            keys.append(_nearest(x[:, nh:nh + nkv], case["format"]))
            values.append(_nearest(x[:, nh + nkv:], case["format"]))
            turned.append(x[:, :nh].reshape(n, -1))
        if case["op"] == "write":
            continue
        L = last[b] + 1
        pages = s["table"][b, :-(-L // PAGE)].long()
        q = torch.as_tensor(x[:, :nh], device=DEVICE)
        o = torch.empty((n, nh, hd), dtype=torch.float64, device=DEVICE)
        i = torch.as_tensor(p, device=DEVICE)[:, None]
        j = torch.arange(L, device=DEVICE)[None]
        hidden = (j > i) | (j <= i - case["window"]) if case["window"] else j > i
        for h in range(nkv):
            kv = []
            for codes, scales, new in ((s["keys"], s["k_scale"], keys), (s["values"], s["v_scale"], values)):
                m = (codes.view(torch.int8)[pages, h].view(codes.dtype).double() * scales[pages, h].double()[..., None]).reshape(-1, hd)[:L]
                if case["op"] == "decode":
                    m[L - 1] = torch.as_tensor(new[b][0, h], device=DEVICE)
                kv.append(m)
            for k in range(h * g, h * g + g):
                w = torch.softmax(((q[:, k] @ kv[0].T) / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1)
                o[:, k] = w @ kv[1]
        outs.append(o.reshape(n, -1).cpu().numpy())
    whole = lambda parts: np.concatenate(parts)                                  # noqa: E731
    if case["op"] == "prompt":
        return whole(outs)
    if case["op"] == "write":
        return whole(turned), whole(keys), whole(values)
    return whole(outs), whole(keys), whole(values)
