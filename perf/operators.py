"""The attention operators of a serving loop, as a program calls them (`metaljax_b200.attention`).

append   rows of a fused q/k/v projection: norm of every query and key head, rotary positions, keys and
         values written into a paged cache (16-bit, or e4m3 with a power-of-two scale per row; the
         latter is read back as values by `read_pages`)
read     rows of a paged cache as a contiguous matrix of values
prompt   causal attention over whole prompts of different lengths packed one behind the other
paged    attention of new tokens (one per sequence, a few, or a chunk) over a paged cache

`run` calls the package where `own` is true, and computes the same in elementary torch operations
in float32 where it is not (angles in float64). `exact` computes it in float64 from the definitions.
"""

from __future__ import annotations

import itertools
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "e4m3": torch.float8_e4m3fn}
EPS = 1e-6


# ---- cases ---------------------------------------------------------------------------------


def _case(name, op, **more):
    base = {"name": name, "op": op, "seqs": 1, "new": 1, "ctx": 0, "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128,
            "dtype": "bf16", "cache": "bf16", "page": 64, "norm": False, "interleaved": False, "rotary": 128, "theta": 500000.0}
    return {**base, **more}


def listed():
    return [
        # one sequence's next token on its way into the cache: launch latency
        _case("append_1_token", "append", ctx=2047),
        # a batch of 64 decoded tokens, q/k norms, half of the head rotated in interleaved pairs
        _case("append_64_tokens", "append", seqs=64, ctx=2047, ragged=True, norm=True, interleaved=True, rotary=64, theta=10000.0),
        # prompts of different lengths written into an 8-bit cache, and its rows read back
        _case("append_prompts_e4m3", "append", seqs=5, new=1638, ragged=True, norm=True, cache="e4m3", page=32),
        # a few short sequences taken out of small pages
        _case("read_3_short", "read", seqs=3, ctx=333, ragged=True, kv_heads=4, dtype="f16", cache="f16", page=16),
        # a batch of sequences taken out of an 8-bit cache
        _case("read_16_e4m3", "read", seqs=16, ctx=4096, ragged=True, cache="e4m3"),
        # four short prompts that arrive together
        _case("prompt_4_short", "prompt", seqs=4, new=150, ragged=True),
        # sixteen prompts of a small model with heads of 64, in f16
        _case("prompt_16_f16_d64", "prompt", seqs=16, new=700, ragged=True, heads=16, kv_heads=4, dim=64, dtype="f16"),
        # one long prompt of an 8B-parameter model's layer
        _case("prompt_8192", "prompt", new=8192),
        # one sequence's next token over 2048 positions
        _case("decode_1", "paged", ctx=2047),
        # 64 sequences of different lengths decoded over an 8-bit cache
        _case("decode_64_e4m3", "paged", seqs=64, ctx=8000, ragged=True, cache="e4m3"),
        # five proposed tokens of each of eight sequences checked at once; seven query heads per key head
        _case("check_8x5", "paged", seqs=8, new=5, ctx=4000, ragged=True, heads=28, kv_heads=4, page=16),
        # a chunk of a long prompt over what is already in the cache
        _case("chunk_1024_over_32768", "paged", new=1024, ctx=31744, page=128),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "read", "prompt", "prompt", "prompt", "paged", "paged", "paged", "paged"])
    dim = rng.choice([64, 128, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 2, 3, 4, 4, 4, 6, 7, 8])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f16"])
    cache = dtype if dtype == "f16" or rng.random() < 0.6 else "e4m3"
    c = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "cache": cache, "page": rng.choice([16, 32, 64, 128, 256]),
         "norm": rng.random() < 0.5, "interleaved": rng.random() < 0.4, "rotary": rng.choice([dim, dim, dim // 2]), "theta": rng.choice([10000.0, 500000.0]),
         "ragged": rng.random() < 0.8, "ctx": 0}
    if op == "append":
        whole = cache == "e4m3"                     # (written as a whole, so that what is read back is what was written)
        c["seqs"] = _spread(rng, 1, 64)
        c["new"] = _spread(rng, 1, 8192 // c["seqs"])
        c["ctx"] = 0 if whole else _spread(rng, 1, 4096)
    elif op == "read":
        c["seqs"] = _spread(rng, 1, 32)
        c["new"], c["ctx"] = 1, _spread(rng, 16, 65536 // c["seqs"])
    elif op == "prompt":
        c["cache"] = dtype
        c["seqs"] = _spread(rng, 1, 24)
        c["new"] = _spread(rng, 1, max(1, int(4096 / math.sqrt(c["seqs"]))))
    else:
        c["seqs"] = _spread(rng, 1, 64)
        c["new"] = 1 if rng.random() < 0.5 else _spread(rng, 1, max(1, 768 // c["seqs"]))
        c["ctx"] = _spread(rng, 1, min(32768, 262144 // c["seqs"]))
    return c


def _lengths(case, gen):
    """(new tokens, positions after them) of every sequence: as given, or down to a quarter of it."""
    n, new, ctx = case["seqs"], case["new"], case["ctx"]
    if not case["ragged"]:
        return [new] * n, [ctx + new] * n
    u = torch.rand((2, n), generator=gen).tolist()
    u[0][0] = u[1][0] = 1.0                          # (the first as long as they get)
    news = [max(1, round(new * (0.25 + 0.75 * a))) for a in u[0]]
    if case["op"] == "paged" and case["new"] <= 8:
        news = [new] * n
    return news, [a + (round(ctx * (0.25 + 0.75 * b)) if ctx else 0) for a, b in zip(news, u[1])]


def _plan(case):
    return _lengths(case, torch.Generator().manual_seed(1234 + case["seqs"] + case["ctx"] + case["new"]))


def _pairs(news, lens):
    """Query and key pairs that causal attention sees."""
    return sum(n * (l - n) + n * (n + 1) // 2 for n, l in zip(news, lens))


def work(case):
    news, lens = _plan(case)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    t, total = sum(news), sum(lens)
    row = kv * d * 2 * (1 if case["cache"] == "e4m3" else 2) + (2 * kv if case["cache"] == "e4m3" else 0)   # bytes of a position in the cache
    if case["op"] == "append":
        out = t * (h + 2 * kv) * d * 2 + t * h * d * 2 + t * row
        back = t * row + t * kv * d * 4 if case["cache"] == "e4m3" else 0
        return {"bytes": out + back, "flops": t * (h + kv) * d * 8}
    if case["op"] == "read":
        return {"bytes": total * (row + kv * d * 4), "flops": 0}
    if case["op"] == "prompt":
        return {"bytes": t * (2 * h + 2 * kv) * d * 2, "flops": 4 * d * h * _pairs(news, lens)}
    return {"bytes": total * row + 2 * t * h * d * 2, "flops": 4 * d * h * _pairs(news, lens)}


# ---- inputs --------------------------------------------------------------------------------


def _starts(counts):
    return torch.tensor([0, *itertools.accumulate(counts)], dtype=torch.int32, device=DEV)


def _quantized(x):
    """e4m3 codes and exponent bytes (E8M0) of the rows of x (float32): the smallest power of two that brings the row's largest within 448."""
    big = x.abs().amax(-1)
    m, e = torch.frexp(big)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-117, 119)
    e = torch.where(big > 0, e, torch.zeros_like(e))
    codes = torch.ldexp(x, -e[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    fine = torch.isfinite(x).all(-1)
    codes = torch.where(fine[..., None], codes.view(torch.uint8), torch.zeros_like(codes.view(torch.uint8))).view(torch.float8_e4m3fn)
    return codes, torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    news, lens = _plan(case)
    h, kv, d, page, n = case["heads"], case["kv_heads"], case["dim"], case["page"], case["seqs"]
    dt = DTYPES[case["dtype"]]
    t = sum(news)
    s = {"case": case, "kv_lens": torch.tensor(lens, dtype=torch.int32, device=DEV), "total": sum(lens),
         "cu_q": None if case["op"] in ("append", "paged") and max(news) == 1 else _starts(news), "cu_kv": _starts(lens), "longest": (max(news), max(lens))}
    if case["op"] in ("append", "prompt"):
        # a projection's output: query, key and value heads of a token side by side
        s["qkv"] = (torch.randn((t, (h + 2 * kv) * d), generator=gen, device=DEV) * 1.5).to(dt)
    if case["op"] == "paged":
        s["q"] = (torch.randn((t, h, d), generator=gen, device=DEV) * 1.5).to(dt)
    if case["op"] == "prompt":
        return s
    # a pool with pages to spare, handed out in no order, full of what earlier sequences left there
    used = [-(-l // page) for l in lens]
    pool = sum(used) + 7
    order = torch.randperm(pool, generator=gen, device=DEV, dtype=torch.int64).to(torch.int32)
    s["table"] = torch.full((n, max(used)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, u in enumerate(used):
        s["table"][i, :u] = order[at: at + u]
        at += u
    values = [torch.randn((pool, kv, page, d), generator=gen, device=DEV) for _ in range(2)]
    if case["cache"] == "e4m3":
        (s["k"], s["k_exp"]), (s["v"], s["v_exp"]) = _quantized(values[0]), _quantized(values[1])
    else:
        s["k"], s["v"] = (x.to(dt) for x in values)
        s["k_exp"] = s["v_exp"] = None
    if case["op"] == "append":
        s["freqs"] = case["theta"] ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=DEV) / case["rotary"])
        s["norms"] = [(1 + 0.2 * torch.randn((d,), generator=gen, device=DEV)).to(dt) for _ in range(2)] if case["norm"] else [None, None]
    return s


# ---- the plain form ------------------------------------------------------------------------


def _where(s):
    """Of every new token: its sequence and its position."""
    t = s["qkv"].shape[0] if "qkv" in s else s["q"].shape[0]
    row = torch.arange(t, device=DEV)
    if s["cu_q"] is None:
        return row, s["kv_lens"].long() - 1
    cu = s["cu_q"].long()
    seq = torch.searchsorted(cu, row, right=True) - 1
    return seq, s["kv_lens"].long()[seq] - (cu[seq + 1] - row)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _rotated(x, pos, freqs, interleaved):
    """Rotates the first 2 * len(freqs) elements of every head of x [T, heads, D]."""
    half = freqs.shape[0]
    angle = pos.double()[:, None] * freqs
    c, s = angle.cos().to(x.dtype)[:, None], angle.sin().to(x.dtype)[:, None]
    if interleaved:
        a, b = x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]
        turned = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half: 2 * half]
        turned = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([turned, x[..., 2 * half:]], dim=-1)


def _values(codes, exps, like=torch.float32):
    """What a cache's entries stand for."""
    if exps is None:
        return codes.to(like)
    x = torch.ldexp(codes.to(like), exps.to(torch.int32)[..., None] - 127)
    return torch.where(exps[..., None] == 255, torch.full_like(x, float("nan")), x)


def _rows(codes, exps, table, seq, pos, page, like=torch.float32):
    """Rows of a paged cache: those of positions `pos` of sequences `seq`, [.., kv_heads, D]."""
    at = table[seq, pos // page].long()
    return _values(codes[at, :, pos % page], None if exps is None else exps[at, :, pos % page], like)


def _append(s):
    c = s["case"]
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].float().view(-1, h + 2 * kv, d)
    seq, pos = _where(s)
    q, k, v = _normed(x[:, :h], s["norms"][0]), _normed(x[:, h: h + kv], s["norms"][1]), x[:, h + kv:]
    q, k = _rotated(q, pos, s["freqs"], c["interleaved"]), _rotated(k, pos, s["freqs"], c["interleaved"])
    at, off = s["table"][seq, pos // page].long(), pos % page
    q = q.to(s["qkv"].dtype)
    if s["k_exp"] is None:
        s["k"][at, :, off], s["v"][at, :, off] = k.to(s["k"].dtype), v.to(s["v"].dtype)
        return {"q": q, "k": s["k"], "v": s["v"]}
    (ck, ek), (cv, ev) = _quantized(k), _quantized(v)
    s["k"].view(torch.uint8)[at, :, off], s["v"].view(torch.uint8)[at, :, off] = ck.view(torch.uint8), cv.view(torch.uint8)
    s["k_exp"][at, :, off], s["v_exp"][at, :, off] = ek, ev
    return {"q": q, **_read(s)}


def _read(s):
    row = torch.arange(s["total"], device=DEV)
    cu = s["cu_kv"].long()
    seq = torch.searchsorted(cu, row, right=True) - 1
    to = DTYPES[s["case"]["dtype"]]
    return {name: _rows(s[name], s[name + "_exp"], s["table"], seq, row - cu[seq], s["case"]["page"]).to(to) for name in ("k", "v")}


def _attend(q, k, v, news, lens):
    """q [S, N, H, D], k and v [S, L, kv_heads, D] in float32, sequences padded to the longest: token i of n stands at
    position len - n + i and sees what is up to there."""
    s, n, h, d = q.shape
    kv, l = k.shape[2], k.shape[1]
    last = lens[:, None] - news[:, None] + torch.arange(n, device=DEV)                       # [S, N]
    seen = torch.arange(l, device=DEV) <= last[..., None]                                    # [S, N, L]
    there = (torch.arange(l, device=DEV) < lens[:, None])[..., None, None]                   # [S, L, 1, 1]
    q = (q / math.sqrt(d)).view(s, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(s, kv, -1, d)    # [S, kv, group * N, D]
    score = (q @ torch.where(there, k, 0).permute(0, 2, 3, 1)).view(s, h, n, l)
    score.masked_fill_(~seen[:, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = score.sum(-1)
    out = score.view(s, kv, -1, l) @ torch.where(there, v, 0).permute(0, 2, 1, 3)            # [S, kv, group * N, D]
    out = out.view(s, h, n, d) / torch.where(total > 0, total, 1)[..., None]
    return out.permute(0, 2, 1, 3)                                                           # [S, N, H, D]


def _prompt(s):
    c = s["case"]
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].view(-1, h + 2 * kv, d)
    cu = s["cu_q"].long()
    news = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + torch.arange(s["longest"][0], device=DEV)).clamp_max(x.shape[0] - 1)
    x = x[at].float()
    out = _attend(x[:, :, :h], x[:, :, h: h + kv], x[:, :, h + kv:], news, news)
    seq, pos = _where(s)
    return out[seq, pos].to(s["qkv"].dtype)


def _paged(s):
    cu = s["cu_q"].long() if s["cu_q"] is not None else torch.arange(s["q"].shape[0] + 1, device=DEV)
    news, lens = cu[1:] - cu[:-1], s["kv_lens"].long()
    pos = torch.arange(s["longest"][1], device=DEV)
    seqs = torch.arange(lens.shape[0], device=DEV)[:, None]
    pos = torch.minimum(pos, lens[:, None] - 1)
    k, v = (_rows(s[name], s[name + "_exp"], s["table"], seqs, pos, s["case"]["page"]) for name in ("k", "v"))
    at = (cu[:-1, None] + torch.arange(s["longest"][0], device=DEV)).clamp_max(s["q"].shape[0] - 1)
    out = _attend(s["q"][at].float(), k, v, news, lens)
    row = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(cu, row, right=True) - 1
    return out[seq, row - cu[seq]].to(s["q"].dtype)


def run(s):
    c = s["case"]
    if not own:
        return {"append": _append, "read": _read, "prompt": _prompt, "paged": _paged}[c["op"]](s)
    from metaljax_b200 import attention
    if c["op"] == "prompt":
        x = s["qkv"].view(-1, c["heads"] + 2 * c["kv_heads"], c["dim"])
        q, k, v = x.split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)
        return attention.prompt_attention(q, k, v, s["cu_q"])
    cache = attention.PagedCache(s["k"], s["v"], s["k_exp"], s["v_exp"])
    if c["op"] == "paged":
        return attention.paged_attention(s["q"], cache, s["table"], s["kv_lens"], s["cu_q"])
    back = None
    if c["op"] == "append":
        q = attention.append(s["qkv"], cache, s["table"], s["kv_lens"], s["cu_q"], heads=c["heads"], freqs=s["freqs"], interleaved=c["interleaved"],
                             q_norm=s["norms"][0], k_norm=s["norms"][1], eps=EPS)
        if s["k_exp"] is None:
            return {"q": q, "k": s["k"], "v": s["v"]}
        back = {"q": q}
    k, v = attention.read_pages(cache, s["table"], s["cu_kv"], s["total"], dtype=DTYPES[c["dtype"]])
    return {**(back or {}), "k": k, "v": v}


# ---- from the definitions, in 64 bits ------------------------------------------------------


def _exact_head(q, k, v, first):
    """softmax(q k^T / sqrt(D)) v of one head's rows; row i sees positions up to first + i."""
    score = q @ k.T / math.sqrt(q.shape[1])
    score += torch.full_like(score, float("-inf")).triu(first + 1)
    return torch.softmax(score, dim=-1) @ v


def _exact_dequantized(codes, exps):
    return codes.double() * torch.exp2(exps.double() - 127)[..., None]


def _exact_quantized(x):
    """Rows of x as an 8-bit cache holds them: the values, in steps of e4m3 (3 bits behind the first, from 2^-9 on) under the row's power of two."""
    big = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp(big, min=1e-300) / 448)).clamp(-117, 119)
    e = torch.where(big > 0, e, torch.zeros_like(e))
    y = x / torch.exp2(e)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(y.abs(), min=1e-300))), min=-6) - 3)
    return torch.round(y / step) * step * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    news, lens = _plan(case)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    group = h // kv
    if case["op"] != "prompt":
        pages = [s["table"][i, : -(-l // page)].long() for i, l in enumerate(lens)]

        def held(name, i):                                         # [kv_heads, len, D] of sequence i
            x = s[name][pages[i]]
            x = x.double() if s[name + "_exp"] is None else _exact_dequantized(x, s[name + "_exp"][pages[i]])
            return x.transpose(0, 1).reshape(kv, -1, d)[:, : lens[i]]
    if case["op"] == "read":
        return {name: torch.cat([held(name, i).transpose(0, 1) for i in range(len(lens))]) for name in ("k", "v")}
    at, outs = 0, []
    if case["op"] == "append":
        k_out, v_out = (None, None) if s["k_exp"] is not None else (s["k"].double(), s["v"].double())
        ks, vs = [], []
        for i, (n, l) in enumerate(zip(news, lens)):
            x = s["qkv"][at: at + n].double().view(n, h + 2 * kv, d)
            parts = [x[:, :h], x[:, h: h + kv]]
            for j in range(2):
                y = parts[j]
                if s["norms"][j] is not None:
                    y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / d + EPS) * s["norms"][j].double()
                turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                                   torch.outer(torch.arange(l - n, l, dtype=torch.float64, device=DEV), s["freqs"]))[:, None]
                rd = case["rotary"]
                z = y[..., :rd].unflatten(-1, (rd // 2, 2)) if case["interleaved"] else y[..., :rd].unflatten(-1, (2, rd // 2)).transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
                z = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
                parts[j] = torch.cat([z, y[..., rd:]], dim=-1)
            outs.append(parts[0])
            v = x[:, h + kv:]
            if k_out is None:
                ks.append(_exact_quantized(parts[1]))
                vs.append(_exact_quantized(v))
            else:
                pos = torch.arange(l - n, l, device=DEV)
                k_out[pages[i][pos // page], :, pos % page] = parts[1]
                v_out[pages[i][pos // page], :, pos % page] = v
            at += n
        return {"q": torch.cat(outs), "k": torch.cat(ks) if k_out is None else k_out, "v": torch.cat(vs) if v_out is None else v_out}
    for i, (n, l) in enumerate(zip(news, lens)):
        if case["op"] == "prompt":
            x = s["qkv"][at: at + n].double().view(n, h + 2 * kv, d)
            q, k, v = x[:, :h], x[:, h: h + kv].transpose(0, 1), x[:, h + kv:].transpose(0, 1)
        else:
            q, k, v = s["q"][at: at + n].double(), held("k", i), held("v", i)
        outs.append(torch.stack([_exact_head(q[:, j], k[j // group], v[j // group], l - n) for j in range(h)], dim=1))
        at += n
    return torch.cat(outs)
