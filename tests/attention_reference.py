"""The attention operators in float64, from their definitions, for the tests."""

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}       # of a rounding, relative


def lengths(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def starts(counts, device):
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    return lengths(at, device)


def attend(q, k, v, first, causal, scale):
    """One sequence: q [n, H, D], k and v [L, kv, D], float64; row i sees positions up to first + i (all, if not causal). Returns the
    result, zero where a row sees nothing, and sum_j p_j |v_j|, which roundings of the weights are relative to."""
    n, h, d = q.shape
    group = h // k.shape[1]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(n):
        seen = min(k.shape[0], first + i + 1) if causal else k.shape[0]
        if seen <= 0:
            continue
        kk, vv = (x[:seen].repeat_interleave(group, dim=1) for x in (k, v))
        p = torch.softmax(torch.einsum("hd,lhd->hl", q[i], kk) * scale, dim=-1)
        out[i] = torch.einsum("hl,lhd->hd", p, vv)
        size[i] = torch.einsum("hl,lhd->hd", p, vv.abs())
    return out, size


def attend_fast(q, k, v, first, causal, scale):
    """The same with whole matrices, for finite inputs of rows that all see something."""
    n, h, d = q.shape
    group = h // k.shape[1]
    kk, vv = (x.repeat_interleave(group, dim=1) for x in (k, v))
    s = torch.einsum("nhd,lhd->hnl", q, kk) * scale
    if causal:
        s = s + torch.full(s.shape[1:], float("-inf"), dtype=s.dtype, device=s.device).triu(first + 1)
    p = torch.softmax(s, dim=-1)
    return torch.einsum("hnl,lhd->nhd", p, vv), torch.einsum("hnl,lhd->nhd", p, vv.abs())


def close(got, want, size, dtype, products=16.0):
    """Within what the kernels' roundings allow: the weights of the values by half a step each, the result by half a step, and scores whose
    float32 sums of 128 products are off by up to 128 * 2^-24 * P, P = sum |q k| * scale (twice, by the weight and by the sum that it is
    divided by). P is `products`: for q, k of N(0, 1) and scale = 128 ** -0.5 its mean is 128 * 0.64 / 11.3 = 7.2, and 16 is far outside
    its spread of 0.7: 2.4e-4. It grows with the scale."""
    bound = (HALF_STEP[dtype] + 256 * 2.0 ** -24 * products) * (want.abs() + size) + 1e-30
    got = got.double()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), "finite at other places"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN at other places"
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), "infinities of another sign"
    off = ((got - want).abs() / bound)[fine]
    assert off.numel() == 0 or off.max().item() <= 1.0, f"{off.max().item():.3f} of the bound at {int(off.argmax())}"


def rotate(x, pos, freqs, interleaved):
    """x [T, heads, D] float64 with the first 2 * len(freqs) elements turned."""
    rd = 2 * freqs.shape[0]
    angle = pos.double()[:, None, None] * freqs
    c, s = torch.cos(angle), torch.sin(angle)
    out = x.clone()
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if interleaved else (x[..., : rd // 2], x[..., rd // 2: rd])
    lo, hi = a * c - b * s, b * c + a * s
    if interleaved:
        out[..., 0:rd:2], out[..., 1:rd:2] = lo, hi
    else:
        out[..., : rd // 2], out[..., rd // 2: rd] = lo, hi
    return out


def norm(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()


def dequantized(codes, exps):
    """What an e4m3 cache's rows stand for, float64."""
    x = codes.double() * torch.exp2(exps.double() - 127)[..., None]
    return torch.where(exps[..., None] == 255, torch.full_like(x, float("nan")), x)


def filled(cache, table, lens, k, v):
    """Writes rows k[s], v[s] [len, kv, D] of every sequence into a 16-bit cache by plain indexing."""
    page = cache.page_size
    for s, n in enumerate(lens):
        pos = torch.arange(n, device=cache.k.device)
        at = table[s].long()[pos // page]
        cache.k[at, :, pos % page] = k[s].to(cache.k.dtype)
        cache.v[at, :, pos % page] = v[s].to(cache.v.dtype)


def quantize(x):
    """float32 rows as an e4m3 cache holds them: codes and exponent bytes."""
    big = x.abs().amax(-1)
    m, e = torch.frexp(big)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-117, 119)
    e = torch.where(big > 0, e, torch.zeros_like(e))
    codes = torch.ldexp(x, -e[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)
