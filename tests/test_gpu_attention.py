"""Attention over prompts and pages, append and read back (needs a B200), against float64 (attention_reference.py)."""

import pytest
import torch

import attention_reference as R
from metaljax_b200 import _lib, attention
from metaljax_b200.attention import E4M3, PagedCache

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _device_ok():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    assert _lib.poll_status() == 0


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _table(lens, page, gen, spare=3, width=None):
    """Pages handed out in no order; entries behind a sequence's last are no pages."""
    used = [-(-n // page) for n in lens]
    pool = sum(used) + spare
    order = torch.randperm(pool, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((len(lens), width or max(max(used), 1)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, u in enumerate(used):
        table[s, :u] = order[at: at + u]
        at += u
    return table, pool


def _rows(lens, kv, dim, dtype, gen):
    return [torch.randn((n, kv, dim), generator=gen, device=DEV).to(dtype) for n in lens]


def _paged(lens, kv, dim, page, dtype, gen, fill=float("nan")):
    """A cache whose unused rows are NaN, its table, and its sequences' rows (as the values it holds)."""
    table, pool = _table(lens, page, gen)
    if dtype != E4M3:
        cache = PagedCache.empty(pool, kv, page, dim, dtype, DEV)
        cache.k.fill_(fill)
        cache.v.fill_(fill)
        k, v = _rows(lens, kv, dim, dtype, gen), _rows(lens, kv, dim, dtype, gen)
        R.filled(cache, table, lens, k, v)
        return cache, table, [x.double() for x in k], [x.double() for x in v]
    cache = PagedCache.empty(pool, kv, page, dim, E4M3, DEV)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).fill_(0x7f)
    for e in (cache.k_exp, cache.v_exp):
        e.fill_(255)
    out = ([], [])
    for s, n in enumerate(lens):
        pos = torch.arange(n, device=DEV)
        at, off = table[s].long()[pos // page], pos % page
        for codes, exps, values in ((cache.k, cache.k_exp, out[0]), (cache.v, cache.v_exp, out[1])):
            x = torch.randn((n, kv, dim), generator=gen, device=DEV)
            x = x * torch.exp2(torch.randint(-3, 3, (n, kv, 1), generator=gen, device=DEV).float())
            c, e = R.quantize(x)
            codes.view(torch.uint8)[at, :, off], exps[at, :, off] = c.view(torch.uint8), e
            values.append(R.dequantized(c, e))
    return cache, table, *out


def _check_paged(news, lens, heads, kv, dim, page, dtype, cache_dtype, *, causal=True, scale=None, seed=0, cu=True, strided=False):
    gen = _gen(seed)
    cache, table, ks, vs = _paged(lens, kv, dim, page, cache_dtype, gen)
    t = sum(news)
    wide = torch.randn((t + 3, heads + 2, dim), generator=gen, device=DEV).to(dtype)
    q = wide[:t, :heads] if strided else wide[:t, :heads].contiguous()
    out = torch.full((t + 3, heads, dim), 7.0, dtype=dtype, device=DEV)
    if not cu:
        out = out[:t]
    q_in = torch.cat([q, wide[t:, :heads]]) if cu else q                # rows behind the last sequence
    if strided and cu:
        q_in = wide[:, :heads]
    got = attention.paged_attention(q_in, cache, table, R.lengths(lens, DEV), R.starts(news, DEV) if cu else None, causal=causal, scale=scale, out=out)
    assert got is out
    at = 0
    sc = dim ** -0.5 if scale is None else scale
    for s, (n, l) in enumerate(zip(news, lens)):
        rows = q[at: at + n].double()
        want, size = (R.attend_fast if l >= n > 0 and l > 0 else R.attend)(rows, ks[s], vs[s], l - n, causal, sc)
        R.close(got[at: at + n], want, size, dtype, products=16.0 * max(1.0, sc * dim ** 0.5))
        at += n
    assert bool((out[t:] == 7.0).all()), "rows behind the last sequence were written"


CACHES = [(BF, BF), (F16, F16), (BF, E4M3)]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype, cache", CACHES)
@pytest.mark.parametrize("group, kv", [(1, 3), (4, 2), (7, 1), (16, 1), (24, 1)])
def test_one_token_each(dim, dtype, cache, group, kv):
    lens = [1, 15, 16, 17, 63, 64, 65, 200, 1000]
    _check_paged([1] * len(lens), lens, group * kv, kv, dim, 32, dtype, cache, cu=False, seed=group)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype, cache", CACHES)
@pytest.mark.parametrize("group, kv", [(1, 4), (3, 6), (16, 4), (5, 9)])
@pytest.mark.parametrize("longest", [60, 640, 8193])
def test_one_token_however_sequences_are_shared(dim, dtype, cache, group, kv, longest):
    """Clusters of eight CTAs, of four, and shares by weight; CTAs without positions among them."""
    lens = [longest, 0, 1, 59, 57, 3, 16, 33, longest // 3]
    _check_paged([1] * len(lens), lens, group * kv, kv, dim, 64, dtype, cache, cu=False, seed=kv)


@pytest.mark.parametrize("dtype, cache", CACHES)
@pytest.mark.parametrize("group, kv", [(2, 1), (5, 2), (7, 6)])
@pytest.mark.parametrize("news", [[1, 1, 0, 3, 1, 2], [5] * 9, [1, 12, 0, 1, 1, 1, 1], [9, 40, 1]])
@pytest.mark.parametrize("longest", [41, 700, 8200])
def test_few_tokens_however_sequences_are_shared(dtype, cache, group, kv, news, longest):
    """Tiles of 16, 32 and 64 rows; sequences of none, of one and of many; CTAs without positions; positions that only some rows see."""
    lens = [max(n, (longest * (3 + 5 * i % 7)) // 9 if i else longest) for i, n in enumerate(news)]
    _check_paged(news, lens, group * kv, kv, 128, 64, dtype, cache, seed=kv + len(news), strided=kv == 2)


@pytest.mark.parametrize("at", [0, 299, 300, 700])
def test_infinite_values_and_scores_of_one_token(at):
    """In a row's sum, on whichever CTA: +inf, NaN, both infinities; keys whose scores are -inf have no weight; none else: no softmax."""
    gen = _gen(at)
    lens = [701] * 4
    cache, table, ks, vs = _paged(lens, 1, 128, 64, BF, gen)
    page, off = table.long()[:, at // 64], at % 64
    cache.v[page[0], 0, off, 5] = torch.inf
    cache.v[page[1], 0, off, 5] = torch.nan
    cache.v[page[1], 0, off, 6] = torch.inf
    other = table.long()[1, (700 - at) // 64]
    cache.v[other, 0, (700 - at) % 64, 6] = -torch.inf
    cache.k[table[2].long(), :, :, 0] = -torch.inf
    cache.k[page[2], 0, off, 0] = 0.0
    cache.k[table[3].long(), :, :, 0] = -torch.inf
    q = torch.randn((4, 2, 128), generator=gen, device=DEV).to(BF)
    q[:, :, 0] = 1.0
    got = attention.paged_attention(q, cache, table, R.lengths(lens, DEV))
    for s in range(2):
        want, size = R.attend(q[s: s + 1].double(), ks[s], vs[s], 700, True, 128 ** -0.5)
        keep = torch.ones(128, dtype=torch.bool, device=DEV)
        keep[5:7] = False
        R.close(got[s: s + 1, :, keep], want[..., keep], size[..., keep], BF)
    assert bool((got[0, :, 5] == torch.inf).all()) and bool(got[1, :, 5].isnan().all())
    if at != 700 - at:
        assert bool(got[1, :, 6].isnan().all())
    assert torch.equal(got[2], vs[2][at].to(BF).expand(2, -1))
    assert bool(got[3].isnan().all())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("dtype, cache", CACHES)
def test_pages_of_every_size(page, dtype, cache):
    _check_paged([1, 5, 40], [page * 3, page * 2 - 1, page + 41], 8, 2, 128, page, dtype, cache, seed=page)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype, cache", CACHES)
@pytest.mark.parametrize("news, extra", [([5] * 6, 300), ([1, 2, 3, 17, 33], 77), ([130, 1, 64, 65], 0), ([300], 1000), ([0, 4, 0, 0, 9, 0], 50)])
@pytest.mark.parametrize("group, kv", [(1, 2), (4, 2), (6, 1)])
def test_chunks(dim, dtype, cache, news, extra, group, kv):
    lens = [n + extra + 13 * i for i, n in enumerate(news)]
    _check_paged(news, lens, group * kv, kv, dim, 64, dtype, cache, seed=len(news), strided=dim == 64)


@pytest.mark.parametrize("dtype, cache", CACHES)
def test_all_positions_seen(dtype, cache):
    _check_paged([4, 70], [90, 200], 4, 1, 128, 16, dtype, cache, causal=False, scale=0.3)


def test_rows_that_see_nothing_are_zero():
    """Sequences of no positions, and ones shorter than their new tokens (the first of which then stand before position 0)."""
    _check_paged([1, 3, 70, 2], [0, 0, 30, 2], 8, 2, 64, 16, BF, BF)
    _check_paged([1, 3, 70, 2], [0, 0, 30, 2], 8, 2, 128, 16, BF, E4M3, causal=False)
    _check_paged([1, 1], [0, 5], 4, 4, 128, 16, F16, F16, cu=False)


def test_many_sequences():
    """More than a warp's lanes, some without tokens."""
    news = [(i * 7) % 5 for i in range(150)]
    lens = [n + (i * 37) % 200 for i, n in enumerate(news)]
    _check_paged(news, lens, 4, 2, 64, 16, BF, BF)


def test_long_cache():
    _check_paged([1, 1, 1], [70000, 3, 20000], 8, 2, 128, 256, BF, E4M3, cu=False)
    _check_paged([64], [30000], 8, 2, 128, 128, BF, BF)


@pytest.mark.parametrize("page", [16, 128])
def test_a_chunk_of_a_long_prompt(page):
    """Thousands of blocks a CTA on the tensor-core kernel, whose roles must not lap one another."""
    gen = _gen(8)
    heads, kv, dim, new, length = 32, 8, 128, 1024, 32768
    cache, table, ks, vs = _paged([length], kv, dim, page, BF, gen)
    q = torch.randn((new, heads, dim), generator=gen, device=DEV).to(BF)
    for _ in range(4):
        got = attention.paged_attention(q, cache, table, R.lengths([length], DEV), R.starts([new], DEV))
    at = torch.tensor([0, 1, 63, 64, 500, 1023], device=DEV)
    for i in at.tolist():
        want, size = R.attend_fast(q[i: i + 1].double(), ks[0][: length - new + i + 1], vs[0][: length - new + i + 1], length - new + i, True, dim ** -0.5)
        R.close(got[i: i + 1], want, size, BF)


def test_calls_one_behind_the_other():
    """Hundreds of calls with nothing between them, so that the copies of keys and values are late now and then: no role of the kernel may take one
    of them for another (a wait that ran out would be reported)."""
    gen = _gen(9)
    heads, kv, dim, n = 32, 8, 128, 4096
    x = torch.randn((n, heads + 2 * kv, dim), generator=gen, device=DEV).to(BF)
    q, k, v = x.split([heads, kv, kv], dim=1)
    cu = R.starts([n], DEV)
    first = attention.prompt_attention(q, k, v, cu)
    outs = [attention.prompt_attention(q, k, v, cu) for _ in range(500)][::50]
    assert all(torch.equal(o, first) for o in outs)
    want, size = R.attend_fast(*(y[:600].double() for y in (q, k, v)), 0, True, dim ** -0.5)
    R.close(first[:600], want, size, BF)


def test_offsets_beyond_32_bits():
    """A sequence in the last pages of a cache of 4.6 GB a side."""
    gen = _gen(5)
    page, kv, dim, pages = 256, 8, 128, 8800                    # 8800 * 8 * 256 rows of 256 bytes
    cache = PagedCache.empty(pages, kv, page, dim, BF, DEV)
    table = torch.tensor([[pages - 1, pages - 5]], dtype=torch.int32, device=DEV)
    k, v = _rows([300], kv, dim, BF, gen), _rows([300], kv, dim, BF, gen)
    R.filled(cache, table, [300], k, v)
    q = torch.randn((1, 16, dim), generator=gen, device=DEV).to(BF)
    got = attention.paged_attention(q, cache, table, R.lengths([300], DEV))
    want, size = R.attend_fast(q.double(), k[0].double(), v[0].double(), 299, True, dim ** -0.5)
    R.close(got, want, size, BF)
    rk, rv = attention.read_pages(cache, table, R.starts([300], DEV), 300)
    assert torch.equal(rk, k[0]) and torch.equal(rv, v[0])


# ---- prompts ----


def _check_prompt(news, heads, kv, dim, dtype, *, causal=True, seed=0, fused=True, scale=None):
    gen = _gen(seed)
    t = sum(news) + 5
    x = torch.randn((t, heads + 2 * kv, dim), generator=gen, device=DEV).to(dtype)
    q, k, v = x.split([heads, kv, kv], dim=1)
    x[sum(news):] = float("nan")                                # tokens of no sequence
    if not fused:
        q, k, v = (y.transpose(0, 1).contiguous().transpose(0, 1) for y in (q, k, v))       # heads first
    out = torch.full((t, heads, dim), 7.0, dtype=dtype, device=DEV)
    attention.prompt_attention(q, k, v, R.starts(news, DEV), causal=causal, out=out, scale=scale)
    at = 0
    for n in news:
        if n:
            sc = dim ** -0.5 if scale is None else scale
            want, size = R.attend_fast(*(y[at: at + n].double() for y in (q, k, v)), 0, causal, sc)
            R.close(out[at: at + n], want, size, dtype, products=16.0 * max(1.0, sc * dim ** 0.5))
        at += n
    assert bool((out[at:] == 7.0).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads, kv", [(3, 3), (8, 2), (7, 1)])
def test_prompts(dim, dtype, causal, heads, kv):
    _check_prompt([1, 2, 63, 64, 65, 0, 127, 128, 129, 300], heads, kv, dim, dtype, causal=causal, fused=heads != 7)


@pytest.mark.parametrize("news", [[1], [1000], [2049, 511], [31] * 40])
def test_prompts_of_other_lengths(news):
    _check_prompt(news, 4, 1, 128, BF, seed=len(news))
    _check_prompt(news, 4, 2, 64, F16, seed=len(news), scale=0.2)


@pytest.mark.parametrize("dim", [64, 128])
def test_large_scores(dim):
    """Scores of hundreds, where all but a few weights vanish."""
    _check_prompt([400, 90], 4, 2, dim, F16, scale=4.0)


@pytest.mark.parametrize("sharp", [False, True])
def test_scores_that_rise(sharp):
    """Every next position's score is higher, so that the running maximum moves all the time."""
    n, h, dim = 700, 2, 128
    gen = _gen(3)
    q = torch.full((n, h, dim), 1.0, device=DEV).to(BF)
    k = (torch.arange(n, device=DEV, dtype=torch.float32)[:, None, None] / (8 if sharp else 128)).expand(n, h, dim).to(BF).contiguous()
    v = torch.randn((n, h, dim), generator=gen, device=DEV).to(BF)
    got = attention.prompt_attention(q, k, v, R.starts([n], DEV), causal=True, scale=1.0 / dim)
    want, size = R.attend_fast(q.double(), k.double(), v.double(), 0, True, 1.0 / dim)
    R.close(got, want, size, BF, products=k.abs().max().item())           # (128 products of 1 and k, over 128)


# ---- what stands at masked positions ----


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_masked_positions_have_no_influence(dim, dtype):
    """Infinities and NaN in keys and values: rows before them are as if they were not there, rows after them are what sums make of them."""
    gen = _gen(11)
    n, heads, kv = 150, 4, 2
    x = torch.randn((2 * n, heads + 2 * kv, dim), generator=gen, device=DEV).to(dtype)
    q, k, v = x.split([heads, kv, kv], dim=1)
    v[40, 0, 3], v[77, 1, 5], v[101, 0, 3], v[20, 1, 9], v[149, 1, 0] = float("nan"), float("inf"), float("inf"), float("-inf"), float("nan")
    v[120, 1, 9] = float("inf")                                  # meets an infinity of the other sign
    k[130, 0, 7] = float("nan")
    x[n:] = float("nan")                                         # the other sequence
    got = attention.prompt_attention(q, k, v, R.starts([n, n], DEV))
    want, size = R.attend(q[:n].double(), k[:n].double(), v[:n].double(), 0, True, dim ** -0.5)
    R.close(got[:n], want, size.nan_to_num(0, 0, 0), dtype)
    assert bool(torch.isnan(got[n:]).all())


@pytest.mark.parametrize("news", [[3], [50], [200]])
@pytest.mark.parametrize("group", [1, 4])
def test_masked_positions_of_a_cache(news, group):
    gen = _gen(12)
    lens, kv, dim = [news[0] + 100], 2, 128
    cache, table, ks, vs = _paged(lens, kv, dim, 64, BF, gen)
    for pos, head, d, x in ((lens[0] - 1, 0, 5, "nan"), (lens[0] - 2, 1, 6, "inf"), (lens[0] - 3, 0, 7, "-inf")):
        vs[0][pos, head, d] = float(x)
        cache.v[table[0, pos // 64].long(), head, pos % 64, d] = float(x)
    q = torch.randn((news[0], group * kv, dim), generator=gen, device=DEV).to(BF)
    got = attention.paged_attention(q, cache, table, R.lengths(lens, DEV), R.starts(news, DEV))
    want, size = R.attend(q.double(), ks[0], vs[0], lens[0] - news[0], True, dim ** -0.5)
    R.close(got, want, size.nan_to_num(0, 0, 0), BF)


def test_e4m3_rows_that_are_no_numbers():
    gen = _gen(13)
    cache, table, ks, vs = _paged([120], 1, 128, 32, E4M3, gen)
    for pos, exps, values in ((100, cache.v_exp, vs), (110, cache.k_exp, ks)):
        exps[table[0, pos // 32].long(), 0, pos % 32] = 255
        values[0][pos] = float("nan")
    q = torch.randn((40, 2, 128), generator=gen, device=DEV).to(BF)
    got = attention.paged_attention(q, cache, table, R.lengths([120], DEV), R.starts([40], DEV))
    want, size = R.attend(q.double(), ks[0], vs[0], 80, True, 128 ** -0.5)
    R.close(got, want, size.nan_to_num(0, 0, 0), BF)


def test_e4m3_values_of_every_size():
    """Rows under powers of two from the smallest to the largest, subnormal codes among them: the sums are those of the values."""
    gen = _gen(14)
    lens = [64]
    cache, table, ks, vs = _paged(lens, 1, 64, 64, E4M3, gen)
    page = int(table[0, 0])
    codes = torch.arange(64 * 64, device=DEV).reshape(64, 64) % 256
    codes = torch.where(codes % 128 == 127, torch.zeros_like(codes), codes).to(torch.uint8)
    cache.v.view(torch.uint8)[page, 0] = codes
    cache.k.view(torch.uint8)[page, 0].zero_()
    for byte in (11, 60, 127, 134, 135, 200, 240):
        cache.v_exp[page, 0] = byte
        cache.k_exp[page, 0] = byte
        want = R.dequantized(cache.v[page, 0], cache.v_exp[page, 0])
        rk, rv = attention.read_pages(cache, table, R.starts(lens, DEV), 64)
        assert torch.equal(rv[:, 0].double(), want) and bool((rk == 0).all())
        q = torch.randn((1, 1, 64), generator=gen, device=DEV).to(BF)
        got = attention.paged_attention(q, cache, table, R.lengths(lens, DEV))         # all keys are zero: the mean of the values
        R.close(got[0], want.mean(0, keepdim=True), want.abs().mean(0, keepdim=True), BF)


@pytest.mark.parametrize("heads", [4, 16])
@pytest.mark.parametrize("spread", [3, 8, 40])
def test_e4m3_rows_of_very_different_sizes(heads, spread):
    """Powers of two that differ between the rows of a sequence, growing along it, falling, and in no order: none loses bits beside the others."""
    gen = _gen(15)
    lens = [333, 333, 333, 1000]
    cache, table, ks, vs = _paged(lens, 1, 128, 32, E4M3, gen)
    for s, n in enumerate(lens):
        pos = torch.arange(n, device=DEV)
        at, off = table[s].long()[pos // 32], pos % 32
        shift = (pos * spread // n, (n - 1 - pos) * spread // n, torch.randint(0, spread, (n,), generator=gen, device=DEV))[s % 3] - spread // 2
        cache.v_exp[at, 0, off] = (cache.v_exp[at, 0, off].int() + shift).to(torch.uint8)
        vs[s] = R.dequantized(cache.v[at, :, off], cache.v_exp[at, :, off])
        # keys shrink as values grow, so that scores stay in their range
        cache.k_exp[at, 0, off] = (cache.k_exp[at, 0, off].int() - (shift > 0).int() * 3).to(torch.uint8)
        ks[s] = R.dequantized(cache.k[at, :, off], cache.k_exp[at, :, off])
    q = (torch.randn((len(lens), heads, 128), generator=gen, device=DEV) * torch.exp2(torch.arange(heads, device=DEV) % 5 - 4.0)[None, :, None]).to(BF)
    got = attention.paged_attention(q, cache, table, R.lengths(lens, DEV))
    for s in range(len(lens)):
        want, size = R.attend_fast(q[s: s + 1].double(), ks[s], vs[s], lens[s] - 1, True, 128 ** -0.5)
        R.close(got[s: s + 1], want, size, BF, products=16.0 * 8)          # (keys here are up to eight times N(0, 1))


# ---- append and read back ----


def _check_append(news, lens, heads, kv, dim, page, dtype, cache_dtype, *, rotary, interleaved, norms, theta=10000.0, cu=True, seed=0):
    gen = _gen(seed)
    table, pool = _table(lens, page, gen)
    cache = PagedCache.empty(pool, kv, page, dim, cache_dtype, DEV)
    cache.k.view(torch.uint8).fill_(0x11)
    cache.v.view(torch.uint8).fill_(0x11)
    before = cache.k.view(torch.uint8).clone()
    t = sum(news)
    x = (torch.randn((t + (2 if cu else 0), heads + 2 * kv, dim), generator=gen, device=DEV) * 2).to(dtype)
    wq, wk = ((1 + 0.3 * torch.randn((dim,), generator=gen, device=DEV)).to(dtype) for _ in range(2)) if norms else (None, None)
    freqs = attention.rotary_frequencies(rotary, theta) if rotary else None
    out = torch.full((x.shape[0], heads, dim), 7.0, dtype=dtype, device=DEV)
    q = attention.append(x.view(x.shape[0], -1), cache, table, R.lengths(lens, DEV), R.starts(news, DEV) if cu else None, heads=heads, freqs=freqs,
                         interleaved=interleaved, q_norm=wq, k_norm=wk, eps=1e-5, out=out)
    assert bool((q[t:] == 7.0).all())
    pos = torch.cat([torch.arange(l - n, l, device=DEV) for n, l in zip(news, lens)])
    seq = torch.cat([torch.full((n,), s, device=DEV) for s, n in enumerate(news)])
    want = {"q": R.norm(x[:t, :heads].double(), wq, 1e-5), "k": R.norm(x[:t, heads: heads + kv].double(), wk, 1e-5), "v": x[:t, heads + kv:].double()}
    # float32: norm, two products and a sum, sine and cosine to 2e-7, half an angle's step of 2^-24 turns: 2e-6 of the pair's size is above their sum
    slack = {name: 2e-6 * (y.abs() + y.abs().amax(-1, keepdim=True)) for name, y in want.items()}
    if rotary:
        for name in ("q", "k"):
            want[name] = R.rotate(want[name], pos, freqs, interleaved)
    assert bool(((q[:t].double() - want["q"]).abs() <= slack["q"] + R.HALF_STEP[dtype] * want["q"].abs() + 1e-7).all())
    at, off = table[seq, pos // page].long(), pos % page
    for name, held, exps in (("k", cache.k, cache.k_exp), ("v", cache.v, cache.v_exp)):
        y = want[name]
        if cache_dtype != E4M3:
            assert bool(((held[at, :, off].double() - y).abs() <= (slack[name] if name == "k" else 0) + R.HALF_STEP[dtype] * y.abs() + 1e-7).all())
            continue
        e = exps[at, :, off].int() - 127
        big = y.abs().amax(-1)
        assert bool((big <= 448 * torch.exp2(e.double()) * (1 + 4e-6)).all()), "an exponent too small"
        assert bool(((big > 224 * torch.exp2(e.double()) * (1 - 4e-6)) | (big == 0)).all()), "an exponent too large"
        got = R.dequantized(held[at, :, off], exps[at, :, off])
        step = torch.exp2(e.double())[..., None]
        # half a step: 2^-4 of the value, 2^-10 of the power of two among the subnormal codes
        assert bool(((got - y).abs() <= slack[name] + torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * step) * (1 + 1e-5)).all())
    # nothing else was written
    kept = torch.ones(before.shape[:3], dtype=torch.bool, device=DEV)
    kept[at, :, off] = False
    assert torch.equal(cache.k.view(torch.uint8)[kept], before[kept])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype, cache", CACHES + [(F16, E4M3)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary, norms", [(0, False), (16, True), (48, False), (64, True)])
def test_append(dim, dtype, cache, interleaved, rotary, norms):
    _check_append([3, 1, 0, 40], [10, 1, 5, 100], 6, 2, dim, 16, dtype, cache, rotary=rotary, interleaved=interleaved, norms=norms)


@pytest.mark.parametrize("interleaved", [False, True])
def test_append_far_on(interleaved):
    """Positions of several hundred thousand, one new token each, whole heads of 128 rotated."""
    _check_append([1, 1, 1], [700001, 131072, 1], 5, 1, 128, 256, BF, BF, rotary=128, interleaved=interleaved, norms=True, theta=500000.0, cu=False)


def test_append_one_head_and_many():
    _check_append([2], [9], 1, 1, 64, 32, BF, E4M3, rotary=64, interleaved=False, norms=False)
    _check_append([2, 7], [9, 7], 70, 10, 128, 32, F16, F16, rotary=128, interleaved=False, norms=True)


def test_append_of_zeros_and_of_no_numbers():
    gen = _gen(2)
    cache = PagedCache.empty(2, 1, 16, 64, E4M3, DEV)
    x = torch.randn((4, 3, 64), generator=gen, device=DEV).to(BF)
    x[0, 1:] = 0
    x[1, 1, 5], x[2, 2, 9], x[3, 1, 0], x[3, 2, 63] = float("nan"), float("inf"), float("-inf"), float("nan")
    table, lens, cu = torch.zeros((1, 1), dtype=torch.int32, device=DEV), R.lengths([4], DEV), R.starts([4], DEV)
    attention.append(x.view(4, -1), cache, table, lens, cu, heads=1)
    assert cache.k_exp[0, 0, 0] == 127 and bool((cache.k[0, 0, 0].float() == 0).all())
    assert cache.k_exp[0, 0, :4].tolist()[1:] == [255, cache.k_exp[0, 0, 2].item(), 255] and cache.v_exp[0, 0, 2:4].tolist() == [255, 255]
    k, v = attention.read_pages(cache, table, cu, 4)
    assert bool(torch.isnan(k[1]).all() and torch.isnan(k[3]).all() and torch.isnan(v[2]).all() and torch.isfinite(k[2]).all())


@pytest.mark.parametrize("dtype", [BF, F16, E4M3])
@pytest.mark.parametrize("dim, page", [(64, 16), (128, 32), (128, 256)])
def test_read_pages(dtype, dim, page):
    gen = _gen(4)
    lens = [1, 0, 33, 300, page]
    cache, table, ks, vs = _paged(lens, 3, dim, page, dtype, gen)
    out = tuple(torch.full((sum(lens) + 2, 3, dim), 7.0, dtype=BF if dtype == E4M3 else dtype, device=DEV) for _ in range(2))
    k, v = attention.read_pages(cache, table, R.starts(lens, DEV), sum(lens) + 2, out=out)
    assert k is out[0] and bool((k[sum(lens):] == 7.0).all())
    assert torch.equal(k[: sum(lens)].double(), torch.cat(ks)) and torch.equal(v[: sum(lens)].double(), torch.cat(vs))
    if dtype == E4M3:
        k, _ = attention.read_pages(cache, table, R.starts(lens, DEV), sum(lens), dtype=F16)
        assert torch.equal(k, torch.cat(ks).to(F16))


# ---- tables and lengths that are wrong ----


def test_bad_pages_and_lengths_are_reported_and_not_followed():
    gen = _gen(6)
    cache, table, _, _ = _paged([40, 40], 1, 64, 16, BF, gen)
    q = torch.randn((2, 2, 64), generator=gen, device=DEV).to(BF)
    kept = cache.k.clone()
    for bad in (-1, cache.k.shape[0], 1 << 30):
        wrong = table.clone()
        wrong[1, 1] = bad
        good = attention.paged_attention(q, cache, table, R.lengths([40, 40], DEV))
        got = attention.paged_attention(q, cache, wrong, R.lengths([40, 40], DEV))
        assert torch.equal(got[0], good[0])
        with pytest.raises(_lib.QmmError):
            _lib.poll_status()
    for lens in ([40, 49], [40, 1 << 30], [40, -7]):
        attention.paged_attention(q, cache, table, R.lengths(lens, DEV))
        with pytest.raises(_lib.QmmError):
            _lib.poll_status()
    x = torch.randn((2, 4 * 64), generator=gen, device=DEV).to(BF)
    wrong = table.clone()
    wrong[:, 2] = cache.k.shape[0]
    for lens in ([40, 40], [49, 49], [0, -3]):
        attention.append(x, cache, wrong, R.lengths(lens, DEV), heads=2)
        with pytest.raises(_lib.QmmError):
            _lib.poll_status()
    assert torch.equal(cache.k.nan_to_num(3.0), kept.nan_to_num(3.0))
    cu = torch.tensor([0, 500, -4], dtype=torch.int32, device=DEV)
    attention.paged_attention(q, cache, table, R.lengths([40, 40], DEV), cu)
    with pytest.raises(_lib.QmmError):
        _lib.poll_status()


# ---- as they are used ----


@pytest.mark.parametrize("cache_dtype", [BF, E4M3])
@pytest.mark.parametrize("chunk", [1, 7, 64, 200])
def test_a_prompt_in_chunks_is_the_prompt(cache_dtype, chunk):
    """Two sequences appended and attended chunk by chunk: with a 16-bit cache the result is that of the whole prompts at
    once, with an e4m3 one that of the rows read back."""
    gen = _gen(21)
    news, heads, kv, dim, page = [200, 123], 8, 2, 128, 32
    freqs = attention.rotary_frequencies(dim, 10000.0)
    x = torch.randn((sum(news), (heads + 2 * kv) * dim), generator=gen, device=DEV).to(BF)
    rows = x.split(news)
    table, pool = _table(news, page, gen)
    cache = PagedCache.empty(pool, kv, page, dim, cache_dtype, DEV)
    done, outs, queries = [0, 0], [[], []], [[], []]
    while done != news:
        take = [min(chunk, n - d) for n, d in zip(news, done)]
        part = torch.cat([r[d: d + n] for r, d, n in zip(rows, done, take)])
        done = [d + n for d, n in zip(done, take)]
        lens, cu = R.lengths(done, DEV), R.starts(take, DEV)
        q = attention.append(part, cache, table, lens, cu, heads=heads, freqs=freqs)
        o = attention.paged_attention(q, cache, table, lens, cu)
        for s, (a, b) in enumerate(zip(q.split(take), o.split(take))):
            queries[s].append(a)
            outs[s].append(b)
    got, q = torch.cat(outs[0] + outs[1]), torch.cat(queries[0] + queries[1])
    k, v = attention.read_pages(cache, table, R.starts(news, DEV), sum(news))
    whole = attention.prompt_attention(q, k, v, R.starts(news, DEV))
    at = 0
    for n in news:
        want, size = R.attend_fast(*(y[at: at + n].double() for y in (q, k, v)), 0, True, dim ** -0.5)
        R.close(got[at: at + n], want, size, BF)
        R.close(whole[at: at + n], want, size, BF)
        at += n


@pytest.mark.parametrize("cache_dtype", [BF, E4M3])
def test_captured_and_replayed_with_other_lengths(cache_dtype):
    """A captured step of append and attention, replayed as the sequences grow; two graphs and an eager call in turn."""
    gen = _gen(22)
    heads, kv, dim, page, width = 8, 2, 128, 16, 8
    lens = [3, 60, 100]
    table = torch.arange(3 * width, dtype=torch.int32, device=DEV).view(3, width)
    freqs = attention.rotary_frequencies(dim)
    cache, other = (PagedCache.empty(3 * width, kv, page, dim, cache_dtype, DEV) for _ in range(2))
    for n in ("k", "v"):
        x = torch.randn(cache.k.shape, generator=gen, device=DEV)
        if cache_dtype == E4M3:
            c, e = R.quantize(x)
            getattr(cache, n).copy_(c)
            getattr(cache, n + "_exp").copy_(e)
            getattr(other, n + "_exp").copy_(e)
        else:
            getattr(cache, n).copy_(x)
        getattr(other, n).copy_(getattr(cache, n))
    x, lens_t = torch.randn((3, (heads + 2 * kv) * dim), generator=gen, device=DEV).to(BF), R.lengths(lens, DEV)

    def step(c):
        q = attention.append(x, c, table, lens_t, heads=heads, freqs=freqs)
        return attention.paged_attention(q, c, table, lens_t)

    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step(cache)
        step(other)                                              # (it writes the last positions, so the other cache gets them too)
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step(cache))
            graphs.append(g)
    torch.cuda.current_stream(DEV).wait_stream(side)
    for i in range(6):
        x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
        lens_t += 1
        want = step(other)
        graphs[i % 2].replay()
        assert torch.equal(outs[i % 2], want)
    a, b = (attention.read_pages(c, table, R.starts([9, 66, 106], DEV), 181) for c in (cache, other))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_calls_on_two_streams_at_once():
    gen = _gen(23)
    cache, table, _, _ = _paged([3000] * 4, 2, 128, 64, BF, gen)
    lens = R.lengths([3000] * 4, DEV)
    q = torch.randn((4, 16, 128), generator=gen, device=DEV).to(BF)
    want = attention.paged_attention(q, cache, table, lens)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(DEV) for _ in range(3)], []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(attention.paged_attention(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_the_same_bits_every_time():
    gen = _gen(24)
    cache, table, _, _ = _paged([5000, 17, 900], 4, 128, 64, E4M3, gen)
    q = torch.randn((3, 16, 128), generator=gen, device=DEV).to(BF)
    lens = R.lengths([5000, 17, 900], DEV)
    first = attention.paged_attention(q, cache, table, lens)
    for _ in range(5):
        assert torch.equal(attention.paged_attention(q, cache, table, lens), first)


def test_rows_that_are_not_aligned():
    """Tensors whose storage starts in the middle of 16 bytes, or whose elements are not side by side, are copied first."""
    gen = _gen(25)
    news, heads, kv, dim = [50, 9], 4, 2, 64
    flat = torch.randn((59 * 8 * dim + 1,), generator=gen, device=DEV).to(BF)
    x = flat[1:].view(59, 8, dim)
    q, k, v = x.split([heads, kv, kv], dim=1)
    cu = R.starts(news, DEV)
    want = attention.prompt_attention(*(y.contiguous() for y in (q, k, v)), cu)
    assert torch.equal(attention.prompt_attention(q, k, v, cu), want)
    turned = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in (q, k, v)]
    assert torch.equal(attention.prompt_attention(*turned, cu), want)
    table, pool = _table(news, 16, gen)
    caches = [PagedCache.empty(pool, kv, 16, dim, BF, DEV) for _ in range(2)]
    a = attention.append(x.reshape(59, -1).clone(), caches[0], table, R.lengths(news, DEV), cu, heads=heads)
    b = attention.append(x.view(59, -1), caches[1], table, R.lengths(news, DEV), cu, heads=heads)
    assert torch.equal(a, b) and all(torch.equal(m, n) for m, n in zip(*(attention.read_pages(c, table, cu, 59) for c in caches)))


@pytest.mark.parametrize("news", [[200, 90], [3, 4]])
def test_layouts_of_heads(news):
    """Heads before tokens, heads that share their rows, rows a fraction of a head apart, dimensions of one with any stride."""
    gen = _gen(31)
    t, heads, kv, dim = sum(news), 4, 2, 64
    cu = R.starts(news, DEV)
    q, k, v = (torch.randn((t, h, dim), generator=gen, device=DEV).to(BF) for h in (heads, kv, kv))
    want = attention.prompt_attention(q, k, v, cu)
    first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(attention.prompt_attention(*first, cu), want)
    padded = []
    for x in (q, k, v):
        rows = torch.full((t, x.shape[1] * dim + 8), torch.nan, dtype=BF, device=DEV)
        rows[:, :-8] = x.flatten(1)
        padded.append(rows[:, :-8].unflatten(1, (-1, dim)))
    assert torch.equal(attention.prompt_attention(*padded, cu), want)
    one = [x[:, :1] for x in (k, v)]
    shared = attention.prompt_attention(q, *(x.expand(-1, 2, -1) for x in one), cu)
    assert torch.equal(shared, attention.prompt_attention(q, *(x.expand(-1, 2, -1).contiguous() for x in one), cu))
    assert torch.equal(shared, attention.prompt_attention(q, *one, cu))
    assert torch.equal(shared, attention.prompt_attention(q, *(x.as_strided(x.shape, (x.stride(0), 8, 1)) for x in one), cu))
    last = [x[t - 1:].as_strided((1,) + tuple(x.shape[1:]), (16, dim, 1)) for x in (q, k, v)]
    assert torch.equal(attention.prompt_attention(*last, R.starts([1], DEV)), last[2].repeat_interleave(2, dim=1))


@pytest.mark.parametrize("offset", [8, 16, 24])
def test_results_at_every_alignment(offset):
    """Results, queries, keys, values and caches that begin at any multiple of 16 bytes."""
    gen = _gen(26)
    news, heads, kv, dim = [150, 9], 4, 2, 128

    def at_offset(t):
        flat = torch.empty((t.numel() + 64,), dtype=t.dtype, device=DEV)
        view = flat[offset * 2 // t.element_size():][: t.numel()].view(t.shape)
        assert view.data_ptr() % 16 == 0 and (offset % 16 == 0 or view.data_ptr() % 32 != 0)
        return view.copy_(t)

    q, k, v = (torch.randn((159, n, dim), generator=gen, device=DEV).to(BF) for n in (heads, kv, kv))
    cu = R.starts(news, DEV)
    want = attention.prompt_attention(q, k, v, cu)
    out = at_offset(torch.zeros_like(q))
    assert torch.equal(attention.prompt_attention(*(at_offset(t) for t in (q, k, v)), cu, out=out), want)
    cache, table, _, _ = _paged([200, 40], kv, dim, 32, BF, gen)
    lens = R.lengths([200, 40], DEV)
    other = PagedCache(at_offset(cache.k), at_offset(cache.v))
    for rows, starts in ((q, cu), (q[:2], None), (q[:5], R.starts([3, 2], DEV))):
        want = attention.paged_attention(rows, cache, table, lens, starts)
        assert torch.equal(attention.paged_attention(at_offset(rows), other, table, lens, starts, out=at_offset(torch.zeros_like(rows))), want)
    x = torch.randn((2, (heads + 2 * kv) * dim), generator=gen, device=DEV).to(BF)
    a = attention.append(x, cache, table, lens, heads=heads)
    assert torch.equal(attention.append(at_offset(x), other, table, lens, heads=heads, out=at_offset(torch.zeros_like(a))), a)
    cu_kv = R.starts([200, 40], DEV)
    outs = tuple(at_offset(torch.zeros((240, kv, dim), dtype=BF, device=DEV)) for _ in range(2))
    assert all(torch.equal(m, n) for m, n in zip(attention.read_pages(other, table, cu_kv, 240, out=outs), attention.read_pages(cache, table, cu_kv, 240)))


def test_no_sequences():
    cache = PagedCache.empty(1, 2, 16, 64, BF, DEV)
    none = torch.zeros((0,), dtype=torch.int32, device=DEV)
    q = torch.zeros((0, 4, 64), dtype=BF, device=DEV)
    assert attention.paged_attention(q, cache, torch.zeros((0, 1), dtype=torch.int32, device=DEV), none).shape == q.shape
    assert attention.prompt_attention(q, q[:, :2], q[:, :2], torch.zeros((1,), dtype=torch.int32, device=DEV)).shape == q.shape


@pytest.mark.parametrize("cache_dtype", [BF, E4M3])
@pytest.mark.parametrize("new", [1, 4, 40])
def test_tables_whose_rows_share_memory(cache_dtype, new):
    """Several sequences over one prefix: one row of pages expanded to all of them, rows that overlap, and the same rows written out."""
    gen = _gen(41)
    seqs, heads, kv, dim, page = 5, 8, 2, 128, 32
    cache, row, _, _ = _paged([320], kv, dim, page, cache_dtype, gen)
    lens, cu = R.lengths([320, 100, 41, 64, 57], DEV), R.starts([new] * seqs, DEV)
    flat = row[0].clone()                                          # ten pages: rows of six entries that begin one behind the other
    q = torch.randn((seqs * new, heads, dim), generator=gen, device=DEV).to(BF)
    few = R.lengths([192, 100, 41, 64, 57], DEV)
    for table, n in ((row.expand(seqs, -1), lens), (row[:, :1].expand(seqs, -1), R.lengths([32] * seqs, DEV)), (flat.as_strided((seqs, 6), (1, 1)), few)):
        whole = table.contiguous()
        assert table.stride(0) < table.shape[1] <= whole.stride(0)
        assert torch.equal(attention.paged_attention(q, cache, table, n, cu), attention.paged_attention(q, cache, whole, n, cu))
        cu_kv, total = R.starts(n.tolist(), DEV), int(n.sum())
        assert all(torch.equal(a, b) for a, b in zip(attention.read_pages(cache, table, cu_kv, total), attention.read_pages(cache, whole, cu_kv, total)))
    # appended through one row of the table: position 10 s of the pages that all sequences share
    x = torch.randn((seqs, (heads + 2 * kv) * dim), generator=gen, device=DEV).to(BF)
    at = R.lengths([10 * s + 1 for s in range(seqs)], DEV)
    caches = [PagedCache(*(t if t is None else t.clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp))) for _ in range(2)]
    a, b = (attention.append(x, c, t, at, heads=heads) for c, t in zip(caches, (row.expand(seqs, -1), row.repeat(seqs, 1))))
    assert torch.equal(a, b)
    for name in ("k", "v") + (("k_exp", "v_exp") if cache_dtype == E4M3 else ()):
        m, n = (getattr(c, name).view(torch.uint8) for c in caches)
        assert torch.equal(m, n) and not torch.equal(m, getattr(cache, name).view(torch.uint8))


# ---- e4m3 pages: heads, rows and positions have nothing to do with one another ----


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("news, heads", [([1, 1, 1], 4), ([1, 1, 1], 16), ([3, 1, 2], 4)])
@pytest.mark.parametrize("longest", [300, 9000])
def test_e4m3_heads_of_very_different_sizes(dim, news, heads, longest):
    """Queries of one head 2^45 or 2^100 above the others, far below them, of zeros or with infinities: the other heads' results are as good as
    without it, and so is its own where it has one."""
    gen = _gen(51)
    lens = [longest, 64, 77]
    cache, table, ks, vs = _paged(lens, 1, dim, 64, E4M3, gen)
    q = torch.randn((sum(news), heads, dim), generator=gen, device=DEV).to(BF)
    cu = None if max(news) == 1 else R.starts(news, DEV)
    for change in (1.0, 2.0 ** 45, 2.0 ** 100, torch.inf, 0.0, 2.0 ** -60):
        x = q.clone()
        x[:, 1] *= change
        keep = torch.ones(heads, dtype=torch.bool, device=DEV)
        keep[1] = change <= 1
        got = attention.paged_attention(x, cache, table, R.lengths(lens, DEV), cu)
        at = 0
        for s, n in enumerate(news):
            k, v = (y.expand(-1, heads, -1)[:, keep] for y in (ks[s], vs[s]))
            want, size = R.attend_fast(x[at: at + n, keep].double(), k, v, lens[s] - n, True, dim ** -0.5)
            R.close(got[at: at + n, keep], want, size, BF, products=16.0 * 8)          # (keys here are up to eight times N(0, 1))
            at += n


@pytest.mark.parametrize("byte", [140, 187, 246, 10, 255])
@pytest.mark.parametrize("news, group", [([2, 3], 4), ([4, 1], 4), ([2, 2], 1), ([7, 3], 2), ([16, 9], 1)])
@pytest.mark.parametrize("longest", [130, 2000, 9000])
def test_e4m3_positions_that_a_token_does_not_see_leave_its_bits(byte, news, group, longest):
    """The last new tokens' rows of values under other powers of two, from the least to the largest, and as no numbers: the tokens before
    them have the bits that they have without."""
    gen = _gen(52)
    lens, kv, dim = [longest, longest // 3 + 20], 2, 128
    cache, table, ks, _ = _paged(lens, kv, dim, 64, E4M3, gen)
    q = torch.randn((sum(news), group * kv, dim), generator=gen, device=DEV).to(BF)
    args = (cache, table, R.lengths(lens, DEV), R.starts(news, DEV))
    first = attention.paged_attention(q, *args)
    for back in (1, 2):
        kept = cache.v_exp.clone()
        for s, n in enumerate(lens):
            if back < news[s]:
                pos = n - back
                cache.v_exp[table[s, pos // 64].long(), 0, pos % 64] = byte
        got = attention.paged_attention(q, *args)
        vs = attention.read_pages(cache, table, R.starts(lens, DEV), sum(lens))[1].split(lens)
        cache.v_exp.copy_(kept)
        at = 0
        for s, n in enumerate(news):
            unseen = max(0, n - back) if back < n else n
            assert torch.equal(got[at: at + unseen], first[at: at + unseen])
            assert torch.equal(got[at: at + n, group:], first[at: at + n, group:])          # (the other key head)
            if unseen < n:                                           # ... and those that see them the sums of what stands there
                want, size = R.attend_fast(q[at + unseen: at + n].double(), ks[s], vs[s].double(), lens[s] - n + unseen, True, dim ** -0.5)
                R.close(got[at + unseen: at + n], want, size.nan_to_num(0, 0, 0), BF, products=16.0 * 8)
            at += n


@pytest.mark.parametrize("heads", [4, 16])
@pytest.mark.parametrize("at, span", [(0, 1), (5, 1), (150, 1), (298, 1), (0, 64), (64, 64), (192, 64)])
def test_e4m3_large_values_of_small_weight(heads, at, span):
    """Rows of values far above the others, at positions whose weights make up for it, or are nothing: their share of the sums is their weights',
    and the other rows keep theirs, whether they come before them or behind."""
    gen = _gen(53)
    # powers of two: of the other rows, of these, and (downwards) of these rows' weights
    cases = [(0, 30, 30.0), (0, 45, 44.0), (0, 60, 62.0), (0, 100, 90.0), (0, 117, 117.0), (0, 117, 124.0), (0, 117, 300.0), (0, 13, 40.0), (-60, 110, 300.0), (-100, 60, 300.0),
             (-60, 50, 112.0), (-40, 80, 118.0)]
    dim, n = 128, 300
    cache, table, ks, vs = _paged([n] * len(cases), 1, dim, 32, E4M3, gen)
    pos = torch.arange(n, device=DEV)
    here = (pos >= at) & (pos < at + span)
    for s, (base, up, _) in enumerate(cases):
        where, off = table[s].long()[pos // 32], pos % 32
        k = torch.zeros((n, 1, dim), device=DEV)                 # keys of one element, zero in the rows in question: their scores are `low` powers of two below
        k[~here, :, 0] = 8.0
        codes, exps = R.quantize(k)
        cache.k.view(torch.uint8)[where, :, off], cache.k_exp[where, :, off] = codes.view(torch.uint8), exps
        ks[s] = R.dequantized(codes, exps)
        assert torch.equal(ks[s], k.double())
        cache.v_exp[where, 0, off] = torch.where(here, torch.full_like(pos, 127 + up), cache.v_exp[where, 0, off].long() + base).to(torch.uint8)
        vs[s] = R.dequantized(cache.v[where, :, off], cache.v_exp[where, :, off])
    scale = 1.0 / 8
    q = torch.zeros((len(cases), heads, dim), device=DEV)
    q[:, :, 0] = torch.tensor([low for _, _, low in cases], device=DEV)[:, None] * 0.6875         # (about ln 2, in five bits: a score of 0.6875 * low)
    q = q.to(BF)
    got = attention.paged_attention(q, cache, table, R.lengths([n] * len(cases), DEV), scale=scale)
    for s in range(len(cases)):
        want, size = R.attend_fast(q[s: s + 1].double(), ks[s], vs[s], n - 1, True, scale)
        # (scores of one exact product, up to 207; in powers of two up to 298, a float32 with a step of 2^-15: far below the bound's part for products of 300)
        R.close(got[s: s + 1], want, size, BF, products=300.0)


@pytest.mark.parametrize("dtype, cache", CACHES)
@pytest.mark.parametrize("group, kv, dim", [(33, 2, 128), (40, 1, 64), (64, 3, 128)])
@pytest.mark.parametrize("longest", [70, 900, 9000])
def test_more_query_heads_than_two_tiles_of_16(dtype, cache, group, kv, dim, longest):
    """Up to 64 query heads a key head, one token each with and without starts, and a few."""
    lens = [longest, 1, 0, 17, longest // 2]
    for cu in (False, True):
        _check_paged([1] * len(lens), lens, group * kv, kv, dim, 32, dtype, cache, cu=cu, seed=group)
    _check_paged([3, 1, 0, 2, 5], lens[:2] + [4] + lens[3:], group * kv, kv, dim, 32, dtype, cache, seed=group)
