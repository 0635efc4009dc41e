"""What the attention entry points refuse, without a GPU: the checks come before anything is launched."""

import ctypes
import math

import pytest
import torch

from metaljax_b200 import _lib, attention
from metaljax_b200.attention import E4M3, PagedCache

BF = torch.bfloat16


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def _cache(dtype=BF, pages=4, kv=2, page=16, dim=64):
    return PagedCache.empty(pages, kv, page, dim, dtype, device="cpu")


def test_caches_that_are_none():
    k = torch.zeros(4, 2, 16, 64, dtype=BF)
    e = torch.zeros(4, 2, 16, dtype=torch.uint8)
    with pytest.raises(ValueError):
        PagedCache(k, k[:2])
    with pytest.raises(TypeError):
        PagedCache(k.float(), k.float())
    with pytest.raises(ValueError):
        PagedCache(k.transpose(1, 2), k.transpose(1, 2))
    with pytest.raises(ValueError):
        PagedCache(k, k, e, e)                                 # a 16-bit cache has no exponents
    with pytest.raises(ValueError):
        PagedCache(k.to(E4M3), k.to(E4M3))
    with pytest.raises(ValueError):
        PagedCache(k.to(E4M3), k.to(E4M3), e, e[:, :1])
    assert PagedCache(k.to(E4M3), k.to(E4M3), e, e).page_size == 16


def test_paged_attention_refuses():
    c, q, table, lens = _cache(), torch.zeros(2, 4, 64, dtype=BF), torch.zeros(2, 2, dtype=torch.int32), _ints(3, 4)
    call = attention.paged_attention
    with pytest.raises(ValueError, match="CUDA"):
        call(q, c, table, lens)
    for bad in (q.float(), q[0], torch.zeros(2, 4, 128, dtype=BF)):
        with pytest.raises(ValueError):
            call(bad, c, table, lens)
    for bad in (table.long(), table[0], table[:1], torch.zeros(2, 2, 2, dtype=torch.int32)[..., 0].t().contiguous().t()):
        with pytest.raises(ValueError):
            call(q, c, bad, lens)
    for bad in (lens.long(), lens[:1], lens[None]):
        with pytest.raises(ValueError):
            call(q, c, table, bad)
    for bad in (_ints(0, 1), _ints(0, 1, 1, 2), torch.tensor([0, 1, 2])):
        with pytest.raises(ValueError):
            call(q, c, table, lens, bad)
    with pytest.raises(ValueError):
        call(q, c, table, lens, out=torch.zeros(2, 4, 64))
    with pytest.raises(RuntimeError, match="backward"):
        call(q.clone().requires_grad_(), c, table, lens)


def test_prompt_attention_refuses():
    q, k, cu = torch.zeros(6, 4, 64, dtype=BF), torch.zeros(6, 2, 64, dtype=BF), _ints(0, 2, 6)
    call = attention.prompt_attention
    with pytest.raises(ValueError, match="CUDA"):
        call(q, k, k, cu)
    for bad in (k.half(), k[:5], k[..., :32], k[0]):
        with pytest.raises(ValueError):
            call(q, bad, bad, cu)
    with pytest.raises(ValueError):
        call(q, k, torch.zeros(6, 4, 64, dtype=BF), cu)
    with pytest.raises(ValueError):
        call(q, k, k, cu.long())
    with pytest.raises(ValueError):
        call(q, k, k, _ints()[:0])
    with pytest.raises(RuntimeError, match="backward"):
        call(q, k.clone().requires_grad_(), k, cu)


def test_append_and_read_refuse():
    c, x, table, lens = _cache(), torch.zeros(2, 8 * 64, dtype=BF), torch.zeros(2, 2, dtype=torch.int32), _ints(3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        attention.append(x, c, table, lens, heads=4)
    for bad in (x.float(), x[0], x[:, :64]):
        with pytest.raises(ValueError):
            attention.append(bad, c, table, lens, heads=4)
    for more in ({"heads": 3}, {"heads": 0}, {"heads": 4, "cu_q": _ints(0, 2)}, {"heads": 4, "q_norm": torch.ones(64)}, {"heads": 4, "k_norm": torch.ones(32, dtype=BF)},
                 {"heads": 4, "freqs": torch.ones(16)}, {"heads": 4, "out": torch.zeros(2, 4, 32, dtype=BF)}):
        with pytest.raises(ValueError):
            attention.append(x, c, table, lens, **more)
    with pytest.raises(ValueError):
        attention.append(x[:1], c, table, lens, heads=4)
    with pytest.raises(ValueError):
        attention.read_pages(c, table, _ints(0, 2), 2)
    with pytest.raises(TypeError):
        attention.read_pages(c, table, _ints(0, 1, 2), 2, dtype=torch.float32)
    with pytest.raises(ValueError, match="CUDA"):
        attention.read_pages(c, table, _ints(0, 1, 2), 2)


def _args(cache=None, **more):
    """Arguments that pass every check (the pointers are never followed: a refusal comes first)."""
    c = _lib.PagedCacheArgs()
    c.struct_size, c.elem, c.k, c.v, c.table = ctypes.sizeof(c), 0, 256, 256, 256
    c.pages, c.kv_heads, c.page_size, c.head_dim, c.table_width, c.table_stride = 4, 2, 16, 64, 2, 2
    a = _lib.AttentionArgs()
    a.struct_size, a.q, a.q_row, a.q_head, a.out = ctypes.sizeof(a), 256, 256, 64, 256
    a.tokens, a.seqs, a.heads, a.kv_heads, a.head_dim, a.causal, a.scale = 2, 2, 4, 2, 64, 1, 0.125
    a.kv_lens, a.workspace, a.workspace_bytes = 256, 256, 1 << 40
    for k, v in (cache or {}).items():
        setattr(c, k, v)
    for k, v in more.items():
        setattr(a, k, v)
    return c, a


@pytest.mark.parametrize("cache, args, status", [
    ({"struct_size": 0}, {}, 1), ({"k": None}, {}, 1), ({"table": None}, {}, 1), ({"elem": 2}, {}, 2), ({"elem": 7}, {}, 1),
    ({"head_dim": 96}, {}, 7), ({"page_size": 24}, {}, 7), ({"page_size": 8}, {}, 7), ({"page_size": 512}, {}, 7), ({"pages": 0}, {}, 3),
    ({"table_stride": 1}, {}, 3), ({"table_width": 1 << 28, "table_stride": 1 << 28}, {}, 10), ({"k": 264}, {}, 4), ({"elem": 1}, {}, 2),
    ({"elem": 7, "k_exp": 256, "v_exp": 256}, {"elem": 1}, 2), ({"kv_heads": 1}, {}, 3),
    ({}, {"struct_size": 1}, 1), ({}, {"tokens": -1}, 3), ({}, {"heads": 5}, 3), ({}, {"heads": 130}, 7), ({}, {"head_dim": 96}, 7),
    ({}, {"elem": 2}, 2), ({}, {"scale": 0.0}, 7), ({}, {"scale": -1.0}, 7), ({}, {"scale": math.nan}, 7), ({}, {"scale": math.inf}, 7),
    ({}, {"q": None}, 1), ({}, {"q": 264}, 4), ({}, {"q_row": 257}, 4), ({}, {"workspace_bytes": 16}, 10), ({}, {"workspace": 264}, 4),
    ({}, {"tokens": 3}, 3), ({}, {"kv_lens": None}, 1),
])
def test_statuses_of_paged_attention(cache, args, status):
    c, a = _args(cache, **args)
    assert _lib.lib().qmm_paged_attention(ctypes.byref(c), ctypes.byref(a), None) == status, _lib.lib().qmm_last_error()


@pytest.mark.parametrize("args, status", [
    ({"kv_lens": 256}, 7), ({"cu_q": None}, 1), ({"k": None}, 1), ({"k": 8}, 4), ({"v_row": 12}, 4), ({"heads": 3}, 3), ({"scale": -0.5}, 7),
])
def test_statuses_of_prompt_attention(args, status):
    _, a = _args(None, **{"kv_lens": None, "cu_q": 256, "k": 256, "v": 256, "k_row": 128, "k_head": 64, "v_row": 128, "v_head": 64, **args})
    assert _lib.lib().qmm_prompt_attention(ctypes.byref(a), None) == status, _lib.lib().qmm_last_error()


@pytest.mark.parametrize("args, status", [
    ({"elem": 2}, 2), ({"elem": 1}, 2), ({"tokens": 3}, 3), ({"rotary_dim": 8}, 3), ({"rotary_dim": 128}, 3), ({"rotary_dim": 32, "freqs": None}, 1),
    ({"row_stride": 500}, 4), ({"row_stride": 513}, 4), ({"qkv": 8}, 4), ({"q_norm": 8}, 4), ({"kv_lens": None}, 1), ({"heads": 0}, 3), ({"struct_size": 4}, 1),
])
def test_statuses_of_append(args, status):
    c, _ = _args()
    a = _lib.AppendArgs()
    a.struct_size, a.qkv, a.row_stride, a.q_out, a.tokens, a.seqs, a.heads = ctypes.sizeof(a), 256, 512, 256, 2, 2, 4
    a.freqs, a.kv_lens = 256, 256
    for k, v in args.items():
        setattr(a, k, v)
    assert _lib.lib().qmm_cache_append(ctypes.byref(c), ctypes.byref(a), None) == status, _lib.lib().qmm_last_error()


@pytest.mark.parametrize("args", [
    {"q_head": 32}, {"q_head": 0}, {"q_row": 0}, {"q_row": 192}, {"q_row": 264}, {"k_head": 0}, {"k_row": 64}, {"v_row": 136}, {"q_row": 64, "q_head": 128},
])
def test_heads_that_overlap_or_lie_between_steps_are_refused(args):
    """(their tensors are copied by the Python calls)"""
    _, a = _args(None, **{"kv_lens": None, "cu_q": 256, "k": 256, "v": 256, "k_row": 128, "k_head": 64, "v_row": 128, "v_head": 64, **args})
    assert _lib.lib().qmm_prompt_attention(ctypes.byref(a), None) == 4, _lib.lib().qmm_last_error()


def test_nothing_to_do_is_no_error():
    c, a = _args(None, tokens=0, seqs=0, q=None, out=None, kv_lens=None)
    assert _lib.lib().qmm_paged_attention(ctypes.byref(c), ctypes.byref(a), None) == 0
    assert _lib.lib().qmm_cache_read(ctypes.byref(c), 0, None, 0, 0, None, None, None) == 0


def test_rotary_frequencies():
    f = attention.rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and f[0] == 1.0 and abs(f[16].item() - 0.01) < 1e-15
    assert torch.allclose(attention.rotary_frequencies(64, 10000.0, factor=4.0, device="cpu"), f / 4, rtol=1e-15)
    g = attention.rotary_frequencies(64, 10000.0, factor=8.0, bands=(1.0, 4.0, 8192), device="cpu")
    waves = 8192 * f / (2 * math.pi)
    assert torch.equal(g[waves >= 4], f[waves >= 4]) and torch.allclose(g[waves <= 1], f[waves <= 1] / 8, rtol=1e-15)
    between = (waves > 1) & (waves < 4)
    assert between.any() and bool(((g < f) & (g > f / 8))[between].all())
    for bad in ((63, {}), (64, {"factor": 0.0}), (64, {"bands": (4.0, 1.0, 8192)})):
        with pytest.raises(ValueError):
            attention.rotary_frequencies(bad[0], device="cpu", **bad[1])


@pytest.mark.parametrize("table", [
    torch.tensor([[2, 0, 3]], dtype=torch.int32).expand(4, 3),                                            # one row for all sequences
    torch.arange(5, dtype=torch.int32).as_strided((2, 4), (1, 1)),                                        # rows that overlap
    torch.tensor([[2]], dtype=torch.int32).expand(3, 1),
    torch.arange(12, dtype=torch.int32).view(3, 4)[:, :2],                                                # rows further apart than they are long
    torch.arange(12, dtype=torch.int32).view(3, 4)[1:2],
])
def test_tables_as_the_kernels_read_them(table):
    """Entry i of sequence s is at s * table_stride + i, whatever the tensor's strides."""
    c = _cache()._with(table)
    assert c.table_stride >= c.table_width == table.shape[1]
    held = (table if c.table == table.data_ptr() else c.table_tensor).untyped_storage()
    last = c.table + 4 * ((table.shape[0] - 1) * c.table_stride + c.table_width)
    assert held.data_ptr() <= c.table and last <= held.data_ptr() + held.nbytes(), "entries behind the table's memory"
    at = ctypes.cast(c.table, ctypes.POINTER(ctypes.c_int32))
    assert [[at[s * c.table_stride + i] for i in range(table.shape[1])] for s in range(table.shape[0])] == table.tolist()


def test_rows_of_more_heads_than_32_bits_count_are_refused():
    """A row of qkv of heads + 2 kv_heads, counted in 64 bits: no such row fits a stride of 512."""
    c, _ = _args({"pages": 1, "kv_heads": 1 << 30})
    a = _lib.AppendArgs()
    a.struct_size, a.qkv, a.row_stride, a.q_out, a.tokens, a.seqs, a.heads = ctypes.sizeof(a), 256, 512, 256, 2, 2, 4
    a.freqs, a.kv_lens = 256, 256
    assert _lib.lib().qmm_cache_append(ctypes.byref(c), ctypes.byref(a), None) == 4, _lib.lib().qmm_last_error()
