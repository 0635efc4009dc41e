"""Attention of a serving loop: prompts, and new tokens over a cache in pages.

`append` takes the output of a fused q/k/v projection -- rows `[q heads | k heads | v heads]` of the new
tokens of all sequences, one behind the other --, normalises and rotates queries and keys, and writes
keys and values into a `PagedCache`; `paged_attention` attends the new tokens (one per sequence, a few,
or a chunk of a prompt) over it; `prompt_attention` attends whole prompts that are not in a cache;
`read_pages` takes rows out of a cache as values. Kernels and definitions: include/qmm_decode.h. The
reference has no counterpart of a cache in pages; its attention recognizer (src/metaljax/sdpa.py) ends in
one dense call.

Lengths and tables are int32 tensors on the device and are read by the kernels, so that nothing waits for
the host and a captured call may be replayed with other lengths. What a kernel finds wrong in them (a page
that the cache does not have, a sequence longer than its table) is reported by `_lib.poll_status` and
never followed. Calls run on the current stream of their tensors' device. Nothing here runs on the CPU.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
_CACHE_ELEM = {torch.bfloat16: 0, torch.float16: 1, E4M3: 7}


def rotary_frequencies(rotary_dim: int, theta: float = 10000.0, *, factor: float = 1.0, bands=None, device="cuda") -> torch.Tensor:
    """Radians per position of the rotary_dim / 2 pairs, float64: `theta ** (-2 i / rotary_dim)`.

    `factor` divides all of them (positions of a longer context brought into the trained range). With
    `bands = (low, high, original)` only long waves are divided: those of which fewer than `low` fit
    into `original` positions by `factor`, those of which more than `high` do not at all, and what
    lies between by a share that is linear in their number."""
    if rotary_dim < 2 or rotary_dim % 2 or not theta > 0 or not factor > 0:
        raise ValueError("rotary_frequencies: rotary_dim is even, theta and factor are positive")
    f = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    if bands is None:
        return (f / factor).to(device)
    low, high, original = bands
    if not 0 < low < high or not original > 0:
        raise ValueError("rotary_frequencies: bands are (low, high, original) with 0 < low < high")
    waves = original * f / (2 * math.pi)
    kept = ((waves - low) / (high - low)).clamp(0, 1)
    return (f * kept + f / factor * (1 - kept)).to(device)


class PagedCache:
    """Keys and values of one layer, `[pages, kv_heads, page_size, head_dim]` each, in bf16, f16 or e4m3.

    An e4m3 cache also has a byte per row (one position of one head), `[pages, kv_heads, page_size]`: the
    row's values are its codes times `2 ** (byte - 127)`, and NaN where the byte is 255. page_size is 16,
    32, 64, 128 or 256, head_dim 64 or 128. Which pages are whose is the caller's: every call takes a table
    `[sequences, pages of a sequence]`."""

    __slots__ = ("k", "v", "k_exp", "v_exp")

    def __init__(self, k, v, k_exp=None, v_exp=None):
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        if _lib.native().is_cache(k, v, k_exp, v_exp):
            return
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("PagedCache: k and v are [pages, kv_heads, page_size, head_dim] of one type and device")
        elem = _CACHE_ELEM.get(k.dtype)
        if elem is None:
            raise TypeError(f"PagedCache: {k.dtype} is none of bfloat16, float16, float8_e4m3fn")
        if not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("PagedCache: k and v have to be contiguous")
        if (elem == 7) != (k_exp is not None) or (k_exp is None) != (v_exp is None):
            raise ValueError("PagedCache: an e4m3 cache has exponent bytes, a 16-bit one has none")
        for e in (k_exp, v_exp) if k_exp is not None else ():
            if e.dtype != torch.uint8 or e.shape != k.shape[:3] or not e.is_contiguous() or e.device != k.device:
                raise ValueError("PagedCache: exponent bytes are uint8 [pages, kv_heads, page_size]")

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, dtype=torch.bfloat16, device="cuda"):
        """A cache that holds nothing yet (its memory is not cleared)."""
        shape = (pages, kv_heads, page_size, head_dim)
        kv = [torch.empty(shape, dtype=dtype, device=device) for _ in range(2)]
        exps = [torch.empty(shape[:3], dtype=torch.uint8, device=device) for _ in range(2)] if dtype == E4M3 else [None, None]
        return cls(*kv, *exps)

    page_size = property(lambda self: self.k.shape[2])
    kv_heads = property(lambda self: self.k.shape[1])
    head_dim = property(lambda self: self.k.shape[3])

    def _with(self, table):
        """The cache as a call takes it, with a table `[sequences, pages]`."""
        _index("page_table", table, self.k.device, 2)
        if table.stride(1) != 1 and table.shape[1] > 1:
            raise ValueError("page_table: a sequence's entries have to lie side by side")
        if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            table = table.contiguous()                          # (rows that share memory, as those of one expanded row do)
        c = _lib.PagedCacheArgs()
        c.struct_size, c.elem = ctypes.sizeof(c), _CACHE_ELEM[self.k.dtype]
        c.k, c.v = self.k.data_ptr(), self.v.data_ptr()
        if self.k_exp is not None:
            c.k_exp, c.v_exp = self.k_exp.data_ptr(), self.v_exp.data_ptr()
        c.pages, c.kv_heads, c.page_size, c.head_dim = self.k.shape
        c.table, c.table_width = table.data_ptr(), table.shape[1]
        c.table_stride = table.stride(0) if table.shape[0] > 1 else table.shape[1]
        c.table_tensor = table                                  # (as long as the call needs it)
        return c


def _index(name, t, device, dim):
    if t.dtype != torch.int32 or t.dim() != dim or t.device != device:
        raise ValueError(f"{name}: an int32 tensor of {dim} dimension{'s' * (dim > 1)} on {device} is wanted")
    if dim == 1 and t.numel() > 1 and t.stride(0) != 1:
        raise ValueError(f"{name}: has to be contiguous")


def _starts(name, cu, device, seqs=None):
    _index(name, cu, device, 1)
    if cu.shape[0] < 1 or (seqs is not None and cu.shape[0] != seqs + 1):
        raise ValueError(f"{name}: one more entry than there are sequences")


def _on(device):
    """The tensors' device as the current one."""
    if device.type != "cuda":
        raise ValueError(f"attention: tensors on a CUDA device are wanted, not on {device}")
    return torch.cuda.device(device)


def _heads_of(name, t, device, dtype):
    """`[tokens, heads, head_dim]` as the kernels read it (a copy, if it lies otherwise): rows of a head side by side, 16-byte steps, tokens
    a whole number of heads apart."""
    if t.dim() != 3 or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name}: [tokens, heads, head_dim] of {dtype} on {device} is wanted")
    (n, h, d), (row, head, one) = t.shape, t.stride()
    lies = (one == 1 or d == 1) and row % 8 == 0 and head % 8 == 0 and t.data_ptr() % 16 == 0 and (n == 1 or row >= d)
    if lies and h > 1:
        lies = head >= d and (n == 1 or (row >= head * h and row % head == 0))
    return t if lies else t.clone(memory_format=torch.contiguous_format)


def _output(out, like, shape):
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if out.shape != torch.Size(shape) or out.dtype != like.dtype or out.device != like.device or not out.is_contiguous():
        raise ValueError(f"out: contiguous {tuple(shape)} of {like.dtype} on {like.device} is wanted")
    return out


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("attention: there is no backward pass here; call it under torch.no_grad() or detach its inputs")


def _native(done):
    """What a native call returned: its result, or the error of its status."""
    if done.__class__ is int:
        _lib.check(done)
    return done


def append(qkv, cache: PagedCache, page_table, kv_lens, cu_q=None, *, heads: int, freqs=None, interleaved: bool = False,
           q_norm=None, k_norm=None, eps: float = 1e-6, out=None):
    """Writes the keys and values of new tokens into `cache` and returns their queries `[tokens, heads, head_dim]`.

    `qkv` `[tokens, (heads + 2 * kv_heads) * head_dim]`, bf16 or f16. `kv_lens[s]` positions are sequence s's with its
    new tokens, rows `cu_q[s]` to `cu_q[s + 1] - 1` (None: one token each). `q_norm`, `k_norm` `[head_dim]`: every
    head divided by its root mean square (plus `eps` under the root) and multiplied by them. `freqs` (float64, see
    `rotary_frequencies`): the first `2 * len(freqs)` elements rotated, pairs half of that apart, or neighbours
    (`interleaved`). float32 arithmetic with angles from float64; rounded once, to the result's type or
    the e4m3 cache's codes. Rows behind the last sequence are neither read nor written. A token before position 0 is
    reported, and not written. (The queries of f16 rows have to be made bf16 to be attended over an e4m3 cache.)"""
    done = _lib.native().append(qkv, cache.k, cache.v, cache.k_exp, cache.v_exp, page_table, kv_lens, cu_q, heads, freqs, interleaved, q_norm, k_norm, eps, out)
    if done is not None:
        return _native(done)
    # (what the native call leaves: tensors to be copied first, empty ones, and what is refused)
    _no_grad(qkv, q_norm, k_norm, out)
    if qkv.dim() != 2 or qkv.dtype not in (torch.bfloat16, torch.float16) or qkv.device != cache.k.device:
        raise ValueError("append: qkv is [tokens, (heads + 2 * kv_heads) * head_dim], bf16 or f16, on the cache's device")
    kv, d = cache.kv_heads, cache.head_dim
    if heads < 1 or qkv.shape[1] != (heads + 2 * kv) * d:
        raise ValueError(f"append: rows of {(heads + 2 * kv) * d} elements are wanted, not {qkv.shape[1]}")
    dev = qkv.device
    _index("kv_lens", kv_lens, dev, 1)
    seqs = kv_lens.shape[0]
    if page_table.shape[0] != seqs:
        raise ValueError("append: a row of page_table for every sequence")
    if cu_q is not None:
        _starts("cu_q", cu_q, dev, seqs)
    elif qkv.shape[0] != seqs:
        raise ValueError("append: without cu_q every sequence has one token")
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None and (w.shape != (d,) or w.dtype != qkv.dtype or w.device != dev):
            raise ValueError(f"append: {name} is [head_dim] of qkv's type")
    if freqs is not None and (freqs.dtype != torch.float64 or freqs.dim() != 1 or freqs.device != dev):
        raise ValueError("append: freqs is a float64 vector on qkv's device")
    if (qkv.shape[1] > 1 and qkv.stride(1) != 1) or qkv.stride(0) % 8 or qkv.stride(0) < qkv.shape[1] or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    q_norm, k_norm = (w if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0) else w.clone(memory_format=torch.contiguous_format)
                      for w in (q_norm, k_norm))
    freqs = freqs if freqs is None else freqs.contiguous()
    q = _output(out, qkv, (qkv.shape[0], heads, d))
    c = cache._with(page_table)
    a = _lib.AppendArgs()
    a.struct_size, a.elem = ctypes.sizeof(a), _lib.ELEM[qkv.dtype]
    a.qkv, a.row_stride, a.q_out = qkv.data_ptr(), qkv.stride(0), q.data_ptr()
    a.tokens, a.seqs, a.heads = qkv.shape[0], seqs, heads
    a.rotary_dim = 0 if freqs is None else 2 * freqs.shape[0]
    a.interleaved, a.eps = int(bool(interleaved)), eps
    a.freqs = None if freqs is None else freqs.data_ptr()
    a.q_norm, a.k_norm = (None if w is None else w.data_ptr() for w in (q_norm, k_norm))
    a.kv_lens, a.cu_q = kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr()
    with _on(dev):
        _lib.check(_lib.lib().qmm_cache_append(ctypes.byref(c), ctypes.byref(a), _lib.stream_ptr(qkv)))
    return q


def read_pages(cache: PagedCache, page_table, cu_kv, total: int, dtype=None, out=None):
    """`(k, v)`, `[total, kv_heads, head_dim]` each: positions 0, 1, ... of sequence s at rows `cu_kv[s]` to `cu_kv[s + 1] - 1`.

    A 16-bit cache is read as it is; an e4m3 one as bf16, which holds its values exactly (`dtype`: f16 instead, rounded,
    infinite above its range). `out`: a pair to write to. Rows from `cu_kv[-1]` on are not written."""
    if out is None and (done := _lib.native().read_pages(cache.k, cache.v, cache.k_exp, cache.v_exp, page_table, cu_kv, total, dtype)) is not None:
        return _native(done)
    dev = cache.k.device
    _starts("cu_kv", cu_kv, dev, page_table.shape[0])
    if dtype is None:
        dtype = torch.bfloat16 if cache.k.dtype == E4M3 else cache.k.dtype
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError("read_pages: values are bf16 or f16")
    shape = (int(total), cache.kv_heads, cache.head_dim)
    like = torch.empty((0,), dtype=dtype, device=dev)
    k, v = (_output(o, like, shape) for o in (out if out is not None else (None, None)))
    c = cache._with(page_table)
    with _on(dev):
        _lib.check(_lib.lib().qmm_cache_read(ctypes.byref(c), page_table.shape[0], ctypes.c_void_p(cu_kv.data_ptr()), int(total), _lib.ELEM[dtype],
                                             ctypes.c_void_p(k.data_ptr()), ctypes.c_void_p(v.data_ptr()), _lib.stream_ptr(k)))
    return k, v


def _attention_args(q, out, seqs, kv_heads, causal, scale):
    a = _lib.AttentionArgs()
    t, h, d = q.shape
    a.struct_size, a.elem = ctypes.sizeof(a), _lib.ELEM.get(q.dtype, -1)
    a.q, a.q_row, a.q_head = q.data_ptr(), q.stride(0), q.stride(1)
    a.out, a.tokens, a.seqs, a.heads, a.kv_heads, a.head_dim = out.data_ptr(), t, seqs, h, kv_heads, d
    a.causal, a.scale = int(bool(causal)), d ** -0.5 if scale is None else scale
    return a


def _run_attention(a, q, call):
    lib = _lib.lib()
    with _on(q.device):
        need = lib.qmm_attention_workspace_bytes(ctypes.byref(a))
        if need < 0:
            raise _lib.QmmError(3, lib.qmm_last_error().decode(errors="replace"))
        work = torch.empty((need,), dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = work.data_ptr(), need
        _lib.check(call(lib, _lib.stream_ptr(q)))


def prompt_attention(q, k, v, cu_seqlens, *, causal: bool = True, scale=None, out=None):
    """Attention within each of the packed sequences `cu_seqlens[s] .. cu_seqlens[s + 1] - 1`: `q` `[tokens, heads, head_dim]`,
    `k` and `v` `[tokens, kv_heads, head_dim]` (kv_heads divides heads), bf16 or f16, which may be views of one projection's
    rows. `scale`: of the scores, `head_dim ** -0.5` unless given. Returns `[tokens, heads, head_dim]`; rows that belong to no
    sequence are not written. A row sees its own sequence's positions, with `causal` up to its own, and nothing else has
    any influence on it."""
    done = _lib.native().prompt_attention(q, k, v, cu_seqlens, causal, scale, out)
    if done is not None:
        return _native(done)
    _no_grad(q, k, v, out)
    if q.dim() != 3 or q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("prompt_attention: q is [tokens, heads, head_dim], bf16 or f16")
    dev = q.device
    _starts("cu_seqlens", cu_seqlens, dev)
    q, k, v = _heads_of("q", q, dev, q.dtype), _heads_of("k", k, dev, q.dtype), _heads_of("v", v, dev, q.dtype)
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError("prompt_attention: k and v are [tokens, kv_heads, head_dim] with q's tokens and head_dim")
    out = _output(out, q, q.shape)
    a = _attention_args(q, out, cu_seqlens.shape[0] - 1, k.shape[1], causal, scale)
    a.k, a.k_row, a.k_head, a.v, a.v_row, a.v_head = k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1)
    a.cu_q = cu_seqlens.data_ptr()
    _run_attention(a, q, lambda lib, stream: lib.qmm_prompt_attention(ctypes.byref(a), stream))
    return out


def paged_attention(q, cache: PagedCache, page_table, kv_lens, cu_q=None, *, causal: bool = True, scale=None, out=None):
    """Attention of new tokens over a cache that holds them already (`append`): `q` `[tokens, heads, head_dim]`, those of sequence s
    being rows `cu_q[s]` to `cu_q[s + 1] - 1` (None: one token each) and the last ones of its `kv_lens[s]` positions. A token
    sees the positions up to its own, or (not `causal`) all of them; one that sees none (before position 0, too: nothing is
    reported) is zero. q has the cache's type, bf16 with an e4m3 cache. Returns `[tokens, heads, head_dim]`; rows that belong to
    no sequence are not written. The kernel is chosen by how many new tokens a sequence has on average: many single tokens and a long
    chunk are better made two calls."""
    done = _lib.native().paged_attention(q, cache.k, cache.v, cache.k_exp, cache.v_exp, page_table, kv_lens, cu_q, causal, scale, out)
    if done is not None:
        return _native(done)
    _no_grad(q, out)
    dev = cache.k.device
    if q.dim() != 3 or q.dtype not in (torch.bfloat16, torch.float16) or q.device != dev:
        raise ValueError("paged_attention: q is [tokens, heads, head_dim], bf16 or f16, on the cache's device")
    _index("kv_lens", kv_lens, dev, 1)
    seqs = kv_lens.shape[0]
    if page_table.shape[0] != seqs:
        raise ValueError("paged_attention: a row of page_table for every sequence")
    if cu_q is not None:
        _starts("cu_q", cu_q, dev, seqs)
    q = _heads_of("q", q, dev, q.dtype)
    out = _output(out, q, q.shape)
    c = cache._with(page_table)
    a = _attention_args(q, out, seqs, cache.kv_heads, causal, scale)
    if q.shape[2] != cache.head_dim:
        raise ValueError("paged_attention: q has another head_dim than the cache")
    a.kv_lens, a.cu_q = kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr()
    _run_attention(a, q, lambda lib, stream: lib.qmm_paged_attention(ctypes.byref(c), ctypes.byref(a), stream))
    return out
