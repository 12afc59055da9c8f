"""Serving a decoder from a paged key/value cache: rotary positions, the write of a step's keys and
values, attention over the pages, copies of pages, and the host's book-keeping of them.

The operators stand between a decoder block's qkv and output projections (`linear`,
`quantized_matmul`); they follow no call of the reference, whose attention runs in MLX
(mlx-gen-sensenova/src/qwen3.rs:463, forward_cached).  One dtype (bf16, f32 or fp16) for queries, keys,
values, cache and result.  A layer's cache is a pair of tensors, with C = 16 bytes of elements,
  keys   [pages, heads, page_size/16, head_dim/C, 16, C]
  values [pages, heads, page_size/C, head_dim, C]
(cache_shapes), the operands of the matrix instructions as they lie; `cache_tokens` gives a
sequence's keys and values back in plain order.  include/mlxq.h has every operator's definition.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _lib
from ._lib import (MLXQ_ROPE_LINEAR, MLXQ_ROPE_LLAMA3, MLXQ_ROPE_NONE, MLXQ_ROPE_NTK, MLXQ_ROPE_YARN, Attention, Heads,
                   PagedBatch, PagedCacheView, RopeScaling, check)
from .ops import _bad, _dt, _need_gpu, _ptr, _stream

_ROPE = {"none": MLXQ_ROPE_NONE, "linear": MLXQ_ROPE_LINEAR, "ntk": MLXQ_ROPE_NTK, "yarn": MLXQ_ROPE_YARN,
         "llama3": MLXQ_ROPE_LLAMA3}
_BOUNDS = {"yarn": (1.0, 32.0), "llama3": (1.0, 4.0)}


class CacheBatch(NamedTuple):
    """The sequences of a step: block_tables [B, width], q_starts [B + 1] and kv_lens [B] (int32, on the
    GPU), and the longest number of new tokens and of cached tokens that the launches are planned for
    (any values give right results; where a plan sums in another order they differ in the last bits)."""
    block_tables: torch.Tensor
    q_starts: torch.Tensor
    kv_lens: torch.Tensor
    max_q: int
    max_kv: int


def _float(op, what, t):
    if t.dtype not in (torch.bfloat16, torch.float32, torch.float16):
        _bad(op, f"{what} must be bfloat16, float32 or float16, got {t.dtype}")


def _heads(op, what, t):
    """A [T, heads, D] tensor as the library reads it: its own strides where features are contiguous
    and every head starts at 16 bytes, else a copy."""
    if t.dim() != 3:
        _bad(op, f"{what} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    C = 16 // t.element_size()
    if t.numel() and (t.stride(2) != 1 or t.stride(0) % C or t.stride(1) % C or t.data_ptr() % 16):
        t = t.contiguous()
        t = t if t.data_ptr() % 16 == 0 else t.clone()
    return t, Heads(t.data_ptr(), t.shape[1], t.stride(0), t.stride(1))


def _result(op, out, like, what="out"):
    """The tensor a result goes to: new, or `out` when the library can write it."""
    if out is None:
        out = torch.empty(like.shape, dtype=like.dtype, device=like.device)
    elif (out.shape != like.shape or out.dtype != like.dtype or out.device != like.device
          or (out.numel() and (out.stride(2) != 1 or out.stride(0) % (16 // out.element_size())
                               or out.stride(1) % (16 // out.element_size()) or out.data_ptr() % 16))):
        _bad(op, f"{what} must be a {like.dtype} tensor of {tuple(like.shape)} on {like.device} with contiguous features and "
                 "heads that start at 16 bytes")
    return out, Heads(out.data_ptr(), out.shape[1], out.stride(0), out.stride(1))


def _ints(op, what, t, shape, device):
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or t.device != device:
        _bad(op, f"{what} must be an int32 tensor of {tuple(shape)} on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def _floats(op, what, t, n, device):
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != (n,) or t.device != device:
        _bad(op, f"{what} must be a float32 tensor of [{n}] on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.contiguous()


def _table(op, table, device):
    if table is None:
        return None, 0, 0
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32 or table.device != device:
        _bad(op, f"table must be a float32 tensor of [positions, rotary_dim/2, 2] on {device}")
    table = table.contiguous()
    table = table if table.data_ptr() % 16 == 0 else table.clone()
    return table, table.shape[0], 2 * table.shape[1]


def cache_shapes(pages: int, heads: int, page_size: int, head_dim: int, dtype=torch.bfloat16):
    """The shapes of a layer's key and value tensors."""
    C = 16 // torch.empty((), dtype=dtype).element_size()
    return ((pages, heads, page_size // 16, head_dim // C, 16, C), (pages, heads, page_size // C, head_dim, C))


def _cache(op, k, v):
    """The (k, v) pair of a layer, checked, as the library reads it.  It is written in place, so nothing
    is copied: each page must be contiguous (pages may be apart)."""
    _float(op, "cache", k)
    C = 16 // k.element_size()
    if k.dim() != 6 or v.dim() != 5 or k.shape[4] != 16 or k.shape[5] != C:
        _bad(op, f"k_cache must be [pages, heads, page_size/16, head_dim/{C}, 16, {C}] and v_cache [pages, heads, "
                 f"page_size/{C}, head_dim, {C}], got {tuple(k.shape)} and {tuple(v.shape)}")
    pages, heads, D, P = k.shape[0], k.shape[1], k.shape[3] * C, k.shape[2] * 16
    if tuple(v.shape) != (pages, heads, P // C, D, C) or v.dtype != k.dtype or v.device != k.device:
        _bad(op, f"v_cache must be {(pages, heads, P // C, D, C)} of {k.dtype} like k_cache, got {tuple(v.shape)} of {v.dtype}")
    for what, t in (("k_cache", k), ("v_cache", v)):
        n = 1
        for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
            if size != 1 and stride != n:
                _bad(op, f"the pages of {what} must be contiguous")
            n *= size
        if pages > 1 and t.stride(0) < n:
            _bad(op, f"the pages of {what} overlap")
    n = heads * P * D  # a single page's stride means nothing
    return PagedCacheView(k.data_ptr(), v.data_ptr(), max(k.stride(0), n), max(v.stride(0), n), pages, P, heads, D, _dt(k))


def _batch(op, batch, device):
    tables, q_starts, kv_lens, max_q, max_kv = batch
    if tables.dim() != 2 or tables.dtype != torch.int32 or tables.device != device:
        _bad(op, f"block_tables must be a 2-D int32 tensor on {device}")
    B = tables.shape[0]
    if tables.numel() and (tables.stride(1) != 1 or (B > 1 and tables.stride(0) < tables.shape[1])):
        tables = tables.contiguous()
    q_starts = _ints(op, "q_starts", q_starts, (B + 1,), device)
    kv_lens = _ints(op, "kv_lens", kv_lens, (B,), device)
    view = PagedBatch(tables.data_ptr(), q_starts.data_ptr(), kv_lens.data_ptr(), B, tables.shape[1], tables.stride(0), int(max_q),
                      int(max_kv))
    return view, (tables, q_starts, kv_lens)


# ---- rotary positions ------------------------------------------------------------------------------


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                       original_context: float = 0.0, low: float | None = None, high: float | None = None):
    """(inverse frequencies, float64 [rotary_dim/2] on the host; the factor of cos and sin).  scaling: "none",
    "linear", "ntk", "yarn" or "llama3"; low and high are the turns over original_context between which the
    last two mix (1 and 32 for yarn, 1 and 4 for llama3 unless given)."""
    if scaling not in _ROPE:
        _bad("rotary_frequencies", f"unknown scaling {scaling!r}")
    bounds = _BOUNDS.get(scaling, (0.0, 0.0))
    s = RopeScaling(_ROPE[scaling], factor, original_context, bounds[0] if low is None else low,
                    bounds[1] if high is None else high)
    out, magnitude = (ctypes.c_double * max(rotary_dim // 2, 1))(), ctypes.c_double()
    check(_lib.load().mlxq_rotary_frequencies(rotary_dim, base, ctypes.byref(s), out, ctypes.byref(magnitude)))
    return torch.tensor(list(out), dtype=torch.float64), magnitude.value


def rotary_table(positions: int, inv_freq: torch.Tensor, magnitude: float = 1.0, device="cuda"):
    """magnitude * (cos, sin) of every position and pair, float32 [positions, rotary_dim/2, 2]."""
    if inv_freq.dim() != 1 or not 1 <= inv_freq.numel() <= 128:
        _bad("rotary_table", "inv_freq must be 1-D, of 1 to 128 values")
    half = inv_freq.numel()
    f = (ctypes.c_double * half)(*inv_freq.double().tolist())
    table = torch.empty((positions, half, 2), dtype=torch.float32, device=device)
    _need_gpu(table)
    with torch.cuda.device(table.device):
        check(_lib.load().mlxq_rotary_table(f, 2 * half, magnitude, positions, _ptr(table), _stream(table.device)))
    return table


def rotary(x, positions, table, interleaved: bool = False, inverse: bool = False, out=None):
    """x [T, heads, D] with its first 2 * table.shape[1] features turned by positions [T] (int32): pairs
    (i, i + half), or neighbours when interleaved.  inverse turns back: the gradient of x from y's (as with the other
    operators, autograd records nothing by itself).  out may be x."""
    if out is None:
        y = _lib.fast().rotary(x, positions, table, interleaved, inverse)
        if y is not None:
            return y
    _float("rotary", "x", x)
    x, xv = _heads("rotary", "x", x)
    positions = _ints("rotary", "positions", positions, x.shape[:1], x.device)
    table, rows, R = _table("rotary", table, x.device)
    if not R:
        _bad("rotary", "a table is needed")
    out, ov = _result("rotary", out, x)
    _need_gpu(x)
    check(_lib.load().mlxq_rotary(ctypes.byref(xv), _dt(x), x.shape[0], x.shape[2], _ptr(positions), _ptr(table), rows, R,
                                  int(interleaved), int(inverse), ctypes.byref(ov), _stream(x.device)))
    return out


# ---- the cache -------------------------------------------------------------------------------------


def cache_append(k, v, k_cache, v_cache, batch, q=None, table=None, positions=None, interleaved: bool = False, out=None):
    """Writes a step's keys and values [T, heads, D] into the cache's pages.  With a table the keys, and q if
    given, are rotated in the same launch, by each token's place in its sequence or by positions [T].  Returns
    the rotated queries (in out, which may be q, or a new tensor), None without q."""
    if out is None:
        y = _lib.fast().cache_append(k, v, k_cache, v_cache, batch, q, table, positions, interleaved)
        if y is not None:
            return None if q is None else y
    op = "cache_append"
    cache = _cache(op, k_cache, v_cache)
    view, keep = _batch(op, batch, k_cache.device)
    ts = {}
    for what, t in (("k", k), ("v", v), ("q", q)):
        if t is None:
            continue
        if t.dtype != k_cache.dtype or t.device != k_cache.device:
            _bad(op, f"{what} must be {k_cache.dtype} on {k_cache.device}, got {t.dtype} on {t.device}")
        ts[what] = _heads(op, what, t)
        if t.shape[2] != cache.head_dim or t.shape[0] != k.shape[0] or (what != "q" and t.shape[1] != cache.heads):
            _bad(op, f"{what} {tuple(t.shape)} does not fit {k.shape[0]} tokens and a cache of {cache.heads} heads of "
                     f"{cache.head_dim}")
    table, rows, R = _table(op, table, k_cache.device)
    if positions is not None:
        positions = _ints(op, "positions", positions, k.shape[:1], k_cache.device)
    ov = None
    if q is not None:
        out, ov = _result(op, out, ts["q"][0])
    elif out is not None:
        _bad(op, "out without q")
    _need_gpu(k_cache)
    check(_lib.load().mlxq_cache_append(ctypes.byref(ts["k"][1]), ctypes.byref(ts["v"][1]), k.shape[0], ctypes.byref(cache),
                                        ctypes.byref(view), _ptr(positions), _ptr(table), rows, R, int(interleaved),
                                        ctypes.byref(ts["q"][1]) if q is not None else None,
                                        ctypes.byref(ov) if ov is not None else None, _stream(k_cache.device)))
    del keep
    return out


def paged_attention(q, k_cache, v_cache, batch, scale: float | None = None, causal: bool = True, window: int = 0,
                    softcap: float = 0.0, prefix_lens=None, alibi_slopes=None, sinks=None, out=None):
    """Attention of a step's new tokens q [T, heads, D] over their sequences' pages: [T, heads, D].

    scale: 1/sqrt(D) unless given.  A row sees the tokens up to its own (causal) or all; prefix_lens [B]
    (int32): and the sequence's first ones in any case; window: and of those only its own and the window - 1
    before.  softcap: scores are softcap * tanh(score / softcap).  alibi_slopes [heads] (f32): less slope times
    the distance.  sinks [heads] (f32): a score without a value in each softmax.  A row that sees nothing is 0."""
    if out is None:
        y = _lib.fast().paged_attention(q, k_cache, v_cache, batch, scale, causal, window, softcap, prefix_lens, alibi_slopes,
                                        sinks)
        if y is not None:
            return y
    op = "paged_attention"
    cache = _cache(op, k_cache, v_cache)
    view, keep = _batch(op, batch, k_cache.device)
    if q.dtype != k_cache.dtype or q.device != k_cache.device:
        _bad(op, f"q must be {k_cache.dtype} on {k_cache.device}, got {q.dtype} on {q.device}")
    q, qv = _heads(op, "q", q)
    T, Hq, D = q.shape
    if D != cache.head_dim or Hq == 0 or Hq % cache.heads:
        _bad(op, f"q {tuple(q.shape)} does not fit a cache of {cache.heads} heads of {cache.head_dim}")
    if prefix_lens is not None:
        prefix_lens = _ints(op, "prefix_lens", prefix_lens, (view.sequences,), q.device)
    alibi_slopes = _floats(op, "alibi_slopes", alibi_slopes, Hq, q.device)
    sinks = _floats(op, "sinks", sinks, Hq, q.device)
    opts = Attention(1.0 / math.sqrt(D) if scale is None else scale, int(causal), window, softcap, _ptr(prefix_lens),
                     _ptr(alibi_slopes), _ptr(sinks))
    out, ov = _result(op, out, q)
    _need_gpu(q)
    lib = _lib.load()
    need = lib.mlxq_paged_attention_workspace_size(T, Hq, ctypes.byref(cache), ctypes.byref(view), ctypes.byref(opts))
    ws = torch.empty((need,), dtype=torch.uint8, device=q.device) if need else None
    check(lib.mlxq_paged_attention(ctypes.byref(qv), T, ctypes.byref(cache), ctypes.byref(view), ctypes.byref(opts),
                                   ctypes.byref(ov), _ptr(ws), need, _stream(q.device)))
    del keep
    return out


def copy_pages(cache, src, dst, block_tables=None, dim: int | None = None):
    """cache[..., dst, :] = cache[..., src, :] in place, over the pages of one pool or of several at once ([planes...,
    pages, heads, ...]: every layer's keys and values, say).  dim is the dimension of the pages: by default the
    sixth from last of key pools, which have 16 tokens next to last, and the fifth from last of value pools (of a
    stack of value pools whose head_dim is 16, which looks alike, dim has to be given).  src and dst: int32, no
    page of dst also in src.  block_tables [B, width] (int32, on the GPU): entries that name a page of src then
    name its copy."""
    if dim is None:
        dim = max(cache.dim() - (6 if cache.dim() > 5 and cache.shape[-2] == 16 else 5), 0)
    if _lib.fast().copy_pages(cache, src, dst, block_tables, dim):
        return
    op = "copy_pages"
    _float(op, "cache", cache)
    if cache.dim() < 5 or not 0 <= dim < cache.dim() - 1 or not cache.is_contiguous():
        _bad(op, f"cache {tuple(cache.shape)} must be a contiguous pool of pages (cache_shapes), dim {dim} their dimension")
    _need_gpu(cache)
    n = src.numel()
    src, dst = _ints(op, "src", src, (n,), cache.device), _ints(op, "dst", dst, (n,), cache.device)
    pages = cache.shape[dim]
    page = cache.element_size() * math.prod(cache.shape[dim + 1:])
    planes = math.prod(cache.shape[:dim])
    rows = width = stride = 0
    if block_tables is not None:
        if block_tables.dim() != 2 or block_tables.dtype != torch.int32 or block_tables.device != cache.device:
            _bad(op, f"block_tables must be a 2-D int32 tensor on {cache.device}")
        rows, width = block_tables.shape
        stride = block_tables.stride(0)
        if block_tables.numel() and (block_tables.stride(1) != 1 or (rows > 1 and stride < width)):
            _bad(op, "the rows of block_tables must be contiguous")
    check(_lib.load().mlxq_cache_copy_pages(_ptr(cache), planes, pages * page, pages, page, page, _ptr(src), _ptr(dst), n,
                                            _ptr(block_tables), rows, width, stride, _stream(cache.device)))


def cache_tokens(k_cache, v_cache, pages, length: int):
    """The first `length` tokens' keys and values [length, heads, D] of a sequence that lies in `pages`."""
    at = torch.as_tensor(pages, dtype=torch.long, device=k_cache.device)
    heads = k_cache.shape[1]
    k = k_cache[at].permute(0, 2, 4, 1, 3, 5).reshape(-1, heads, k_cache.shape[3] * k_cache.shape[5])
    v = v_cache[at].permute(0, 2, 4, 1, 3).reshape(-1, heads, v_cache.shape[3])
    return k[:length], v[:length]


class PagedCache:
    """The pages of a decoder's layers and which sequence holds them.

    All layers' pools are one tensor; the host keeps each sequence's pages and every page's number of
    holders.  A step: `batch` makes room for its new tokens and returns the CacheBatch for cache_append and
    paged_attention of every layer.  fork() shares a sequence's full pages and copies its last, partly filled
    one; a page that several sequences hold is never written.  free() gives pages back; compact() moves the
    held pages to the front of the pool.  A call that fails changes nothing.  Calls on one cache are ordered on the
    current stream."""

    def __init__(self, layers: int, pages: int, heads: int, head_dim: int, page_size: int = 16, dtype=torch.bfloat16,
                 device="cuda"):
        if dtype not in (torch.bfloat16, torch.float32, torch.float16):
            _bad("PagedCache", f"dtype must be bfloat16, float32 or float16, got {dtype}")
        if layers < 1 or pages < 1 or heads < 1:
            _bad("PagedCache", f"layers={layers}, pages={pages} and heads={heads} must be positive")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            _bad("PagedCache", f"page_size {page_size} is not a power of two from 16 to 1024")
        if head_dim < 16 or head_dim % 16 or head_dim > 256:
            _bad("PagedCache", f"head_dim {head_dim} is not a multiple of 16 up to 256")
        self.page_size, self.pages = page_size, pages
        ks, self._v_shape = cache_shapes(pages, heads, page_size, head_dim, dtype)
        self.pool = torch.empty((layers, 2, *ks), dtype=dtype, device=device)
        self._free = list(range(pages - 1, -1, -1))  # the lowest is taken first
        self._holders = [0] * pages
        self._seqs = {}  # id -> (pages, length)
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def layer(self, i: int):
        """The key and value tensors of layer i."""
        return self.pool[i, 0], self.pool[i, 1].view(self._v_shape)

    def new(self) -> int:
        """An empty sequence."""
        self._seqs[self._next] = ([], 0)
        self._next += 1
        return self._next - 1

    def _of(self, op, seq):
        if seq not in self._seqs:
            _bad(op, f"no sequence {seq}")
        return self._seqs[seq]

    def length(self, seq: int) -> int:
        return self._of("PagedCache", seq)[1]

    def pages_of(self, seq: int) -> list[int]:
        return list(self._of("PagedCache", seq)[0])

    def _take(self, n):
        got = [self._free.pop() for _ in range(n)]
        for p in got:
            self._holders[p] = 1
        return got

    def _drop(self, pages):
        for p in pages:
            self._holders[p] -= 1
            if self._holders[p] == 0:
                self._free.append(p)
        self._free.sort(reverse=True)

    def batch(self, seqs, new) -> CacheBatch:
        """Room for new[i] tokens of seqs[i], and the step's CacheBatch."""
        seqs, new = list(seqs), [int(n) for n in new]
        if not seqs or len(seqs) != len(new) or min(new) < 0 or len(set(seqs)) != len(seqs):
            _bad("PagedCache.batch", "one number of new tokens is needed for each of some different sequences")
        need = []
        for s, n in zip(seqs, new):
            pages, length = self._of("PagedCache.batch", s)
            need.append(-(-(length + n) // self.page_size) - len(pages))
        if sum(need) > len(self._free):
            _bad("PagedCache.batch", f"{sum(need)} pages are needed and {len(self._free)} are free")
        got = [self._take(more) for more in need]
        held = [(self._seqs[s][0] + pages, self._seqs[s][1] + n) for s, n, pages in zip(seqs, new, got)]
        try:
            step = self._describe(held, new)
        except BaseException:
            self._drop([p for pages in got for p in pages])
            raise
        self._seqs.update(zip(seqs, held))
        return step

    def _describe(self, held, new):
        width = max(max(len(p) for p, _ in held), 1)
        rows = [p + [-1] * (width - len(p)) for p, _ in held]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        lens = [n for _, n in held]
        flat = torch.tensor([*starts, *lens, *(p for r in rows for p in r)], dtype=torch.int32).to(self.pool.device)
        B = len(held)
        return CacheBatch(flat[2 * B + 1:].view(B, width), flat[:B + 1], flat[B + 1:2 * B + 1], max(new), max(lens))

    def fork(self, seqs):
        """A new sequence for each of seqs (a list, entries may repeat) with the same tokens; the last, partly
        filled pages are copied in all layers by one launch.  Returns their ids."""
        held = [self._of("PagedCache.fork", s) for s in seqs]
        part = [n % self.page_size != 0 for _, n in held]
        if sum(part) > len(self._free):
            _bad("PagedCache.fork", f"{sum(part)} pages are needed and {len(self._free)} are free")
        src = [pages[-1] for (pages, _), copied in zip(held, part) if copied]
        dst = self._take(len(src))
        try:
            if src:
                self._copy(src, dst)
        except BaseException:
            self._drop(dst)
            raise
        ids, copies = [], iter(dst)
        for (pages, length), copied in zip(held, part):
            shared = pages[:-1] if copied else list(pages)
            for p in shared:
                self._holders[p] += 1
            ids.append(self.new())
            self._seqs[ids[-1]] = (shared + [next(copies)] if copied else shared, length)
        return ids

    def _copy(self, src, dst, tables=None):
        pair = torch.tensor([src, dst], dtype=torch.int32).to(self.pool.device)
        copy_pages(self.pool, pair[0], pair[1], tables)

    def free(self, seq: int) -> None:
        """Forgets a sequence; pages that no other holds are free again."""
        pages, _ = self._of("PagedCache.free", seq)
        del self._seqs[seq]
        self._drop(pages)

    def truncate(self, seq: int, length: int) -> None:
        """Drops a sequence's tokens from `length` on (rejected drafts).  A page cut short that other sequences
        hold too is copied, so that writing on does not reach them."""
        pages, old = self._of("PagedCache.truncate", seq)
        if not 0 <= length <= old:
            _bad("PagedCache.truncate", f"length {length} of a sequence of {old}")
        keep = -(-length // self.page_size)
        mine = pages[:keep]
        last = pages[keep:]
        if length % self.page_size and self._holders[mine[-1]] > 1:
            # The copy goes to a page that the sequence gives back, if there is one.
            copy = next((p for p in reversed(last) if self._holders[p] == 1), None)
            if copy is None and not self._free:
                _bad("PagedCache.truncate", "1 page is needed and 0 are free")
            to = self._free[-1] if copy is None else copy
            self._copy([mine[-1]], [to])
            if copy is None:
                self._take(1)
            else:
                last.remove(copy)
            last.append(mine[-1])
            mine[-1] = to
        self._drop(last)
        self._seqs[seq] = (mine, length)

    def compact(self, block_tables=None) -> int:
        """Moves the held pages to the lowest numbers, in all layers by one launch, and returns how many pages
        from the front are then in use.  block_tables: a step's tables, redirected in place."""
        used = self.pages - len(self._free)
        dst = sorted(p for p in self._free if p < used)
        src = [p for p in range(used, self.pages) if self._holders[p]]
        if src:
            self._copy(src, dst, block_tables)
            to = dict(zip(src, dst))
            for s, (pages, length) in self._seqs.items():
                self._seqs[s] = ([to.get(p, p) for p in pages], length)
            for a, b in to.items():
                self._holders[b], self._holders[a] = self._holders[a], 0
            self._free = list(range(self.pages - 1, used - 1, -1))
        return used
