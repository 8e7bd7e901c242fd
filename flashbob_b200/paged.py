"""A paged cache of keys and values, and attention over it: generation with the heads that `sdpa_bob` trains.

    cache = PagedCache.allocate(pages, kv_heads, page_size, head_dim)              # or bits=4
    lengths += 1                                                                   # a step: one new token per sequence
    append_kv(k, v, cache, page_table, lengths, rotary=rotary)
    out = sdpa_paged(q, cache, page_table, lengths, rotary=rotary)

Position t of sequence b lies in page page_table[b, t // page_size], row t % page_size.  `lengths` counts the positions
that are there with the call's new tokens, `counts` (default: all rows of the call) the new ones: row i of sequence b sits
at position lengths[b] - counts[b] + i in `append_kv` and in `sdpa_paged` alike.  Both live on the GPU and are never
read by the host, so a step can be captured in a CUDA graph (after one eager call on the device) and replayed as sequences grow.

A cache of 4 bits keeps a row of a head as codes 0 ... 15 (element 2 j in the low half of byte j) and fp32 (scale, zero):
value = code * scale + zero, with zero the row's minimum and scale 1/15 of its range (1 where that is nothing), fp32 throughout.  Keys
are turned and rounded to the cache's 16-bit type before they are coded.  A row with a NaN or infinity, or a range beyond fp32's,
reads as not finite.

CUDA tensors go through libbob_sm100.so (csrc/cache.cuh, csrc/paged.cuh); there is no fallback.  CPU tensors take plain
tensor operations.  Nothing here records gradients: `read_kv` brings a cached context back to contiguous keys and values,
which `sdpa_bob` takes.

What only the GPU knows is checked there.  A page table entry within a sequence's length that is no page of the cache, a
length that the table has no room for, or a count that exceeds the call's rows or (but for attention without `is_causal`)
the length raises `BobSm100Error` at the next call on that device (`BOB_SM100_CHECK_STATUS=1`: at the call itself); what it
concerns - of a page its rows, of a length or count the whole sequence, whose results are zero - is neither read nor written.
On the CPU the call raises `ValueError`.  Entries outside the reach of a sequence's rows - behind its length, before its
window - are never looked at.
"""

from __future__ import annotations

import math

import torch

from . import _native, ops
from .interface import _CUDA_DTYPES, _CUDA_HEAD_DIMS, _MAX_GROUP, _as_count, _check_scalars
from .rotary import Rotary, check_heads, check_plain_call, check_rotary, turn

__all__ = ["PagedCache", "append_kv", "read_kv", "sdpa_paged"]

_PAGE_SIZES = tuple(1 << n for n in range(4, 13))


class PagedCache:
    """The storage: k and v [pages, kv_heads, page_size, head_dim], fp16 or bf16; or uint8 [..., head_dim / 2] with k_scales
    and v_scales fp32 [pages, kv_heads, page_size, 2] and the 16-bit `dtype` of what goes in and comes out.

    Tensors may be views in another order (as [pages, page_size, kv_heads, head_dim] transposed) with unit stride in the last
    dimension, rows that start at multiples of 16 bytes (scales: 8) and no two rows in one place.
    """

    __slots__ = ("k", "v", "k_scales", "v_scales", "dtype", "bits", "_args", "_on_gpu")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, *, k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                 dtype: torch.dtype | None = None):
        for name, t in (("k", k), ("v", v)):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"{name} must be a torch.Tensor")
            if t.ndim != 4 or t.numel() == 0:
                raise ValueError(f"{name} must be [pages, kv_heads, page_size, head_dim] with positive sizes, got {tuple(t.shape)}")
            if t.requires_grad:
                raise ValueError(f"{name} must not require gradients")
        if (k_scales is None) != (v_scales is None):
            raise ValueError("k_scales and v_scales go together")
        self.bits = 16 if k_scales is None else 4
        if dtype is None and self.bits == 16:
            dtype = k.dtype
        if dtype not in _CUDA_DTYPES:
            raise TypeError(f"dtype must be one of {', '.join(map(str, _CUDA_DTYPES))}; got {dtype}")
        if k.shape != v.shape or k.device != v.device:
            raise ValueError(f"k and v must share shape and device, got {tuple(k.shape)} {k.device} and {tuple(v.shape)} {v.device}")
        stored = dtype if self.bits == 16 else torch.uint8
        if k.dtype != stored or v.dtype != stored:
            raise TypeError(f"k and v of a {self.bits}-bit {dtype} cache must be {stored}, got {k.dtype} and {v.dtype}")
        head_dim = k.shape[3] * (1 if self.bits == 16 else 2)
        if head_dim not in _CUDA_HEAD_DIMS:
            raise ValueError(f"head dimension must be one of {_CUDA_HEAD_DIMS}, got {head_dim}")
        if k.shape[2] not in _PAGE_SIZES:
            raise ValueError(f"page size must be a power of two from {_PAGE_SIZES[0]} to {_PAGE_SIZES[-1]}, got {k.shape[2]}")
        checked = [("k", k, 16), ("v", v, 16)]
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            if t is None:
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != torch.float32:
                raise TypeError(f"{name} must be a float32 torch.Tensor")
            if t.shape != (*k.shape[:3], 2) or t.device != k.device or t.requires_grad:
                raise ValueError(f"{name} must be {(*k.shape[:3], 2)} on {k.device} without gradients, got {tuple(t.shape)} on {t.device}")
            checked.append((name, t, 8))
        for name, t, align in checked:
            size = t.element_size()
            if t.stride(3) != 1 or t.data_ptr() % align or any(s * size % align for s in t.stride()[:3]):
                raise ValueError(f"{name} needs unit stride in its last dimension and rows at multiples of {align} bytes, got strides {t.stride()}")
            reach = t.shape[3]                       # rows in one place: each dimension has to step over those inside it
            for s, n in sorted((s, n) for s, n in zip(t.stride()[:3], t.shape[:3]) if n > 1):
                if s < reach:
                    raise ValueError(f"{name} has rows that overlap, got strides {t.stride()}")
                reach = s * (n - 1) + reach
        if len({t.data_ptr() for _, t, _ in checked}) < len(checked):
            raise ValueError("keys and values (and their scales) must not lie in one place")
        self.k, self.v, self.k_scales, self.v_scales, self.dtype = k, v, k_scales, v_scales, dtype
        self._args = (k, v, k_scales, v_scales, dtype == torch.bfloat16)
        self._on_gpu = k.is_cuda

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, *, dtype: torch.dtype = torch.bfloat16, bits: int = 16,
                 device="cuda") -> "PagedCache":
        """A cache of its own storage, zeroed."""
        if bits not in (16, 4):
            raise ValueError(f"bits must be 16 or 4, got {bits!r}")
        shape = tuple(_as_count(n, x) for n, x in (("pages", pages), ("kv_heads", kv_heads), ("page_size", page_size), ("head_dim", head_dim)))
        if bits == 16:
            return cls(*(torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)))
        k, v = (torch.zeros((*shape[:3], shape[3] // 2), dtype=torch.uint8, device=device) for _ in range(2))
        ks, vs = (torch.zeros((*shape[:3], 2), dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, k_scales=ks, v_scales=vs, dtype=dtype)

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3] * (1 if self.bits == 16 else 2)

    @property
    def device(self) -> torch.device:
        return self.k.device


# --------------------------------------------------------------------------------------
# argument checks
# --------------------------------------------------------------------------------------
def _plain_rotary(rotary):
    """The native calls' form of `rotary`; None if it is none of the kind."""
    if rotary is None:
        return None, None
    return (rotary._packed, rotary.head_dim) if isinstance(rotary, Rotary) else None


def _native_call(cache, turn_args) -> bool:
    return turn_args is not None and isinstance(cache, PagedCache) and cache._on_gpu and not torch._C._are_functorch_transforms_active()


def _check_cache(cache) -> None:
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache must be a PagedCache, got {type(cache).__name__}")


def _check_rows(name: str, t, cache: PagedCache) -> None:
    check_heads(name, t)
    if t.dtype != cache.dtype:
        raise TypeError(f"{name} must have the cache's dtype {cache.dtype}, got {t.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on the cache's device {cache.device}, got {t.device}")
    if t.shape[3] != cache.head_dim:
        raise ValueError(f"{name} must have the cache's head dimension {cache.head_dim}, got {t.shape[3]}")
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"the paged cache records no gradients: detach {name}, call under torch.no_grad(), or use sdpa_bob")


def _check_sequences(cache: PagedCache, page_table, lengths, counts, batch: int | None = None):
    for name, t, ndim in (("page_table", page_table, 2), ("lengths", lengths, 1), ("counts", counts, 1)):
        if t is None and name == "counts":
            continue
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
            raise TypeError(f"{name} must be an int32 torch.Tensor")
        if t.ndim != ndim or t.numel() == 0:
            raise ValueError(f"{name} must have rank {ndim} and positive sizes, got {tuple(t.shape)}")
        if t.device != cache.device:
            raise ValueError(f"{name} must be on the cache's device {cache.device}, got {t.device}")
        if batch is None:
            batch = t.shape[0]
        if t.shape[0] != batch:
            raise ValueError(f"{name} must have one entry per sequence, got {t.shape[0]} for {batch}")
    if page_table.shape[1] * cache.page_size > 1 << 28:
        raise ValueError("page_table has room for more than 2**28 positions per sequence")
    return page_table, lengths, counts


# --------------------------------------------------------------------------------------
# CPU route
# --------------------------------------------------------------------------------------
def _quantise(x: torch.Tensor):
    """Codes [..., D / 2] and (scale, zero) [..., 2] of 16-bit rows [..., D]; fp32 arithmetic, as the kernels'."""
    x = x.float()
    zero, top = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = torch.where(top > zero, (top - zero) * (1 / 15), 1.0)
    codes = ((x - zero) / scale).round().nan_to_num(0.0).clamp(0, 15).to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.cat((scale, zero), -1)


def _cpu_rows(cache: PagedCache, which: str, pages, places):
    """Rows of k or v at (page, place), [H, n, D], fp32."""
    x = getattr(cache, which)[pages, :, places].transpose(0, 1)
    if cache.bits == 16:
        return x.float()
    scales = getattr(cache, which + "_scales")[pages, :, places].transpose(0, 1)
    return torch.stack((x & 15, x >> 4), -1).flatten(-2).float() * scales[..., :1] + scales[..., 1:]


def _cpu_sequences(cache: PagedCache, page_table, lengths, counts, n_rows: int, apart: bool = False):
    """(sequence, length, count) one by one, checked.  apart: the rows have no positions in the sequence, and may be more."""
    room = page_table.shape[1] * cache.page_size
    for b, length in enumerate(lengths.tolist()):
        count = n_rows if counts is None else int(counts[b])
        if not 0 <= length <= room or not 0 <= count <= (n_rows if apart else min(n_rows, length)):
            raise ValueError(f"sequence {b}: length {length} (room for {room}) or count {count} (of {n_rows} rows) out of range")
        yield b, length, count


def _cpu_places(cache: PagedCache, page_table, b: int, first: int, last: int):
    at = torch.arange(first, last)
    pages = page_table[b].long()[at // cache.page_size]
    if bool(((pages < 0) | (pages >= cache.pages)).any()):
        raise ValueError(f"sequence {b}: a page table entry within its length is outside the cache of {cache.pages} pages")
    return pages, at % cache.page_size


# --------------------------------------------------------------------------------------
# public operations
# --------------------------------------------------------------------------------------
def append_kv(k: torch.Tensor, v: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, *,
              counts: torch.Tensor | None = None, rotary: Rotary | None = None) -> None:
    """Writes new rows k, v [B, H_KV, N, D] into the pages, k turned to its positions where `rotary` is given.

    Row i < counts[b] of sequence b goes to position lengths[b] - counts[b] + i; the rows from counts[b] on are padding and not
    looked at, and no other row of the cache changes.  Pages may be shared between sequences as long as nothing is
    written to them: of two new rows for one place, parts of both may be left there.
    """
    # The usual valid CUDA call is recognised natively; everything else takes the checks below.
    turn_args = _plain_rotary(rotary)
    if _native_call(cache, turn_args) and _native.load().try_append(k, v, *cache._args, page_table, lengths, counts, *turn_args, ops._CHECK_STATUS):
        return
    check_plain_call()
    _check_cache(cache)
    _check_rows("k", k, cache)
    _check_rows("v", v, cache)
    if k.shape != v.shape:
        raise ValueError(f"k and v must share one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[1] != cache.kv_heads:
        raise ValueError(f"k and v must have the cache's {cache.kv_heads} heads, got {k.shape[1]}")
    sequences = _check_sequences(cache, page_table, lengths, counts, k.shape[0])
    packed = check_rotary(rotary, cache.head_dim, optional=True)
    if k.is_cuda:
        _native.load().cache_append(k, v, *cache._args, *sequences, packed, ops._CHECK_STATUS)
        return
    writes = []
    for b, length, count in _cpu_sequences(cache, *sequences, k.shape[2]):
        if count:
            writes.append((b, length - count, count, *_cpu_places(cache, page_table, b, length - count, length)))
    with torch.no_grad():
        for b, start, count, pages, places in writes:
            for name, x in (("k", k[b, :, :count]), ("v", v[b, :, :count])):
                if name == "k" and rotary is not None:
                    wide = x.double() if cache.bits == 4 else x
                    x = turn(wide, torch.arange(start, start + count), rotary).to(cache.dtype)
                if cache.bits == 4:
                    x, scales = _quantise(x)
                    getattr(cache, name + "_scales")[pages, :, places] = scales.transpose(0, 1)
                getattr(cache, name)[pages, :, places] = x.transpose(0, 1)


def read_kv(cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, n: int):
    """Positions 0 ... n - 1 of every sequence as contiguous (k, v) [B, H_KV, n, D]; rows from lengths[b] on are zero.

    The keys come as they lie in the cache, turned.  For `sdpa_bob` over a cached context.
    """
    check_plain_call()
    _check_cache(cache)
    n = _as_count("n", n)
    if not 0 < n <= 1 << 28:
        raise ValueError(f"n must be positive and at most 2**28, got {n}")
    sequences = _check_sequences(cache, page_table, lengths, None)
    if cache.k.is_cuda:
        return _native.load().cache_read(*cache._args, *sequences, n, ops._CHECK_STATUS)
    out = tuple(torch.zeros(page_table.shape[0], cache.kv_heads, n, cache.head_dim, dtype=cache.dtype) for _ in range(2))
    for b, length, _ in _cpu_sequences(cache, *sequences, 0):
        m = min(n, length)
        if m:
            places = _cpu_places(cache, page_table, b, 0, m)
            for t, which in zip(out, ("k", "v")):
                t[b, :, :m] = _cpu_rows(cache, which, *places).to(cache.dtype)
    return out


def sdpa_paged(q: torch.Tensor, cache: PagedCache, page_table: torch.Tensor, lengths: torch.Tensor, *, counts: torch.Tensor | None = None,
               is_causal: bool = True, scale: float | None = None, window_size: int = 0, rotary: Rotary | None = None) -> torch.Tensor:
    """Attention of q [B, H_Q, N, D] over the cached keys and values: [B, H_Q, N, D], contiguous, without gradients.

    Query i < counts[b] of sequence b sits at position lengths[b] - counts[b] + i, to which `rotary` turns it.  `is_causal`
    keeps keys at positions up to the query's, `window_size` w > 0 further keeps only the last w of them; without
    `is_causal` every query sees all lengths[b] keys, as in cross attention to cached encoder states (such queries have no
    position among the keys: there may be more of them, and `rotary` is refused).  Rows from counts[b] on, and rows without keys, are zero.
    Key and value rows that no query of its sequence attends to have no part in the result, whatever they hold; a NaN in a query or
    in a key that it attends to makes its result NaN and no other; a NaN or infinity among the values that some queries of a
    sequence attend to may reach its other queries of the same call, as in any product of probabilities and values.  H_Q is a multiple of H_KV, up to 32 times.

    Up to 16 rows (tokens of the call x H_Q / H_KV), in fp16 over 4 bits up to 64, only the result is rounded to 16 bits; beyond,
    turned queries, probabilities and rows of 4 bits are too, as in `apply_rotary` and `read_kv` followed by `sdpa_bob`.
    """
    turn_args = _plain_rotary(rotary)
    if _native_call(cache, turn_args):
        out = _native.load().try_paged(q, *cache._args, page_table, lengths, counts, *turn_args, is_causal, scale, window_size, ops._CHECK_STATUS)
        if out is not None:
            return out
    check_plain_call()
    _check_cache(cache)
    _check_rows("q", q, cache)
    if q.shape[1] % cache.kv_heads:
        raise ValueError(f"query heads H_Q={q.shape[1]} must be divisible by the cache's KV heads H_KV={cache.kv_heads}")
    if q.shape[1] // cache.kv_heads > _MAX_GROUP:
        raise NotImplementedError(f"grouping factors up to {_MAX_GROUP} are supported, got {q.shape[1] // cache.kv_heads}")
    window, _, _ = _check_scalars(is_causal, scale, window_size, None, 0)
    if rotary is not None and not is_causal:
        raise ValueError("rotary needs is_causal=True: without it queries have no position among the keys")
    sequences = _check_sequences(cache, page_table, lengths, counts, q.shape[0])
    packed = check_rotary(rotary, cache.head_dim, optional=True)
    if q.is_cuda:
        return _native.load().paged(q, *cache._args, *sequences, packed, is_causal, min(window, 1 << 28), None if scale is None else float(scale),
                                    ops._CHECK_STATUS)
    out = torch.zeros(q.shape, dtype=q.dtype)
    group, n_rows = q.shape[1] // cache.kv_heads, q.shape[2]
    tau = 1.0 / math.sqrt(q.shape[3]) if scale is None else float(scale)
    with torch.no_grad():
        for b, length, count in _cpu_sequences(cache, *sequences, n_rows, not is_causal):
            first = max(0, length - count - window + 1) if window else 0
            if not count or first >= length:
                continue
            position = torch.arange(length - count, length)
            x = q[b, :, :count].float()
            if rotary is not None:
                x = turn(x, position, rotary)
            places = _cpu_places(cache, page_table, b, first, length)
            keys, values = (_cpu_rows(cache, w, *places).repeat_interleave(group, 0) for w in ("k", "v"))
            s = (x @ keys.transpose(-1, -2)) * tau
            distance = position[:, None] - torch.arange(first, length)
            keep = torch.ones_like(distance, dtype=torch.bool)
            if is_causal:
                keep = distance >= 0
                if window:
                    keep &= distance < window
            out[b, :, :count] = (torch.softmax(s.masked_fill(~keep, -math.inf), -1) @ values).to(q.dtype)
    return out
