"""Paged key/value cache in 8 bits: quantizing append, attention over the cache, gather, page copies.

One layer's cache (:class:`FP8KVCache`) holds e4m3 codes ``[pages, heads, page_size, d]`` and fp32 scales
``[pages, heads, page_size / 16]``: every 16 tokens of a head share one scale, the smallest power of two (kept within
2^-60 .. 2^60) with ``max|x| <= 448 * scale`` over the block's finite values.  Appending to a partly filled block may raise
its scale; the codes it held are then rounded again, which changes only those that become subnormal.  Infinities
saturate, NaN stays NaN.

On CUDA every function runs the kernels of ``csrc/attn/kv_cache.cu`` and ``csrc/attn/fp8_attend.cu`` on the current
stream (head dims 64, 128, 256); the PyTorch bodies below are the CPU path and the oracle of the kernel tests (any head
dim).  Sequence i owns row i of ``page_table`` (int32 ``[n, width]``, the page of every ``page_size`` tokens, -1 where
none is held) and ``kv_lens[i]`` tokens.  Ids outside the cache and lengths that do not fit are skipped by the kernels and
reported by :func:`transformerengine_b200.check_status`; attention takes the keys and values of a page that is not held for
zeros, and reports it where a query sees it.  No function synchronizes with the device.
"""
from __future__ import annotations

import math
from typing import List, NamedTuple, Optional, Sequence, Tuple, Union

import torch

from ..ops import _ext
from ..ops import flash as _flash

BLOCK = 16            # tokens that share a scale
HEAD_DIMS = (64, 128, 256)
_MAX_EXP = 60


class FP8KVCache(NamedTuple):
    """The 8-bit cache of one layer (:meth:`allocate` makes an empty one, :func:`append` fills it: scales that are not
    powers of two give wrong results).  On CUDA the codes start on a multiple of 16 bytes."""

    k: torch.Tensor          # float8_e4m3fn [pages, heads, page_size, d]
    v: torch.Tensor
    k_scale: torch.Tensor    # fp32 [pages, heads, page_size / 16]
    v_scale: torch.Tensor

    @classmethod
    def allocate(cls, num_pages: int, num_heads: int, page_size: int, head_dim: int, device=None) -> "FP8KVCache":
        _check_geometry(page_size, head_dim, device)
        mk = lambda: torch.zeros(num_pages, num_heads, page_size, head_dim, dtype=torch.uint8,  # noqa: E731
                                 device=device).view(torch.float8_e4m3fn)
        sc = lambda: torch.zeros(num_pages, num_heads, page_size // BLOCK, dtype=torch.float32, device=device)  # noqa: E731
        return cls(mk(), mk(), sc(), sc())

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


def _check_geometry(page_size: int, head_dim: int, device) -> None:
    if page_size < BLOCK or page_size % BLOCK:
        raise ValueError(f"the 8-bit cache needs a page size that is a multiple of {BLOCK}, got {page_size}")
    if device is not None and torch.device(device).type == "cuda" and head_dim not in HEAD_DIMS:
        raise ValueError(f"the 8-bit cache kernels take head dims {HEAD_DIMS}, got {head_dim}")


def _cuda(cache: FP8KVCache) -> bool:
    return cache.k.is_cuda


# ------------------------------------------------------------------------------------------------ reference pieces
def block_scale(top: torch.Tensor) -> torch.Tensor:
    """The smallest power of two with ``top <= 448 * scale``, within 2^-60 .. 2^60 (2^-60 for zero)."""
    m, e = torch.frexp(top.float())
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-_MAX_EXP, _MAX_EXP)
    e = torch.where(top > 0, e, torch.full_like(e, -_MAX_EXP)).to(torch.int32)
    return ((e + 127) << 23).view(torch.float32)


def _round_e4m3(x: torch.Tensor) -> torch.Tensor:
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _append_ref(cache: FP8KVCache, new_k, new_v, table, cu_new, kv_lens) -> None:
    ps = cache.page_size
    cu, lens, tab = cu_new.tolist(), kv_lens.tolist(), table.tolist()
    for i in range(len(lens)):
        n = cu[i + 1] - cu[i]
        old = lens[i] - n
        if n <= 0:
            continue
        assert old >= 0 and cu[i + 1] <= new_k.shape[0], "kv_lens counts the new tokens"
        for blk in range(old // BLOCK, (lens[i] - 1) // BLOCK + 1):
            page, at = tab[i][blk * BLOCK // ps], blk * BLOCK % ps
            if not 0 <= page < cache.k.shape[0]:
                raise ValueError(f"sequence {i} holds no page for token {blk * BLOCK}")
            a, b = max(old, blk * BLOCK), min(lens[i], (blk + 1) * BLOCK)
            for codes, scales, new in ((cache.k, cache.k_scale, new_k), (cache.v, cache.v_scale, new_v)):
                x = new[cu[i] + a - old:cu[i] + b - old].float().transpose(0, 1)                  # [h, rows, d]
                mag = x.abs()
                now = block_scale(torch.where(mag < math.inf, mag, torch.zeros_like(mag)).amax((1, 2)))
                rows = codes[page].view(torch.uint8)
                if a > blk * BLOCK:
                    was = scales[page, :, at // BLOCK]
                    now = torch.maximum(now, was)
                    kept = slice(at, at + a - blk * BLOCK)
                    held = rows[:, kept].view(torch.float8_e4m3fn).float() * (was / now)[:, None, None]
                    rows[:, kept] = _round_e4m3(held).view(torch.uint8)
                rows[:, at + a - blk * BLOCK:at + b - blk * BLOCK] = _round_e4m3(x / now[:, None, None]).view(torch.uint8)
                scales[page, :, at // BLOCK] = now


def _values_ref(cache: FP8KVCache, pages: List[int], length: int, dtype) -> Tuple[torch.Tensor, torch.Tensor]:
    """One sequence's keys and values ``[length, h, d]``; pages that are not held give zeros."""
    ps, out = cache.page_size, []
    need = -(-length // ps)
    ids = torch.tensor([p for p in pages[:need]] + [-1] * max(0, need - len(pages)), dtype=torch.long, device=cache.k.device)
    top = torch.finfo(dtype).max
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = codes.view(torch.uint8)[ids.clamp(min=0)].view(torch.float8_e4m3fn).float()
        x = x * scales[ids.clamp(min=0)].repeat_interleave(BLOCK, dim=2)[..., None]
        x = torch.where((ids >= 0)[:, None, None, None], x, torch.zeros_like(x))
        x = x.transpose(1, 2).reshape(need * ps, codes.shape[1], codes.shape[3])[:length]
        out.append(x.clamp(-top, top).to(dtype))
    return out[0], out[1]


def _attend_ref(q, cache, table, cu_q, kv_lens, scale, causal, window_left, sink_tokens):
    from ..ops.attention import attention_ref

    out = torch.zeros_like(q, memory_format=torch.contiguous_format)
    cu, lens, tab = cu_q.tolist(), kv_lens.tolist(), table.tolist()
    for i in range(len(lens)):
        if cu[i + 1] <= cu[i] or lens[i] <= 0:
            continue
        k, v = (x.transpose(0, 1).unsqueeze(0) for x in _values_ref(cache, tab[i], lens[i], torch.float32))
        o = attention_ref(q[cu[i]:cu[i + 1]].transpose(0, 1).unsqueeze(0).float(), k, v, scale=scale, causal=causal,
                          window=(window_left, 0 if causal else -1), sink_tokens=sink_tokens, bottom_right=True)
        out[cu[i]:cu[i + 1]] = o.squeeze(0).transpose(0, 1).to(q.dtype)
    return out


# ------------------------------------------------------------------------------------------------------ entry points
def append(cache: FP8KVCache, new_k: torch.Tensor, new_v: torch.Tensor, page_table: torch.Tensor, cu_new: torch.Tensor,
           kv_lens: torch.Tensor, *, max_new: Optional[int] = None) -> None:
    """Quantize the packed new tokens ``[t, h, d]`` (fp32, fp16 or bf16; any strides with d contiguous) into the cache.

    Sequence i's new tokens are rows ``cu_new[i] .. cu_new[i + 1]`` and end at token ``kv_lens[i]`` of the sequence: the
    lengths COUNT the new tokens.  ``max_new`` (longest run of new tokens) sizes the launch; longer runs are handled too.
    No page may belong to two sequences that both append to it (``fork_sequence`` of the paged managers copies first)."""
    if not _cuda(cache):
        _append_ref(cache, new_k, new_v, page_table, cu_new, kv_lens)
        return
    _ext.get().fp8_cache_append(*cache, new_k, new_v, page_table, cu_new, kv_lens,
                                new_k.shape[0] if max_new is None else max_new)


def gather(cache: FP8KVCache, page_table: torch.Tensor, kv_lens: torch.Tensor, offsets: torch.Tensor, rows: int,
           dtype: torch.dtype, *, max_kv: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of all sequences as ``[rows, h, d]`` in 16 bits or fp32; sequence i starts at row
    ``offsets[i]``.  Tokens whose page is not held give zeros, rows that belong to no sequence are not written."""
    h, d = cache.k.shape[1], cache.k.shape[3]
    k = torch.empty(rows, h, d, dtype=dtype, device=cache.k.device)
    v = torch.empty_like(k)
    if _cuda(cache):
        _ext.get().fp8_cache_gather(*cache, page_table, kv_lens, offsets, k, v, rows if max_kv is None else max_kv)
        return k, v
    for i, (n, o, pages) in enumerate(zip(kv_lens.tolist(), offsets.tolist(), page_table.tolist())):
        k[o:o + n], v[o:o + n] = _values_ref(cache, pages, n, dtype)
    return k, v


_EXPAND_BYTES = 4 << 30      # of expanded keys and values at a time, 2 % of the device's memory; needs beyond are read in place


def _expansion_bytes(hq: int, hk: int, d: int, max_q: int, max_kv: int) -> int:
    """Buffers that one sequence takes where its codes are expanded: keys and values in 16 bits, row sums."""
    return 4 * hk * d * (-(-max_kv // 128) * 128) + 4 * hq * (-(-max_q // 128) * 128)


def _expands(n: int, hq: int, hk: int, d: int, max_q: int, tokens: int, max_kv: int) -> bool:
    """Whether expanding the codes once for the packed 16-bit attention kernel beats the kernel that reads them in place.

    The latter walks the cache once for every 16 query rows of a key head (4.3e-5 us per tile and token on all SMs), the
    former takes 0.02 us per token and wave of its CTAs (256 queries of a head each).  Measured, us in place / expanded,
    32 / 8 heads: 8 sequences of 8000 tokens, 32 queries 187 / 328, 64 queries 350 / 330, 128 queries 670 / 333; one of
    100000, 128 queries 985 / 1597; 64 of 2000, 64 queries 790 / 649.  Both counts are bounded by the packed queries
    (``tokens``) too: beside a prompt chunk the other sequences may have a token each (1024 queries beside 63 single ones on
    500 - 8000 tokens: 1016 / 1485).  Sequences whose expansion would
    not fit ``_EXPAND_BYTES`` one at a time (a ``max_kv`` far above the lengths, say) are read in place."""
    rows = hq // hk * max_q
    if rows <= 64 or _expansion_bytes(hq, hk, d, max_q, max_kv) > _EXPAND_BYTES:
        return False
    waves = -(-hq * min(n * -(-max_q // 256), tokens // 256 + n) // 148)
    return hk * min(n * -(-rows // 16), hq // hk * tokens // 16 + n) > 470 * waves


def attend(q: torch.Tensor, cache: FP8KVCache, page_table: torch.Tensor, cu_q: torch.Tensor, kv_lens: torch.Tensor, *,
           max_q: int, max_kv: int, scale: Optional[float] = None, causal: bool = True,
           window: Optional[Tuple[int, int]] = None, sink_tokens: int = 0) -> torch.Tensor:
    """Attention of packed queries ``[t, hq, d]`` (fp16 or bf16) over the cached tokens; returns ``[t, hq, d]``.

    Sequence i's queries are rows ``cu_q[i] .. cu_q[i + 1]`` (``cu_q[0]`` is 0) and, under the causal mask, the LAST tokens of its
    ``kv_lens[i]`` (bottom-right alignment).  ``window = (left, right)`` limits what the query at position p sees to keys
    ``p - left .. p``, plus the first ``sink_tokens`` tokens; -1 leaves a side open, and the right side is the causal
    one.  ``max_q`` / ``max_kv`` bound the queries and tokens of a sequence: a longer one is cut there and reported.  Rows
    that see nothing, rows behind the last sequence, and rows that were cut off are zero.  With fp16 queries, prompt chunks
    at head dim 128 may read keys and values as fp16 (beyond 65504, in a cache filled from another type, they saturate).
    There is no backward pass."""
    if q.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("attention over the 8-bit cache has no backward pass: call it under torch.no_grad()")
    left = -1
    if window is not None:
        left, right = window
        if right >= 0 and not (causal and right == 0):
            raise ValueError("attention over the 8-bit cache takes windows with a left side only (right: -1, or 0 with causal)")
        if left >= 0 and not causal:
            raise ValueError("a sliding window over the 8-bit cache needs the causal mask")
    if sink_tokens < 0:
        raise ValueError("sink_tokens must not be negative")
    _, hq, d = q.shape
    if scale is None:
        scale = d ** -0.5
    if not _cuda(cache):
        return _attend_ref(q, cache, page_table, cu_q, kv_lens, scale, causal, left, sink_tokens)
    max_q = min(max_q, q.shape[0])     # it sizes launches and buffers: no sequence has more
    # (the packed kernels take the maximum of the raw scores: a positive scale)
    if d == 128 and scale > 0.0 and max_q > 0 and max_kv > 0 and _expands(page_table.shape[0], hq, cache.k.shape[1], d, max_q,
                                                                                q.shape[0], max_kv):
        return _attend_expanded(q, cache, page_table, cu_q, kv_lens, max_q, max_kv, scale, causal, left, sink_tokens)
    return _ext.get().fp8_cache_attend(q, *cache, page_table, cu_q, kv_lens, max_q, max_kv, scale, causal, left, sink_tokens)


def _attend_expanded(q, cache, page_table, cu_q, kv_lens, max_q, max_kv, scale, causal, left, sink_tokens):
    """Codes expanded to 16 bits (every sequence padded to whole 128-token blocks with zeros), then the packed attention
    kernel: prompt chunks are bound by its products, not by the cache.  As many sequences at a time as fit the buffers."""
    C_ = _ext.get()
    n, hq, d = page_table.shape[0], q.shape[1], q.shape[2]
    group = max(1, _EXPAND_BYTES // _expansion_bytes(hq, cache.k.shape[1], d, max_q, max_kv))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for i in range(0, n, group):
        table, cu, lens = (page_table, cu_q, kv_lens) if group >= n else \
            (page_table[i:i + group], cu_q[i:i + group + 1], kv_lens[i:i + group])
        k, v, cu_k, first_k, cut_q, first_q = C_.fp8_cache_expand(q, *cache, table, cu, lens, out, max_q, max_kv, left, sink_tokens,
                                                                  i + group >= n)
        _flash.flash_varlen_forward(q, k, v, out, cut_q, cu_k, first_q, first_k, max_q, max_kv, scale, causal, left, sink_tokens)
        del k, v
    return out


def copy_pages(caches: Sequence[Union[torch.Tensor, FP8KVCache]], src: Union[Sequence[int], torch.Tensor],
               dst: Union[Sequence[int], torch.Tensor]) -> None:
    """``pages[dst[i]] = pages[src[i]]`` in every cache of the list, one launch for up to 128 tensors and 1024 pages.

    The caches are :class:`FP8KVCache` or plain tensors whose first dimension counts pages (16-bit caches); the page ids
    are host data (lists or CPU tensors).  No page may be written twice, or both read and written."""
    tensors: List[torch.Tensor] = []
    for c in caches:
        if isinstance(c, FP8KVCache):
            tensors.extend(c)
        else:
            tensors.append(c)
    src, dst = (torch.as_tensor(x, dtype=torch.int64, device="cpu").contiguous() for x in (src, dst))
    if src.dim() != 1 or src.shape != dst.shape:
        raise ValueError("copy_pages: as many source pages as destination pages")
    if not tensors or src.numel() == 0:
        return
    if tensors[0].is_cuda:
        _ext.get().copy_pages(tensors, src, dst)
        return
    pages = min(t.shape[0] for t in tensors)
    s, d = src.tolist(), dst.tolist()
    if min(s + d) < 0 or max(s + d) >= pages:
        raise ValueError("copy_pages: page id out of range")
    if len(set(d)) != len(d) or set(s) & set(d):
        raise ValueError("copy_pages: a page is written twice, or read and written")
    for t in tensors:
        raw = t.view(torch.uint8) if t.element_size() == 1 else t
        raw[dst] = raw[src]
