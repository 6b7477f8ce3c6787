"""KV cache for incremental decoding: ``InferenceParams`` with a contiguous (non-paged), a paged and an
8-bit paged cache manager (reference: ``pytorch/attention/inference.py:57, 405, 596``).

Usage, per generation step::

    params = InferenceParams(max_batch_size=8, max_sequence_length=4096, num_heads_kv=8,
                             head_dim_k=128, dtype=torch.bfloat16, is_paged=True, page_size=64,
                             total_num_pages=512)
    params.pre_step(OrderedDict((seq_id, new_tokens) ...))   # which sequences advance, by how much
    y = transformer_layer(x, inference_params=params, ...)      # every layer calls params.step(...)

``step`` appends the new K/V tokens of the step to the layer's cache and hands attention the
packed ("thd") queries together with every sequence's full cached K/V and the cumulative
lengths, so that the causal mask is aligned bottom-right per sequence.

With ``cache_dtype=torch.float8_e4m3fn`` the paged cache holds 8-bit codes (``attention/kv_cache.py``) and attention reads
them in place.  Paged sequences can be forked (pages are shared and copied when one of the owners writes), cut back, and
the pool compacted.
"""
from __future__ import annotations

from collections import OrderedDict
from typing import Dict, List, Optional, Tuple

import torch

from . import kv_cache as _kv
from . import thd as _thd


def _step_metadata(lens_old: List[int], lens_new: List[int], tables: List[List[int]], device):
    """Device-side description of one decoding step, shared by all layers: page table
    ``[sequences, width]`` (-1 where unused) and the cumulative new / resulting lengths."""
    width = max((len(t) for t in tables), default=1) or 1
    pt = [list(t) + [-1] * (width - len(t)) for t in tables]
    cu_new, cu_kv = [0], [0]
    for o, n in zip(lens_old, lens_new):
        cu_new.append(cu_new[-1] + n)
        cu_kv.append(cu_kv[-1] + o + n)
    mk = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return mk(pt).reshape(len(tables), width), mk(cu_new), mk(cu_kv), cu_kv[-1]


class KVCacheManager:
    """Interface of a cache manager (custom managers may subclass it)."""

    def reset(self) -> None:
        """Forget every sequence (the cache memory stays allocated)."""
        raise NotImplementedError

    def allocate_memory(self, layer_number: int) -> None:
        raise NotImplementedError

    def pre_step(self, step_dict: "OrderedDict[int, int]") -> None:
        raise NotImplementedError

    def step(self, layer_number: int, new_k: torch.Tensor, new_v: torch.Tensor, cu_new: List[int]):
        """Append packed new tokens ``[t_new, h, d]``; return packed full K, V and their lengths."""
        raise NotImplementedError


class NonPagedKVCacheManager(KVCacheManager):
    """One ``[max_batch, max_seq, h, d]`` slab per layer; a sequence owns one batch slot."""

    def __init__(self, max_batch_size, max_sequence_length, num_heads_kv, head_dim_k, dtype, head_dim_v=None,
                 device=None):
        self.max_batch_size, self.max_seq = max_batch_size, max_sequence_length
        self.h, self.dk, self.dv = num_heads_kv, head_dim_k, head_dim_v or head_dim_k
        self.dtype, self.device = dtype, device
        self.cache: Dict[int, Tuple[torch.Tensor, torch.Tensor]] = {}
        self.slots: "OrderedDict[int, int]" = OrderedDict()   # seq id -> batch slot
        self.lengths: Dict[int, int] = {}                       # seq id -> tokens cached BEFORE this step
        self.step_dict: "OrderedDict[int, int]" = OrderedDict()
        self.free_slots = list(range(max_batch_size - 1, -1, -1))
        self._meta = None  # device metadata of the current step (built by the first layer)

    def allocate_memory(self, layer_number):
        dev = self.device or ("cuda" if torch.cuda.is_available() else "cpu")
        k = torch.zeros(self.max_batch_size, self.max_seq, self.h, self.dk, dtype=self.dtype, device=dev)
        v = torch.zeros(self.max_batch_size, self.max_seq, self.h, self.dv, dtype=self.dtype, device=dev)
        self.cache[layer_number] = (k, v)

    def pre_step(self, step_dict):
        # sequences that are not part of this step have finished: release their slots
        for sid in [s for s in self.slots if s not in step_dict]:
            self.free_slots.append(self.slots.pop(sid))
            self.lengths.pop(sid, None)
        for sid in step_dict:
            if sid not in self.slots:
                assert self.free_slots, "KV cache is full: more live sequences than max_batch_size"
                self.slots[sid] = self.free_slots.pop()
                self.lengths[sid] = 0
        self.step_dict = OrderedDict(step_dict)
        self._meta = None

    def post_step(self):
        for sid, n in self.step_dict.items():
            self.lengths[sid] += n

    def reset(self) -> None:
        self.slots.clear()
        self.lengths.clear()
        self.step_dict = OrderedDict()
        self.free_slots = list(range(self.max_batch_size - 1, -1, -1))
        self._meta = None

    def step(self, layer_number, new_k, new_v, cu_new):
        if layer_number not in self.cache:
            self.allocate_memory(layer_number)
        kc, vc = self.cache[layer_number]
        olds = [self.lengths[sid] for sid in self.step_dict]
        news = list(self.step_dict.values())
        assert all(o + n <= self.max_seq for o, n in zip(olds, news)), "sequence exceeds max_sequence_length"
        if self._meta is None or self._meta[0].device != kc.device:
            # the whole slab is one "page" per slot: page size = max_seq, page table = slot
            self._meta = _step_metadata(olds, news, [[self.slots[sid]] for sid in self.step_dict], kc.device)
        pt, cu_n, cu_kv, total = self._meta
        k, v = _thd.kv_cache_step(new_k[:cu_new[-1]], new_v[:cu_new[-1]], kc, vc, pt, cu_n, cu_kv, total)
        return k, v, [o + n for o, n in zip(olds, news)]


class PagedKVCacheManager(KVCacheManager):
    """Pages of ``page_size`` tokens shared by all sequences, a page table per sequence."""

    def __init__(self, total_num_pages, page_size, num_heads_kv, head_dim_k, dtype, max_batch_size,
                 max_sequence_length, head_dim_v=None, device=None):
        self.total_num_pages, self.page_size = total_num_pages, page_size
        self.h, self.dk, self.dv = num_heads_kv, head_dim_k, head_dim_v or head_dim_k
        self.dtype, self.device = dtype, device
        self.max_batch_size, self.max_seq = max_batch_size, max_sequence_length
        self.cache: Dict[int, Tuple[torch.Tensor, torch.Tensor]] = {}
        self.free_pages = list(range(total_num_pages - 1, -1, -1))
        self.page_table: "OrderedDict[int, List[int]]" = OrderedDict()
        self.page_refs: Dict[int, int] = {}                  # owners of a page that several sequences share
        self.lengths: Dict[int, int] = {}
        self.step_dict: "OrderedDict[int, int]" = OrderedDict()
        self._meta = None

    def allocate_memory(self, layer_number):
        dev = self.device or ("cuda" if torch.cuda.is_available() else "cpu")
        k = torch.zeros(self.total_num_pages, self.page_size, self.h, self.dk, dtype=self.dtype, device=dev)
        v = torch.zeros(self.total_num_pages, self.page_size, self.h, self.dv, dtype=self.dtype, device=dev)
        self.cache[layer_number] = (k, v)

    def pre_step(self, step_dict):
        for sid in [s for s in self.page_table if s not in step_dict]:
            self._release(self.page_table.pop(sid))
            self.lengths.pop(sid, None)
        copies: List[Tuple[int, int]] = []
        try:
            for sid, n in step_dict.items():
                if sid not in self.page_table:
                    assert len(self.page_table) < self.max_batch_size, "more live sequences than max_batch_size"
                    self.page_table[sid] = []
                    self.lengths[sid] = 0
                table, first = self.page_table[sid], self.lengths[sid] // self.page_size
                need = -(-(self.lengths[sid] + n) // self.page_size) - len(table)
                # the page that the first new token goes to may be shared with a fork: this sequence gets its own
                own = n > 0 and first < len(table) and self.page_refs.get(table[first], 1) > 1
                assert max(need, 0) + own <= len(self.free_pages), "KV cache is out of pages"
                if own:
                    page = self.free_pages.pop()
                    if self.lengths[sid] % self.page_size:
                        copies.append((table[first], page))
                    self._release([table[first]])
                    table[first] = page
                for _ in range(max(need, 0)):
                    table.append(self.free_pages.pop())
        finally:
            self._copy(copies)    # also where a later sequence finds no page: the tables name the copies already
        self.step_dict = OrderedDict(step_dict)
        self._meta = None

    def _release(self, pages) -> None:
        """One owner less for each page; those without one return to the pool (-1: a page given back before)."""
        for p in pages:
            refs = self.page_refs.get(p, 1)
            if refs > 2:
                self.page_refs[p] = refs - 1
            elif refs == 2:
                del self.page_refs[p]
            elif p >= 0:
                self.free_pages.append(p)

    def _cache_tensors(self) -> List[torch.Tensor]:
        return [t for pair in self.cache.values() for t in pair]

    def _copy(self, pairs: List[Tuple[int, int]]) -> None:
        if pairs and self.cache:
            _kv.copy_pages(self._cache_tensors(), [s for s, _ in pairs], [d for _, d in pairs])

    # ---- sharing, cutting back, compacting (between steps: ``InferenceParams`` completes the step in flight first)
    def fork_sequence(self, seq: int, new_seq: int) -> None:
        """``new_seq`` starts as a copy of ``seq``.  Both share the pages that hold tokens; the page that one of them
        next writes to is copied then, in one launch over all layers."""
        if seq not in self.page_table:
            raise ValueError(f"unknown sequence {seq}")
        if new_seq in self.page_table:
            raise ValueError(f"sequence {new_seq} exists already")
        if len(self.page_table) >= self.max_batch_size:
            raise ValueError("more live sequences than max_batch_size")
        pages = self.page_table[seq][:-(-self.lengths[seq] // self.page_size)]
        for p in pages:
            if p >= 0:
                self.page_refs[p] = self.page_refs.get(p, 1) + 1
        self.page_table[new_seq], self.lengths[new_seq] = list(pages), self.lengths[seq]
        self._meta = None

    def truncate_sequence(self, seq: int, length: int) -> None:
        """Forget the tokens from ``length`` on (rejected drafts); pages that hold none of the rest are given back."""
        if seq not in self.page_table:
            raise ValueError(f"unknown sequence {seq}")
        if not 0 <= length <= self.lengths[seq]:
            raise ValueError(f"sequence {seq} holds {self.lengths[seq]} tokens, cannot cut it to {length}")
        keep = -(-length // self.page_size)
        table = self.page_table[seq]
        self._release(table[keep:])
        del table[keep:]
        self.lengths[seq] = length
        self._meta = None

    def compact(self) -> int:
        """Move the pages in use to the lowest page numbers (one launch over all layers) and return how many moved, so
        that the upper part of the pool can be handed to something else."""
        used = sorted({p for t in self.page_table.values() for p in t if p >= 0})
        holes = sorted(set(range(len(used))) - set(used))
        moved = dict(zip([p for p in used if p >= len(used)], holes))
        self._copy(list(moved.items()))
        for table in self.page_table.values():
            table[:] = [moved.get(p, p) for p in table]
        self.page_refs = {moved.get(p, p): n for p, n in self.page_refs.items()}
        self.free_pages = list(range(self.total_num_pages - 1, len(used) - 1, -1))
        self._meta = None
        return len(moved)

    def post_step(self):
        for sid, n in self.step_dict.items():
            self.lengths[sid] += n

    def get_page_table(self, sequences: Optional[List[int]] = None, device=None) -> torch.Tensor:
        """``[num_sequences, max_pages_per_seq]`` int32 table of the live sequences (or of ``sequences``, in that
        order), -1 where unused."""
        tables = [self.page_table[s] for s in sequences] if sequences is not None else list(self.page_table.values())
        width = max((len(p) for p in tables), default=0)
        t = torch.full((len(tables), width), -1, dtype=torch.int32, device=device)
        for i, pages in enumerate(tables):
            t[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        return t

    # ---- bookkeeping queries and manual page management (reference: attention/inference.py, PagedKVCacheManager)
    def reset(self) -> None:
        self.free_pages = list(range(self.total_num_pages - 1, -1, -1))
        self.page_table = OrderedDict()
        self.page_refs = {}
        self.lengths = {}
        self.step_dict = OrderedDict()
        self._meta = None

    def get_sequence_count(self) -> int:
        return len(self.page_table)

    def get_sequence_lengths(self) -> List[int]:
        """Cached tokens of every live sequence (before the step in flight)."""
        return [self.lengths[s] for s in self.page_table]

    def has_free_page(self) -> bool:
        return len(self.free_pages) > 0

    def get_page_count(self, seq: int) -> int:
        return len(self.page_table.get(seq, ()))

    def get_page_list(self, seq: int) -> List[int]:
        return list(self.page_table.get(seq, ()))

    def allocate_page(self, seq: int) -> None:
        if not self.free_pages:
            raise RuntimeError("KV cache is full!")
        self.page_table.setdefault(seq, []).append(self.free_pages.pop())
        self.lengths.setdefault(seq, 0)

    def allocate_sequence(self, seq: int, context_len: int) -> None:
        """Reserve the pages ``context_len`` tokens of a new sequence need."""
        for _ in range(-(-context_len // self.page_size)):
            self.allocate_page(seq)

    def deallocate_sequence(self, seq: int) -> None:
        self._release(self.page_table.pop(seq, ()))
        self.lengths.pop(seq, None)

    def print_cache(self) -> None:
        import logging

        log = logging.getLogger("PagedKVCacheManager")
        used = self.total_num_pages - len(self.free_pages)
        log.debug("total pages: %s (used %s, free %s); sequences: %s", self.total_num_pages, used,
                  len(self.free_pages), len(self.page_table))
        for i, (seq, pages) in enumerate(self.page_table.items()):
            log.debug("  batch index %s: seq_id %s, tokens %s, pages %s", i, seq, self.lengths.get(seq, 0), pages)

    def step(self, layer_number, new_k, new_v, cu_new):
        if layer_number not in self.cache:
            self.allocate_memory(layer_number)
        kc, vc = self.cache[layer_number]
        olds = [self.lengths[sid] for sid in self.step_dict]
        news = list(self.step_dict.values())
        if self._meta is None or self._meta[0].device != kc.device:
            self._meta = _step_metadata(olds, news, [self.page_table[sid] for sid in self.step_dict], kc.device)
        pt, cu_n, cu_kv, total = self._meta
        k, v = _thd.kv_cache_step(new_k[:cu_new[-1]], new_v[:cu_new[-1]], kc, vc, pt, cu_n, cu_kv, total)
        return k, v, [o + n for o, n in zip(olds, news)]


class FP8PagedKVCacheManager(PagedKVCacheManager):
    """The paged cache in 8 bits: e4m3 codes with a power-of-two scale for every 16 tokens of a head.

    ``attend`` appends a step's tokens and runs attention on the codes in place; ``step`` (attention variants that the
    cache kernels do not have) appends and returns all keys and values expanded to the step's dtype.  With
    ``window_size`` (left side of the layers' sliding window, the same in all of them) and ``sink_tokens``, pages that
    no later token can see return to the pool."""

    def __init__(self, total_num_pages, page_size, num_heads_kv, head_dim_k, dtype, max_batch_size, max_sequence_length,
                 head_dim_v=None, device=None, window_size: Optional[int] = None, sink_tokens: int = 0):
        if head_dim_v is not None and head_dim_v != head_dim_k:
            raise ValueError("the 8-bit cache holds keys and values of one head dim")
        device = device or ("cuda" if torch.cuda.is_available() else "cpu")
        _kv._check_geometry(page_size, head_dim_k, device)
        if sink_tokens < 0 or (window_size is not None and window_size < 0):
            raise ValueError("window_size and sink_tokens must not be negative")
        super().__init__(total_num_pages, page_size, num_heads_kv, head_dim_k, dtype, max_batch_size, max_sequence_length,
                         head_dim_v, device)
        self.window_size, self.sink_tokens = window_size, sink_tokens

    def allocate_memory(self, layer_number):
        self.cache[layer_number] = _kv.FP8KVCache.allocate(self.total_num_pages, self.h, self.page_size, self.dk, self.device)

    def pre_step(self, step_dict):
        if self.window_size is not None:
            # before the step's pages are taken: what its first query no longer sees, no later one does
            for sid, table in self.page_table.items():
                last = min((self.lengths[sid] - self.window_size) // self.page_size, len(table))
                for i in range(-(-self.sink_tokens // self.page_size), last):
                    if table[i] >= 0:
                        self._release([table[i]])
                        table[i] = -1
        super().pre_step(step_dict)

    def truncate_sequence(self, seq, length):
        if self.window_size is not None and seq in self.page_table:
            # the next query's window (a sequence cut to nothing starts anew) must still be there
            first = max(0, length - self.window_size) // self.page_size
            if any(p < 0 for p in self.page_table[seq][first:-(-length // self.page_size)]):
                raise ValueError(f"sequence {seq} cannot be cut to {length}: its window has been given back")
        super().truncate_sequence(seq, length)

    def _layer(self, layer_number) -> "_kv.FP8KVCache":
        if layer_number not in self.cache:
            self.allocate_memory(layer_number)
        return self.cache[layer_number]

    def _step_meta(self):
        """Device tensors of the step (page table, cumulative new tokens, resulting lengths), uploaded once for all
        layers, and the host's numbers."""
        if self._meta is None:
            tables = [self.page_table[sid] for sid in self.step_dict]
            news = list(self.step_dict.values())
            lens = [self.lengths[sid] + n for sid, n in self.step_dict.items()]
            n, width = len(news), max((len(t) for t in tables), default=1) or 1
            flat = [p for t in tables for p in t + [-1] * (width - len(t))]
            cu, cu_kv = [0], [0]
            for a, b in zip(news, lens):
                cu.append(cu[-1] + a)
                cu_kv.append(cu_kv[-1] + b)
            dev = torch.tensor(flat + cu + lens + cu_kv, dtype=torch.int32, device=self.device)
            at = [n * width, n * width + n + 1, n * width + 2 * n + 1]
            self._meta = (dev[:at[0]].view(n, width), dev[at[0]:at[1]], dev[at[1]:at[2]], dev[at[2]:], max(news, default=0),
                          max(lens, default=0), cu_kv[-1])
        return self._meta

    def step(self, layer_number, new_k, new_v, cu_new):
        cache = self._layer(layer_number)
        table, cu, lens, cu_kv, max_new, max_kv, total = self._step_meta()
        _kv.append(cache, new_k[:cu_new[-1]], new_v[:cu_new[-1]], table, cu, lens, max_new=max_new)
        k, v = _kv.gather(cache, table, lens, cu_kv[:-1], total, new_k.dtype, max_kv=max_kv)
        return k, v, [self.lengths[sid] + n for sid, n in self.step_dict.items()]

    def check_window(self, layer_number, window, sink_tokens) -> None:
        """Refuse a layer that looks further back than the pages that are kept."""
        if self.window_size is not None:
            left = -1 if window is None else window[0]
            if left < 0 or left > self.window_size or sink_tokens > self.sink_tokens:
                raise ValueError(f"the cache keeps a window of {self.window_size} and {self.sink_tokens} sinks; layer {layer_number} "
                                 f"looks at a window of {left} and {sink_tokens}")

    def attend(self, layer_number, q, new_k, new_v, *, scale, causal, window, sink_tokens):
        """Append the packed new tokens ``[t, h, d]`` and attend: packed output ``[t, hq, d]``."""
        self.check_window(layer_number, window, sink_tokens)
        cache = self._layer(layer_number)
        table, cu, lens, _, max_new, max_kv, _ = self._step_meta()
        _kv.append(cache, new_k, new_v, table, cu, lens, max_new=max_new)
        return _kv.attend(q, cache, table, cu, lens, max_q=max_new, max_kv=max_kv, scale=scale, causal=causal, window=window,
                          sink_tokens=sink_tokens)


class InferenceParams:
    """State of incremental decoding shared by all layers of a model.

    ``cache_dtype=torch.float8_e4m3fn`` keeps the (paged) cache in 8 bits; ``window_size`` / ``sink_tokens`` then tell it
    the sliding window and the first tokens that all layers attend to, so that pages out of sight are reused."""

    def __init__(self, max_batch_size: int, max_sequence_length: int, num_heads_kv: Optional[int] = None,
                 head_dim_k: Optional[int] = None, dtype: Optional[torch.dtype] = None,
                 head_dim_v: Optional[int] = None, is_paged: bool = False, total_num_pages: Optional[int] = None,
                 page_size: Optional[int] = None, max_ctx_len: Optional[int] = None, qkv_format: str = "bshd",
                 custom_cache_manager=None, device=None, cache_dtype: Optional[torch.dtype] = None,
                 window_size: Optional[int] = None, sink_tokens: int = 0):
        if cache_dtype not in (None, dtype, torch.float8_e4m3fn):
            raise ValueError(f"cache_dtype must be {dtype} or torch.float8_e4m3fn, got {cache_dtype}")
        fp8 = cache_dtype == torch.float8_e4m3fn
        if fp8 and (not is_paged or custom_cache_manager is not None):
            raise ValueError("the 8-bit cache is paged: is_paged=True, and no custom cache manager")
        if not fp8 and (window_size is not None or sink_tokens):
            raise ValueError("window_size and sink_tokens are for the 8-bit cache")
        self.max_batch_size, self.max_sequence_length = max_batch_size, max_sequence_length
        self.num_heads_kv, self.head_dim_k, self.head_dim_v = num_heads_kv, head_dim_k, head_dim_v or head_dim_k
        self.dtype, self.is_paged, self.page_size = dtype, is_paged, page_size
        self.total_num_pages, self.max_ctx_len, self.input_qkv_format = total_num_pages, max_ctx_len, qkv_format
        if custom_cache_manager is not None:
            self.cache_manager = custom_cache_manager
        elif fp8:
            assert page_size and total_num_pages, "a paged cache needs page_size and total_num_pages"
            self.cache_manager = FP8PagedKVCacheManager(total_num_pages, page_size, num_heads_kv, head_dim_k, dtype,
                                                        max_batch_size, max_sequence_length, head_dim_v, device,
                                                        window_size, sink_tokens)
        elif is_paged:
            assert page_size and total_num_pages, "a paged cache needs page_size and total_num_pages"
            self.cache_manager = PagedKVCacheManager(total_num_pages, page_size, num_heads_kv, head_dim_k, dtype,
                                                     max_batch_size, max_sequence_length, head_dim_v, device)
        else:
            self.cache_manager = NonPagedKVCacheManager(max_batch_size, max_sequence_length, num_heads_kv,
                                                        head_dim_k, dtype, head_dim_v, device)
        self.step_dict: "OrderedDict[int, int]" = OrderedDict()
        self.sequences: "OrderedDict[int, int]" = OrderedDict()   # seq id -> length before the current step
        self._layers_seen: set = set()
        self._pending_post = False
        self._orig: Optional[Tuple[str, int, int]] = None

    # ---- step bookkeeping
    def reset(self):
        self.pre_step(OrderedDict())
        self.sequences = OrderedDict()
        if hasattr(self.cache_manager, "reset"):
            try:
                self.cache_manager.reset()
            except NotImplementedError:
                pass

    def allocate_memory(self, layer_number: int):
        self.cache_manager.allocate_memory(layer_number)

    def pre_step(self, step_dict: "OrderedDict[int, int]"):
        self._complete_step()
        self.cache_manager.pre_step(step_dict)
        self.step_dict = OrderedDict(step_dict)
        self.sequences = OrderedDict((sid, self.cache_manager.lengths[sid]) for sid in step_dict)
        self._layers_seen = set()
        self._pending_post = bool(step_dict)

    def _complete_step(self):
        if self._pending_post:
            self.cache_manager.post_step()
            self._pending_post = False

    def _pages(self) -> PagedKVCacheManager:
        if not isinstance(self.cache_manager, PagedKVCacheManager):
            raise ValueError("forking, cutting back and compacting need a paged cache")
        self._complete_step()
        return self.cache_manager

    def fork_sequence(self, seq: int, new_seq: int) -> None:
        """After a step: ``new_seq`` continues from what ``seq`` holds (paged caches; pages are shared until written)."""
        self._pages().fork_sequence(seq, new_seq)

    def truncate_sequence(self, seq: int, length: int) -> None:
        """After a step: cut a sequence back to its first ``length`` tokens (paged caches)."""
        self._pages().truncate_sequence(seq, length)

    def compact(self) -> int:
        """After a step: move the pages in use to the front of the pool (paged caches); returns how many moved."""
        return self._pages().compact()

    def get_seqlens_pre_step(self) -> torch.Tensor:
        return torch.tensor(list(self.sequences.values()), dtype=torch.int32)

    def convert_paged_to_nonpaged(self, layer_number: int):
        """The paged cache of one layer as contiguous ``[sequences, pages_per_seq * page_size, h, d]`` tensors
        (sequences in batch order; positions past a sequence's length hold whatever its last page holds)."""
        assert self.is_paged, "the cache is not paged"
        m = self.cache_manager
        if isinstance(m, FP8PagedKVCacheManager):
            cache, table = m.cache[layer_number], m.get_page_table(device=m.device)
            n, rows = table.shape[0], table.shape[1] * m.page_size
            mk = lambda x: torch.tensor(x, dtype=torch.int32, device=m.device)  # noqa: E731
            k, v = _kv.gather(cache, table, mk([len(t) * m.page_size for t in m.page_table.values()]),
                              mk([i * rows for i in range(n)]), n * rows, m.dtype, max_kv=rows)
            return tuple(t.view(n, rows, *t.shape[1:]) for t in (k, v))
        k, v = m.cache[layer_number]
        table = m.get_page_table(device=k.device).clamp(min=0).long()
        n, w = table.shape
        gather = lambda c: c[table.reshape(-1)].reshape(n, w * c.shape[1], *c.shape[2:]).contiguous()  # noqa: E731
        return gather(k), gather(v)

    def __repr__(self) -> str:
        kind = f"paged (page_size={self.page_size}, total_num_pages={self.total_num_pages})" if self.is_paged \
            else "non-paged"
        return (f"InferenceParams({kind}, max_batch_size={self.max_batch_size}, "
                f"max_sequence_length={self.max_sequence_length}, num_heads_kv={self.num_heads_kv}, "
                f"head_dim_k={self.head_dim_k}, head_dim_v={self.head_dim_v}, dtype={self.dtype}, "
                f"sequences={dict(self.sequences)})")

    def sequence_start_positions(self, batch: int, device) -> torch.Tensor:
        """Position of each sequence's first new token (RoPE offset)."""
        starts = list(self.sequences.values())
        starts += [0] * (batch - len(starts))
        return torch.tensor(starts[:batch], dtype=torch.int32, device=device)

    # ---- per-layer cache update
    def step(self, layer_number, q, k, v, qkv_format, mask_type):
        """Returns (q, k, v, "thd", mask type, cu_seqlens_q, cu_seqlens_kv) for attention."""
        lens_new = list(self.step_dict.values())
        nb = len(lens_new)
        if qkv_format == "thd":
            cu = [0]
            for n in lens_new:
                cu.append(cu[-1] + n)
            qp, kp, vp = q, k[:cu[-1]], v[:cu[-1]]
            self._orig = ("thd", q.shape[0], 0)
        else:
            if qkv_format == "sbhd":
                q, k, v = (t.transpose(0, 1) for t in (q, k, v))
            b, s = q.shape[0], q.shape[1]
            assert nb <= b, "step_dict names more sequences than the batch holds"
            cu = [0]
            for n in lens_new:
                cu.append(cu[-1] + n)
            cu_t = torch.tensor(cu, dtype=torch.int32, device=q.device)
            qp, kp, vp = (_thd.convert_bshd_to_thd(t, cu_t, cu[-1]) for t in (q, k, v))
            self._orig = (qkv_format, b, s)
            self._cu_new = cu_t
        kf, vf, lens_kv = self.cache_manager.step(layer_number, kp, vp, cu)
        cu_kv = [0]
        for n in lens_kv:
            cu_kv.append(cu_kv[-1] + n)
        dev = q.device
        mt = "padding_causal_bottom_right" if "causal" in mask_type else "padding"
        return (qp, kf, vf, "thd", mt, torch.tensor(cu, dtype=torch.int32, device=dev),
                torch.tensor(cu_kv, dtype=torch.int32, device=dev))

    def check_window(self, layer_number, window, sink_tokens) -> None:
        """Raise if the layer attends to tokens that the cache has given back (8-bit cache with ``window_size``)."""
        if hasattr(self.cache_manager, "check_window"):
            self.cache_manager.check_window(layer_number, window, sink_tokens)

    def attends(self) -> bool:
        """Whether the cache itself runs attention (``attend``) instead of handing out keys and values (``step``)."""
        return hasattr(self.cache_manager, "attend")

    def attend(self, layer_number, q, k, v, qkv_format, mask_type, *, scale, window, sink_tokens):
        """Append the step's keys and values to the layer's cache and attend to it; the output has the layout of ``q``
        with heads and head dim merged."""
        news = list(self.step_dict.values())
        causal = "causal" in mask_type
        kw = dict(scale=scale, causal=causal, window=window, sink_tokens=sink_tokens)
        if qkv_format == "thd":
            o = self.cache_manager.attend(layer_number, q, k, v, **kw)
            return o.reshape(o.shape[0], -1)
        if qkv_format == "sbhd":
            q, k, v = (t.transpose(0, 1) for t in (q, k, v))
        b, s = q.shape[:2]
        assert len(news) <= b, "step_dict names more sequences than the batch holds"
        if all(n == s for n in news) and len(news) == b and (s == 1 or q.is_contiguous()):
            # nothing is padding: the packed rows are the batch's own
            o = self.cache_manager.attend(layer_number, *(t.reshape(b * s, *t.shape[2:]) for t in (q, k, v)), **kw).view(b, s, -1)
        else:
            cu, total = self.cache_manager._step_meta()[1], sum(news)
            q, k, v = (_thd.convert_bshd_to_thd(t, cu, total) for t in (q, k, v))
            o = self.cache_manager.attend(layer_number, q, k, v, **kw)
            o = _thd.convert_thd_to_bshd(o.view(total, -1), cu, b, s)
        return o.transpose(0, 1) if qkv_format == "sbhd" else o

    def unpack_output(self, out: torch.Tensor) -> torch.Tensor:
        """Packed attention output ``[t, h*d]`` back to the layout the caller passed in."""
        fmt, b, s = self._orig
        if fmt == "thd":
            return out
        res = _thd.convert_thd_to_bshd(out, self._cu_new, b, s)
        return res.transpose(0, 1) if fmt == "sbhd" else res
