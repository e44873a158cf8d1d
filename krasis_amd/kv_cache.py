"""Paged KV cache bookkeeping with the reference's class surface (python/krasis/kv_cache.py:38-272: `PagedKVCache`, `SequenceKVState`) and the hand-off of
a paged cache to the decode store (`CpuDecoder._copy_kv_cache`, decode_setup.py:653-711).

On MI355X a request's cache is ONE contiguous `[max_seq, kv_heads * head_dim]` allocation per layer inside the decode store (288 GB of HBM: nothing has to
be paged to make room for the experts), and the prompt pass of this library writes that flat cache directly.  What is here is the part of the reference a
CALLER sees: the page pool, the per-sequence page list with its index arrays, the store method of the combined MLA layout -- same constructor arguments,
same tensor shapes / dtypes, same error texts -- and `unpage_into_store`, which gathers a sequence's pages into the flat caches the decode store takes
(FP8-E4M3 pages are widened to FP16 exactly, or handed over as E4M3 bytes when the store runs `kr_decode_set_kv_dtype(FP8)`).  The attention kernels of the stores do
NOT read through this page table: a caller that keeps its own paged cache unpages once, at the prompt -> decode hand-off, as the reference does.

A caller that runs its own layers on the paged cache uses `KVBatch`, the plan of one step over some sequences: new rows quantised into the pages, read back, and attended to where
they lie -- prompts and their portions, single tokens, both at once, with or without a sliding window and first tokens that stay visible, and trees of drafted tokens.  Pages are
16-bit, E4M3, or microscaled to eight or four bits (`kv_format`)."""
import array
import ctypes
import math
from typing import List, Optional, Sequence

import torch

from . import _lib

PAGE_SIZE = 16                   # tokens per page (kv_cache.py:25)
TRTLLM_BLOCK_CONSTRAINT = 128    # block_num % (128 / page_size) == 0 (kv_cache.py:28)
_ROWS = {torch.bfloat16: 0, torch.float16: 1}            # KR_KV_*
_PAGES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}
_MICROSCALED = {"mx8": 3, "mx4": 4}
_INT_MAX = 2 ** 31 - 1           # of an argument that the library takes as a C int
MAX_DRAFTS = 64                  # of one sequence in a tree
_Strides = ctypes.c_int64 * 4


class PagedKVCache:
    """A fixed pool of pages for a set of layers on one device (kv_cache.py:31-181).  `cfg` needs: is_mla / is_gqa, attention_type, and
    kv_lora_rank + qk_rope_head_dim (MLA) or num_key_value_heads + gqa_head_dim (GQA).

    kv_format "mx8" or "mx4" (GQA, heads of a multiple of 32 channels; not in the reference class) keeps E4M3 or E2M1 codes with one E8M0 scale byte for every 32 channels in k_scale /
    v_scale: 8.25 and 4.25 bits a channel.  k_cache / v_cache then hold codes (mx4: two a byte, the even channel in the low half) and only KVBatch knows what they stand for."""

    def __init__(self, cfg, num_layers: int, device, max_pages: Optional[int] = None, kv_dtype: torch.dtype = torch.float8_e4m3fn,
                 page_size: int = PAGE_SIZE, combined: bool = False, max_mb: Optional[int] = None,
                 kv_format: Optional[str] = None):
        if kv_format is not None:
            if kv_format not in _MICROSCALED:
                raise ValueError(f"kv_format {kv_format!r}: None, 'mx8' or 'mx4'")
            if not cfg.is_gqa or cfg.gqa_head_dim % 32:
                raise ValueError(f"kv_format {kv_format!r} needs key / value heads of a multiple of 32 channels")
            kv_dtype = torch.float8_e4m3fn if kv_format == "mx8" else torch.uint8
        self.kv_format = kv_format
        self.cfg, self.num_layers, self.device, self.page_size, self.kv_dtype, self.combined = cfg, num_layers, device, page_size, kv_dtype, combined
        self.attention_type = cfg.attention_type
        if cfg.is_mla:
            self.ckv_dim, self.kpe_dim = cfg.kv_lora_rank, cfg.qk_rope_head_dim
            self.kv_cache_dim = self.ckv_dim + self.kpe_dim
            self.num_kv_heads = self.gqa_head_dim = None
        else:
            self.ckv_dim = self.kpe_dim = None
            self.num_kv_heads, self.gqa_head_dim = cfg.num_key_value_heads, cfg.gqa_head_dim
            self.kv_cache_dim = cfg.num_key_value_heads * cfg.gqa_head_dim * 2
        if max_pages is None:
            budget = (2000 if max_mb is None else max_mb) * 1024 * 1024
            max_pages = max(64, budget // self._bytes_per_page())
        self.max_pages = max_pages
        self.k_cache = self.v_cache = self.ckv_cache = self.kpe_cache = self.kv_cache = None
        self.k_scale = self.v_scale = None
        z = lambda *shape: torch.zeros(*shape, dtype=kv_dtype, device=device)
        if cfg.is_gqa:
            width = self.gqa_head_dim // 2 if kv_format == "mx4" else self.gqa_head_dim
            self.k_cache = z(num_layers, max_pages, page_size, self.num_kv_heads, width)
            self.v_cache = z(num_layers, max_pages, page_size, self.num_kv_heads, width)
            if kv_format is not None:
                self.k_scale = torch.zeros(num_layers, max_pages, page_size, self.num_kv_heads, self.gqa_head_dim // 32, dtype=torch.uint8, device=device)
                self.v_scale = torch.zeros_like(self.k_scale)
        elif combined:
            self.kv_cache = z(num_layers, max_pages, page_size, self.kv_cache_dim)
        else:
            self.ckv_cache = z(num_layers, max_pages, page_size, self.ckv_dim)
            self.kpe_cache = z(num_layers, max_pages, page_size, self.kpe_dim)
        self._free_pages: List[int] = list(range(max_pages))
        self._free_pages.reverse()          # pop from the end: pages are handed out in ascending order

    def _bytes_per_page(self) -> int:
        if self.kv_format is not None:
            return self.page_size * self.kv_cache_dim * (33 if self.kv_format == "mx8" else 17) // 32 * self.num_layers
        return self.page_size * self.kv_cache_dim * (1 if self.kv_dtype == torch.float8_e4m3fn else 2) * self.num_layers

    @property
    def max_context_tokens(self) -> int:
        return self.max_pages * self.page_size

    @property
    def free_page_count(self) -> int:
        return len(self._free_pages)

    def alloc_pages(self, n: int) -> List[int]:
        if n > len(self._free_pages):
            raise RuntimeError(f"KV cache exhausted: need {n} pages, have {len(self._free_pages)}")
        return [self._free_pages.pop() for _ in range(n)]

    def free_pages(self, pages: Sequence[int]) -> None:
        self._free_pages.extend(pages)

    def get_layer_caches(self, layer_offset: int):
        assert self.attention_type == "mla" and not self.combined
        return self.ckv_cache[layer_offset], self.kpe_cache[layer_offset]

    def get_combined_layer_cache(self, layer_offset: int) -> torch.Tensor:
        assert self.attention_type == "mla" and self.combined
        return self.kv_cache[layer_offset].unsqueeze(0)

    def get_gqa_layer_caches(self, layer_offset: int):
        assert self.attention_type == "gqa"
        return self.k_cache[layer_offset], self.v_cache[layer_offset]


class SequenceKVState:
    """The pages of one request and its length (kv_cache.py:184-272)."""

    def __init__(self, cache: PagedKVCache, seq_id: int = 0):
        self.cache, self.seq_id = cache, seq_id
        self.pages: List[int] = []
        self.seq_len = 0

    def ensure_capacity(self, new_tokens: int) -> None:
        need = (self.seq_len + new_tokens + self.cache.page_size - 1) // self.cache.page_size
        if need > len(self.pages):
            self.pages.extend(self.cache.alloc_pages(need - len(self.pages)))

    def advance(self, num_tokens: int) -> None:
        self.seq_len += num_tokens

    def free(self) -> None:
        if self.pages:
            self.cache.free_pages(self.pages)
            self.pages = []
            self.seq_len = 0

    def kv_indices(self, device) -> torch.Tensor:
        return torch.tensor(self.pages, dtype=torch.int32, device=device) if self.pages else torch.zeros(0, dtype=torch.int32, device=device)

    def kv_indptr(self, device) -> torch.Tensor:
        return torch.tensor([0, len(self.pages)], dtype=torch.int32, device=device)

    def kv_len_arr(self, device) -> torch.Tensor:
        return torch.tensor([self.seq_len], dtype=torch.int32, device=device)

    def last_page_len(self) -> int:
        if self.seq_len == 0:
            return 0
        rem = self.seq_len % self.cache.page_size
        return rem if rem > 0 else self.cache.page_size

    def last_page_len_tensor(self, device) -> torch.Tensor:
        return torch.tensor([self.last_page_len()], dtype=torch.int32, device=device)

    def block_tables(self, device, pad_to_multiple: int = 8) -> torch.Tensor:
        n = len(self.pages)
        c = TRTLLM_BLOCK_CONSTRAINT // self.cache.page_size
        padded = math.ceil(n / c) * c if n > 0 else c
        table = torch.full((1, padded), -1, dtype=torch.int32, device=device)
        if n > 0:
            table[0, :n] = torch.tensor(self.pages, dtype=torch.int32, device=device)
        return table

    def store_kv_combined(self, layer_offset: int, kv_combined: torch.Tensor, positions: torch.Tensor) -> None:
        assert self.cache.combined, "store_kv_combined requires combined cache"
        ps = self.cache.page_size
        pages = torch.tensor(self.pages, dtype=torch.long, device=kv_combined.device)
        self.cache.kv_cache[layer_offset, pages[positions.long() // ps], positions.long() % ps] = kv_combined.to(self.cache.kv_dtype)

    # ---- not in the reference class: the gather its CpuDecoder._copy_kv_cache does page by page (decode_setup.py:653-711)
    def unpage(self, paged_layer: torch.Tensor, out_dtype: Optional[torch.dtype] = torch.float16) -> torch.Tensor:
        """rows 0 .. seq_len-1 of one layer's paged tensor `[pages, page_size, ...]` as a flat `[seq_len, prod(...)]` tensor; out_dtype None keeps the
        page dtype (E4M3 bytes for a store that runs an FP8 cache), else the exact widening the reference applies (`.to(torch.float16)`)."""
        if getattr(self.cache, "kv_format", None) is not None:
            raise ValueError("microscaled pages hold codes that mean nothing without their scales: KVBatch.stored(cache, [state]).read(layer)")
        if self.seq_len == 0:
            return paged_layer.new_zeros((0, int(paged_layer[0, 0].numel())), dtype=out_dtype or paged_layer.dtype)
        n_pages = (self.seq_len + self.cache.page_size - 1) // self.cache.page_size
        idx = torch.tensor(self.pages[:n_pages], dtype=torch.long, device=paged_layer.device)
        flat = paged_layer[idx].reshape(n_pages * self.cache.page_size, -1)[: self.seq_len]
        return flat if out_dtype is None else flat.to(out_dtype)


def unpage_into_store(store, seq_state: SequenceKVState, layer_map, kv_max_seq: int, conv_states=None, recur_states=None, keep_alive: Optional[list] = None):
    """Hand a paged prompt-pass cache to the decode store (the GPU-paged -> flat copy of decode_setup.py:653-711 followed by set_decode_state).
    layer_map: one entry per decode layer -- None (linear-attention layer: no KV), or the KV layer offset inside `seq_state.cache`.  The flat caches are
    `[kv_max_seq, dim]` in the store's KV element type (FP16, or E4M3 bytes when the store was switched with set_kv_dtype(True) and the pages are FP8).
    Returns the list of (k, v) host arrays (keep them alive as long as the store uses them -- `keep_alive` gets them appended)."""
    import numpy as np
    cache = seq_state.cache
    fp8_store = bool(getattr(store, "_kv_fp8", False))
    microscaled = getattr(cache, "kv_format", None) is not None       # a caller's own cache object may know nothing of it
    if microscaled and fp8_store:
        raise ValueError("microscaled pages go to a store with an FP16 cache (set_kv_dtype(False)): E4M3 without scales does not hold their values")
    batch = KVBatch.stored(cache, [seq_state]) if microscaled and any(off is not None for off in layer_map) else None
    ks, vs, held = [], [], []
    for off in layer_map:
        if off is None:
            ks.append(0); vs.append(0); continue
        if batch is not None:
            a, b = batch.read(off)
        elif cache.attention_type == "gqa":
            a, b = cache.get_gqa_layer_caches(off)
        elif cache.combined:
            both = cache.kv_cache[off]
            a, b = both[..., : cache.ckv_dim], both[..., cache.ckv_dim:]
        else:
            a, b = cache.get_layer_caches(off)
        pair = []
        for t in (a, b):
            keep_bytes = fp8_store and t.dtype == torch.float8_e4m3fn
            flat = (t.flatten(1) if batch is not None else seq_state.unpage(t, None if keep_bytes else torch.float16)).cpu().contiguous()
            host = flat.view(torch.uint8).numpy() if keep_bytes else flat.view(torch.int16).numpy().view(np.uint16)
            full = np.zeros((kv_max_seq, host.shape[1]), host.dtype)
            full[: host.shape[0]] = host
            pair.append(full)
        held.append(tuple(pair)); ks.append(pair[0].ctypes.data); vs.append(pair[1].ctypes.data)
    n = len(layer_map)
    conv = [(c.ctypes.data if c is not None else 0) for c in (conv_states or [None] * n)]
    rec = [(r.ctypes.data if r is not None else 0) for r in (recur_states or [None] * n)]
    store.set_decode_state(seq_state.seq_len, kv_max_seq, ks, vs, conv, rec)
    if keep_alive is not None:
        keep_alive.extend(held)
    return held


class KVBatch:
    """One step over some sequences of a GQA cache on a GPU: `counts[i]` new tokens at the end of `states[i]`, whose pages are taken from the cache here (all or none: a cache that has
    too few raises as `ensure_capacity` does and nothing changes).  Rows of new tokens, one sequence's after the other, are what `write` stores, `read` returns and `attend` asks for;
    `commit` (or, for drafts, `keep`) makes them part of the sequences.  Every call works on torch's current stream of the cache's device and only enqueues.  The calls may be captured
    into a graph (the batch is made before, outlives the graph, and a replay finds the pages as they are then); making a batch copies its plan to the device and may not.
    Making one is host work, 0.07 ms for 8 sequences of 4096 tokens and 0.2 for 32 of 8192: once a step, for all layers.
    Row tensors may have any strides; where a row's channels do not lie together, or rows do not begin at multiples of 16 bytes, a copy is made."""

    def __init__(self, cache: PagedKVCache, states: Sequence[SequenceKVState], counts: Sequence[int], _stored: bool = False):
        states, counts = list(states), [int(c) for c in counts]
        if cache.attention_type != "gqa":
            raise ValueError("KVBatch needs a GQA cache")
        if len(states) != len(counts):
            raise ValueError(f"{len(states)} sequences, {len(counts)} counts")
        if any(c < 0 for c in counts):
            raise ValueError("counts must not be negative")
        if any(s.cache is not cache for s in states):
            raise ValueError("a sequence belongs to another cache")
        if len({id(s) for s in states}) != len(states):
            raise ValueError("a sequence is listed twice")
        if cache.kv_format is None and cache.kv_dtype not in _PAGES:
            raise ValueError(f"pages of {cache.kv_dtype}: bfloat16, float16, float8_e4m3fn, or kv_format 'mx8' / 'mx4'")
        self.cache, self.states, self.counts, self._done = cache, states, counts, _stored
        if not _stored:
            need = [max(0, -(-(s.seq_len + c) // cache.page_size) - len(s.pages)) for s, c in zip(states, counts)]
            if sum(need) > cache.free_page_count:
                raise RuntimeError(f"KV cache exhausted: need {sum(need)} pages, have {cache.free_page_count}")
        if not cache.k_cache.is_cuda:
            raise _lib.KrasisHipError("KVBatch needs its cache on a GPU: krasis_amd has no CPU fallback")
        self.device = cache.k_cache.device
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a KVBatch is made before the capture that uses it")
        if not _stored:
            for s, c in zip(states, counts):
                s.ensure_capacity(c)
        self._lib = _lib.load_library()
        self._host = plan_of(cache, states, counts, _stored)
        self.rows = int(self._host[1])
        self._lens = [x.seq_len for x in states]
        with torch.cuda.device(self.device):
            self._dev = self._host.to(self.device)
            self._stream = torch.cuda.current_stream().cuda_stream
        self._plan = self._host.data_ptr(), self._dev.data_ptr()
        self._format = _MICROSCALED[cache.kv_format] if cache.kv_format is not None else _PAGES[cache.kv_dtype]
        self._pages, self._need = {}, {}

    @classmethod
    def stored(cls, cache: PagedKVCache, states: Sequence[SequenceKVState]) -> "KVBatch":
        """All rows that the sequences hold, to be read back (or attended from, every token as if it were new).  Takes no pages and commits nothing."""
        states = list(states)
        return cls(cache, states, [s.seq_len for s in states], _stored=True)

    def _layer(self, layer: int):
        p = self._pages.get(layer)
        if p is None:
            c = self.cache
            if not 0 <= layer < c.num_layers:
                raise ValueError(f"layer {layer} of {c.num_layers}")
            at = lambda t: None if t is None else t[layer].data_ptr()
            p = _lib.KvPagesC(at(c.k_cache), at(c.v_cache), at(c.k_scale), at(c.v_scale), self._format, c.page_size, c.max_pages, c.num_kv_heads, c.gqa_head_dim)
            self._pages[layer] = p = ctypes.byref(p)
        return p

    def _call(self, fn, *args) -> None:
        stream = torch._C._cuda_getCurrentRawStream(self.device.index)      # torch.cuda.current_stream() without the objects around it: steps are made of calls of a few microseconds
        if stream != self._stream:
            self._dev.record_stream(torch.cuda.current_stream(self.device))      # the plan's memory is not given to anyone else before this stream is done with it
        if torch._C._cuda_getDevice() == self.device.index:
            rc = fn(*args, stream or 1)
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args, stream or 1)
        if rc:
            _lib.check(rc)

    def _rows_of(self, name: str, t: torch.Tensor, heads: int):
        """the rows as a kernel takes them, the two strides and the number of heads; heads 0: any number"""
        d, shape = self.cache.gqa_head_dim, t.shape
        if t.device != self.device or t.dtype not in _ROWS:
            raise ValueError(f"{name}: bfloat16 or float16 rows on {self.device}, not {t.dtype} on {t.device}")
        if len(shape) == 2 and shape[1] % d == 0:
            t = t.unflatten(1, (shape[1] // d, d))
            shape = t.shape
        if len(shape) != 3 or shape[0] != self.rows or shape[2] != d or (heads and shape[1] != heads):
            raise ValueError(f"{name}: {tuple(shape)} for {self.rows} rows of {heads or 'any'} heads of {d} channels")
        st, sh, sd = t.stride()
        if (sd != 1 or st % 8 or sh % 8 or t.data_ptr() % 16) and t.numel():
            t = t.clone(memory_format=torch.contiguous_format)
            st, sh, sd = t.stride()
        return t, st, sh, shape[1]

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor) -> None:
        """The new tokens' keys and values `[rows, kv_heads, dim]` (or `[rows, kv_heads * dim]`) into the pages, in the pages' format."""
        h = self.cache.num_kv_heads
        k, kt, kh, _ = self._rows_of("k", k, h)
        v, vt, vh, _ = self._rows_of("v", v, h)
        if k.dtype != v.dtype:
            raise ValueError(f"k is {k.dtype}, v is {v.dtype}")
        self._call(self._lib.kr_kv_write, self._layer(layer), *self._plan, k.data_ptr(), v.data_ptr(), _Strides(kt, kh, vt, vh), _ROWS[k.dtype])

    def read(self, layer: int, dtype: torch.dtype = torch.float16):
        """The new tokens' keys and values as the pages hold them, `[rows, kv_heads, dim]` each, rounded once to `dtype` (bfloat16 or float16)."""
        if dtype not in _ROWS:
            raise ValueError(f"rows are read as bfloat16 or float16, not {dtype}")
        h, d = self.cache.num_kv_heads, self.cache.gqa_head_dim
        # one allocation, its strides given: a call on few rows takes the time of its host code
        k, v = torch.empty_strided((2, self.rows, h, d), (self.rows * h * d, h * d, d, 1), dtype=dtype, device=self.device).unbind(0)
        self._call(self._lib.kr_kv_read, self._layer(layer), *self._plan, k.data_ptr(), v.data_ptr(), _Strides(h * d, d, h * d, d), _ROWS[dtype])
        return k, v

    def attend(self, layer: int, q: torch.Tensor, scale: Optional[float] = None, window: int = 0, keep_first: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the new tokens' queries `[rows, heads, dim]` over the pages (the new tokens' own keys and values written before): `[rows, heads, dim]` of q's type.
        `window` > 0: a token sees the last `window` tokens up to itself and the sequence's first `keep_first`.  `scale`: dim ** -0.5.  Over 16-bit pages q has their type.
        The order of the sums is fixed by the step's lengths and the sizes: equal calls give equal bits."""
        return self._attend(layer, q, None, scale, window, keep_first, out)

    def attend_tree(self, layer: int, q: torch.Tensor, parents, scale: Optional[float] = None, window: int = 0, keep_first: int = 0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The same where the new tokens are drafts, at most 64 a sequence: `parents` gives for every row the draft of its sequence (counted from 0) that it follows, an earlier one, or
        -1 for the last token before the drafts.  A draft sees what is before the drafts, its ancestors and itself, and stands at its depth after the last token (for the window).
        parents: integers, flat over all rows, or one list for each sequence; what is not on the GPU is checked and copied there, in an int32 tensor on the GPU a number that is no
        earlier draft's counts as -1."""
        return self._attend(layer, q, self._parents(parents), scale, window, keep_first, out)

    def _parents(self, parents) -> torch.Tensor:
        if any(c > MAX_DRAFTS for c in self.counts):
            raise ValueError(f"{max(self.counts)} drafts of a sequence, at most {MAX_DRAFTS}")
        if isinstance(parents, torch.Tensor) and parents.is_cuda:
            if parents.device != self.device or parents.dtype != torch.int32 or parents.shape != (self.rows,):
                raise ValueError(f"parents: int32 [{self.rows}] on {self.device}, not {parents.dtype} {tuple(parents.shape)} on {parents.device}")
            return parents.contiguous()
        parents = parents.tolist() if isinstance(parents, torch.Tensor) else list(parents)
        if parents and hasattr(parents[0], "__len__"):
            if [len(p) for p in parents] != self.counts:
                raise ValueError("parents: one list for each sequence, one number for each of its drafts")
            parents = [x for p in parents for x in p]
        parents = [int(x) for x in parents]
        if len(parents) != self.rows:
            raise ValueError(f"parents: {len(parents)} numbers for {self.rows} rows")
        at = 0
        for c in self.counts:
            for i in range(c):
                if not -1 <= parents[at + i] < i:
                    raise ValueError(f"parents: draft {i} follows {parents[at + i]}, which is no earlier draft")
            at += c
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("parents that are not on the GPU cannot be copied there during a capture")
        return torch.tensor(parents, dtype=torch.int32, device=self.device)

    def _attend(self, layer, q, parents, scale, window, keep_first, out):
        q, qt, qh, heads = self._rows_of("q", q, 0)
        d = self.cache.gqa_head_dim
        if not 0 <= window <= _INT_MAX or not 0 <= keep_first <= _INT_MAX:
            raise ValueError(f"window {window}, keep_first {keep_first}: 0 to {_INT_MAX}")
        if out is None:
            out = torch.empty_strided((self.rows, heads, d), (heads * d, d, 1), dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"out: contiguous {q.dtype} {tuple(q.shape)} on {q.device}, aligned to 16 bytes")
        pages, key = self._layer(layer), (heads, q.dtype, window, keep_first, parents is not None)
        need = self._need.get(key)
        if need is None:
            size = ctypes.c_size_t()
            _lib.check(self._lib.kr_kv_attend_workspace(pages, self._plan[0], heads, _ROWS[q.dtype], window, keep_first, int(parents is not None), ctypes.byref(size)))
            self._need[key] = need = size.value
        ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=self.device) if need else None      # of this call alone: two streams, or two graphs, never share one
        self._call(self._lib.kr_kv_attend, pages, *self._plan, q.data_ptr(), qt, qh, out.data_ptr(), _ROWS[q.dtype], heads, d ** -0.5 if scale is None else scale,
                   window, keep_first, None if parents is None else parents.data_ptr(), None if ws is None else ws.data_ptr(), need)
        return out

    def commit(self) -> None:
        """The new tokens are part of the sequences from here on."""
        self._unfinished()
        self._done = True
        for s, c in zip(self.states, self.counts):
            s.advance(c)

    def keep(self, paths: Sequence[Sequence[int]]) -> None:
        """Of the drafts only a path for each sequence, the accepted ones from the root on (numbers of its drafts, rising): their rows move down in all layers to the places after the
        last token, and the sequences grow by them.  An empty path keeps none.  Pages that are not needed any more stay with the sequence."""
        paths = [[int(i) for i in p] for p in paths]
        if len(paths) != len(self.states):
            raise ValueError(f"{len(paths)} paths for {len(self.states)} sequences")
        for p, c in zip(paths, self.counts):
            if any(not 0 <= i < c for i in p) or any(a >= b for a, b in zip(p, p[1:])):
                raise ValueError(f"path {p}: rising numbers of {c} drafts")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("keep copies its paths to the device: not during a capture")
        self._unfinished()
        start, src, dst, at, slots = [0], [], [], 0, self._host[len(self._host) - self.rows:].tolist()
        for p, c in zip(paths, self.counts):
            for to, i in enumerate(p):
                if to != i:
                    src.append(slots[at + i]); dst.append(slots[at + to])
            start.append(len(src)); at += c
        if src:
            n = len(start)
            moves = torch.tensor(start + src + dst, dtype=torch.int32, device=self.device)
            self._call(self._lib.kr_kv_move, self._layer(0), self.cache.num_layers, len(paths), moves.data_ptr(), moves.data_ptr() + 4 * n, moves.data_ptr() + 4 * (n + len(src)))
        self._done = True                                # not before: a launch that is refused leaves everything as it was
        for s, p in zip(self.states, paths):
            s.advance(len(p))

    def _unfinished(self) -> None:
        if self._done:
            raise RuntimeError("the batch's tokens are part of their sequences already")
        if self._lens != [s.seq_len for s in self.states]:
            raise RuntimeError("a sequence has changed since the batch was made: its new tokens are not where it ends")


def plan_of(cache: PagedKVCache, states: Sequence[SequenceKVState], counts: Sequence[int], stored: bool = False) -> torch.Tensor:
    """What the calls of a step share (kr_kv_plan in include/krasis_hip.h), on the host."""
    ints = lambda x: torch.tensor(list(x), dtype=torch.int32, device="cpu")      # the library follows these: never on a program's default device
    lens = ints(s.seq_len + (0 if stored else c) for s, c in zip(states, counts))
    cnt, sizes, need = ints(counts), ints(len(s.pages) for s in states), ctypes.c_size_t()
    tables = array.array("i")                        # 32 sequences of 500 pages: 0.33 ms; through a tensor of a Python list 1.2
    for s in states:
        tables.fromlist(list(s.pages))
    lib = _lib.load_library()
    args = (cache.max_pages, cache.page_size, len(states), lens.data_ptr(), cnt.data_ptr(), tables.buffer_info()[0] if tables else lens.data_ptr(), sizes.data_ptr())
    _lib.check(lib.kr_kv_plan(*args, None, 0, ctypes.byref(need)))
    plan = torch.empty(need.value, dtype=torch.int32, device="cpu")
    _lib.check(lib.kr_kv_plan(*args, plan.data_ptr(), need.value, ctypes.byref(need)))
    return plan
