"""A paged KV cache and decoding from it: sequences of any lengths in one batch, memory
by the page, prompts that several samples share (the reference's paged design,
cache/kv_cache.py:293-760, is not wired into its models).

* ``PagedKVCache``    pages of every layer, taken, shared and given back on the host;
* ``RotaryTable``     the position rotation's angles: layout, rotated part, scaling;
* ``PagedBatch``      which sequences a step advances, by which rows, on which pages;
* ``paged_append``    a step's queries and keys rotated, keys and values into pages;
* ``paged_attention`` a step's rows over their sequences' pages;
* ``generate``        ragged prompts, admitted as pages allow, sampled with penalties
  (MixtralDecoder.generate_paged).

A sequence's length is an entry of a device tensor lens [B] (int64, before the step;
negative: it takes no part), so a captured step can be replayed as sequences grow.  On
the GPU each function is one library call (include/hn_int4.h); on the CPU, the same
definitions in torch, also of what is no number: a position that a row does not see has
no effect on it, whatever it holds.
"""
from __future__ import annotations

import ctypes
import math
from typing import Dict, List, Optional, Sequence

import torch

from .. import _lib
from .sampling import adjust_logits
from .speculative import DraftTree, verify_tree

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


class PagedKVCache:
    """Pages of `page_size` positions (a power of two from 16 to 1024) of every layer
    and KV head: k[layer] [pages, kv_heads, page_size, hd], v[layer] [pages, kv_heads,
    page_size / 8, hd, 8] (eight consecutive positions of a dimension side by side, as
    the value product reads them).  The host keeps who uses a page: take, share and
    give count references."""

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int,
                 page_size: int = 64, device=None, dtype=torch.float16):
        shape = (num_pages, num_kv_heads, page_size, head_dim)
        self._set([torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)],
                  [torch.zeros(shape[:2] + (page_size // 8, head_dim, 8), dtype=dtype,
                               device=device) for _ in range(num_layers)])

    @classmethod
    def wrap(cls, k: List[torch.Tensor], v: List[torch.Tensor]) -> "PagedKVCache":
        """A cache over given tensors, one of each kind per layer."""
        c = cls.__new__(cls)
        c._set(list(k), list(v))
        return c

    def _set(self, k, v):
        assert len(k) == len(v) > 0 and k[0].dim() == 4, "k, v: a tensor per layer"
        n, nkv, page, hd = k[0].shape
        assert 16 <= page <= 1024 and page & (page - 1) == 0, \
            f"pages of 16 to 1024 positions, a power of two (got {page})"
        dt, dev = k[0].dtype, k[0].device
        assert all(t.shape == (n, nkv, page, hd) for t in k) \
            and all(t.shape == (n, nkv, page // 8, hd, 8) for t in v) \
            and all(t.dtype == dt and t.device == dev and t.is_contiguous() for t in k + v), \
            "keys [pages, kv_heads, page, hd], values [pages, kv_heads, page / 8, hd, 8], " \
            "contiguous, of one type on one device, in every layer"
        self.k, self.v = k, v
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = n, nkv, page, hd
        self._free = list(range(n - 1, -1, -1))
        self._users = [0] * n

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def pages_for(self, positions: int) -> int:
        return -(-positions // self.page_size)

    def take(self, n: int) -> List[int]:
        """n pages of the free ones."""
        if n > len(self._free):
            raise RuntimeError(f"KV cache full ({n} pages, {len(self._free)} of "
                               f"{self.num_pages} free)")
        got = [self._free.pop() for _ in range(n)]
        for p in got:
            self._users[p] = 1
        return got

    def share(self, pages: Sequence[int]) -> None:
        """One more user of each page."""
        assert all(0 <= p < self.num_pages and self._users[p] > 0 for p in pages), \
            "only pages that are taken can be shared"
        for p in pages:
            self._users[p] += 1

    def give(self, pages: Sequence[int]) -> None:
        """One user less; a page that has none is free again."""
        left: Dict[int, int] = {}
        for p in pages:
            assert 0 <= p < self.num_pages, f"pages 0 to {self.num_pages - 1}"
            left[p] = left.get(p, self._users[p]) - 1
            assert left[p] >= 0, f"page {p} is free already"
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)

    def fork(self, pages: Sequence[int], length: int) -> List[int]:
        """The pages of a further sequence with the same first `length` positions: the
        full ones shared, the last one, which either may go on writing, copied."""
        full, rest = divmod(length, self.page_size)
        used = pages[:full + (rest > 0)]
        assert 0 <= length and len(used) == full + (rest > 0), \
            f"{len(pages)} pages for {length} positions"
        assert all(0 <= p < self.num_pages and self._users[p] > 0 for p in used), \
            "only pages that are taken can be shared"
        mine = self.take(1) if rest else []
        self.share(pages[:full])
        if rest:
            self.copy([pages[full]], mine)
        return list(pages[:full]) + mine

    def copy(self, src: Sequence[int], dst: Sequence[int]) -> None:
        """Page src[i] copied to page dst[i] in every layer.  A page may be a source
        several times, a destination once, and none both."""
        assert len(src) == len(dst) and len(set(dst)) == len(dst) and not set(src) & set(dst), \
            "as many sources as destinations, each destination once and no source"
        assert all(0 <= p < self.num_pages for p in (*src, *dst)), \
            f"pages 0 to {self.num_pages - 1}"
        k0 = self.k[0]
        if not k0.is_cuda:
            for t in self.k + self.v:
                t[list(dst)] = t[list(src)]
            return
        n = len(self.k)
        ptrs, ints = ctypes.c_void_p * n, ctypes.c_int * max(1, len(src))
        _lib.call_on(k0.device, "hn_page_copy", ptrs(*(t.data_ptr() for t in self.k)),
                     ptrs(*(t.data_ptr() for t in self.v)), n,
                     k0[0].numel() * k0.element_size(), self.num_pages, ints(*src), ints(*dst),
                     len(src))

    def table(self, pages: Sequence[Sequence[int]], columns: Optional[int] = None) -> torch.Tensor:
        """int32 [sequences, columns] of the sequences' pages, -1 where there is none."""
        n = max([len(p) for p in pages] + [1]) if columns is None else columns
        rows = [list(p) + [-1] * (n - len(p)) for p in pages]
        return torch.tensor(rows, dtype=torch.int32, device=self.k[0].device).view(len(rows), n)


class RotaryTable:
    """Angles of the position rotation: cos, sin [positions, dim / 2] fp32, angle i of
    position p being p * base^(-2 i / dim), computed in 64 bits.  dim: how many of a
    head's dimensions (the first ones) are rotated, in pairs (i, i + dim / 2) ("half") or
    (2 i, 2 i + 1) ("interleaved").

    scaling, for texts longer than the `original` positions a model was trained on:
      {"type": "linear", "factor": f}    positions divided by f;
      {"type": "ntk", "factor": f}       base * f^(dim / (dim - 2)), which divides the
                                         slowest angle by f and leaves the fastest;
      {"type": "yarn", "factor": f, "original": n, "fast": 32, "slow": 1}
                                         angles that turn more than `fast` times in n
                                         positions stay, those below `slow` turns are
                                         divided by f, between them a linear blend over
                                         the index; cos and sin times 0.1 ln f + 1."""

    LAYOUTS = ("half", "interleaved")

    def __init__(self, dim: int, positions: int, base: float = 1e4, layout: str = "half",
                 scaling: Optional[dict] = None, device=None):
        assert dim >= 0 and dim % 2 == 0 and positions >= 0 and base > 0, \
            f"{dim} rotated dimensions (even), {positions} positions, base {base}"
        i = torch.arange(0, dim, 2, dtype=torch.float64)
        amount, f = 1.0, 1.0
        kind = None if scaling is None else scaling["type"]
        if kind is not None:
            f = float(scaling["factor"])
            assert f >= 1.0 and math.isfinite(f), f"scaling factor {f}"
        if kind == "ntk":
            assert dim > 2, "ntk scaling needs more than one angle"
            base = base * f ** (dim / (dim - 2))
        inv = float(base) ** (-i / max(dim, 1))
        if kind == "linear":
            inv = inv / f
        elif kind == "yarn":
            n = float(scaling["original"])
            fast, slow = float(scaling.get("fast", 32)), float(scaling.get("slow", 1))
            assert n > 0 and fast > slow > 0 and base > 1, \
                f"yarn: original {n}, fast {fast}, slow {slow}, base {base}"

            def index(turns):  # of the angle that turns so often in n positions
                return dim * math.log(n / (2 * math.pi * turns)) / (2 * math.log(base))
            low = max(math.floor(index(fast)), 0)
            high = min(math.ceil(index(slow)), dim - 1)
            keep = 1.0 - ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
            inv = inv * (keep + (1 - keep) / f)
            amount = 0.1 * math.log(f) + 1.0
        else:
            assert kind in (None, "ntk"), f"scaling {kind}: linear, ntk or yarn"
        a = torch.outer(torch.arange(positions, dtype=torch.float64), inv)
        self._set((a.cos() * amount).float().to(device), (a.sin() * amount).float().to(device),
                  layout)

    @classmethod
    def wrap(cls, cos: torch.Tensor, sin: torch.Tensor, layout: str = "half") -> "RotaryTable":
        """Over given tables [positions, dim / 2] fp32 (copies, if they are not contiguous)."""
        r = cls.__new__(cls)
        r._set(cos, sin, layout)
        return r

    def _set(self, cos, sin, layout):
        assert layout in self.LAYOUTS, f"layout {layout}: half or interleaved"
        assert cos.dim() == 2 and cos.shape == sin.shape and cos.device == sin.device \
            and cos.dtype == sin.dtype == torch.float32, "cos, sin: fp32 [positions, dim / 2]"
        self.cos, self.sin, self.layout = cos.contiguous(), sin.contiguous(), layout
        self.dim, self.device = 2 * cos.shape[1], cos.device

    def _args(self):
        """The angles' arguments of a library call."""
        return (self.cos.data_ptr(), self.sin.data_ptr(), self.cos.shape[0], self.dim,
                self.layout == "interleaved")


class PagedBatch:
    """What a step advances, for all of its layers.  table int32 [B, columns]: row b
    names the pages of sequence b in order (PagedKVCache.table); lens int64 [B]: its
    cached positions before the step, negative: it takes no part.  starts int32 [B + 1]
    (not decreasing, from 0): sequence b's new tokens are rows starts[b] to starts[b +
    1] - 1 of the step's `rows`, at most max_new each; None: one row each.  kv_bound: about
    the most positions of a sequence (with the new ones), for the launches' sizes, and so
    the order in which sums are added; the results do not go by it otherwise.  The tensors
    are read when the kernels run, so a captured step may be replayed after they were
    changed in place."""

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, kv_bound: int,
                 starts: Optional[torch.Tensor] = None, rows: Optional[int] = None,
                 max_new: int = 1):
        dev = table.device
        assert table.dtype == torch.int32 and table.dim() == 2 \
            and (table.shape[1] <= 1 or table.stride(1) == 1) \
            and (table.shape[0] <= 1 or table.stride(0) >= table.shape[1]), \
            "table: int32 [B, columns], dense rows"
        B = table.shape[0]
        assert lens.dtype == torch.int64 and tuple(lens.shape) == (B,) and lens.device == dev \
            and lens.is_contiguous(), f"lens: int64 [{B}] on {dev}, contiguous"
        if starts is None:
            assert rows in (None, B) and max_new == 1, f"one row for each of {B} sequences"
            rows = B
        else:
            assert starts.dtype == torch.int32 and tuple(starts.shape) == (B + 1,) \
                and starts.device == dev and starts.is_contiguous(), \
                f"starts: int32 [{B + 1}] on {dev}, contiguous"
            assert rows is not None and rows >= 0 and max_new >= 1 and (B or not rows), \
                "starts needs the step's rows and max_new, rows need a sequence"
        assert kv_bound >= 1, f"kv_bound {kv_bound}"
        self.table, self.lens, self.starts = table, lens, starts
        self.size, self.rows, self.max_new, self.kv_bound = B, rows, max_new, kv_bound
        self.device, self.index = dev, table.get_device()
        self._made = None

    def _step(self, cache: PagedKVCache, num_heads: int):
        """(the C struct of this step over a cache, its address, the attention's workspace),
        made once for all layers."""
        old = self._made
        if old is not None and old[0] is cache and old[1] == num_heads:
            return old[2]
        nkv, hd = cache.kv_heads, cache.head_dim
        assert num_heads > 0 and num_heads % nkv == 0, f"{num_heads} heads over {nkv} KV heads"
        assert hd in (64, 128, 256), f"heads of 64, 128 or 256 (got {hd})"
        assert self.device == cache.k[0].device, \
            f"the batch on {self.device}, the cache on {cache.k[0].device}"
        t = self.table
        s = _lib.PagedStep(t.data_ptr(), max(t.stride(0), t.shape[1]), t.shape[1],
                           cache.num_pages, self.lens.data_ptr(),
                           None if self.starts is None else self.starts.data_ptr(), self.size,
                           self.rows, num_heads, nkv, hd, cache.page_size, self.max_new,
                           self.kv_bound)
        at = ctypes.addressof(s)
        with torch.cuda.device(self.device):  # (it goes by the device's CUs)
            made = (s, at, _lib.lib().hn_paged_attention_workspace_bytes(at))
        self._made = (cache, num_heads, made)
        return made

    def __getstate__(self):  # (a copy's tensors are elsewhere)
        return dict(self.__dict__, _made=None)

    def _runs(self):
        """On the CPU: (sequence, first row, rows, cached positions) of each run."""
        lens = self.lens.tolist()
        ends = list(range(self.size + 1)) if self.starts is None else self.starts.tolist()
        for b, C in enumerate(lens):
            first, end = max(ends[b], 0), min(ends[b + 1], self.rows)
            if end > first:
                yield b, first, end - first, C

    def _pages(self, cache: PagedKVCache, b: int):
        """On the CPU: the named pages of sequence b up to the first that is none."""
        ids = self.table[b].tolist()
        for n, i in enumerate(ids):
            if not 0 <= i < cache.num_pages:
                return ids[:n]
        return ids


def _check(batch: PagedBatch, cache: PagedKVCache, layer: int, x: torch.Tensor,
           columns: int, name: str) -> torch.Tensor:
    """The layer's keys, if the call's tensors fit."""
    assert 0 <= layer < len(cache.k), f"layer {layer} of {len(cache.k)}"
    k = cache.k[layer]
    assert x.shape == (batch.rows, columns), \
        f"{name} {tuple(x.shape)} vs {batch.rows} rows of {columns}"
    at = x.get_device()
    assert at == batch.index and at == k.get_device(), \
        f"{name} on {x.device}, the batch on {batch.device}, the cache on {k.device}"
    assert x.dtype is k.dtype, f"{name} {x.dtype}, the cache {k.dtype}"
    return k


def paged_append(qkv: torch.Tensor, rope: RotaryTable, batch: PagedBatch, cache: PagedKVCache,
                 layer: int, num_heads: int) -> torch.Tensor:
    """The position rotation and the cache append of a step.  qkv [rows, (heads + 2
    kv_heads) * hd]: the fused projection's rows (query heads, keys, values); each is
    rotated at its sequence's length + its place among the sequence's new rows, and its
    key and value go to that position's page.  Returns the rotated queries [rows, heads *
    hd].  fp32 products, rounded once.  Rows of a sequence that takes no part write no
    page and have zero queries, rows of no sequence too; a row past the table of angles,
    or whose page is not named, writes no page and has NaN queries."""
    nkv, hd, T = cache.kv_heads, cache.head_dim, batch.rows
    assert num_heads > 0 and num_heads % nkv == 0, f"{num_heads} heads over {nkv} KV heads"
    columns = (num_heads + 2 * nkv) * hd
    k, v = _check(batch, cache, layer, qkv, columns, "qkv"), cache.v[layer]
    assert rope.device == qkv.device and rope.dim <= hd, \
        f"{rope.dim} rotated dimensions of {hd}, the angles on {rope.device}"
    if qkv.is_cuda:
        assert qkv.dtype in _DTYPES, f"fp16 or bf16 rows (got {qkv.dtype})"
        ld, last = qkv.stride()
        if last != 1 or ld < columns:
            qkv, ld = qkv.contiguous(), columns
        q = qkv.new_empty((T, num_heads * hd))
        held, step, _ = batch._step(cache, num_heads)  # (held: until the call has read it)
        _lib.call_on(qkv.device, "hn_paged_append", step, qkv.data_ptr(), ld,
                     _DTYPES[qkv.dtype], *rope._args(), q.data_ptr(), k.data_ptr(), v.data_ptr())
        return q
    wide = torch.float64 if qkv.dtype == torch.float64 else torch.float32
    q = torch.zeros((T, num_heads, hd), dtype=qkv.dtype)
    n, rd = cache.page_size, rope.dim
    a, b_ = (slice(0, rd, 2), slice(1, rd, 2)) if rope.layout == "interleaved" else \
        (slice(0, rd // 2), slice(rd // 2, rd))
    for b, first, m, C in batch._runs():
        if C < 0:
            continue
        pages, ids = cache.num_pages, batch.table[b]
        pos = min(C, 2 ** 62) + torch.arange(m)
        col = (pos // n).clamp(max=max(ids.shape[0] - 1, 0))
        page = ids[col].long() if ids.shape[0] else torch.full((m,), -1)
        ok = (pos < rope.cos.shape[0]) & (pos // n < ids.shape[0]) & (page >= 0) & (page < pages)
        x = qkv[first:first + m].view(m, num_heads + 2 * nkv, hd)
        q[first:first + m] = math.nan
        x, pos, page = x[ok], pos[ok], page[ok]
        y = x[:, :num_heads + nkv].to(wide)
        cos, sin = rope.cos[pos][:, None].to(wide), rope.sin[pos][:, None].to(wide)
        ya = y[..., a] * cos - y[..., b_] * sin
        y[..., b_] = y[..., b_] * cos + y[..., a] * sin
        y[..., a] = ya
        y = y.to(qkv.dtype)
        q[first:first + m][ok] = y[:, :num_heads]
        slot = pos % n
        k[page, :, slot] = y[:, num_heads:]
        v[page, :, slot // 8, :, slot % 8] = x[:, num_heads + nkv:]
    return q.view(T, num_heads * hd)


def paged_attention(q: torch.Tensor, batch: PagedBatch, cache: PagedKVCache, layer: int,
                    scale: Optional[float] = None) -> torch.Tensor:
    """Attention of a step's rows (paged_append's queries [rows, heads * hd], their keys
    and values in the pages) over the positions up to their own -> [rows, heads * hd].
    scale: of the scores, 1 / sqrt(hd) by default.  Rows of a sequence that takes no
    part and of no sequence are zero; a row that sees a position whose page is not named
    is NaN, and so are the rows of a run of more than the batch's max_new.  An infinite or
    NaN value is in its dimension of the rows that see it, whatever its weight."""
    nkv, hd, T = cache.kv_heads, cache.head_dim, batch.rows
    assert q.dim() == 2 and q.shape[1] % hd == 0, f"q [rows, heads * {hd}]"
    columns = q.shape[1]
    nh = columns // hd
    assert nh > 0 and nh % nkv == 0, f"{nh} heads over {nkv} KV heads"
    k, v = _check(batch, cache, layer, q, columns, "q"), cache.v[layer]
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    assert 0.0 < scale < 2e38, f"scale {scale}"
    if q.is_cuda:
        assert q.dtype in _DTYPES, f"fp16 or bf16 rows (got {q.dtype})"
        ld, last = q.stride()
        if last != 1 or ld % 8 or ld < columns or q.data_ptr() % 16:
            q, ld = _lib.aligned_rows(q.contiguous()), columns
        out = q.new_empty((T, columns))
        held, step, n = batch._step(cache, nh)  # (held: until the call has read it)
        work = q.new_empty((n // 2,)) if n else None  # (two bytes each)
        _lib.call_on(q.device, "hn_paged_attention", step, q.data_ptr(), ld, _DTYPES[q.dtype],
                     k.data_ptr(), v.data_ptr(), scale, out.data_ptr(), columns,
                     None if work is None else work.data_ptr(), n)
        return out
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = torch.zeros((T, nkv, nh // nkv, hd), dtype=q.dtype)
    for b, first, m, C in batch._runs():
        if C < 0:
            continue
        pages = batch._pages(cache, b)
        out[first:first + m] = math.nan
        if m > batch.max_new:
            continue
        m = min(m, len(pages) * cache.page_size - C)  # rows all of whose pages are named
        if m <= 0:
            continue
        L = C + m
        at = torch.tensor(pages[:cache.pages_for(L)])
        kk = k[at].transpose(0, 1).reshape(nkv, -1, hd)[:, :L].to(wide)
        vv = v[at].permute(1, 0, 2, 4, 3).reshape(nkv, -1, hd)[:, :L].to(wide)
        x = torch.einsum("mgrd,gpd->gmrp", q[first:first + m].view(m, nkv, -1, hd).to(wide), kk)
        see = torch.arange(L) <= C + torch.arange(m)[:, None]
        x = (x * scale).masked_fill(~see[None, :, None], -math.inf)
        p = torch.softmax(x, -1)
        # a value that is no number reaches the rows that see it, not the product, where
        # 0 times it would reach every row
        odd = ~vv.isfinite()
        o = torch.einsum("gmrp,gpd->mgrd", p, torch.where(odd, 0.0, vv))
        for g, j, d in odd.nonzero().tolist():
            o[see[:, j], g, :, d] += vv[g, j, d]
        out[first:first + m] = o.to(q.dtype)
    return out.view(T, nh * hd)


class _Slots:
    """The sequences that decode together, in buffers that stay where they are, so that a
    step over them is one captured graph.  Slot i without a sequence has lens[i] = -1."""

    def __init__(self, model, cache: PagedKVCache, n: int, width: int, sampling: dict,
                 temperature: float, words: int, bound: int, graph: bool):
        dev = cache.k[0].device
        long = {"dtype": torch.int64, "device": dev}
        self.model, self.cache, self.n = model, cache, n
        self.sampling, self.temperature = sampling, temperature
        self.tok, self.lens = torch.zeros(n, **long), torch.full((n,), -1, **long)
        self.text, self.prompt = torch.zeros((n, width), **long), torch.zeros(n, **long)
        self.table = torch.full((n, cache.pages_for(width)), -1, dtype=torch.int32, device=dev)
        self.allowed = torch.full((n, words), -1, dtype=torch.int32, device=dev) if words else None
        self.uniforms = torch.zeros((n, 1), device=dev)
        self.batch = PagedBatch(self.table, self.lens, bound)
        self.one = DraftTree.chain(1, dev)
        self.graph = None
        if graph and dev.type == "cuda":
            s = torch.cuda.Stream(device=dev)
            s.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(s):
                self._body()  # warm-up (allocator, library handles): no slot takes part
            torch.cuda.current_stream(dev).wait_stream(s)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.device(dev), torch.cuda.graph(self.graph):  # (on the current device)
                self._body()

    def draw(self, logits, text, lens, prompt, allowed, uniforms):
        """The next token of each row of logits [n, V], whose text so far is given."""
        if self.sampling or allowed is not None:
            logits = adjust_logits(logits, text, lens, prompt, allowed=allowed, **self.sampling)
        zero = torch.zeros_like(uniforms, dtype=torch.int64)
        return verify_tree(logits[:, None], zero, self.one, uniforms, None,
                           self.temperature).token

    def _body(self):
        logits = self.model.forward_paged(self.tok, self.batch, self.cache)
        new = self.draw(logits, self.text, self.lens + 1, self.prompt, self.allowed,
                        self.uniforms)
        live = self.lens >= 0
        self.tok.copy_(torch.where(live, new, 0))
        self.lens.add_(live)
        at = self.lens.clamp(0, self.text.shape[1] - 1)[:, None]
        old = torch.gather(self.text, 1, at)
        self.text.scatter_(1, at, torch.where(live[:, None], new[:, None], old))
        self.tok.clamp_(min=0)  # (a row without a finite logit draws -1)

    def step(self, generator) -> List[int]:
        """One token further for every sequence; the tokens, in the slots' order."""
        if self.temperature > 0:
            self.uniforms.copy_(torch.rand((self.n, 1), generator=generator,
                                           device=self.uniforms.device))
        if self.graph is None:
            self._body()
        else:
            self.graph.replay()
        at = self.lens.clamp(min=0)[:, None]
        return torch.gather(self.text, 1, at)[:, 0].tolist()


@torch.no_grad()
def generate(model, prompts, max_new_tokens: int, temperature: float = 0.0, samples: int = 1,
             generator: Optional[torch.Generator] = None, stop: Sequence[int] = (),
             repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0,
             bias: Optional[Dict[int, float]] = None, allowed=None, max_batch: int = 64,
             cache: Optional[PagedKVCache] = None, page_size: int = 64, chunk: int = 4096,
             graph: bool = True) -> List[List[int]]:
    """Up to max_new_tokens after each of the prompts (sequences of token ids, of any
    lengths) by a MixtralDecoder from a paged cache -> lists of tokens, entry s * prompts
    + b the s-th continuation of prompt b.  A text ends with a token of `stop` (which is
    its last) or at max_new_tokens.

    Up to max_batch texts decode together; a prompt is admitted, with its samples, when
    slots and pages for the whole of them are free, passes in chunks of up to `chunk`
    rows together with others, once for all samples, which share its full pages.
    repetition, presence, frequency, bias {token: value}: as adjust_logits.  allowed(text)
    -> int32 words of the allowed tokens' bits (ceil(vocab / 32)), or None for all: asked
    before each token with the text so far.  cache: pages to use (returned afterwards);
    None: enough for max_batch texts.  graph: decode steps replayed from one captured
    graph.  The device is read back once per step."""
    prompts = [[int(t) for t in p] for p in prompts]
    B, V = len(prompts), model.cfg.vocab_size
    assert samples >= 1 and max_new_tokens >= 1 and max_batch >= samples and chunk >= 1, \
        "samples, tokens, chunk >= 1, max_batch >= samples"
    assert all(p and all(0 <= t < V for t in p) for p in prompts), \
        f"prompts of at least one token, tokens 0 to {V - 1}"
    if not prompts:
        return []
    rows = model.rotary.cos_cached.shape[0]
    longest = max(map(len, prompts)) + max_new_tokens - 1  # (the last token is not cached)
    assert longest <= rows, f"{max_new_tokens} tokens after {max(map(len, prompts))}: the model " \
                            f"has {rows} positions"
    n = min(max_batch, B * samples)
    weight = model.embed_tokens.weight
    dev = weight.device
    if cache is None:
        cfg = model.cfg
        cache = PagedKVCache(cfg.num_layers, n * -(-longest // page_size), cfg.num_kv_heads,
                             cfg.head_dim, page_size, dev, weight.dtype)
    sampling = {}
    if repetition != 1.0 or presence or frequency:
        sampling = {"repetition": repetition, "presence": presence, "frequency": frequency}
    ids = None
    if bias:
        ids = torch.tensor(list(bias), dtype=torch.int64, device=dev)
        values = torch.tensor(list(bias.values()), dtype=torch.float32, device=dev)
        sampling["bias"] = (ids.expand(n, -1).contiguous(), values.expand(n, -1).contiguous())
    words = -(-V // 32) if allowed is not None else 0
    slots = _Slots(model, cache, n, longest + 1, sampling, temperature, words, longest, graph)
    every = torch.full((words,), -1, dtype=torch.int32)

    def bits(text):
        w = allowed(text)
        w = every if w is None else torch.as_tensor(w, dtype=torch.int32).cpu()
        assert tuple(w.shape) == (words,), f"allowed: {words} words (got {tuple(w.shape)})"
        return w

    out: List[List[int]] = [[] for _ in range(B * samples)]
    texts = {}                    # slot -> (entry of out, prompt, pages)
    free = list(range(n - 1, -1, -1))
    waiting = list(range(B - 1, -1, -1))
    coming: List[list] = []       # admitted, not decoding: [prompt, its slots, tokens passed]

    def finish(slot):
        cache.give(texts.pop(slot)[2])
        free.append(slot)

    def emit(slot, token) -> bool:
        entry, b, _ = texts[slot]
        if token < 0:
            raise RuntimeError(f"prompt {b}: no logit is finite")
        out[entry].append(token)
        return len(out[entry]) >= max_new_tokens or token in stop

    def admit():
        while waiting and len(free) >= samples:
            b = waiting[-1]
            P = len(prompts[b])
            whole = cache.pages_for(P + max_new_tokens - 1)
            need = whole + (samples - 1) * (whole - P // cache.page_size)
            if need > cache.free_pages:
                if not texts:
                    raise RuntimeError(f"KV cache full (prompt {b} needs {need} pages, "
                                       f"{cache.free_pages} are free)")
                return
            waiting.pop()
            mine = [free.pop() for _ in range(samples)]
            for s, slot in enumerate(mine):
                if s == 0:
                    pages = first = cache.take(whole)
                else:
                    cache.share(first[:P // cache.page_size])
                    pages = first[:P // cache.page_size]
                    pages = pages + cache.take(whole - len(pages))
                texts[slot] = (s * B + b, b, pages)
            coming.append([b, mine, 0])

    def prefill():
        """One step over rows of the prompts that were admitted; those that it ends draw
        their first tokens and decode from then on."""
        step, left = [], chunk
        for job in coming:
            m = min(left, len(prompts[job[0]]) - job[2])
            if m > 0:
                step.append((job, m))
                left -= m
        starts, tokens, last = [0], [], []
        for (b, mine, done), m in step:
            tokens += prompts[b][done:done + m]
            starts.append(len(tokens))
            if done + m == len(prompts[b]):
                last.append(len(tokens) - 1)
        lens = torch.tensor([done for (_, _, done), _ in step], device=dev)
        batch = PagedBatch(cache.table([texts[mine[0]][2] for (_, mine, _), _ in step]), lens,
                           max(done + m for (_, _, done), m in step),
                           torch.tensor(starts, dtype=torch.int32, device=dev), len(tokens),
                           max(m for _, m in step))
        logits = model.forward_paged(torch.tensor(tokens, device=dev), batch, cache,
                                     2, torch.tensor(last, dtype=torch.int64, device=dev))
        ended = []
        for job, m in step:
            job[2] += m
            if job[2] == len(prompts[job[0]]):
                coming.remove(job)
                ended.append(job)
        if not ended:
            return
        src, dst = [], []  # the samples' own copies of the last page
        for b, mine, P in ended:
            full, rest = divmod(P, cache.page_size)
            if rest:
                src += [texts[mine[0]][2][full]] * (samples - 1)
                dst += [texts[s][2][full] for s in mine[1:]]
        if src:
            cache.copy(src, dst)
        at = [s for _, mine, _ in ended for s in mine]
        where = torch.tensor(at, device=dev)
        width = slots.text.shape[1]
        rows_ = [prompts[b] + [0] * (width - len(prompts[b])) for b, _, _ in ended]
        text = torch.tensor(rows_, dtype=torch.int64, device=dev).repeat_interleave(samples, 0)
        size = torch.tensor([P for _, _, P in ended], device=dev).repeat_interleave(samples)
        grammar = None
        if allowed is not None:
            grammar = torch.stack([bits(prompts[b]) for b, _, _ in ended]).to(dev)
            grammar = grammar.repeat_interleave(samples, 0)
        uniforms = torch.rand((len(at), 1), generator=generator, device=dev)
        mine = slots.sampling
        if ids is not None:
            slots.sampling = dict(mine, bias=tuple(x[:len(at)] for x in mine["bias"]))
        new = slots.draw(logits.repeat_interleave(samples, 0), text, size, size, grammar,
                         uniforms)
        slots.sampling = mine
        text.scatter_(1, size[:, None], new[:, None])
        slots.text[where], slots.prompt[where] = text, size
        slots.tok[where] = new.clamp(min=0)
        slots.table[where] = cache.table([texts[s][2] for s in at], slots.table.shape[1])
        slots.lens[where] = size
        over = [s for s, t in zip(at, new.tolist()) if emit(s, t)]
        leave(over)

    def leave(over):
        for s in over:
            finish(s)
        if over:
            slots.lens[torch.tensor(over, device=dev)] = -1

    try:
        while waiting or texts:
            admit()
            if coming:
                prefill()
                continue
            if allowed is not None:
                rows_ = [every] * n
                for s, (entry, b, _) in texts.items():
                    rows_[s] = bits(prompts[b] + out[entry])
                slots.allowed.copy_(torch.stack(rows_))
            tokens = slots.step(generator)
            leave([s for s in list(texts) if emit(s, tokens[s])])
    finally:
        for _, _, pages in texts.values():
            cache.give(pages)
    return out
