"""Attention between a decoder layer's quantized projections: rotary
positions, attention of packed sequences (with its gradient), a paged cache
of keys and values, and attention of new tokens over it.  The reference has no
counterpart: it leaves a model's attention to the model's own modules.

Layouts.  Heads are rows of packed tokens: queries (T, heads, head_dim), keys
and values (T, kv_heads, head_dim), one sequence after the other; query head h
reads key head h // (heads / kv_heads).  The heads may be parts of a fused
projection's output (any strides, the last dimension contiguous): nothing is
copied then.  ``cu_seqlens`` holds the B + 1 offsets of the sequences (int32
on the GPU, the first 0); tokens past the last one give zeros.  A cache is
(pages, page_size, kv_heads, head_dim); a sequence's block table row names its
pages in order.  Offsets, positions, slots, lengths and page numbers may be int64
too, which takes two small launches more.

The functions run on the current stream, allocate from torch's caching
allocator, do not wait for the GPU, and can be captured in a graph
(``PagedKVCache.extend`` waits, and can not).  There is no CPU path.  Forward-mode
derivatives raise, as do gradients of what has none.
"""
from __future__ import annotations

import itertools
import math
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Tuple

import torch
import torch.nn as nn

from .. import _lib as L

CODES = (torch.int8, torch.float8_e4m3fn)  # what a quantised cache holds, beside fp32 scales

_ops: dict = {}  # name -> operator, once its library is loaded


def _op(name: str, *args):
    """Call operator gptq::name; a status of the library is raised as its own
    error type."""
    op = _ops.get(name)
    if op is None:
        L.load_torch_ops()
        op = _ops[name] = getattr(torch.ops.gptq, name).default
    try:
        return op(*args)
    except NotImplementedError:
        raise RuntimeError(f"gptq::{name}: expected GPU tensors (there is no CPU path)") from None
    except RuntimeError as e:
        L.reraise(e)


def _needs_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t.requires_grad for t in ts)


def _scale(q: torch.Tensor, scale: Optional[float]) -> float:
    return 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)


# ------------------------------------------------------------------ rotary --

def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                       device=None) -> Tuple[torch.Tensor, float]:
    """The angle per position of each pair of channels, base^(-2 i / rotary_dim)
    (float64), and the factor of cosines and sines.  ``scaling`` (for contexts
    longer than those of training) is one of

    * ``{"type": "linear", "factor": f}``: every angle divided by f;
    * ``{"type": "ntk", "factor": f}``: base times f^(d / (d - 2)), which leaves
      the highest frequency and divides the lowest by f;
    * ``{"type": "bands", "factor": f, "low": a, "high": b, "context": n}``:
      frequencies of fewer than a turns over the n positions of training are
      divided by f, those of more than b kept, those between mixed linearly in
      their turns;
    * ``{"type": "yarn", "factor": f, "context": n, "low": 1, "high": 32}``
      (Peng et al., "YaRN"): the same mixed linearly in the channel's number
      between the two bounds, and cosines and sines times 0.1 ln f + 1 (or
      ``"attention_factor"``)."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim has to be even, got {rotary_dim}")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    kind = (scaling or {}).get("type")
    factor = float((scaling or {}).get("factor", 1.0))
    if scaling and factor < 1.0:
        raise ValueError(f"a scaling factor of {factor}: it has to be at least 1")
    if kind == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs rotary_dim >= 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    inv = float(base) ** (-i / rotary_dim)
    if not scaling or kind == "ntk":
        return inv, 1.0
    if kind == "linear":
        return inv / factor, 1.0
    n = float(scaling["context"]) if kind in ("bands", "yarn") else 0.0
    if kind == "bands":
        low, high = float(scaling["low"]), float(scaling["high"])
        keep = ((n * inv / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        return inv / factor * (1 - keep) + inv * keep, 1.0
    if kind == "yarn":
        low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 32.0))

        def channel(turns):  # the pair of channels that turns so often over the context
            return rotary_dim * math.log(n / (turns * 2 * math.pi)) / (2 * math.log(base))
        first, last = max(math.floor(channel(high)), 0), min(math.ceil(channel(low)), rotary_dim - 1)
        drop = ((i / 2 - first) / max(last - first, 1e-3)).clamp(0.0, 1.0)
        mscale = float(scaling.get("attention_factor", 0.1 * math.log(factor) + 1.0))
        return inv / factor * drop + inv * (1 - drop), mscale
    raise ValueError(f"unknown rotary scaling {kind!r}")


def rotary_table(rotary_dim: int, positions: int, base: float = 10000.0, scaling: Optional[dict] = None,
                 device="cuda") -> torch.Tensor:
    """Cosines and sines (positions, 2, rotary_dim / 2) of positions 0, 1, ...,
    computed in float64 (a float32 angle of a late position is off by 1e-3)."""
    inv, factor = rotary_frequencies(rotary_dim, base, scaling, device)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return (torch.stack([a.cos(), a.sin()], 1) * factor).float()


def rotary(q: torch.Tensor, k: torch.Tensor, table: torch.Tensor, positions: torch.Tensor,
           interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """q (T, heads, head_dim) and k (T, kv_heads, head_dim), fp32, fp16 or
    bf16, with the first 2 * table.shape[2] channels of each head turned by the
    angles of ``positions`` (T): pairs (i, i + half), or with ``interleaved``
    (2i, 2i + 1).  ``table`` is ``rotary_table``'s; positions outside it are
    turned by the angles of its ends."""
    return _op("rotary", q, k, table, positions, interleaved, False)


def norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                table: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                interleaved: bool = False, eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor]:
    """``rotary`` of normed heads in one pass: each head of q and k over its root
    mean square, x (mean x^2 + eps)^-1/2, times ``q_weight`` or ``k_weight``
    (head_dim values, the same for all heads; fp32, fp16 or bf16), then turned.
    ``table`` None: only normed.  head_dim a multiple of 8 up to 256, the turned
    channels of 4; ``eps`` within [1e-12, 1].  Computed in fp32 and rounded once;
    differentiable in q, k and the weights (once), whose gradients are the same
    bits from call to call."""
    return _op("norm_rotary", q, k, q_weight, k_weight, table, positions, interleaved, eps)


def rotary_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: Optional[torch.Tensor],
                  positions: Optional[torch.Tensor], k_cache: torch.Tensor, v_cache: torch.Tensor,
                  slots: torch.Tensor, interleaved: bool = False, *, k_scale: Optional[torch.Tensor] = None,
                  v_scale: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                  k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6) -> torch.Tensor:
    """``rotary`` for new tokens in one launch with the cache's update: returns
    the turned queries and writes the turned keys and the values of token t into
    place ``slots[t]`` (page * page_size + row) of the cache.  Tokens with a
    negative slot (padding) are not written.  ``table`` None: positions are not
    rotary, nothing is turned; positions outside it are turned by the angles of
    its ends.  For serving: no gradient is recorded.

    ``q_weight`` and ``k_weight``: the heads are normed first, as in
    ``norm_rotary``.  A cache of int8 or float8_e4m3fn holds codes (head_dim a
    multiple of 16, the turned channels of 8), and ``k_scale`` and ``v_scale``
    (pages, page_size, kv_heads; float32) the scale of each token's head: its
    largest value over 127 or 448.  Codes are of the fp32 values, rounded to the
    nearest; heads up to 2^-120 read back as zeros, ones with values that are not
    finite as NaN."""
    if _needs_grad(q, k, v):
        raise RuntimeError("rotary_append records no gradient: call it under torch.no_grad()")
    if k_scale is None and v_scale is None and q_weight is None and k_weight is None and k_cache.dtype not in CODES:
        return _op("rotary_append", q, k, v, table, positions, k_cache, v_cache, slots, interleaved)
    return _op("norm_rotary_append", q, k, v, q_weight, k_weight, table, positions, k_cache, v_cache, slots, k_scale,
               v_scale, interleaved, eps)


# --------------------------------------------------------------- attention --

def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
              cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True,
              scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of each packed sequence and head, fp16 or bf16,
    head_dim a multiple of 8 up to 128; differentiable in q, k and v (once).

    ``cu_seqlens``: offsets of the sequences' queries (None: one sequence), and
    of their keys unless ``cu_seqlens_k`` gives those.  ``causal``: the last
    query sees the last key, the one before it one key less, and so on; a query
    without a key gives zeros, and gradients of zero.  ``scale``: 1 / sqrt(head_dim)
    by default, else within [1e-7, 1e7].  Infinities and NaN reach only the rows
    and gradients whose sums they are terms of; sums that are infinite are made
    a second time, at up to 20 times a finite call's time."""
    return _op("attention", q, k, v, cu_seqlens, cu_seqlens_k, causal, _scale(q, scale))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                    context_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None, max_context: Optional[int] = None, *,
                    k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of new tokens, q (T, heads, head_dim), over the cache,
    which holds their own keys and values already (``rotary_append``).

    ``context_lens`` (B): cached tokens of each sequence, the new ones among
    them; the last new token sees them all, the one before it one less.
    ``block_table`` (B, pages): the sequence's pages, entries past its context
    unused.  ``cu_seqlens``: offsets of the sequences' new tokens (None: one
    token each).  ``max_context``: the longest context where it is known, for
    the choice of kernel (by default what the block table could hold).

    ``k_scale`` and ``v_scale``: those of a cache of codes (``rotary_append``),
    whose rows are code times scale; q is fp16 or bf16.  A row whose scale is NaN
    reaches the queries that see it only.  A value's code that is NaN, which
    ``rotary_append`` never writes, may reach those before it too.  One kernel, by
    the average number of new tokens, takes all sequences: a long chunk beside many
    single tokens is faster as a call for each kind."""
    if _needs_grad(q, k_cache, v_cache):
        raise RuntimeError("paged_attention records no gradient: call it under torch.no_grad()")
    if max_context is None:
        max_context = block_table.shape[-1] * k_cache.shape[1]
    if k_cache.dtype in CODES or k_scale is not None or v_scale is not None:
        if k_scale is None or v_scale is None or k_cache.dtype not in CODES:
            raise ValueError(f"paged_attention: a cache of {k_cache.dtype} "
                             + ("needs the scales of its keys and values" if k_cache.dtype in CODES else "has no scales"))
        return _op("code_attention", q, k_cache, v_cache, block_table, context_lens, cu_seqlens, k_scale, v_scale,
                   _scale(q, scale), max_context)
    return _op("paged_attention", q, k_cache, v_cache, block_table, context_lens, cu_seqlens, _scale(q, scale),
               max_context)


def cached_rows(k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor,
                cu_seqlens: torch.Tensor, tokens: int, dtype: Optional[torch.dtype] = None, *,
                k_scale: Optional[torch.Tensor] = None,
                v_scale: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values (tokens, kv_heads, head_dim) read back from the cache: of
    sequence b the last cu_seqlens[b + 1] - cu_seqlens[b] of its
    ``context_lens[b]`` cached tokens.  Rows that a sequence does not have, and
    rows behind the last sequence, are zeros.  A cache of codes (``k_scale``,
    ``v_scale``) is read as code times scale in fp32, rounded to ``dtype`` (fp16,
    bf16 or fp32; bf16 by default); another cache has its own type.  No gradient
    is recorded."""
    if dtype is None:
        dtype = torch.bfloat16 if k_cache.dtype in CODES else k_cache.dtype
    return _op("cached_rows", k_cache, v_cache, block_table, context_lens, cu_seqlens, tokens, k_scale, v_scale, dtype)


# ------------------------------------------------------------------- cache --

@dataclass
class PagedBatch:
    """What one step over a cache needs on the GPU, for new tokens of B
    sequences, T together: views of one int32 tensor."""
    positions: torch.Tensor      # (T) place of each token in its sequence
    slots: torch.Tensor          # (T) place of each token in the cache
    context_lens: torch.Tensor   # (B)
    block_table: torch.Tensor    # (B, pages of the longest)
    cu_seqlens: Optional[torch.Tensor]  # (B + 1), None where every sequence has one token
    max_context: int


class PagedKVCache:
    """Keys and values of ``layers`` layers in pages of ``page_size`` tokens,
    (pages, page_size, kv_heads, head_dim) each, and which page belongs to which
    sequence (on the host).  All layers share the pages' numbers.  Places that
    no token was written to are never read.

    ``dtype`` int8 or float8_e4m3fn: a quantised cache of codes, with ``k_scale``
    and ``v_scale`` (layers, pages, page_size, kv_heads), None of another cache;
    head_dim is a multiple of 16.  A head's rows of a page lie next to each other
    then: 2 KB at a time for pages of 16 tokens and heads of 128, where a token's
    heads side by side would leave 128 bytes."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, layers: int = 1,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        if pages < 1 or page_size < 1 or layers < 1:
            raise ValueError(f"a cache of {layers} layers, {pages} pages of {page_size} tokens")
        if pages * page_size > 1 << 31:
            raise ValueError(f"{pages} pages of {page_size} tokens: a cache has at most 2^31 places, which slots can name")
        self.k_scale: Optional[torch.Tensor] = None
        self.v_scale: Optional[torch.Tensor] = None
        if dtype in CODES:
            if head_dim % 16:
                raise ValueError(f"a quantised cache of heads of {head_dim} values (multiples of 16 are supported)")
            rows = (layers, pages, kv_heads, page_size)
            self.k, self.v = (torch.empty(*rows, head_dim, dtype=dtype, device=device).transpose(2, 3) for _ in "kv")
            self.k_scale, self.v_scale = (torch.empty(rows, device=device).transpose(2, 3) for _ in "kv")
        else:
            shape = (layers, pages, page_size, kv_heads, head_dim)
            self.k = torch.empty(shape, dtype=dtype, device=device)
            self.v = torch.empty(shape, dtype=dtype, device=device)
        self.page_size = page_size
        self._free: List[int] = list(range(pages - 1, -1, -1))
        self._pages: Dict[object, List[int]] = {}
        self._lens: Dict[object, int] = {}

    def __contains__(self, seq) -> bool:
        return seq in self._lens

    def length(self, seq) -> int:
        """Cached tokens of a sequence."""
        return self._lens[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def scales(self, layer: int = 0) -> Dict[str, torch.Tensor]:
        """``k_scale`` and ``v_scale`` of a layer as the functions' arguments (none
        of a cache that has none)."""
        if self.k_scale is None:
            return {}
        return {"k_scale": self.k_scale[layer], "v_scale": self.v_scale[layer]}

    def rows(self, seqs: Sequence, layer: int = 0,
             dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """All cached keys and values of some sequences as packed rows
        (``cached_rows``), and the sequences' offsets.  Waits for the GPU as
        ``extend`` does."""
        seqs = list(seqs)
        if not seqs or not all(s in self._lens for s in seqs):
            raise ValueError("rows: some sequences of the cache")
        lens = [self._lens[s] for s in seqs]
        width = max(len(self._pages[s]) for s in seqs)
        table = [p for s in seqs for p in self._pages[s] + [0] * (width - len(self._pages[s]))]
        parts = [table, lens, [0, *itertools.accumulate(lens)]]
        t = torch.tensor(list(itertools.chain(*parts)), dtype=torch.int32).to(self.k.device)
        b, c, o = t.split([len(x) for x in parts])
        k, v = cached_rows(self.k[layer], self.v[layer], b.view(len(seqs), width), c, o, sum(lens), dtype,
                           **self.scales(layer))
        return k, v, o

    def free(self, seq) -> None:
        """Forget a sequence; its pages can be given to others."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lens[seq]

    def extend(self, seqs: Sequence, new: Sequence[int]) -> PagedBatch:
        """Places for ``new[b]`` more tokens of sequence ``seqs[b]`` (unknown ones
        begin here), and the step's tensors.  Raises MemoryError, and changes
        nothing, when the pages do not suffice.

        The host makes all sequences' whole block tables on each call (0.3-0.6 ms
        for one of 8192 pages, 0.9-1.7 ms for 48 of 512) and copies them from pageable
        memory, which waits for what the current stream has been given."""
        seqs, new = list(seqs), [int(n) for n in new]
        if not seqs or len(seqs) != len(new) or len(set(seqs)) != len(seqs) or min(new) < 1:
            raise ValueError("extend: one count of new tokens, at least 1, for each of some different sequences")
        ps = self.page_size
        need = [-(-(self._lens.get(s, 0) + n) // ps) - len(self._pages.get(s, ())) for s, n in zip(seqs, new)]
        if sum(need) > len(self._free):
            raise MemoryError(f"the cache has {len(self._free)} free pages, {sum(need)} are needed")
        positions: List[int] = []
        slots: List[int] = []
        for s, n, k in zip(seqs, new, need):
            pages = self._pages.setdefault(s, [])
            pages.extend(self._free.pop() for _ in range(k))
            first = self._lens.get(s, 0)
            self._lens[s] = first + n
            positions.extend(range(first, first + n))
            slots.extend(pages[p // ps] * ps + p % ps for p in range(first, first + n))
        context = [self._lens[s] for s in seqs]
        width = max(len(self._pages[s]) for s in seqs)
        table = [p for s in seqs for p in self._pages[s] + [0] * (width - len(self._pages[s]))]
        cu = [0, *itertools.accumulate(new)] if max(new) > 1 else []
        parts = [positions, slots, context, table, cu]
        # one copy for all of them
        t = torch.tensor(list(itertools.chain(*parts)), dtype=torch.int32).to(self.k.device)
        p, s, c, b, o = t.split([len(x) for x in parts])
        return PagedBatch(p, s, c, b.view(len(seqs), width), o if cu else None, max(context))


def packed_positions(cu_seqlens: torch.Tensor, tokens: int) -> torch.Tensor:
    """Each packed token's place in its sequence (int32, on the GPU)."""
    at = torch.arange(tokens, device=cu_seqlens.device, dtype=torch.int32)
    first = cu_seqlens[torch.searchsorted(cu_seqlens, at, right=True).sub_(1).clamp_(min=0)]
    return at - first.to(torch.int32)


class QuantizedAttention(nn.Module):
    """A decoder layer's attention over quantized projections: ``qkv`` gives
    queries, keys and values of packed tokens (a ``FusedQuantizedLinear`` of the
    three), ``o`` takes the heads' outputs.  ``table`` (``rotary_table``) None:
    positions are not rotary.  ``q_norm`` and ``k_norm`` (head_dim weights each, or
    neither): the heads are normed before they are turned (``norm_rotary``); they
    become parameters.

    ``forward`` runs whole packed sequences, for prompts, calibration and
    training; ``step`` runs new tokens over a ``PagedKVCache``, a quantised one
    too.  Both raise ValueError where the host knows that a position is past the
    table: one sequence longer than it, a step whose longest context is.
    Sequences by ``cu_seqlens`` and given positions are not looked at; positions
    past the table are turned by its last angles."""

    def __init__(self, qkv: nn.Module, o: nn.Module, heads: int, kv_heads: int, head_dim: int,
                 table: Optional[torch.Tensor] = None, interleaved: bool = False, scale: Optional[float] = None,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6):
        super().__init__()
        if (q_norm is None) != (k_norm is None):
            raise ValueError("QuantizedAttention: the queries' norm without the keys', or these without those")
        for w in (q_norm, k_norm):
            if w is not None and tuple(w.shape) != (head_dim,):
                raise ValueError(f"QuantizedAttention: a norm of {tuple(w.shape)} weights for heads of {head_dim}")
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads over {kv_heads} key heads")
        self.qkv, self.o = qkv, o
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.interleaved, self.scale, self.eps = interleaved, scale, eps
        self.q_norm = None if q_norm is None else nn.Parameter(q_norm.detach().clone())
        self.k_norm = None if k_norm is None else nn.Parameter(k_norm.detach().clone())
        self.register_buffer("table", table, persistent=False)

    def _apply(self, fn, recurse=True):
        # a cast of the module's dtype leaves the angles in 32 bits
        table = self.table
        super()._apply(fn, recurse)
        if table is not None and table.dtype == torch.float32 and self.table.dtype != torch.float32:
            self.table = table.to(self.table.device)
        return self

    def _check_length(self, n: int) -> None:
        if self.table is not None and n > self.table.shape[0]:
            raise ValueError(f"a sequence of {n} tokens: the rotary table has {self.table.shape[0]} positions")

    def _heads(self, x: torch.Tensor):
        q, k, v = self.qkv(x)
        d = self.head_dim
        return q.unflatten(-1, (self.heads, d)), k.unflatten(-1, (self.kv_heads, d)), \
            v.unflatten(-1, (self.kv_heads, d))

    def forward(self, x: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x (T, hidden): packed sequences (None: one), causal."""
        if cu_seqlens is None and positions is None:
            self._check_length(x.shape[0])
        q, k, v = self._heads(x)
        if self.table is not None:
            if positions is None:
                positions = (torch.arange(x.shape[0], device=x.device, dtype=torch.int32) if cu_seqlens is None
                             else packed_positions(cu_seqlens, x.shape[0]))
        if self.q_norm is not None:
            q, k = norm_rotary(q, k, self.q_norm, self.k_norm, self.table, positions if self.table is not None else None,
                               self.interleaved, self.eps)
        elif self.table is not None:
            q, k = rotary(q, k, self.table, positions, self.interleaved)
        y = attention(q, k, v, cu_seqlens, scale=self.scale)
        return self.o(y.flatten(-2))

    @torch.no_grad()
    def step(self, x: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, layer: int = 0) -> torch.Tensor:
        """x (T, hidden): the batch's new tokens (``cache.extend``), whose keys
        and values are stored on the way."""
        self._check_length(batch.max_context)
        q, k, v = self._heads(x)
        kc, vc = cache.k[layer], cache.v[layer]
        scales = cache.scales(layer)
        norms = {} if self.q_norm is None else {"q_weight": self.q_norm, "k_weight": self.k_norm, "eps": self.eps}
        q = rotary_append(q, k, v, self.table, batch.positions, kc, vc, batch.slots, self.interleaved, **scales, **norms)
        y = paged_attention(q, kc, vc, batch.block_table, batch.context_lens, batch.cu_seqlens, self.scale,
                            batch.max_context, **scales)
        return self.o(y.flatten(-2))
