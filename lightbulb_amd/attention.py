"""The 8-bit paged key/value cache and attention over it: a decoder layer between its
q/k/v projections and its o projection.

The reference runs this in f32 (``BatchedAttention::forward``, src/model/custom_attention.rs:250-671,
over the paged cache of src/cache/).  Here keys and values are held in 8 bits, int8 or e4m3, with
one scale for each block of tokens (a page) and head:

* ``PageTable``        block tables and free pages on the GPU; ``step`` turns the requests' lengths
                       into tables, slots and positions, ``release`` gives pages back
* ``KvCache``          one layer's codes and scales; ``append`` rotates, quantises and writes
* ``paged_attention``  prompts, single tokens, sliding windows, cross attention
* ``Attention``        projections, append and attention of a layer, beside ``quantized.Mlp``

The arithmetic runs in liblbq's HIP kernels; torch provides memory and the current stream.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .int8 import int8_linear_group
from .quantized import GROUP_MAX, QuantizableLinear, _expect_values, _stream, context, qmatmul_group

#: element types of queries, keys, values and outputs -> the library's type ids
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_KINDS = {"int8": (0, torch.int8), "e4m3": (1, torch.float8_e4m3fn)}
PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 96, 128, 192, 256)
#: lengths and counts go to the library in 32 bits; a bound above that is this one
_MOST = 2 ** 31 - 1


def _expect(name: str, t: torch.Tensor, dtype, device, numel: int | None = None) -> None:
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} on {t.device}, expected {device}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} values, expected {numel}")


def _expect_tables(tables: torch.Tensor) -> None:
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.stride(1) != 1 or not all(tables.shape):
        raise ValueError("block tables must be an int32 tensor [sequences, blocks] with contiguous rows")


class _Fixed:
    """What the library is given as addresses and sizes when the object is made: setting such an attribute
    anew would leave the library with the old ones.  The tensors' contents may change."""

    def __setattr__(self, name, value):
        raise AttributeError(f"a {type(self).__name__}'s {name} is fixed when it is made")


class Step(_Fixed):
    """One step's view of the cache: which pages hold the sequences, and which rows are new.

    ``tables`` int32 [batch, blocks], ``seq_lens`` int32 [batch] (new tokens included) and
    ``cu_new`` int32 [batch + 1] (rows ``cu_new[b]:cu_new[b + 1]`` of q, k and v are sequence b's
    new tokens); ``slots`` int64 and ``positions`` int32 [num_tokens] for an append.  ``max_len``
    and ``max_new`` bound the sequences and their new tokens where the caller knows them: work is
    laid out by them, and what lies beyond them is not served.  0 leaves them open.
    ``granted`` and ``free_count`` are set by ``PageTable.step``; ``taken`` is false for one that took no
    pages (``commit=False``); ``crosses`` says that the rows are another step's (``across``).
    """

    crosses, taken = False, True

    def __init__(self, tables: torch.Tensor, seq_lens: torch.Tensor, cu_new: torch.Tensor, slots: torch.Tensor | None,
                 positions: torch.Tensor | None, *, page_size: int, num_tokens: int, max_len: int = 0, max_new: int = 0,
                 granted: torch.Tensor | None = None, free_count: torch.Tensor | None = None):
        _expect_tables(tables)
        dev, b = tables.device, tables.shape[0]
        _expect("seq_lens", seq_lens, torch.int32, dev, b)
        _expect("cu_new", cu_new, torch.int32, dev, b + 1)
        if slots is not None:
            _expect("slots", slots, torch.int64, dev, num_tokens)
        if positions is not None:
            _expect("positions", positions, torch.int32, dev, num_tokens)
        if min(num_tokens, max_len, max_new) < 0:
            raise ValueError("num_tokens, max_len and max_new must not be negative")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size} is none of {PAGE_SIZES}")
        vars(self).update(
            tables=tables, seq_lens=seq_lens, cu_new=cu_new, slots=slots, positions=positions, page_size=page_size, num_tokens=num_tokens,
            max_len=max_len, max_new=max_new, granted=granted, free_count=free_count, device=tables.device, _struct=_lib.KvStepStruct(
                tables.data_ptr(), tables.stride(0), seq_lens.data_ptr(), cu_new.data_ptr(), slots.data_ptr() if slots is not None else None,
                positions.data_ptr() if positions is not None else None, num_tokens, tables.shape[0], tables.shape[1],
                min(max_len, _MOST), min(max_new, _MOST)),
            _ws={})  # bytes of workspace by heads and head_dim: every layer asks

    def across(self, source: "Step") -> "Step":
        """This step's rows over ``source``'s sequences: cross attention of a decoder's queries
        to an encoder's states, whose lengths and pages are ``source``'s."""
        if source.tables.shape[0] != self.tables.shape[0]:
            raise ValueError(f"{self.tables.shape[0]} sequences across {source.tables.shape[0]}")
        s = Step(source.tables, source.seq_lens, self.cu_new, None, None, page_size=source.page_size, num_tokens=self.num_tokens,
                 max_len=source.max_len, max_new=self.max_new)
        vars(s)["crosses"] = True
        return s


class PageTable(_Fixed):
    """Block tables of ``max_seqs`` sequences over a pool of ``num_pages`` pages, on the GPU.

    ``tables`` int32 [max_seqs, max_blocks] (-1: no page; what stands behind the blocks that a sequence's
    length needs is of no meaning); ``free`` int32 [num_pages], of which the first ``free_count`` are the
    free pages, the last of them taken first.  Several layers' caches share one table.
    """

    def __init__(self, num_pages: int, page_size: int, max_seqs: int, max_blocks: int, device="cuda"):
        if min(num_pages, max_seqs, max_blocks) < 1:
            raise ValueError("a page table needs pages, sequences and blocks")
        dev = torch.device(device)
        self._init(torch.full((max_seqs, max_blocks), -1, dtype=torch.int32, device=dev),
                   torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev),
                   torch.full((1,), num_pages, dtype=torch.int32, device=dev), page_size)

    @classmethod
    def wrap(cls, tables: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, page_size: int) -> "PageTable":
        """Over tensors that the caller holds."""
        self = cls.__new__(cls)
        self._init(tables, free, free_count, page_size)
        return self

    def _init(self, tables, free, free_count, page_size):
        _expect_tables(tables)
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size {page_size} is none of {PAGE_SIZES}")
        _expect("free", free, torch.int32, tables.device)
        _expect("free_count", free_count, torch.int32, tables.device, 1)
        dev, (rows, blocks) = tables.device, tables.shape
        vars(self).update(
            tables=tables, free=free, free_count=free_count, page_size=page_size, device=dev, _ctx=context(dev),
            _ticket=torch.zeros(1, dtype=torch.int32, device=dev), _longs=torch.empty(0, dtype=torch.int64, device=dev),
            # (what a call would ask the tensors for each time: 2 us of a token step's 12)
            _rows=rows, _blocks=blocks, _places=(tables.data_ptr(), tables.stride(0), blocks, page_size, free.data_ptr(), free.numel()))

    def step(self, ctx_lens: torch.Tensor, new_lens: torch.Tensor, num_tokens: int, *, commit: bool = True, max_len: int = 0,
             max_new: int = 0) -> Step:
        """Pages, slots and positions for ``new_lens`` more tokens of sequences that hold ``ctx_lens``
        (int32 [batch] on the GPU; batch row b uses table row b).  Rows 0 .. num_tokens - 1 of q, k
        and v hold the sequences' new tokens in order; what is left over is padding.  A sequence that
        does not fit the free pages, its table row or ``num_tokens`` has ``granted`` 0 and sees nothing; one of a negative
        length has no rows either.  ``commit=False`` works the step out without taking the pages: they stand in the
        tables until another step is worked out, but stay free, and nothing can be appended to them."""
        b, dev = ctx_lens.numel(), self.device
        _expect("ctx_lens", ctx_lens, torch.int32, dev)
        _expect("new_lens", new_lens, torch.int32, dev, b)
        if not 1 <= b <= self._rows:
            raise ValueError(f"a batch of {b} sequences over {self._rows} table rows")
        if num_tokens < 0 or max_len < 0 or max_new < 0:
            raise ValueError("num_tokens, max_len and max_new must not be negative")
        slots = self._longs.new_empty(num_tokens)
        ints = ctx_lens.new_empty(3 * b + 2 + num_tokens)
        seq_lens, cu, granted, positions, left = ints.split_with_sizes((b, b + 1, b, num_tokens, 1))
        p_lens, p_slots = ints.data_ptr(), slots.data_ptr()
        p_cu = p_lens + 4 * b
        p_granted = p_cu + 4 * (b + 1)
        p_pos = p_granted + 4 * b
        p_count = self.free_count.data_ptr()
        if commit:
            left, p_left = self.free_count, p_count
        else:
            p_left = p_pos + 4 * num_tokens
        _lib.check(_lib.lib().lbq_kv_step_build(
            self._ctx, ctx_lens.data_ptr(), new_lens.data_ptr(), b, *self._places, p_count, p_left, self._ticket.data_ptr(), num_tokens,
            p_lens, p_cu, p_granted, p_slots, p_pos, _stream(dev)))
        s = Step.__new__(Step)
        vars(s).update(
            tables=self.tables if b == self._rows else self.tables[:b], seq_lens=seq_lens, cu_new=cu, slots=slots, positions=positions,
            page_size=self.page_size, num_tokens=num_tokens, max_len=max_len, max_new=max_new, granted=granted, free_count=left, device=dev, taken=commit,
            _struct=_lib.KvStepStruct(self._places[0], self._places[1], p_lens, p_cu, p_slots, p_pos, num_tokens, b, self._blocks,
                                      min(max_len, _MOST), min(max_new, _MOST)),
            _ws={})
        return s

    def release(self, lens: torch.Tensor, which: torch.Tensor) -> None:
        """The pages of the sequences b with ``which[b] != 0``, which hold ``lens[b]`` tokens, are free
        again (int32 [batch] on the GPU).  Entries of pages that another sequence still holds are set
        to -1 by the caller first."""
        b = lens.numel()
        _expect("lens", lens, torch.int32, self.device)
        _expect("which", which, torch.int32, self.device, b)
        if not 1 <= b <= self._rows:
            raise ValueError(f"a batch of {b} sequences over {self._rows} table rows")
        _lib.check(_lib.lib().lbq_kv_release(self._ctx, lens.data_ptr(), which.data_ptr(), b, *self._places, self.free_count.data_ptr(),
                                             _stream(self.device)))


class Rotary(_Fixed):
    """Rotary position angles: ``cos`` and ``sin`` f32 [max_pos, rot_dim / 2].  Pairs are channels
    (i, i + rot_dim / 2), or neighbours (2 i, 2 i + 1) where ``interleaved`` (candle's ``rope`` and
    ``rope_i``)."""

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False):
        if cos.dim() != 2 or cos.shape != sin.shape or not all(cos.shape):
            raise ValueError(f"angles must be two tensors [positions, pairs], got {tuple(cos.shape)} and {tuple(sin.shape)}")
        _expect("cos", cos, torch.float32, cos.device)
        _expect("sin", sin, torch.float32, cos.device)
        vars(self).update(cos=cos, sin=sin, interleaved=bool(interleaved), max_pos=cos.shape[0], rot_dim=2 * cos.shape[1])

    @classmethod
    def from_theta(cls, rot_dim: int, max_pos: int, theta: float = 10000.0, interleaved: bool = False, device="cuda") -> "Rotary":
        """Angles pos * theta^(-2 i / rot_dim), formed in 64 bits."""
        half = torch.arange(rot_dim // 2, dtype=torch.float64, device=device)
        angle = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * theta ** (-2 * half / rot_dim)
        return cls(angle.cos().float(), angle.sin().float(), interleaved)


def _rows(name: str, x: torch.Tensor, heads: int | None, dim: int, step: Step) -> int:
    """Checks q, k or v [num_tokens, heads, head_dim]; its type id."""
    t = _DTYPES.get(x.dtype)
    if t is None:
        raise ValueError(f"{name} must be f32, f16 or bf16, got {x.dtype}")
    shape, stride = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != step.num_tokens or shape[2] != dim or (heads is not None and shape[1] != heads):
        raise ValueError(f"{name} {tuple(shape)} is not [{step.num_tokens}, {heads or 'heads'}, {dim}]")
    if stride[2] != 1 and x.numel():
        raise ValueError(f"{name}'s channels are not contiguous")
    if x.device != step.device:
        raise ValueError(f"{name} on {x.device}, step on {step.device}")
    return t


class KvCache(_Fixed):
    """One layer's keys and values: codes ``k`` [pages, kv_heads, page_size, head_dim] and ``v``
    [pages, kv_heads, head_dim, page_size] (values are held transposed), int8 or e4m3, and f32 scales
    ``k_scales`` and ``v_scales`` [pages, kv_heads]; a value is code * scale."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, kind: str = "int8", device="cuda"):
        if kind not in _KINDS:
            raise ValueError(f"cache kind {kind!r} is none of {tuple(_KINDS)}")
        dt, dev = _KINDS[kind][1], torch.device(device)
        shape = (num_pages, kv_heads, page_size, head_dim), (num_pages, kv_heads, head_dim, page_size)
        k, v = (torch.zeros(s, dtype=torch.int8, device=dev).view(dt) for s in shape)
        ks, vs = (torch.zeros(num_pages, kv_heads, device=dev) for _ in range(2))
        self._init(k, v, ks, vs)

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor) -> "KvCache":
        """Over tensors that the caller holds."""
        self = cls.__new__(cls)
        self._init(k, v, k_scales, v_scales)
        return self

    def _init(self, k, v, k_scales, v_scales):
        kinds = {dt: (name, i) for name, (i, dt) in _KINDS.items()}
        if k.dtype not in kinds:
            raise ValueError(f"a cache holds int8 or float8_e4m3fn codes, got {k.dtype}")
        if k.dim() != 4 or not all(k.shape):
            raise ValueError(f"k {tuple(k.shape)} is not [pages, kv_heads, page_size, head_dim]")
        pages, heads, page, dim = k.shape
        if page not in PAGE_SIZES or dim not in HEAD_DIMS:
            raise ValueError(f"page_size {page} and head_dim {dim} must be among {PAGE_SIZES} and {HEAD_DIMS}")
        if tuple(v.shape) != (pages, heads, dim, page):
            raise ValueError(f"v {tuple(v.shape)} is not [pages, kv_heads, head_dim, page_size] of k {tuple(k.shape)}")
        _expect("k", k, k.dtype, k.device)
        _expect("v", v, k.dtype, k.device)
        for name, s in (("k_scales", k_scales), ("v_scales", v_scales)):
            _expect(name, s, torch.float32, k.device, pages * heads)
        name, kind = kinds[k.dtype]
        vars(self).update(
            k=k, v=v, k_scales=k_scales, v_scales=v_scales, kind=name, page_size=page, kv_heads=heads, head_dim=dim, device=k.device,
            _ctx=context(k.device),
            _struct=_lib.KvCacheStruct(k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), pages, kind, page, heads, dim))

    def _fits(self, step: Step) -> None:
        if step.page_size != self.page_size:
            raise ValueError(f"a step of {step.page_size}-token pages over a cache of {self.page_size}-token pages")
        if step.device != self.device:
            raise ValueError(f"step on {step.device}, cache on {self.device}")

    def append(self, k: torch.Tensor, v: torch.Tensor, step: Step, rotary: Rotary | None = None,
               q: torch.Tensor | None = None) -> torch.Tensor | None:
        """Writes the step's keys and values ([num_tokens, kv_heads, head_dim]) into their pages, keys
        rotated by ``rotary`` first, and gives ``q`` [num_tokens, heads, head_dim] rotated likewise.
        Pages that are not there take nothing, and rows of ``q`` without a position are left unset."""
        self._fits(step)
        if not step.taken:
            raise ValueError("the step took no pages (commit=False): they are free, and the next step's")
        t = _rows("k", k, self.kv_heads, self.head_dim, step)
        if _rows("v", v, self.kv_heads, self.head_dim, step) != t:
            raise ValueError(f"k is {k.dtype}, v {v.dtype}")
        if step.slots is None or step.positions is None:
            raise ValueError("an append needs the step's slots and positions")
        out = None
        qp, qs, heads, op = None, (0, 0), 0, None
        if q is not None:
            if _rows("q", q, None, self.head_dim, step) != t:
                raise ValueError(f"k is {k.dtype}, q {q.dtype}")
            heads = q.shape[1]
            out = q.new_empty(q.shape)
            qp, qs, op = q.data_ptr(), q.stride(), out.data_ptr()
        if rotary is None:
            cos = sin = None
            max_pos = rot = inter = 0
        else:
            if rotary.cos.device != self.device:
                raise ValueError(f"angles on {rotary.cos.device}, cache on {self.device}")
            if rotary.rot_dim > self.head_dim:
                raise ValueError(f"{rotary.rot_dim} rotated channels of {self.head_dim}")
            cos, sin, max_pos, rot, inter = rotary.cos.data_ptr(), rotary.sin.data_ptr(), rotary.max_pos, rotary.rot_dim, rotary.interleaved
        if step.num_tokens:
            ks, vs = k.stride(), v.stride()
            _lib.check(_lib.lib().lbq_kv_append(
                self._ctx, self._struct, step._struct, t, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], qp, qs[0], qs[1], heads,
                cos, sin, max_pos, rot, inter, op, _stream(self.device)))
        return out


def paged_attention(q: torch.Tensor, cache: KvCache, step: Step, *, scale: float | None = None, causal: bool | None = None, window: int = 0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """``softmax(scale q k^T) v`` of the step's queries [num_tokens, heads, head_dim] over the cache; each
    ``heads / kv_heads`` query heads share a key/value head.  Causal: row i of a sequence's n new ones is at
    position ``seq_len - n + i`` and sees the tokens up to it, or the last ``window`` of them.  Not causal: all
    of the sequence.  ``causal`` defaults to true, and to false for a step ``across`` other sequences: cross
    attention.  A row that sees nothing is zero; rows behind the last sequence are left as they are.  ``scale``
    defaults to head_dim ** -0.5."""
    cache._fits(step)
    dim, kv = cache.head_dim, cache.kv_heads
    t = _rows("q", q, None, dim, step)
    heads = q.shape[1]
    if heads < 1 or heads % kv:
        raise ValueError(f"{heads} query heads over {kv} key/value heads")
    if causal is None:
        causal = not step.crosses
    if window < 0 or (window and not causal):
        raise ValueError(f"a window of {window} needs a causal mask")
    if out is None:
        out = q.new_empty(q.shape)
    elif out.dtype != q.dtype or out.shape != q.shape or not out.is_contiguous() or out.device != q.device:
        raise ValueError(f"out must be a contiguous {q.dtype} tensor {tuple(q.shape)} on {q.device}")
    if step.num_tokens:
        lib, size = _lib.lib(), step._ws.get((heads, kv, dim))
        if size is None:
            n = ctypes.c_size_t()
            _lib.check(lib.lbq_kv_attention_workspace(cache._ctx, cache._struct, step._struct, heads, n))
            size = step._ws[heads, kv, dim] = n.value
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        qs = q.stride()
        _lib.check(lib.lbq_kv_attention(
            cache._ctx, cache._struct, step._struct, t, q.data_ptr(), qs[0], qs[1], heads, dim ** -0.5 if scale is None else scale, causal,
            window, out.data_ptr(), ws.data_ptr() if ws is not None else None, size, _stream(q.device)))
    return out


class Attention:
    """A layer's attention over ``QuantizableLinear`` projections (``BatchedAttention``,
    src/model/custom_attention.rs:250-282, :671): q, k and v of the input, the append of k and v
    (rotated) to the layer's cache, attention of the rotated queries over it, and the o projection."""

    def __init__(self, q_proj: QuantizableLinear, k_proj: QuantizableLinear, v_proj: QuantizableLinear, o_proj: QuantizableLinear,
                 heads: int, kv_heads: int, head_dim: int, rotary: Rotary | None = None, scale: float | None = None, window: int = 0):
        if heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError(f"{heads} query heads over {kv_heads} key/value heads")
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = q_proj, k_proj, v_proj, o_proj
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.rotary, self.scale, self.window = rotary, scale, window

    def _project(self, xs: torch.Tensor) -> list[torch.Tensor]:
        """q, k and v; quantized projections of one type, or 8-bit integer ones, in one call."""
        projs = (self.q_proj, self.k_proj, self.v_proj)
        groups: dict = {}
        for i, p in enumerate(projs):
            groups.setdefault(p.inner.qtensor().dtype() if p.is_quantized() else "int8" if p.is_int8() else ("dense", i), []).append(i)
        out: list = [None] * 3
        for kind, at in groups.items():
            if not 1 < len(at) <= GROUP_MAX:
                ys = [projs[at[0]].forward(xs)]
            elif kind == "int8":
                ys = int8_linear_group([projs[i].inner for i in at], xs)
            else:
                _expect_values(xs)
                ys = qmatmul_group([projs[i].inner for i in at], xs)
            for i, y in zip(at, ys):
                out[i] = y
        return out

    def forward(self, xs: torch.Tensor, cache: KvCache, step: Step) -> torch.Tensor:
        """``xs`` [.., hidden], ``step.num_tokens`` rows: the step's new tokens in order, as values or, over 8-bit
        integer projections, as ``int8.Int8Tokens``.  Rows behind the last sequence's come out unset."""
        n = step.num_tokens
        q, k, v = (y.view(n, h, self.head_dim) for y, h in zip(self._project(xs), (self.heads, self.kv_heads, self.kv_heads)))
        if self.rotary is None:
            cache.append(k, v, step)
        else:
            q = cache.append(k, v, step, rotary=self.rotary, q=q)
        o = paged_attention(q, cache, step, scale=self.scale, window=self.window)
        return self.o_proj.forward(o.view(*xs.shape[:-1], self.heads * self.head_dim))

    __call__ = forward
