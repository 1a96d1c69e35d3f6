"""Paged key / value cache over the C ABI: claim, write, fork, copy, compact and free pages, and attention over them.

K and V are pools ``[layers, pages, Hkv, page tokens, D]`` (bf16, f16, or E4M3 with one factor per layer and kv head).
A slot is one sequence: its row of ``page_table`` names its pages in order (-1 behind them), ``seq_lens`` its tokens,
``ref_counts`` how many slots hold a page.  Everything lives on the device and no call synchronises, so a serving step
(extend, write, attend) can be captured into a graph; lists of slots and pages are int32 CUDA tensors.  Calls on one
cache have to be ordered on the device, as they change it."""

from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib
from ._lib import check, lib, ptr

# A decoding step makes several calls of a few microseconds: what one costs on the host counts.  Arguments are packed in one
# go (native alignment: the layout of the C structs), and a call of the current device takes no device guard.
_WRITE = struct.Struct("@PP3q3q4iPP")
_ATTEND = struct.Struct("@P3qP3qP5ifP2iPPP")

_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream

_LARGEST = torch.finfo(torch.float32).max
KV_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float8_e4m3fn: 2}


def _pool(t, name: str):
    if not isinstance(t, torch.Tensor) or t.ndim != 5:
        raise ValueError(f"{name} must be a [layers, pages, Hkv, page tokens, D] tensor")
    if t.dtype not in KV_DTYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float8_e4m3fn, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on a CUDA device (there is no CPU path)")
    _, _, heads, tokens, d = t.shape
    if t.stride()[2:] != (tokens * d, d, 1):
        raise ValueError(f"the inner three dimensions of {name} must be contiguous")


def _ints(t, name: str, ndim: int, device) -> None:
    if not isinstance(t, torch.Tensor) or t.ndim != ndim:
        raise ValueError(f"{name} must be a {ndim}-D tensor")
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} must live on {device}, got {t.device}")
    if t.stride(ndim - 1) != 1 and t.shape[ndim - 1] > 1:
        raise ValueError(f"{name} must have a contiguous last dimension")


class PagedKVCache:
    """A cache over tensors that the caller made (:meth:`empty` makes them).

    ``k``, ``v`` ``[layers, pages, Hkv, page tokens, D]``: inner three dimensions contiguous, any layer and page strides
    (two views of one ``[layers, pages, 2, Hkv, page tokens, D]`` tensor serve).  ``k_scale``, ``v_scale`` f32
    ``[layers, Hkv]``: what an E4M3 code is multiplied with."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor, *,
                 k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
        _pool(k, "k")
        _pool(v, "v")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise ValueError(f"k and v must be alike, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        layers, pages, heads, tokens, d = k.shape
        _ints(page_table, "page_table", 2, k.device)
        _ints(seq_lens, "seq_lens", 1, k.device)
        _ints(ref_counts, "ref_counts", 1, k.device)
        if seq_lens.shape[0] != page_table.shape[0]:
            raise ValueError(f"page_table has {page_table.shape[0]} rows, seq_lens {seq_lens.shape[0]} entries")
        if ref_counts.shape[0] != pages:
            raise ValueError(f"ref_counts must have {pages} entries, got {ref_counts.shape[0]}")
        e4m3 = k.dtype == torch.float8_e4m3fn
        for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if (t is not None) != e4m3:
                raise ValueError(f"{name} goes with a float8_e4m3fn cache, and with no other")
            if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (layers, heads) or not t.is_contiguous() or t.device != k.device):
                raise ValueError(f"{name} must be a contiguous float32 [{layers}, {heads}] tensor on {k.device}")
        self.k, self.v, self.page_table, self.seq_lens, self.ref_counts = k, v, page_table, seq_lens, ref_counts
        self.k_scale, self.v_scale = k_scale, v_scale
        self.device = k.device
        self._index = k.device.index
        self._c = _lib.KvCache(ptr(k), ptr(v), k.stride(0), k.stride(1), v.stride(0), v.stride(1), layers, pages, heads, tokens, d,
                               KV_DTYPES[k.dtype], ptr(k_scale), ptr(v_scale), ptr(page_table), page_table.stride(0), page_table.shape[0],
                               page_table.shape[1], ptr(seq_lens), ptr(ref_counts), 0)
        self._at = C.addressof(self._c)
        self._lib = lib()
        self._heads, self._d, self._takes = heads, d, (torch.bfloat16, torch.float16) if e4m3 else (k.dtype,)
        self._ws_bytes: dict = {}
        self._floats = torch.empty(0, dtype=torch.float32, device=self.device)
        self._work = torch.zeros((self._lib.fa4b_kv_workspace_bytes(self._at) + 3) // 4, dtype=torch.int32, device=self.device)
        self._c.work = ptr(self._work)
        self._call("fa4b_kv_copy_pages", 0, 0, 0)  # empty lists: the checks of the C side

    def _call(self, name: str, *args) -> None:
        """One C call on the cache's device and that device's current stream."""
        index = self._index
        if _current_device() == index:
            status = getattr(self._lib, name)(self._at, *args, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                status = getattr(self._lib, name)(self._at, *args, _raw_stream(index))
        if status:
            check(status, name)

    @classmethod
    def empty(cls, num_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, max_seqs: int, max_pages_per_seq: int, *, n_layers: int = 1,
              dtype: torch.dtype = torch.bfloat16, device="cuda", k_scale=None, v_scale=None) -> "PagedKVCache":
        """A cache with every page free and every slot empty; the pools are not initialised (nothing reads a token that
        was not written)."""
        if dtype not in KV_DTYPES:
            raise TypeError(f"dtype must be bfloat16, float16 or float8_e4m3fn, got {dtype}")
        shape = (n_layers, num_pages, n_kv_heads, page_tokens, head_dim)
        if min(shape) < 1 or max_seqs < 1 or max_pages_per_seq < 1:
            raise ValueError("all sizes must be positive")
        pools = [torch.empty(shape, dtype=dtype, device=device) for _ in range(2)]
        return cls(*pools, torch.full((max_seqs, max_pages_per_seq), -1, dtype=torch.int32, device=device),
                   torch.zeros(max_seqs, dtype=torch.int32, device=device), torch.zeros(num_pages, dtype=torch.int32, device=device),
                   k_scale=k_scale, v_scale=v_scale)

    # ------------------------------------------------------------------------------------------------ pages
    def _list(self, t, name: str, n: int = -1) -> int:
        if type(t) is not torch.Tensor or t.dtype is not torch.int32 or t.dim() != 1 or t.get_device() != self._index or not t.is_contiguous():
            _ints(t, name, 1, self.device)
        if n >= 0 and t.numel() != n:
            raise ValueError(f"{name} has {t.numel()} entries, expected {n}")
        return t.data_ptr()

    def free(self, seqs: torch.Tensor) -> None:
        """The slots ``seqs`` give their pages back and are empty then.  Empty slots and repeated ones do no harm."""
        self._call("fa4b_kv_free", self._list(seqs, "seqs"), seqs.numel())

    def extend(self, seqs: torch.Tensor, n_new: torch.Tensor) -> None:
        """Slot ``seqs[i]`` grows by ``n_new[i]`` tokens (:meth:`write` fills them) and claims pages for them: the lowest
        free ones, in the order of the list.  All or nothing; :meth:`check_status` tells.  The slots of a list that was refused take no
        writes until one of their calls (an ``extend``, by 0 tokens too, or a ``free``, or a ``fork`` into them) succeeds."""
        a, n = self._list(seqs, "seqs"), seqs.numel()
        self._call("fa4b_kv_extend", a, self._list(n_new, "n_new", n), n)

    def write(self, k: torch.Tensor, v: torch.Tensor, seqs: torch.Tensor, *, n_new: torch.Tensor | None = None, layer: int = 0) -> None:
        """Keys and values ``[n, Hkv, T, D]`` (any batch / head / token strides) of the newest tokens: token ``t < n_new[i]``
        goes to position ``seq_lens[seqs[i]] - n_new[i] + t`` (``n_new`` None: T for every row).  A 16-bit cache takes its
        own type, an E4M3 cache bf16 or f16, divided by the scale, clamped to +-448 and rounded.  A slot whose last :meth:`extend` was
        refused is left out and reported, and so are tokens whose page several slots hold: those from before a :meth:`fork` (write them
        before it).  A slot named twice gets either row's values."""
        a, n = self._list(seqs, "seqs"), seqs.numel()
        b = 0 if n_new is None else self._list(n_new, "n_new", n)
        if type(k) is not torch.Tensor or type(v) is not torch.Tensor:
            self._check_new(k, v, n)
        dtype, index, (k_shape, k_strides), (v_shape, v_strides) = k.dtype, self._index, (k.shape, k.stride()), (v.shape, v.stride())
        if (len(k_shape) != 4 or k_shape != v_shape or k_shape[0] != n or k_shape[1] != self._heads or k_shape[3] != self._d or dtype is not v.dtype or
                dtype not in self._takes or k.get_device() != index or v.get_device() != index or k_strides[3] != 1 or v_strides[3] != 1):
            self._check_new(k, v, n)
        args = _WRITE.pack(k.data_ptr(), v.data_ptr(), *_strides(k_shape, k_strides), *_strides(v_shape, v_strides), k_shape[2], KV_DTYPES[dtype], layer, n, a, b)
        self._call("fa4b_kv_write", args)

    def _check_new(self, k, v, n: int) -> None:
        for t, name in ((k, "k"), (v, "v")):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[0] != n or t.shape[1] != self._heads or t.shape[3] != self._d:
                raise ValueError(f"{name} must be a [{n}, {self._heads}, T, {self._d}] tensor")
            if t.dtype not in self._takes:
                raise TypeError(f"{name} is {t.dtype}, the cache {self.k.dtype}")
            if t.get_device() != self._index:
                raise RuntimeError(f"{name} must live on {self.device}, got {t.device}")
            if t.stride(3) != 1:
                raise ValueError(f"{name} must have a contiguous head dimension")
        if k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be alike")

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Slot ``children[i]``, which is empty, becomes a copy of ``parents[i]``: full pages are shared, the page that is
        still being filled is copied.  All or nothing; :meth:`check_status` tells."""
        a, n = self._list(parents, "parents"), parents.numel()
        self._call("fa4b_kv_fork", a, self._list(children, "children", n), n)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Pages ``src[i]`` to pages ``dst[i]`` in every layer; tables and counts stay.  A pair with a negative entry is
        skipped, and one whose pages another pair writes, or whose destination another reads, is left out and reported."""
        a, n = self._list(src, "src"), src.numel()
        self._call("fa4b_kv_copy_pages", a, self._list(dst, "dst", n), n)

    def compact(self) -> None:
        """Moves the used pages behind the first ``n`` (``n``: pages in use) to the free ones among them, in order, so
        that the pages in use are ``0..n-1``; tables and counts follow."""
        self._call("fa4b_kv_compact")

    # ------------------------------------------------------------------------------------------------ attention
    def attend(self, q: torch.Tensor, seqs: torch.Tensor | None = None, *, layer: int = 0, group_offsets: torch.Tensor | None = None,
               shared_lens: torch.Tensor | None = None, softmax_scale: float | None = None, out: torch.Tensor | None = None):
        """O ``[n, Hq, T, D]`` and LSE ``[n, Hq, T]`` f32 of the newest ``T <= 16`` tokens of ``n`` sequences: ``q [n, Hq, T, D]``
        (any batch / head / token strides) over the pages of slots ``seqs`` (None: slot ``i`` for row ``i``).  Query ``t``
        sees keys ``j < len - (T - 1 - t)``; a row that sees none, or whose slot is out of range (padding), is 0 with LSE -inf.

        ``group_offsets [groups + 1]``, ``shared_lens [groups]``: rows ``group_offsets[g]`` up to ``group_offsets[g + 1]`` hold
        the same pages for their first ``shared_lens[g]`` tokens (as :meth:`fork` leaves them), which are read once for
        the group; rows in no group have LSE -inf, and O 0 or what ``out`` held.  ``out`` receives O when given (any strides but 0).  There is no
        gradient: a backward pass that comes to a ``q`` which requires one is refused.  ``softmax_scale`` None: ``1 / sqrt(D)``."""
        if not isinstance(q, torch.Tensor) or len(shape := q.shape) != 4 or shape[3] != self._d:
            raise ValueError(f"q must be a [n, Hq, T, {self._d}] tensor")
        dtype, strides = q.dtype, q.stride()
        if dtype not in self._takes:
            raise TypeError(f"q is {dtype}, the cache {self.k.dtype}")
        if q.get_device() != self._index:
            raise RuntimeError(f"q must live on {self.device}, got {q.device}")
        n, hq, t, d = shape
        if strides[3] != 1:
            raise ValueError("q must have a contiguous head dimension")
        if (group_offsets is None) != (shared_lens is None):
            raise ValueError("group_offsets and shared_lens go together")
        slots = 0 if seqs is None else self._list(seqs, "seqs", n)
        groups = offsets = shared = 0
        if group_offsets is not None:
            shared, groups = self._list(shared_lens, "shared_lens"), shared_lens.numel()
            if group_offsets.numel() != groups + 1:
                raise ValueError(f"group_offsets must have {groups + 1} entries, got {group_offsets.numel()}")
            if groups == 0 and n > 0:
                raise ValueError("no groups: without group_offsets and shared_lens every row stands by itself")
            offsets = self._list(group_offsets, "group_offsets")
        flags = 2  # of rows in no group the LSE says that nothing was computed, and a new O is 0
        if out is None:
            out, o_strides, flags = q.new_empty(shape), (hq * t * d, t * d, d), 3
        elif out.shape != shape or out.dtype != q.dtype or out.device != self.device or out.stride(3) != 1:
            raise ValueError(f"out must be a {tuple(shape)} tensor like q with a contiguous head dimension")
        else:
            o_strides = _strides(shape, out.stride())
        lse = self._floats.new_empty((n, hq, t))
        code, scale = KV_DTYPES[dtype], 0.0 if softmax_scale is None else softmax_scale
        if softmax_scale is not None and not 2.0 ** -149 <= scale <= _LARGEST:
            raise ValueError(f"softmax_scale must be positive and finite in 32 bits, got {softmax_scale}")
        q_strides = _strides(shape, strides)
        size = self._ws_bytes.get((n, hq, t, groups))
        if size is None:
            args = _ATTEND.pack(q.data_ptr(), *q_strides, out.data_ptr(), *o_strides, lse.data_ptr(), n, t, hq, layer, code, scale, slots, groups, flags, offsets, shared, 0)
            with torch.cuda.device(self._index):  # the size goes by the number of SMs
                size = self._lib.fa4b_attn_paged_workspace_bytes(self._at, args)
            if size:
                self._ws_bytes[n, hq, t, groups] = size
        ws = self._floats.new_empty(size >> 2)  # of this call alone: calls on two streams, or of two captured graphs, may overlap
        args = _ATTEND.pack(q.data_ptr(), *q_strides, out.data_ptr(), *o_strides, lse.data_ptr(), n, t, hq, layer, code, scale, slots, groups, flags, offsets, shared,
                            ws.data_ptr())
        self._call("fa4b_attn_paged_fwd", args)
        if q.requires_grad and torch.is_grad_enabled():
            out, lse = _WithoutGradient.apply(q, out, lse)
        return out, lse

    def check_status(self) -> None:
        """Synchronise and raise on what the calls since the last check found wrong on the device (slots out of range, too
        few free pages, ...)."""
        self._call("fa4b_kv_check_status")


class _WithoutGradient(torch.autograd.Function):
    """Hands results on, and refuses the backward pass instead of leaving a gradient out."""

    @staticmethod
    def forward(ctx, q, out, lse):
        return out, lse

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("attention over a paged cache has no gradient")


def _strides(shape, strides) -> tuple:
    a, b, c, _ = shape
    x, y, z, _ = strides
    return x if a > 1 else 0, y if b > 1 else 0, z if c > 1 else 0  # a dimension of one entry carries no stride of its own
