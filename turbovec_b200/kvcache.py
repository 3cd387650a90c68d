"""Paged key/value cache on one GPU: appending keys and values with their position rotation, attention for a batch that may share
a long prefix, and attention over pages that a cheap score selects (tv_kv_* of include/turbovec_b200.h).

    cache = PagedKVCache.empty(pages=4096, page_size=64, kv_heads=8, head_dim=128, dtype=torch.bfloat16, device="cuda:0")
    batch = KVBatch(table, lens, offsets)            # int32 tensors; lens counts the tokens of the call
    q = cache.append(batch, k, v, q=q, cos=cos, sin=sin)
    out = cache.attend(batch, q, prefix_pages=document_pages, prefix_len=30_000)
    out, pages = cache.attend_selected(batch, q, budget=64, first=1, recent=4)

Row t of a call is token j of sequence b, offsets[b] <= t < offsets[b + 1]; it stands at position lens[b] - (offsets[b + 1] -
offsets[b]) + j of the sequence's own pages, table[b][position // page_size].  Rows behind the last sequence are left as they are: in a
result that the call makes itself they hold anything.

Everything runs on torch's current stream of the cache's device, without a synchronisation, and may be captured into a CUDA graph;
results and workspaces come from torch's allocator.  Tensors are read when the kernels run: table, lens and offsets may be changed
in place between calls, and a captured graph sees the new values.  There is no CPU path.  No gradient passes through: tensors
that require one are refused unless gradients are off (torch.no_grad, torch.inference_mode).
"""
from __future__ import annotations

import torch

from . import _native

__all__ = ["PagedKVCache", "KVBatch", "OPT_TENSOR_PREFIX", "set_option"]

OPT_TENSOR_PREFIX = 1
_options = 0                                            # how often an option was set: workspace sizes follow options

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}


def _stream(index: int) -> int:
    """torch's current stream of a device, as a number."""
    return torch.cuda.current_stream(index).cuda_stream


# the same without a Stream object around it: 0.2 us instead of 2.4
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def _fail(lib, rc: int):
    msg = lib.tv_last_error(None).decode()
    raise (ValueError if rc == 90 else RuntimeError)(msg)


def _tensor(name: str, t, dtype, ndim: int, device=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be of {dtype}, got {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got {t.dim()}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t


def _no_gradient(name: str):
    raise RuntimeError(f"{name} requires a gradient, and none passes through the cache: detach it, or call under torch.no_grad()")


def _last_adjacent(name: str, t: torch.Tensor) -> None:
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the elements of the last dimension must be adjacent")


def set_option(option: int, value: int) -> None:
    """An option of the cache's calls, for the whole process (TV_KV_OPT_* of include/turbovec_b200.h).  Not while another thread is in a call."""
    global _options
    lib = _native.load()
    rc = lib.tv_kv_set_option(int(option), int(value))
    if rc:
        _fail(lib, rc)
    _options += 1


def _kept(name: str) -> property:
    """A tensor whose address calls use: what it holds may be changed, it may not be replaced."""
    place = "_" + name

    def get(self):
        return getattr(self, place)

    def put(self, t):
        if t is not getattr(self, place):               # (`batch.lens += 1` gives the tensor itself)
            raise AttributeError(f"{name} is changed in place; for another tensor make another {type(self).__name__}")
    return property(get, put)


class KVBatch:
    """The sequences of a call: `table` int32 [sequences, width], page numbers of each; `lens` int32 [sequences], tokens in its own
    pages, those of the call among them; `offsets` int32 [sequences + 1], first row of each (None: one row each).  The tensors
    are kept and read when the kernels run: change them in place."""

    table, lens, offsets = _kept("table"), _kept("lens"), _kept("offsets")

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, offsets: torch.Tensor | None = None):
        _tensor("lens", lens, torch.int32, 1)
        if not lens.is_contiguous():
            raise ValueError("lens must be contiguous")
        self.device = lens.device
        n = lens.numel()
        _tensor("table", table, torch.int32, 2, self.device)
        if table.shape[0] != n:
            raise ValueError(f"table must have a row for each of the {n} sequences, got {table.shape[0]}")
        _last_adjacent("table", table)
        if offsets is None:
            offsets = torch.arange(n + 1, dtype=torch.int32, device=self.device)
        _tensor("offsets", offsets, torch.int32, 1, self.device)
        if offsets.numel() != n + 1 or not offsets.is_contiguous():
            raise ValueError(f"offsets must hold {n + 1} adjacent numbers, got {offsets.numel()}")
        self._table, self._lens, self._offsets = table, lens, offsets
        width = table.shape[1]
        stride = table.stride(0) if n > 1 else width
        if stride < width:
            raise ValueError("the rows of table must not overlap")
        self._view = _native.KvBatchView(n, width, stride, table.data_ptr(), lens.data_ptr(), offsets.data_ptr())

    def __len__(self) -> int:
        return self._view.sequences


class PagedKVCache:
    """A pool of pages over tensors that the caller owns: k and v [pages, kv_heads, page_size, head_dim] with any strides but adjacent
    channels (a pool laid out [pages, page_size, kv_heads, head_dim] is passed as its transpose(1, 2)), bfloat16 or float16, head_dim
    64 or 128, page_size 16, 32, 64 or 128.  bounds int8 [pages, kv_heads, 2, head_dim] and scales float32 [pages, kv_heads] hold
    the lowest and highest key of every channel of a page, as multiples of scales; both None where no pages are selected by score."""

    k, v, bounds, scales = _kept("k"), _kept("v"), _kept("bounds"), _kept("scales")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, bounds: torch.Tensor | None = None, scales: torch.Tensor | None = None):
        if not isinstance(k, torch.Tensor):
            raise TypeError(f"k must be a torch tensor, got {type(k).__name__}")
        if k.dtype not in _DTYPES:
            raise TypeError(f"k must be of bfloat16 or float16, got {k.dtype}")
        _tensor("k", k, k.dtype, 4)
        _tensor("v", v, k.dtype, 4, k.device)
        if k.shape != v.shape:
            raise ValueError("k and v must have the same shape")
        _last_adjacent("k", k)
        _last_adjacent("v", v)
        pages, heads, page_size, dim = k.shape
        if dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {dim}")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page_size must be 16, 32, 64 or 128, got {page_size}")
        if pages < 1 or heads < 1:
            raise ValueError("the pool must have at least one page and one key head")
        if (bounds is None) != (scales is None):
            raise ValueError("bounds and scales must be given together")
        if bounds is not None:
            _tensor("bounds", bounds, torch.int8, 4, k.device)
            _tensor("scales", scales, torch.float32, 2, k.device)
            if tuple(bounds.shape) != (pages, heads, 2, dim) or not bounds.is_contiguous():
                raise ValueError(f"bounds must be contiguous with shape {(pages, heads, 2, dim)}, got {tuple(bounds.shape)}")
            if tuple(scales.shape) != (pages, heads) or not scales.is_contiguous():
                raise ValueError(f"scales must be contiguous with shape {(pages, heads)}, got {tuple(scales.shape)}")
        self._lib = _native.load()
        if k.device.type != "cuda":
            raise RuntimeError("turbovec_b200 has no CPU path: the cache must be in the memory of a CUDA device")
        self._k, self._v, self._bounds, self._scales = k, v, bounds, scales
        self.device, self.dtype = k.device, k.dtype
        self.pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page_size, dim
        self._index, self._scale, self._sizes = k.device.index, dim ** -0.5, {}

        def stride(t, i, natural):                      # of a dimension of one, whatever it says
            return t.stride(i) if t.shape[i] > 1 else natural
        sk = [stride(k, i, heads * page_size * dim) for i in range(3)]
        sv = [stride(v, i, heads * page_size * dim) for i in range(3)]
        self._view = _native.KvCacheView(
            k.device.index, _DTYPES[k.dtype], dim, heads, page_size, pages, k.data_ptr(), v.data_ptr(), *sk, *sv,
            bounds.data_ptr() if bounds is not None else None, scales.data_ptr() if scales is not None else None)
        for name, strides, t in (("k", sk, k), ("v", sv, v)):
            if any(s <= 0 or s % 8 for s in strides) or t.data_ptr() % 16:
                raise ValueError(f"{name}: strides must be positive multiples of 8 elements, and the tensor 16-byte aligned")

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype=torch.bfloat16, device="cuda", bounds: bool = True):
        """A pool of its own, contiguous, without contents; bounds=False leaves out what attend_selected needs."""
        shape = (pages, kv_heads, page_size, head_dim)
        k, v = torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)
        b = torch.zeros(pages, kv_heads, 2, head_dim, dtype=torch.int8, device=device) if bounds else None
        s = torch.full((pages, kv_heads), 2.0 ** -24, dtype=torch.float32, device=device) if bounds else None
        return cls(k, v, b, s)

    # ---- helpers (on the path of every call: a tensor's attributes cost 0.2 us each, a check by a function of its own 0.3) ----
    def _rows(self, name: str, t, tokens: int | None, heads: int | None):
        """(rows, heads, view) of a [rows, heads, head_dim] tensor, of `tokens` and `heads` where given."""
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
        if t.dtype != self.dtype:
            raise TypeError(f"{name} must be of {self.dtype}, got {t.dtype}")
        shape = t.shape
        if len(shape) != 3:
            raise ValueError(f"{name} must have 3 dimensions, got {len(shape)}")
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}")
        n, h, d = shape
        if d != self.head_dim:
            raise ValueError(f"{name} must have {self.head_dim} channels, got {d}")
        if (tokens is not None and n != tokens) or (heads is not None and h != heads):
            raise ValueError(f"{name} must have {n if tokens is None else tokens} rows of {h if heads is None else heads} heads, got {n} of {h}")
        st = t.stride()
        if st[2] != 1:
            raise ValueError(f"{name}: the elements of the last dimension must be adjacent")
        if t.requires_grad and torch.is_grad_enabled():
            _no_gradient(name)
        return n, h, _native.KvRowsView(t.data_ptr(), st[0] if n > 1 else h * d, st[1] if h > 1 else d)

    def _query(self, q, tokens: int | None = None):
        n, heads, view = self._rows("q", q, tokens, None)
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"the number of query heads must be a positive multiple of {self.kv_heads}, got {heads}")
        return n, heads, view

    def _batch(self, batch) -> _native.KvBatchView:
        if not isinstance(batch, KVBatch):
            raise TypeError(f"batch must be a KVBatch, got {type(batch).__name__}")
        if batch.device != self.device:
            raise ValueError(f"batch must be on {self.device}, got {batch.device}")
        if (self._k.requires_grad or self._v.requires_grad) and torch.is_grad_enabled():
            _no_gradient("the pool")
        return batch._view

    def _array(self, name: str, t, dtype, shape) -> int:
        """Address of a contiguous tensor of that type and shape (None: any length of one dimension)."""
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
        if t.dtype != dtype:
            raise TypeError(f"{name} must be of {dtype}, got {t.dtype}")
        if (len(t.shape) != 1 if shape is None else t.shape != shape) or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous with {'one dimension' if shape is None else f'shape {tuple(shape)}'}, got {tuple(t.shape)}")
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            _no_gradient(name)
        return t.data_ptr()

    def _workspace(self, op: str, batch, *sizes):
        """A workspace for an operator; its size for these sizes is asked for once.  None where there is none: the operator says why."""
        key = (op, _options, batch._view.sequences, *sizes)
        n = self._sizes.get(key)
        if n is None:
            n = getattr(self._lib, f"tv_kv_{op}_workspace")(self._view, batch._view, *sizes)
            if n == 0:
                return None
            if len(self._sizes) >= 256:
                self._sizes.clear()
            self._sizes[key] = n
        return torch.empty(n, dtype=torch.uint8, device=self.device)

    # ---- operators ----
    def append(self, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, *, q: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
               cos: torch.Tensor | None = None, sin: torch.Tensor | None = None, interleaved: bool = False, position_offset: int = 0):
        """Writes the rows of k and v [tokens, kv_heads, head_dim] into the pages of their sequences, keys rotated by the angles of
        position + position_offset; rotates q [tokens, heads, head_dim] into q_out (a new tensor by default; q itself is allowed) and
        returns it.  cos and sin: float32 [positions, rotary / 2], rotary a multiple of 16 up to head_dim; None: no rotation.  Pairs are
        channels i and i + rotary / 2, or 2i and 2i + 1 where `interleaved`.  Tokens at positions below 0 or without an angle are left out: their
        pages, bounds and rows of q_out stay as they are."""
        b = self._batch(batch)
        tokens, heads, kr = self._rows("k", k, None, self.kv_heads)
        vr = self._rows("v", v, tokens, heads)[2]
        qr = qo = None
        if q is not None:
            _, heads, qr = self._query(q, tokens)
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
            qo = self._rows("q_out", q_out, tokens, heads)[2]
        elif q_out is not None:
            raise ValueError("q_out must not be given without q")
        positions = rotary = 0
        cos_at = sin_at = None
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin must be given together")
        if cos is not None:
            if not isinstance(cos, torch.Tensor) or len(cos.shape) != 2:
                raise ValueError("cos must be a tensor of two dimensions")
            cos_at, sin_at = self._array("cos", cos, torch.float32, cos.shape), self._array("sin", sin, torch.float32, cos.shape)
            positions, rotary = cos.shape[0], 2 * cos.shape[1]
        if not -(1 << 40) <= position_offset <= 1 << 40:         # (ctypes cuts to 64 bits what is more)
            raise ValueError(f"position_offset is out of range: {position_offset}")
        rc = self._lib.tv_kv_append(self._view, b, tokens, heads, kr, vr, qr, qo, cos_at, sin_at, positions, rotary,
                                    1 if interleaved else 0, position_offset, _stream(self._index))
        if rc:
            _fail(self._lib, rc)
        return q_out

    def attend(self, batch: KVBatch, q: torch.Tensor, *, prefix_pages: torch.Tensor | None = None, prefix_len: int = 0,
               scale: float | None = None, out: torch.Tensor | None = None, lse: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of the rows of q [tokens, heads, head_dim] over the first prefix_len keys of prefix_pages (int32 [n], read once for the
        whole batch) and the keys of their own sequence up to their position.  Returns out (a new tensor by default); lse, where given,
        receives the logarithm of each row's sum of exponentials.  scale: head_dim ** -0.5 by default.  Rows that see no key: zeros
        and -inf.  Many rows on a long prefix go to a kernel that rounds the weights to the type (1.4 times the error of one rounding of the
        result); set_option(OPT_TENSOR_PREFIX, 0) keeps to the other one."""
        b = self._batch(batch)
        tokens, heads, qr = self._query(q)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        orow = self._rows("out", out, tokens, heads)[2]
        width, pages_at = 0, None
        if prefix_pages is not None:
            pages_at = self._array("prefix_pages", prefix_pages, torch.int32, None)
            width = prefix_pages.shape[0]
        if not 0 <= prefix_len <= width * self.page_size:
            raise ValueError(f"prefix_len must be between 0 and the {width * self.page_size} tokens of prefix_pages, got {prefix_len}")
        lse_at = None if lse is None else self._array("lse", lse, torch.float32, (tokens, heads))
        ws_at, ws_n = None, 0
        if tokens and len(batch):
            ws = self._workspace("attend", batch, tokens, heads, prefix_len)
            if ws is not None:
                ws_at, ws_n = ws.data_ptr(), ws.shape[0]
        rc = self._lib.tv_kv_attend(self._view, b, tokens, heads, qr, pages_at, width, prefix_len, self._scale if scale is None else scale,
                                    orow, lse_at, ws_at, ws_n, _stream(self._index))
        if rc:
            _fail(self._lib, rc)
        return out

    def attend_selected(self, batch: KVBatch, q: torch.Tensor, *, budget: int, first: int = 1, recent: int = 1, scale: float | None = None,
                        out: torch.Tensor | None = None, lse: torch.Tensor | None = None, pages: torch.Tensor | None = None):
        """Attention of every row over at most `budget` pages of its sequence: the `first` and the `recent` ones and the best of the others by
        a score, what a key at a page's bounds would give the query rounded to int8 (include/turbovec_b200.h), chosen for each token and
        key head.  Returns (out, pages): the chosen page numbers within the sequence, int32 [tokens, kv_heads, budget], ascending, then -1."""
        if self._bounds is None:
            raise ValueError("the cache has no bounds to choose pages by")
        b = self._batch(batch)
        tokens, heads, qr = self._query(q)
        if budget < 1 or first < 0 or recent < 0 or first + recent > budget:
            raise ValueError(f"budget must be positive and first + recent at most budget, got {budget}, {first} and {recent}")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        orow = self._rows("out", out, tokens, heads)[2]
        if pages is None:
            pages = torch.empty(tokens, self.kv_heads, budget, dtype=torch.int32, device=self.device)
        pages_at = self._array("pages", pages, torch.int32, (tokens, self.kv_heads, budget))
        lse_at = None if lse is None else self._array("lse", lse, torch.float32, (tokens, heads))
        ws_at, ws_n = None, 0
        if tokens and len(batch):
            ws = self._workspace("attend_selected", batch, tokens, heads, budget)
            if ws is not None:
                ws_at, ws_n = ws.data_ptr(), ws.shape[0]
        rc = self._lib.tv_kv_attend_selected(self._view, b, tokens, heads, qr, budget, first, recent, self._scale if scale is None else scale,
                                             orow, lse_at, pages_at, ws_at, ws_n, _stream(self._index))
        if rc:
            _fail(self._lib, rc)
        return out, pages

    def check(self) -> None:
        """Waits for the device and raises RuntimeError if a kernel of the cache gave up a wait since the last check."""
        rc = self._lib.tv_kv_status(self._index)
        if rc:
            _fail(self._lib, rc)
