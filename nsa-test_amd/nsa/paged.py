"""Paged K/V cache in 4 bits (no counterpart in the reference): what a server of NSA layers keeps
between steps when every request has its own length.

* ``build_block_tables``: block tables and slot maps of a step, on the GPU from the requests'
  lengths.
* ``PagedKV4``: a pool of K/V pages in OCP MXFP4 (e2m1 elements, an e8m0 scale for each 32
  features: 4.25 bits a value); ``store_kv4`` writes rows to slots, ``load_kv4`` reads contexts
  back for the prompt kernels.
* ``NSAPagedKVCache``: the decode state of one NSAAttention layer in such pages, each sequence at a
  length of its own; NSAAttention.prefill and .decode take it in NSAKVCache's place.
* ``attend_kv4``: causal attention of the last tokens of each request over the pages, whole
  context, a window, or selected blocks; ``nsa_attend_kv4``: the three branches of an NSA layer
  with their gates.

The functions take lengths, counts and tables from the device and wait for nothing, so that a step
of them can be captured into a graph and replayed.  None of it is differentiable: tensors that
require a gradient are refused outside torch.no_grad().
"""
from __future__ import annotations

import ctypes
from typing import List, NamedTuple, Optional, Sequence

import torch
import torch.nn.functional as F

from . import _lib, _ops

PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)
MAX_REQUESTS = 4096
MAX_BLOCKS = 4096  # compressed blocks a query can score
MAX_PAIRS = 65535  # (request, group) pairs of a call
MAX_BLOCK_SIZE = 1 << 20  # tokens of a selection block
MAX_TOKENS = 1 << 30  # tokens of a block table


# A call is one or two launches of a few us each, so small ones wait for its host side (10 to 17 us, a
# launch 3.3 of them): conditions are tested in line, sizes and strides read once, addresses passed plain.
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch(dev: int, name: str, *args) -> None:
    """The C call on device `dev` (whichever is current) and its current stream."""
    if _current_device() == dev:
        rc = getattr(_lib.load(), name)(*args, _raw_stream(dev))
        if rc:
            raise _lib.error(name, rc)
    else:
        with torch.cuda.device(dev):
            _launch(dev, name, *args)


def _need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def _refuse(name: str, t: torch.Tensor, want: str) -> None:
    if not t.is_cuda:
        raise RuntimeError("NSA kernels run on the GPU only: got a tensor on " + str(t.device))
    raise ValueError(f"{name} must be {want}, got {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")


def _refuse_grad(name: str) -> None:
    # the calls work on addresses: a gradient that is asked for would be lost
    raise RuntimeError(f"{name} is not differentiable: call it under torch.no_grad(), or detach its tensors")


def _check_vector(name: str, t: torch.Tensor, n: int, dtype: torch.dtype, dev: int) -> None:
    if t.dtype is not dtype or t.shape != (n,) or not t.is_contiguous() or t.get_device() != dev:
        _refuse(name, t, f"contiguous {dtype} [{n}] on cuda:{dev}")


def _check_tables(name: str, t: torch.Tensor, batch: int, dev: int) -> int:
    """The table's width."""
    if t.dtype is torch.int32 and t.dim() == 2 and t.get_device() == dev:
        n, w = t.shape
        if n == batch and w and (t.stride(1) == 1 or w == 1):
            return w
    _refuse(name, t, f"int32 [{batch}, pages] with rows of unit stride on cuda:{dev}")


def _rows16(t: torch.Tensor, cdt: torch.dtype, width: int) -> torch.Tensor:
    """t in cdt with rows of `width` unit-stride features, zeros past its own, 16-byte aligned."""
    if t.dtype is not cdt:
        t = t.to(cdt)
    if t.shape[-1] != width:
        t = F.pad(t, (0, width - t.shape[-1]))
    st = t.stride()
    m = t.data_ptr()
    for x in st[:-1]:
        m |= x * (4 if cdt is torch.float32 else 2)
    return t if not m & 15 and st[-1] == 1 else _ops._compact(t)


class BlockTables(NamedTuple):
    """What build_block_tables gives: for each row of the step's batch its slot (int64), position and
    request (int32), -1 for rows without a token; the requests' first rows [B + 1]; the lengths
    after the step [B]; info [3]: tokens placed, entries of the free list used so far, tokens
    refused."""

    slots: torch.Tensor
    positions: torch.Tensor
    sequences: torch.Tensor
    offsets: torch.Tensor
    lengths: torch.Tensor
    info: torch.Tensor


def build_block_tables(tables: torch.Tensor, lengths: torch.Tensor, new: torch.Tensor, free: torch.Tensor,
                       used: torch.Tensor, page_size: int, rows: int, row_stride: int = 0) -> BlockTables:
    """Places the new tokens of a step in pages (nsa_block_tables).

    tables [B,W] int32: the pages of each request in order, extended in place; lengths [B], new [B]
    int32: tokens cached and to come; free [F] int32: free pages, taken in order from entry
    used[0] (int32 [1]) on.  The step's batch has `rows` rows: packed request after request, or with
    row_stride those of request b from b * row_stride on (rows = B * row_stride).  Tokens that the
    table, the rows or the free pages have no room for are refused: -1 in their rows, not counted in
    the lengths, counted in info[2].  Neither lengths nor used is changed: the next step takes the
    returned lengths and info[1:2]."""
    dev, B = tables.get_device(), lengths.shape[0] if lengths.dim() else 0
    if not 1 <= B <= MAX_REQUESTS:
        raise ValueError(f"between 1 and {MAX_REQUESTS} requests, got {B}")
    if dev < 0:
        _refuse("tables", tables, "on the GPU")
    W = _check_tables("tables", tables, B, dev)
    _check_vector("lengths", lengths, B, torch.int32, dev)
    _check_vector("new", new, B, torch.int32, dev)
    n_free = free.numel()
    _check_vector("free", free, n_free, torch.int32, dev)
    _check_vector("used", used, 1, torch.int32, dev)
    if page_size not in PAGE_SIZES:
        raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {page_size}")
    if rows < 0 or row_stride < 0 or (row_stride and rows != B * row_stride):
        raise ValueError(f"{rows} rows of {B} requests do not agree with row_stride {row_stride}")
    slots = torch.empty(rows, device=tables.device, dtype=torch.int64)
    ints = torch.empty(2 * (rows + B) + 4, device=tables.device, dtype=torch.int32)  # one allocation for the rest
    at = ints.data_ptr()
    off = at + 8 * rows
    _launch(dev, "nsa_block_tables", tables.data_ptr(), tables.stride(0), B, W, lengths.data_ptr(), new.data_ptr(),
            free.data_ptr(), n_free, used.data_ptr(), page_size, rows, row_stride, slots.data_ptr(), at, at + 4 * rows, off,
            off + 4 * (B + 1), off + 4 * (2 * B + 1))
    return BlockTables(slots, *ints.split_with_sizes((rows, rows, B + 1, B, 3)))


class PagedKV4:
    """A pool of K/V pages in 4 bits: codes k [pages,G,page,dk/2] and v [pages,G,page,dv/2] (element 2i
    in the low nibble of byte i), scales k_scale [pages,G,page,dk/32] and v_scale [pages,G,page,dv/32],
    all uint8 and contiguous.  (dk, dv) is a compiled head-width pair; head_dims names the narrower
    widths of the rows where they are padded to it (``empty`` pads)."""

    def __init__(self, k: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor, v_scale: torch.Tensor, head_dims=None):
        ts = (k, k_scale, v, v_scale)
        _need(all(t.dtype == torch.uint8 and t.dim() == 4 and t.is_contiguous() for t in ts),
              "pages are four contiguous uint8 tensors [pages, groups, page, bytes]")
        _need(all(t.device == k.device and t.shape[:3] == k.shape[:3] for t in ts),
              "the page tensors differ in device, pages, groups or page size")
        dk, dv = 2 * k.shape[3], 2 * v.shape[3]
        _need((dk, dv) in _ops.HEAD_DIM_PAIRS and 32 * k_scale.shape[3] == dk and 32 * v_scale.shape[3] == dv,
              f"page rows of {k.shape[3]} / {v.shape[3]} bytes and {k_scale.shape[3]} / {v_scale.shape[3]} scales are "
              f"of no compiled head widths {_ops.HEAD_DIM_PAIRS}")
        _need(k.shape[2] in PAGE_SIZES, f"page size must be one of {PAGE_SIZES}, got {k.shape[2]}")
        _need(min(k.shape) > 0, "a pool needs pages and groups")
        _need(all(t.data_ptr() % 16 == 0 for t in ts), "page tensors must be 16-byte aligned")
        self._tensors = ts
        self.n_pages, self.n_kv_groups, self.page_size = k.shape[:3]
        self.kernel_dims = (dk, dv)
        self.head_dims = (dk, dv) if head_dims is None else tuple(head_dims)
        _need(0 < self.head_dims[0] <= dk and 0 < self.head_dims[1] <= dv, f"head_dims {head_dims} exceed {dk}, {dv}")
        self.device, self._dev = k.device, k.get_device()
        self._pages = _lib.Kv4Pages(*(t.data_ptr() for t in ts), self.n_pages, self.page_size)
        self._at = ctypes.addressof(self._pages)
        # what pools that one call reads must share
        self._kind = (self._dev, self.n_kv_groups, self.kernel_dims, self.head_dims)

    # read only: the calls use the addresses of the tensors given at the start
    k = property(lambda self: self._tensors[0])
    k_scale = property(lambda self: self._tensors[1])
    v = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])

    @classmethod
    def empty(cls, n_pages: int, page_size: int, n_kv_groups: int, head_dim_qk: int, head_dim_v: int, device) -> "PagedKV4":
        """A pool of zeros."""
        dk, dv = _ops.kernel_dims(head_dim_qk, head_dim_v)
        codes, scales = ([torch.zeros(n_pages, n_kv_groups, page_size, d // n, device=device, dtype=torch.uint8)
                          for d in (dk, dv)] for n in (2, 32))
        return cls(codes[0], scales[0], codes[1], scales[1], (head_dim_qk, head_dim_v))

def store_kv4(kv: PagedKV4, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Rows k [N,G,dk] and v [N,G,dv] into slots [N] (int64: page * page_size + offset) of the pool
    (nsa_kv4_store).  Each block of 32 features gets the scale 2^(floor(log2 max|x|) - 2) and its elements
    the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it (ties to even, saturating); a block with an
    infinity or NaN becomes NaN.  Slots below 0 or outside the pool are skipped; the others of a call
    have to differ (of a slot named twice, codes and scales may be of different rows)."""
    N, dev = slots.shape[0] if slots.dim() else 0, kv._dev
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        _refuse_grad("store_kv4")
    if dev < 0:
        _refuse("the pool", kv.k, "on the GPU")
    _check_vector("slots", slots, N, torch.int64, dev)
    G, (dk, dv), (DK, DV) = kv.n_kv_groups, kv.head_dims, kv.kernel_dims
    if k.shape != (N, G, dk) or k.get_device() != dev:
        _refuse("k", k, f"[{N}, {G}, {dk}] on cuda:{dev}")
    if v.shape != (N, G, dv) or v.get_device() != dev or v.dtype is not k.dtype:
        _refuse("v", v, f"{k.dtype} [{N}, {G}, {dv}] on cuda:{dev}")
    if N == 0:
        return
    cdt = _ops.compute_dtype(k.dtype)
    k, v = _rows16(k, cdt, DK), _rows16(v, cdt, DV)
    _launch(dev, "nsa_kv4_store", kv._at, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
            slots.data_ptr(), N, G, DK, DV, _lib.NSA_F32 if cdt is torch.float32 else _lib.NSA_BF16)


def load_kv4(kv: PagedKV4, tables: torch.Tensor, lengths: torch.Tensor, max_len: int, dtype=torch.bfloat16):
    """(k [B,G,max_len,dk], v [B,G,max_len,dv]) of the cached tokens (nsa_kv4_load): token t < lengths[b]
    (int32 [B]) from page tables[b, t // page_size]; zeros behind a length and where the table names
    no page of the pool."""
    dev, B = kv._dev, lengths.shape[0] if lengths.dim() else 0
    if dev < 0:
        _refuse("the pool", kv.k, "on the GPU")
    if B < 1 or max_len < 0:
        raise ValueError(f"{B} requests, max_len {max_len}")
    _check_vector("lengths", lengths, B, torch.int32, dev)
    W = _check_tables("tables", tables, B, dev)
    cdt = _ops.compute_dtype(dtype)
    G, (DK, DV) = kv.n_kv_groups, kv.kernel_dims
    k = torch.empty((B, G, max_len, DK), device=kv.device, dtype=cdt)
    v = torch.empty((B, G, max_len, DV), device=kv.device, dtype=cdt)
    _launch(dev, "nsa_kv4_load", kv._at, tables.data_ptr(), tables.stride(0), W, lengths.data_ptr(), k.data_ptr(),
            v.data_ptr(), B, G, max_len, DK, DV, _lib.NSA_F32 if cdt is torch.float32 else _lib.NSA_BF16)
    if kv.head_dims != kv.kernel_dims:
        k, v = k[..., :kv.head_dims[0]], v[..., :kv.head_dims[1]]
    return (k, v) if dtype is cdt else (k.to(dtype), v.to(dtype))


# packed in one go: the fields one at a time through ctypes took 8 us of a call
_ATTN, _STEP, _BLOCKS = (_lib.packer(t) for t in (_lib.Kv4AttnArgs, _lib.PagedStepArgs, _lib.PagedBlocksArgs))
_INT_MAX = (1 << 31) - 1


def _attend(q, sources, lengths, scale, window=1, indices=None, block_size=64, l=1, d=1, gates=None, gate_act=0,
            max_length=None):
    """The call of nsa_kv4_attn: sources (pool, tables) or (None, None), three of them in the order of the gates."""
    kv = sources[2][0] or sources[1][0]
    dev, G, (DK, DV), (dk, dv) = kv._kind
    if (q.requires_grad or gates is not None and gates.requires_grad) and torch.is_grad_enabled():
        _refuse_grad("attention over 4-bit pages")
    if dev < 0:
        _refuse("the pool", kv.k, "on the GPU")
    if q.dim() != 4 or q.get_device() != dev:
        _refuse("q", q, f"[B, H, T, {dk}] on cuda:{dev}")
    B, H, T, width = q.shape
    if width != dk or H % G or not (B and H and T):
        raise ValueError(f"q {tuple(q.shape)} does not go with {G} groups of width {dk}")
    _check_vector("lengths", lengths, B, torch.int32, dev)
    pages, tabs, strides, widths, widest = [], [], [], [], 0
    for pool, tab in sources:
        if pool is None:
            pages.append(0), tabs.append(0), strides.append(0), widths.append(0)
            continue
        if pool is not kv and pool._kind != kv._kind:
            raise ValueError("the pools differ in device, groups or head widths")
        w = _check_tables("tables", tab, B, dev)
        pages.append(pool._at), tabs.append(tab.data_ptr()), strides.append(tab.stride(0)), widths.append(w)
        widest = max(widest, w * pool.page_size)
    cdt = _ops.compute_dtype(q.dtype)
    qk = _rows16(q, cdt, DK)
    n_slots, idx = 0, 0
    if indices is not None:
        n_slots = indices.shape[-1] if indices.dim() else 0
        if (indices.shape != (B, G, T, n_slots) or not 1 <= n_slots <= 64 or indices.is_floating_point()
                or indices.get_device() != dev):
            _refuse("indices", indices, f"whole numbers [{B}, {G}, {T}, 1 to 64] on cuda:{dev}")
        if indices.dtype is not torch.int64:
            indices = indices.long()
        indices = indices.contiguous()
        idx = indices.data_ptr()
    gate, sg = 0, (0, 0, 0, 0)
    if gates is not None:
        if gates.shape != (B, H, T, 3) or gates.get_device() != dev:
            _refuse("gates", gates, f"[{B}, {H}, {T}, 3] on cuda:{dev}")
        if gates.dtype is not cdt:
            gates = gates.to(cdt)
        gate, sg = gates.data_ptr(), gates.stride()
    if max_length is None:
        max_length = widest
    elif max_length < 1:
        raise ValueError(f"max_length {max_length}")
    # [B,T,H,dv] storage
    out = torch.empty_strided((B, H, T, DV), (T * H * DV, DV, H * DV, 1), device=kv.device, dtype=cdt)
    sq, so = qk.stride(), out.stride()
    a = _ATTN.pack(qk.data_ptr(), out.data_ptr(), gate, idx, lengths.data_ptr(), *pages, *tabs, *strides, *sq[:3], *so[:3], *sg,
                   *widths, B, H, G, T, DK, DV, min(max_length, 1 << 30), l, d, n_slots, block_size, min(window, _INT_MAX),
                   gate_act, _lib.NSA_F32 if cdt is torch.float32 else _lib.NSA_BF16, scale)
    n = _lib.load().nsa_kv4_attn_workspace_size(a)
    ws = torch.empty(n, device=kv.device, dtype=torch.uint8) if n else None
    _launch(dev, "nsa_kv4_attn", a, ws.data_ptr() if n else 0, n)
    if dv != DV:
        out = out[..., :dv]
    return out if q.dtype is cdt else out.to(q.dtype)


def attend_kv4(q: torch.Tensor, kv: PagedKV4, tables: torch.Tensor, lengths: torch.Tensor, scale: float, *,
               window: Optional[int] = None, indices: Optional[torch.Tensor] = None, block_size: int = 64,
               max_length: Optional[int] = None) -> torch.Tensor:
    """Causal attention over 4-bit pages (nsa_kv4_attn): q [B,H,T,dk] are the last T tokens of each
    request, row i at position lengths[b] - T + i; it sees every position up to its own, the last
    `window` of them, or those in its blocks indices [B,G,T,n] of block_size tokens (negative = none, a
    repeat counts once; a row without any takes its own block).  Rows at negative positions and rows
    that see nothing are zero.  tables [B,W], lengths [B] int32.  max_length: a bound that the lengths
    are expected to keep (default: what the tables hold); it decides how the work is split, not the
    result.  Returns [B,H,T,dv] in q's dtype, of [B,T,H,dv] storage."""
    if indices is not None:
        if window is not None or block_size < 16 or block_size % 16:
            raise ValueError(f"indices take no window (got {window}) and a block_size that is a multiple of 16 (got {block_size})")
        return _attend(q, (_NO, (kv, tables), _NO), lengths, scale, indices=indices, block_size=block_size,
                       max_length=max_length)
    if window is None:
        window = _INT_MAX
    elif window < 1:
        raise ValueError(f"window {window} must be at least 1")
    return _attend(q, (_NO, _NO, (kv, tables)), lengths, scale, window, max_length=max_length)


_NO = (None, None)  # a source that is not there
GATE_ACT = {"sigmoid": 1, "softmax": 2}  # gate_act codes of nsa_kv4_attn and nsa_paged_step


def nsa_attend_kv4(q: torch.Tensor, cmp: PagedKV4, sel: PagedKV4, win: PagedKV4, cmp_tables: torch.Tensor,
                   tables: torch.Tensor, lengths: torch.Tensor, indices: torch.Tensor, gates: torch.Tensor, scale: float,
                   config, max_length: Optional[int] = None) -> torch.Tensor:
    """The attention of an NSA layer over 4-bit pages: the compressed tokens completed at each query's
    position (cmp through cmp_tables), its selected blocks (sel) and its window (win; sel and win
    share tables and have pages of one size), each as attend_kv4 takes them, mixed by the activated gates [B,H,T,3] (config's
    gate_mode), in one pass.  A branch that sees nothing adds zero."""
    c = config
    if c.l_prime % 16:
        raise ValueError(f"l_prime {c.l_prime} must be a multiple of 16")
    if sel.page_size != win.page_size:  # the table's pages would stand for other tokens in one of them
        raise ValueError(f"sel and win share tables, but have pages of {sel.page_size} and {win.page_size} tokens")
    return _attend(q, ((cmp, cmp_tables), (sel, tables), (win, tables)), lengths, scale, c.w, indices, c.l_prime, c.l, c.d, gates,
                   GATE_ACT[c.gate_mode], max_length)


# ------------------------------------------------------------------------ a layer's cache
# what a layer and its cache share
_CONFIG = ("head_dim_qk", "head_dim_v", "n_heads", "n_kv_groups", "l", "d", "l_prime", "n", "n_fixed",
           "include_fixed_in_selection", "w", "gate_mode")


def _n_blocks(tokens: int, l: int, d: int) -> int:
    """Compressed tokens completed by that many tokens."""
    return (tokens - l) // d + 1 if tokens >= l else 0


class _Pages:
    """Block tables of one token sequence kind and the free list they draw on: free[used:] are the
    pages nobody holds.  The host keeps the lengths as well, so that a step that does not fit is
    refused before anything is launched."""

    def __init__(self, batch: int, width: int, n_pages: int, page_size: int, device):
        self.page_size, self.n_pages = page_size, n_pages
        self.tables = torch.full((batch, width), -1, device=device, dtype=torch.int32)
        self.free = torch.arange(n_pages, device=device, dtype=torch.int32)
        # What a step leaves (offsets, lengths and info of nsa_block_tables), for every other step: memory that
        # is kept, since the next step may run on another stream than the one that would get it back.
        self._states = [torch.zeros(2 * batch + 4, device=device, dtype=torch.int32) for _ in range(2)]
        self._views = [(t[batch + 1:2 * batch + 1], t[2 * batch + 2:2 * batch + 3]) for t in self._states]
        self._side = 0
        self.lengths, self.used = self._views[0]
        self.host: List[int] = [0] * batch

    @property
    def next_state(self) -> torch.Tensor:
        return self._states[1 - self._side]

    def placed(self, host: List[int]) -> None:
        """next_state is written (or about to be, on this stream), the lengths then being host."""
        self._side = 1 - self._side
        self.lengths, self.used = self._views[self._side]
        self.host = host

    def held(self, tokens: int) -> int:
        return -(-tokens // self.page_size)

    def pages_after(self, new: Sequence[int]) -> int:
        return sum(self.held(m + n) for m, n in zip(self.host, new))

    def place(self, new: Sequence[int], new_dev: torch.Tensor, stride: int) -> BlockTables:
        """Slots of the rows [B, stride] whose first new[b] are sequence b's next tokens."""
        t = build_block_tables(self.tables, self.lengths, new_dev, self.free, self.used, self.page_size,
                               len(self.host) * stride, row_stride=stride)
        B = len(self.host)
        self.next_state[B + 1:].copy_(torch.cat([t.lengths, t.info]))
        self.placed([m + n for m, n in zip(self.host, new)])
        return t

    def release(self, b: int) -> None:
        n, used = self.held(self.host[b]), self.pages_after([0] * len(self.host))
        self.free[used - n:used] = self.tables[b, :n]
        self.tables[b] = -1
        self.used -= n
        self.lengths[b] = 0
        self.host[b] = 0


class NSAPagedKVCache:
    """Decode state of one NSAAttention layer in 4-bit pages (not in the reference), every sequence at a
    length of its own: the keys and values of the selection and window branches (sel, win: one table
    for both) and the compressed tokens (cmp) in PagedKV4 pools, the compressed keys once more in the
    layer's dtype for the block scores (K_cmp), and of the compression branch only the last tokens that
    blocks still to come need.  A token costs 2 (dk + dv) 17/32 bytes a group (bf16 NSAKVCache: 6 (dk +
    dv)), a page only once a sequence reaches it.

    batch sequences of at most max_len tokens share n_pages pages of page_size tokens (default: enough
    for all at max_len).  NSAAttention.prefill / decode raise ValueError, and change nothing, when the
    tokens of a step do not fit; ``release(b)`` empties sequence b for another request."""

    def __init__(self, config, batch: int, max_len: int, device, dtype, page_size: int = 64,
                 n_pages: Optional[int] = None):
        c = self.config = config
        _need(batch >= 1 and max_len >= 1, f"batch {batch}, max_len {max_len}")
        _need(c.l_prime % 16 == 0, f"l_prime {c.l_prime} must be a multiple of 16")
        _need(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}, got {page_size}")
        _need(1 <= c.n <= 64 and c.heads_per_group <= 64, f"n {c.n} or {c.heads_per_group} heads a group outside [1, 64]")
        _need(batch <= MAX_REQUESTS, f"batch {batch} exceeds {MAX_REQUESTS}")
        # what the kernels of a decode step would refuse once its token is stored
        _need(batch * c.n_kv_groups <= MAX_PAIRS, f"{batch} sequences of {c.n_kv_groups} groups: more than {MAX_PAIRS} pairs")
        _need(c.l_prime <= MAX_BLOCK_SIZE, f"l_prime {c.l_prime} exceeds {MAX_BLOCK_SIZE}")
        _need(-(-max_len // page_size) * page_size <= MAX_TOKENS, f"max_len {max_len} exceeds {MAX_TOKENS} tokens")
        _need(_n_blocks(max_len, c.l, c.d) <= MAX_BLOCKS,
              f"{max_len} tokens make {_n_blocks(max_len, c.l, c.d)} compressed blocks, the scoring takes {MAX_BLOCKS}")
        self.batch, self.max_len, self.page_size = batch, max_len, page_size
        with torch.inference_mode(False):  # (tensors made under it could not be written outside)
            self._allocate(device, dtype, n_pages)

    def _allocate(self, device, dtype, n_pages: Optional[int]) -> None:
        c, batch, max_len, page_size = self.config, self.batch, self.max_len, self.page_size
        G, dk, dv = c.n_kv_groups, c.head_dim_qk, c.head_dim_v
        width, n_max = -(-max_len // page_size), max(_n_blocks(max_len, c.l, c.d), 1)
        n_pages = batch * width if n_pages is None else n_pages
        cmp_width = -(-n_max // page_size)
        # sequences of T tokens in all hold at most T / d compressed tokens, and a part page each
        n_cmp = min(batch * cmp_width, n_pages // c.d + batch)
        self.sel = PagedKV4.empty(n_pages, page_size, G, dk, dv, device)
        self.win = PagedKV4.empty(n_pages, page_size, G, dk, dv, device)
        self.cmp = PagedKV4.empty(n_cmp, page_size, G, dk, dv, device)
        self._tokens = _Pages(batch, width, n_pages, page_size, device)
        self._blocks = _Pages(batch, cmp_width, n_cmp, page_size, device)
        # one row more, where the rows of no sequence go
        self._K_cmp = torch.zeros(batch, G, n_max + 1, dk, device=device, dtype=dtype)
        self.block_ends = torch.arange(n_max, device=device, dtype=torch.int32) * c.d + (c.l - 1)
        self._ones = torch.ones(batch, device=device, dtype=torch.int32)
        self._steps = torch.arange(max(batch, c.l), device=device, dtype=torch.int32)
        # the last l tokens of each sequence, token m at place m % l
        self._tail = torch.zeros(batch, c.l, G * (dk + dv), device=device, dtype=dtype)

    @property
    def lengths(self) -> List[int]:
        """Tokens of each sequence."""
        return list(self._tokens.host)

    @property
    def K_cmp(self) -> torch.Tensor:
        """Compressed keys [B,G,dk,blocks] in the layer's dtype (zeros past a sequence's own)."""
        return self._K_cmp[:, :, :-1].transpose(-1, -2)

    def _not_captured(self) -> None:
        if self.sel._dev >= 0 and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a step of an NSAPagedKVCache cannot be captured into a graph: the host keeps its lengths too")

    def check(self, new: Sequence[int], x: Optional[torch.Tensor] = None, config=None) -> None:
        """Raises ValueError unless sequence b has room for new[b] tokens more (and rows x are on the cache's device, a
        layer's config is the cache's), RuntimeError in a graph's capture: the host keeps the lengths too, and
        a replay would not move them."""
        if x is not None and x.device != self._tail.device:
            raise ValueError(f"rows on {x.device} for a cache on {self._tail.device}")
        if config is not None and config is not self.config:
            for f in _CONFIG:
                _need(getattr(config, f) == getattr(self.config, f),
                      f"a layer with {f} {getattr(config, f)} and a cache made for {getattr(self.config, f)}")
        self._not_captured()
        _need(len(new) == self.batch, f"{len(new)} counts for {self.batch} sequences")
        most, page, need = self.max_len, self.page_size, 0
        for b, (m, n) in enumerate(zip(self._tokens.host, new)):
            if n < 0 or m + n > most:
                raise ValueError(f"sequence {b}: cache holds {most} tokens, {m + n} requested")
            need -= -(m + n) // page
        if need > self._tokens.n_pages:
            raise ValueError(f"the cache's {self._tokens.n_pages} pages do not hold these tokens: {need} needed")

    def append(self, kv, new: Sequence[int], compress, weights=lambda cache: None) -> None:
        """The first new[b] tokens of each sequence's rows (which `check` has let through) join the cache: kv = the
        selection's and the window's k and v [B,T,G,d] and the compression's [B,T,G dk + G dv], k then v;
        compress(keys [B,G,n,dk], values) -> (K_cmp [B,G,dk,blocks], V_cmp [B,G,blocks,dv], ...) over n tokens;
        weights(self) -> its layers' (E, W1, b1, W2, b2) for nsa_paged_blocks, or None."""
        if not any(new):
            return
        c, B, T, dev = self.config, self.batch, kv[0].shape[1], self._tail.device
        before, had = self._tokens.lengths, self._blocks.host
        t = self._tokens.place(new, self._counts(new), T)
        for pool, k, v in ((self.sel, kv[0], kv[1]), (self.win, kv[2], kv[3])):
            store_kv4(pool, k.flatten(0, 1), v.flatten(0, 1).to(k.dtype), t.slots)
        fresh = [_n_blocks(m, c.l, c.d) - h for m, h in zip(self._tokens.host, had)]
        n = max(fresh)
        tail, x = self._tail, kv[4] if kv[4].dtype is self._tail.dtype else kv[4].to(self._tail.dtype)
        if T == 1:
            # Token m of a sequence has the place m % l.  A sequence without a token gets a row too, where
            # its next one goes: the token there, l before it, is in no block to come.
            tail.scatter_(1, before.remainder(c.l).long().view(B, 1, 1).expand_as(x), x)
            if n:
                self._close_blocks(fresh, compress, weights(self))
            return
        old = torch.cat([tail, x], 1)
        if n:  # the tokens from each sequence's first open block on
            span = (n - 1) * c.d + c.l
            at = (self._blocks.lengths * c.d)[:, None] + torch.arange(span, device=dev)
            j = torch.where(at < before[:, None], at % c.l, c.l + at - before[:, None]).clamp_(max=c.l + T - 1)
            buf = old.gather(1, j[:, :, None].expand(-1, -1, old.shape[2]))
        # each place's last token
        at = t.lengths[:, None] - 1 - (t.lengths[:, None] - 1 - self._steps[:c.l]) % c.l
        j = torch.where(at >= before[:, None], c.l + at - before[:, None], self._steps[:c.l]).long()
        tail.copy_(old.gather(1, j[:, :, None].expand_as(tail)))
        if n:
            self._add_blocks(fresh, buf, compress)

    def _counts(self, new: Sequence[int]) -> torch.Tensor:
        """new on the device [B] int32."""
        dev = self._tail.device
        if min(new) == max(new):
            return self._ones if new[0] == 1 else torch.full((self.batch,), new[0], device=dev, dtype=torch.int32)
        # copied as the stream comes to it: the host does not wait
        return torch.tensor(new, dtype=torch.int32, pin_memory=True).to(dev, non_blocking=True)

    def step(self, x: torch.Tensor, layers, new: Sequence[int], scale: float, compress, weights, project: bool) -> torch.Tensor:
        """A decode step in one library call (nsa_paged_step; two around `compress` when it completes a block and
        weights(self) is None, see append): the token rows x [B,D]
        (16-byte aligned) through the layers (q, the six of the caches, the gate's two, the output's), sequences with
        new[b] = 1 (which `check` has let through) taking theirs.  Returns [B,D], or with project False the mixed
        heads [B,H dv]."""
        c, tk, bk = self.config, self._tokens, self._blocks
        B, D = x.shape
        H, G, dk, dv = c.n_heads, c.n_kv_groups, c.head_dim_qk, c.head_dim_v
        n_out = D if project else H * dv
        out, state = x.new_empty(B, n_out), tk.next_state
        counts, host, l, d = self._counts(new), [m + n for m, n in zip(tk.host, new)], c.l, c.d
        fresh = [1 if n and m >= l and (m - l) % d == 0 else 0 for m, n in zip(host, new)]
        ends = max(_n_blocks(max(host), l, d), 1)
        ends = min(1 << (ends - 1).bit_length(), self.block_ends.shape[0])
        ps = [m._parameters for m in layers]
        kc = self._K_cmp
        w = [p["weight"].data_ptr() for p in ps]
        if not project:
            w[9] = 0
        a = [x.data_ptr(), *w, *(0 if p["bias"] is None else p["bias"].data_ptr() for p in ps), self.cmp._at, self.sel._at,
             self.win._at, tk.tables.data_ptr(), bk.tables.data_ptr(), tk.lengths.data_ptr(), counts.data_ptr(),
             tk.free.data_ptr(), tk.used.data_ptr(), state.data_ptr(), self._tail.data_ptr(), kc.data_ptr(),
             self.block_ends.data_ptr(), out.data_ptr(), x.stride(0), n_out, *[D] * 8, layers[8].in_features, H * dv,
             tk.tables.stride(0), bk.tables.stride(0), *kc.stride()[:3], B, H, G, D, dk, dv, layers[8].in_features,
             tk.tables.shape[1], bk.tables.shape[1], tk.n_pages, ends, max(host) or 1, c.l, c.d, c.l_prime, c.n,
             int(bool(c.include_fixed_in_selection)), int(c.n_fixed), min(c.w, _INT_MAX), GATE_ACT[c.gate_mode],
             _lib.NSA_F32 if x.dtype is torch.float32 else _lib.NSA_BF16, 3, scale, 0]
        blocks = None
        if any(fresh):
            mlp = weights(self)
            if mlp is None:
                a[-3] = 1
            else:
                blocks = self._blocks_args(fresh, mlp, state.data_ptr() + 4 * (B + 1))
                a[-1] = ctypes.addressof(blocks)
        args = _STEP.pack(*a)
        nb = _lib.load().nsa_paged_step_workspace_size(args)
        ws = torch.empty(nb, device=x.device, dtype=torch.uint8)
        dev = self.sel._dev
        _launch(dev, "nsa_paged_step", args, ws.data_ptr(), nb)
        tk.placed(host)
        if blocks is not None:
            bk.placed([n + f for n, f in zip(bk.host, fresh)])
        elif any(fresh):
            self._close_blocks(fresh, compress, None)
            a[-3] = 2
            _launch(dev, "nsa_paged_step", _STEP.pack(*a), ws.data_ptr(), nb)
        return out

    def _blocks_args(self, fresh: Sequence[int], ws, token_lengths: int):
        """nsa_paged_blocks' packed arguments for the blocks of fresh (0 or 1 each)."""
        c, bk, kc, B = self.config, self._blocks, self._K_cmp, self.batch
        p = [0 if t is None else t.data_ptr() for t in ws]
        args = _BLOCKS.pack(self.cmp._at, bk.tables.data_ptr(), token_lengths, bk.lengths.data_ptr(), bk.free.data_ptr(),
                            bk.used.data_ptr(), bk.next_state.data_ptr(), self._tail.data_ptr(), kc.data_ptr(), *p,
                            sum(1 << b for b, f in enumerate(fresh) if f), bk.tables.stride(0), *kc.stride()[:3], B,
                            c.n_kv_groups, c.head_dim_qk, c.head_dim_v, bk.tables.shape[1], bk.n_pages, c.l,
                            _lib.NSA_F32 if kc.dtype is torch.float32 else _lib.NSA_BF16)
        return ctypes.create_string_buffer(args, len(args))

    def _close_blocks(self, fresh: Sequence[int], compress, ws) -> None:
        """The blocks that a step of single tokens completed (fresh[b]: 0 or 1): each the last l tokens."""
        if ws is not None:
            args, bk = self._blocks_args(fresh, ws, self._tokens.lengths.data_ptr()), self._blocks
            nb = _lib.load().nsa_paged_blocks_workspace_size(args)
            buf = torch.empty(nb, device=self._tail.device, dtype=torch.uint8)
            _launch(self.sel._dev, "nsa_paged_blocks", args, buf.data_ptr(), nb)
            return bk.placed([n + f for n, f in zip(bk.host, fresh)])
        j = (self._tokens.lengths[:, None] + self._steps[:self.config.l]).remainder_(self.config.l).long()
        self._add_blocks(fresh, self._tail.gather(1, j[:, :, None].expand_as(self._tail)), compress)

    def _add_blocks(self, fresh: Sequence[int], buf: torch.Tensor, compress) -> None:
        """The next fresh[b] compressed tokens of each sequence, from its tokens buf [B,n,G dk + G dv] (from its first
        open block on)."""
        c, n, B, dev = self.config, max(fresh), self.batch, buf.device
        G, (dk, dv) = c.n_kv_groups, (c.head_dim_qk, c.head_dim_v)
        buf = [y.unflatten(2, (G, -1)).transpose(1, 2) for y in buf.split_with_sizes((G * dk, G * dv), 2)]
        kc, vc = compress(*buf)[:2]
        kc, vc = kc[..., :n].permute(0, 3, 1, 2).flatten(0, 1), vc[:, :, :n].transpose(1, 2).flatten(0, 1)  # [B n,G,d]
        kc, vc = kc.to(self._K_cmp.dtype), vc.to(self._K_cmp.dtype)  # (under autocast they differ)
        fresh_dev = torch.div(self._tokens.lengths + (c.d - c.l), c.d, rounding_mode="floor").clamp_(min=0) - self._blocks.lengths
        bt = self._blocks.place(fresh, fresh_dev, n)
        store_kv4(self.cmp, kc, vc, bt.slots)
        none = self._K_cmp.shape[2] - 1
        pos = torch.where(bt.positions < 0, none, bt.positions)
        rows = self._steps[:B] if n == 1 else torch.arange(B, device=dev).repeat_interleave(n)
        self._K_cmp[rows, :, pos] = kc

    def release(self, b: int) -> None:
        """Empties sequence b: its pages are free again (not in a graph's capture, as for a step)."""
        _need(0 <= b < self.batch, f"sequence {b} of {self.batch}")
        self._not_captured()
        self._tokens.release(b)
        self._blocks.release(b)
        # a request without a completed block is scored against block 0, which must not be the last one's
        self._K_cmp[b].zero_()
