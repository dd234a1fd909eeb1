"""Paged key-value cache and beam search's selection on PyTorch tensors (cudallm_paged_*, cudallm_beam_select).

A `PagedCache` is a pool of pages for every layer. A sequence is a row of a page table (int32 [rows][width], -1 where
there is no page) with a length; any number of rows may share pages, counted in `refs` (int32 [pages]). A decode loop
over beams, per step:

    tables, lens, refs, missing = cache.fork(tables, lens, refs, parents.view(-1), room=1)   # who continues whom
    for layer in range(layers):
        turned = cache.append(q, k, v, lens, tables, rope, layer=layer)   # q, k, v of the layer; rotate, store at position lens
        out = cache.attend(turned, tables, lens + 1, layer=layer)
    lens = lens + 1                                                       # the token that was stored counts from here on
    scores, parents, tokens = beam_select(logits, scores, keep=beams)

Every call enqueues its work on the current stream of the cache's device, reads lengths, tables and parents there
(nothing is copied to the host or waited for) and returns new tensors unless `out` is given. Errors in what the
host can see raise CudaLLMError (INVALID_ARG) before anything runs; contents out of range are bounded as
include/cudallm.h states. A cache serves one host thread at a time. No gradient flows through these calls: outputs are detached from
inputs that require one.
"""
from __future__ import annotations

import ctypes
import functools
import math
import threading

import torch

from . import abi
from .abi import CudaLLMError, check, lib

__all__ = ["PagedCache", "Rope", "beam_select"]

try:  # a tenth of the time of torch.cuda.current_stream, half of torch.cuda.current_device
    from torch._C import _cuda_getCurrentRawStream as _stream_of
    from torch._C import _cuda_getDevice as _current_device
except ImportError:
    def _stream_of(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream

    _current_device = torch.cuda.current_device

_X = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_KV = {torch.float16: 0, torch.bfloat16: 1}
_INVALID_ARG = 1
_INT_MAX = 2 ** 31 - 1
_BEAM_COUNTERS = 16384  # CUDALLM_BEAM_COUNTER_BYTES


def _refuse(message: str):
    raise CudaLLMError(_INVALID_ARG, message)


def _need(ok: bool, message: str) -> None:
    if not ok:
        _refuse(message)


def _args(name: str):
    """A zeroed argument struct with its struct_size, and its reference."""
    a = abi.struct(name)()
    a.struct_size = ctypes.sizeof(a)
    return a, ctypes.byref(a)


_beam = threading.local()


@functools.cache
def _beam_calls():
    return lib().cudallm_beam_select, lib().cudallm_beam_workspace_bytes


def _beam_args():
    """This thread's argument struct of beam_select, its reference, and this thread's workspaces by device: two launches make up a call, and those
    of two threads on one stream may come in between each other."""
    if not hasattr(_beam, "args"):
        _beam.args = (*_args("cudallm_beam_args"), {})
    return _beam.args


class _Workspaces:
    """A workspace for each of a device's streams (calls on different streams may overlap)."""

    def __init__(self, device: torch.device, counters: int = 0):
        self.device, self.counters = device, counters  # leading bytes that start at zero
        self.by_stream: dict[int, torch.Tensor] = {}

    def _new(self, size: int) -> torch.Tensor:
        w = torch.empty(size, dtype=torch.uint8, device=self.device)
        if self.counters:
            w[:self.counters].zero_()
        return w

    def _capturing(self) -> bool:
        """Whether this device's current stream is being captured (torch answers for the current device)."""
        if _current_device() == self.device.index:
            return torch.cuda.is_current_stream_capturing()
        with _OnDevice(self.device.index):
            return torch.cuda.is_current_stream_capturing()

    def get(self, stream: int, size: int) -> torch.Tensor:
        if self._capturing():  # the graph's own, which later calls must not replace
            return self._new(size)
        w = self.by_stream.get(stream)
        if w is None or w.numel() < size:
            w = self.by_stream[stream] = self._new(size)
        return w


class _OnDevice:
    """Makes a device current for a call where another one is."""

    __slots__ = ("index", "was")

    def __init__(self, index: int):
        self.index = index

    def __enter__(self):
        self.was = torch.cuda.current_device()
        if self.was != self.index:
            torch.cuda.set_device(self.index)

    def __exit__(self, *exc):
        if self.was != self.index:
            torch.cuda.set_device(self.was)


def _int32(t: torch.Tensor, device: torch.device, shape: tuple, name: str) -> int:
    if t.dtype is not torch.int32 or t.get_device() != device.index or t.shape != shape or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous int32 tensor {list(shape)} on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    return t.data_ptr()


def _table(t: torch.Tensor, device: torch.device, name: str) -> tuple[int, int, int]:
    """(rows, width, row stride) of a page table."""
    if t.dtype is not torch.int32 or t.get_device() != device.index or t.dim() != 2:
        _refuse(f"{name} must be an int32 tensor [rows][width] on {device}")
    rows, width = t.shape
    if rows | width > _INT_MAX:  # all ones below 2^31: either of them is
        _refuse(f"{name} must have fewer than 2^31 rows and entries a row")
    stride, inner = t.stride()
    if inner != 1 and rows and width > 1:
        _refuse(f"{name} must have its entries side by side")
    return rows, width, stride


def _heads(t: torch.Tensor, device: torch.device, dtype: torch.dtype, dim: int, name: str) -> tuple[int, int, int, int]:
    """(tokens, heads, token stride, head stride) of [tokens][heads][dim]."""
    if t.dtype is not dtype or t.get_device() != device.index or t.dim() != 3:
        _refuse(f"{name} must be a {dtype} tensor [tokens][heads][{dim}] on {device}, got {t.dtype} {list(t.shape)} on {t.device}")
    n, heads, d = t.shape
    if n | heads > _INT_MAX:
        _refuse(f"{name} must have fewer than 2^31 tokens and heads")
    ts, hs, inner = t.stride()
    if d != dim or (inner != 1 and n and heads):
        _refuse(f"{name} must be [tokens][heads][{dim}] with its dims side by side, got {list(t.shape)} with strides {list(t.stride())}")
    return n, heads, ts, hs


class Rope:
    """Rotary positions: inverse frequencies (fp32 tensor on the GPU; twice as many dims turn, the rest of a head is
    copied), pairs (2j, 2j + 1) if `interleaved` else (j, j + n), and a factor of cos and sin."""

    def __init__(self, inv_freq: torch.Tensor, *, interleaved: bool = False, factor: float = 1.0):
        _need(inv_freq.dtype is torch.float32 and inv_freq.dim() == 1 and inv_freq.is_contiguous() and inv_freq.is_cuda,
              "inv_freq must be a contiguous fp32 vector on the GPU")
        self.inv_freq, self.interleaved, self.factor = inv_freq, bool(interleaved), float(factor)
        self.rotary = 2 * inv_freq.numel()

    @classmethod
    def make(cls, rotary: int, *, theta: float = 500000.0, scaling: str = "none", scale: float = 1.0, original: float = 8192.0,
             low: float = 1.0, high: float | None = None, interleaved: bool = False, device="cuda") -> "Rope":
        """Frequencies theta^(-2j / rotary), for contexts `scale` times the `original` length: "linear" divides all of them by
        `scale`; "llama3" and "yarn" divide those that turn fewer than `low` times within `original` positions, keep
        those that turn more than `high` times (4 and 32) and blend between, linearly in the number of turns; yarn also
        multiplies cos and sin by 0.1 ln(scale) + 1. Some loaders of yarn checkpoints blend linearly in the index of the
        pair between the same two ends instead, which gives other frequencies: pass theirs to Rope itself."""
        _need(rotary > 0 and rotary % 2 == 0, "rotary must be positive and even")
        _need(scaling in ("none", "linear", "llama3", "yarn"), "scaling must be none, linear, llama3 or yarn")
        f = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
        factor = 1.0
        if scaling == "linear":
            f = f / scale
        elif scaling != "none":
            high = high if high is not None else 4.0 if scaling == "llama3" else 32.0
            keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
            f = f * (keep + (1 - keep) / scale)
            if scaling == "yarn" and scale > 1:
                factor = 0.1 * math.log(scale) + 1.0
        return cls(f.to(torch.float32).to(device), interleaved=interleaved, factor=factor)


class PagedCache:
    """Pages of keys and values: tensors [layers][pages][kv heads][page size][head dim], fp16 or bf16, on one GPU, with any
    strides (multiples of 8 elements, the same for both) as long as a head's dims lie side by side; pages whose memory is
    token by token are passed as their transposed view."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        _need(k.dim() == 5 and k.shape == v.shape and k.dtype == v.dtype and k.dtype in _KV and k.is_cuda and k.device == v.device,
              "k and v must be fp16 or bf16 tensors [layers][pages][kv heads][page size][head dim] of one shape on one GPU")
        _need(max(k.shape) <= _INT_MAX, "sizes must be below 2^31")
        _need(k.stride() == v.stride() and k.stride(4) == 1, "k and v must have the same strides, and a head's dims side by side")
        self.k, self.v, self.device = k, v, k.device
        self._index = k.device.index
        self.n_layers, self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        p, self._pages = _args("cudallm_pages")
        p.kv_dtype = _KV[k.dtype]
        p.n_layers, p.n_pages, p.n_kv_heads, p.page_size, p.head_dim = k.shape
        p.k, p.v = k.data_ptr(), v.data_ptr()
        p.layer_stride, p.page_stride, p.head_stride, p.token_stride = k.stride()[:4]
        self._lib = lib()
        self._call_attend, self._call_append = self._lib.cudallm_paged_attend, self._lib.cudallm_paged_append
        self._call_fork, self._call_compact = self._lib.cudallm_paged_fork, self._lib.cudallm_paged_compact
        self._attend, self._attend_ref = _args("cudallm_attend_args")
        self._append, self._append_ref = _args("cudallm_append_args")
        self._fork, self._fork_ref = _args("cudallm_fork_args")
        self._compact, self._compact_ref = _args("cudallm_compact_args")
        self._workspaces = _Workspaces(self.device)
        self._scale = self.head_dim ** -0.5
        self._pages_bytes: dict[int, int] = {}  # workspace of fork and compact by rows
        self._attend_bytes = self._lib.cudallm_attend_workspace_bytes()
        check(self._lib.cudallm_paged_attend(self._pages, self._attend_ref, None))  # no rows: checks the pool alone

    @classmethod
    def allocate(cls, n_layers: int, n_pages: int, n_kv_heads: int, page_size: int, head_dim: int, *, dtype=torch.float16,
                 device="cuda") -> "PagedCache":
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    def rows(self, n: int, width: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """(tables, lens, refs) of n empty rows of up to `width` pages, with no page in use."""
        new = lambda shape, v: torch.full(shape, v, dtype=torch.int32, device=self.device)  # noqa: E731
        return new((n, width), -1), new((n,), 0), new((self.n_pages,), 0)

    def _run(self, fn, args_ref, stream: int) -> None:
        if _current_device() == self._index:
            rc = fn(self._pages, args_ref, stream)
        else:
            with _OnDevice(self._index):
                rc = fn(self._pages, args_ref, stream)
        if rc:
            check(rc)

    def _workspace(self, a, size: int, stream: int):
        w = self._workspaces.get(stream, size)
        a.workspace, a.workspace_bytes = w.data_ptr(), w.numel()
        return w

    def _pages_size(self, rows: int) -> int:
        size = self._pages_bytes.get(rows)
        if size is None:
            size = self._pages_bytes[rows] = self._lib.cudallm_pages_workspace_bytes(self.n_pages, rows)
        return size

    def attend(self, q: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, *, layer: int = 0, scale: float | None = None,
               window: int = 0, out: torch.Tensor | None = None, with_lse: bool = False):
        """Attention of one new token per row: q [rows][heads][head dim] (fp32, fp16 or bf16) over the first lens[row] tokens of
        the row's pages, the last `window` of them if that is not 0; scale None is head_dim ** -0.5. Returns out (q's type),
        or (out, lse fp32 [rows][heads])."""
        n, heads, a_seq, a_head = _heads(q, self.device, q.dtype, self.head_dim, "q")
        x = _X.get(q.dtype)
        if x is None:
            _refuse("q must be fp32, fp16 or bf16")
        rows, width, stride = _table(tables, self.device, "tables")
        if rows != n:
            _refuse(f"tables has {rows} rows for {n} queries")
        if not (0 <= layer < self.n_layers and 0 <= window <= _INT_MAX):
            _refuse(f"layer must be in [0, {self.n_layers}), window not negative and below 2^31")
        a = self._attend
        a.lens = _int32(lens, self.device, (n,), "lens")
        if out is None:
            contiguous = a_head == self.head_dim and a_seq == heads * a_head
            out = torch.empty_like(q) if contiguous else q.new_empty(n, heads, self.head_dim)
        elif out.dtype is not q.dtype or out.device != self.device or out.shape != q.shape or not out.is_contiguous():
            _refuse("out must be contiguous, with q's shape and type")
        lse = None if not with_lse else q.new_empty(n, heads, dtype=torch.float32)
        a.layer, a.x_dtype, a.n_seq, a.n_heads, a.table_width, a.window = layer, x, n, heads, width, window
        a.scale = self._scale if scale is None else scale
        a.q, a.q_seq_stride, a.q_head_stride = q.data_ptr(), a_seq, a_head
        a.tables, a.table_stride, a.out = tables.data_ptr(), stride, out.data_ptr()
        a.lse = None if lse is None else lse.data_ptr()
        stream = _stream_of(self._index)
        keep = self._workspace(a, self._attend_bytes, stream)  # noqa: F841  lives until the launch
        self._run(self._call_attend, self._attend_ref, stream)
        return (out, lse) if with_lse else out

    def append(self, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, tables: torch.Tensor,
               rope: Rope | None, *, layer: int = 0, rows: torch.Tensor | None = None, out: torch.Tensor | None = None):
        """Rotates q [tokens][heads][head dim] and k, and stores k and v [tokens][kv heads][head dim] (all of one type, any strides
        with dims side by side) at `positions` (int32) of the table rows `rows` (int32; None: token i is row i). A negative
        position is padding. Returns the rotated q (`out` may be q itself), None without a q; rope None: no rotation."""
        dev, dim, a = self.device, self.head_dim, self._append
        x = _X.get(k.dtype)
        if x is None:
            _refuse("q, k and v must be fp32, fp16 or bf16")
        if not 0 <= layer < self.n_layers:
            _refuse(f"layer must be in [0, {self.n_layers})")
        n, kv_heads, a.k_token_stride, a.k_head_stride = _heads(k, dev, k.dtype, dim, "k")
        nv, v_heads, a.v_token_stride, a.v_head_stride = _heads(v, dev, k.dtype, dim, "v")
        if kv_heads != self.n_kv_heads or v_heads != kv_heads or nv != n:
            _refuse(f"k and v must be [tokens][{self.n_kv_heads}][{dim}]")
        n_rows, width, stride = _table(tables, dev, "tables")
        heads = 0
        a.q = a.q_out = None
        if q is not None:
            nq, heads, a.q_token_stride, a.q_head_stride = _heads(q, dev, k.dtype, dim, "q")
            if nq != n:
                _refuse("q, k and v must have the same number of tokens")
            if out is None:
                out = q.new_empty(n, heads, dim)
                a.out_token_stride, a.out_head_stride = heads * dim, dim
            elif out.shape != q.shape:
                _refuse("out must have q's shape")
            else:
                _, _, a.out_token_stride, a.out_head_stride = _heads(out, dev, k.dtype, dim, "out")
            a.q, a.q_out = q.data_ptr(), out.data_ptr()
        elif out is not None:
            _refuse("out needs a q")
        a.positions = _int32(positions, dev, (n,), "positions")
        a.rows = None if rows is None else _int32(rows, dev, (n,), "rows")
        a.layer, a.x_dtype, a.n_tokens, a.n_heads, a.n_rows, a.table_width = layer, x, n, heads, n_rows, width
        if rope is None:
            a.rotary, a.inv_freq, a.factor = 0, None, 1.0
        else:
            if rope.inv_freq.device != dev:
                _refuse("the rotation's frequencies must be on the cache's device")
            a.rotary, a.interleaved, a.factor, a.inv_freq = rope.rotary, rope.interleaved, rope.factor, rope.inv_freq.data_ptr()
        a.k, a.v, a.tables, a.table_stride = k.data_ptr(), v.data_ptr(), tables.data_ptr(), stride
        self._run(self._call_append, self._append_ref, _stream_of(self._index))
        return out

    def fork(self, tables: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, *, room: int = 1,
             out: tuple | None = None):
        """The next step's rows: row i continues row parents[i] (outside the rows: empty, which frees), sharing its full pages,
        with its own copy of the page being filled, and with pages for `room` more tokens. Returns (tables, lens, refs,
        missing); missing [1] is how many pages there were too few (the inputs are unchanged and can be used again).
        `out` = such a tuple to write, which must not overlap the inputs (a program keeps two and swaps them)."""
        dev, a = self.device, self._fork
        n_rows, width, a.table_stride = _table(tables, dev, "tables")
        if parents.dim() != 1 or not 0 <= room <= _INT_MAX:
            _refuse("parents must be a vector, room not negative and below 2^31")
        n_out = parents.shape[0]
        if n_out > _INT_MAX:
            _refuse("parents must have fewer than 2^31 entries")
        a.lens = _int32(lens, dev, (n_rows,), "lens")
        a.refs = _int32(refs, dev, (self.n_pages,), "refs")
        a.parents = _int32(parents, dev, (n_out,), "parents")
        a.tables = tables.data_ptr()
        if out is None:
            out = t, n, r, missing = tables.new_empty(n_out, width), torch.empty_like(parents), torch.empty_like(refs), refs.new_empty(1)
            a.tables_out, a.table_out_stride = t.data_ptr(), width
            a.lens_out, a.refs_out, a.missing = n.data_ptr(), r.data_ptr(), missing.data_ptr()
        else:
            t_rows, t_width, a.table_out_stride = _table(out[0], dev, "out tables")
            if t_rows != n_out or t_width != width:
                _refuse(f"out tables must be [{n_out}][{width}]")
            a.tables_out = out[0].data_ptr()
            a.lens_out = _int32(out[1], dev, (n_out,), "out lens")
            a.refs_out = _int32(out[2], dev, (self.n_pages,), "out refs")
            a.missing = _int32(out[3], dev, (1,), "missing")
        a.n_rows, a.n_out, a.table_width, a.room = n_rows, n_out, width, room
        stream = _stream_of(self._index)
        keep = self._workspace(a, self._pages_size(n_rows if n_rows > n_out else n_out), stream)  # noqa: F841
        self._run(self._call_fork, self._fork_ref, stream)
        return out

    def compact(self, tables: torch.Tensor, refs: torch.Tensor, *, out: tuple | None = None):
        """Moves the pages in use (refs > 0) to the front of the pool, all layers. Returns (tables, refs, live): the entries'
        and references' new places and how many pages are in use (int32 [1]); pages from `live` on are free."""
        dev, a = self.device, self._compact
        n_rows, width, a.table_stride = _table(tables, dev, "tables")
        a.refs = _int32(refs, dev, (self.n_pages,), "refs")
        a.tables = tables.data_ptr()
        if out is None:
            out = t, r, live = tables.new_empty(n_rows, width), torch.empty_like(refs), refs.new_empty(1)
            a.tables_out, a.table_out_stride, a.refs_out, a.live = t.data_ptr(), width, r.data_ptr(), live.data_ptr()
        else:
            t_rows, t_width, a.table_out_stride = _table(out[0], dev, "out tables")
            if t_rows != n_rows or t_width != width:
                _refuse(f"out tables must be [{n_rows}][{width}]")
            a.tables_out = out[0].data_ptr()
            a.refs_out = _int32(out[1], dev, (self.n_pages,), "out refs")
            a.live = _int32(out[2], dev, (1,), "live")
        a.n_rows, a.table_width = n_rows, width
        stream = _stream_of(self._index)
        keep = self._workspace(a, self._pages_size(n_rows), stream)  # noqa: F841
        self._run(self._call_compact, self._compact_ref, stream)
        return out


def beam_select(logits: torch.Tensor, scores: torch.Tensor, *, keep: int, finished: torch.Tensor | None = None, eos: int = 0,
                out: tuple | None = None):
    """The `keep` best continuations of each group of beams: logits [groups * beams][vocab] (fp32, fp16 or bf16), scores fp32
    [groups][beams] (the beams' log-probabilities so far), finished int32 [groups][beams] (a beam with a nonzero value only
    continues with `eos`, at its score). Returns (scores fp32, parents int32, tokens int32), each [groups][keep], best
    first; parents are rows of logits, as PagedCache.fork takes them (flattened). Equal candidates go to the lower row, then
    token. Any thread may call it."""
    x = _X.get(logits.dtype)
    if x is None or logits.dim() != 2 or not logits.is_cuda:
        _refuse("logits must be an fp32, fp16 or bf16 tensor [groups * beams][vocab] on the GPU")
    dev = logits.device
    if scores.dtype is not torch.float32 or scores.device != dev or scores.dim() != 2 or not scores.is_contiguous():
        _refuse("scores must be a contiguous fp32 tensor [groups][beams] on the logits' device")
    groups, beams = scores.shape
    rows, vocab = logits.shape
    row_stride, inner = logits.stride()
    if rows != groups * beams or (rows and vocab > 1 and inner != 1):
        _refuse("logits must have groups * beams rows with their values side by side")
    if not (1 <= keep <= _INT_MAX and 0 <= eos <= _INT_MAX and rows | vocab <= _INT_MAX):
        _refuse("keep must be positive, eos a token, and sizes below 2^31")
    a, ref, spaces_of = _beam_args()
    a.finished = None if finished is None else _int32(finished, dev, (groups, beams), "finished")
    if out is None:
        best = scores.new_empty(groups, keep)
        parents = torch.empty_like(best, dtype=torch.int32)
        tokens = torch.empty_like(parents)
        out = best, parents, tokens
        a.out_scores, a.out_parents, a.out_tokens = best.data_ptr(), parents.data_ptr(), tokens.data_ptr()
    else:
        if out[0].dtype is not torch.float32 or out[0].device != dev or out[0].shape != (groups, keep) or not out[0].is_contiguous():
            _refuse("out scores must be a contiguous fp32 tensor [groups][keep]")
        a.out_scores = out[0].data_ptr()
        a.out_parents = _int32(out[1], dev, (groups, keep), "out parents")
        a.out_tokens = _int32(out[2], dev, (groups, keep), "out tokens")
    a.x_dtype, a.n_groups, a.beams, a.keep, a.vocab, a.eos = x, groups, beams, keep, vocab, eos
    a.logits, a.row_stride, a.scores = logits.data_ptr(), row_stride, scores.data_ptr()
    select, size = _beam_calls()
    index = dev.index
    stream = _stream_of(index)
    spaces = spaces_of.get(index)
    if spaces is None:
        spaces = spaces_of[index] = _Workspaces(dev, _BEAM_COUNTERS)
    w = spaces.get(stream, size(rows, vocab, keep))
    a.workspace, a.workspace_bytes = w.data_ptr(), w.numel()
    if _current_device() == index:
        rc = select(ref, stream)
    else:
        with _OnDevice(index):
            rc = select(ref, stream)
    if rc:
        check(rc)
    return out
