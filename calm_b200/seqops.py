"""Operators of the layer-list library on the caller's own GPU tensors (include/calm_b200_seq.h, second half): the n best continuations of beams, copies of
cache pages and state slots, caches of keys and values in 8 and in 16 bits and attention over them, prefixes that sequences share, rotary positions.  The serving runtime (seqlib.SeqDeviceModel, serving.Scheduler) runs
on the kernels of the beams, the copies and the 8-bit cache; rotary positions, the 16-bit cache and shared prefixes are for callers with a loop of their own.

Calls run on torch's current stream of the tensors' device, return before the work is done and can be captured into CUDA graphs.  What a call refuses raises
ValueError before anything is launched.  None has a gradient: results require none, whatever the inputs do.  Like everywhere in this package there is no CPU path."""
from __future__ import annotations

import ctypes as C
import math
from array import array
from operator import index as index_of
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from . import seqlib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # enum SeqType
_int, _ll, _ptr, _size = C.c_int, C.c_longlong, C.c_void_p, C.c_size_t


class _Beam(C.Structure):
    _fields_ = [("logits", _ptr), ("type", _int), ("group_stride", _ll), ("row_stride", _ll), ("scores", _ptr), ("groups", _int), ("beams", _int), ("vocab", _int), ("n", _int),
                ("tokens", _ptr), ("parents", _ptr), ("best", _ptr), ("workspace", _ptr), ("workspace_bytes", _size)]


class _Units(C.Structure):
    _fields_ = [("src", _ptr), ("dst", _ptr), ("unit_bytes", _ll), ("row_bytes", _ll), ("src_units", _int), ("dst_units", _int), ("kind", _int)]


class _Cache8(C.Structure):
    _fields_ = [("k", _ptr), ("k_scale", _ptr), ("v", _ptr), ("v_scale", _ptr), ("pages", _int), ("heads", _int), ("page", _int), ("dim", _int), ("table", _ptr), ("slots", _int),
                ("table_pages", _int)]


class _Portions(C.Structure):
    _fields_ = [("n", _int), ("start", _ptr), ("count", _ptr), ("slot", _ptr), ("pos0", _ptr), ("longest", _int)]


class _Rows(C.Structure):
    _fields_ = [("p", _ptr), ("type", _int), ("row_stride", _ll), ("head_stride", _ll), ("rows", _int)]


class _Attend8(C.Structure):
    _fields_ = [("q", _Rows), ("out", _Rows), ("heads", _int), ("scale", C.c_float), ("window", _int), ("keep_first", _int), ("chunk", _int), ("softcap", C.c_float), ("sinks", _ptr),
                ("slopes", _ptr), ("gate", _ptr), ("gate_row", _ll), ("gate_head", _ll), ("gate_dim", _ll), ("most_keys", _int), ("workspace", _ptr), ("workspace_bytes", _size)]


class _Rotation(C.Structure):
    _fields_ = [("turns", _ptr), ("dims", _int), ("neighbours", _int), ("gain", C.c_float)]


class _Cache16(C.Structure):
    _fields_ = [("k", _ptr), ("v", _ptr), ("type", _int), ("pages", _int), ("heads", _int), ("page", _int), ("dim", _int), ("table", _ptr), ("slots", _int), ("table_pages", _int)]


class _Shared(C.Structure):
    _fields_ = [("n", _int), ("first", _ptr), ("count", _ptr), ("positions", _ptr), ("group", _ptr), ("n_alone", _int), ("alone", _ptr), ("longest", _int), ("tokens", _int), ("most_own", _int),
                ("most_alone", _int), ("lengths", _ptr)]


class _Groups(C.Structure):
    """struct SeqShared whole: `likely` lies where _Shared has padding, which is zero."""
    _fields_ = _Shared._fields_[:6] + [("likely", _int)] + _Shared._fields_[6:]


class _Attend16(C.Structure):
    _fields_ = [("q", _Rows), ("out", _Rows), ("heads", _int), ("scale", C.c_float), ("window", _int), ("softcap", C.c_float), ("sinks", _ptr), ("most_keys", _int), ("row_tiles", _ll),
                ("workspace", _ptr), ("workspace_bytes", _size), ("few", _int)]


_lib = None


def _load() -> C.CDLL:
    global _lib
    if _lib is None:
        L = seqlib.load()
        L.calm_b200_seq_error.argtypes, L.calm_b200_seq_error.restype = [], C.c_char_p
        L.calm_b200_seq_beam_workspace.argtypes, L.calm_b200_seq_beam_workspace.restype = [_int] * 4, _size
        L.calm_b200_seq_beam_select.argtypes, L.calm_b200_seq_beam_select.restype = [C.POINTER(_Beam), _ptr], _int
        L.calm_b200_seq_copy_units.argtypes = [_int, C.POINTER(_Units), _int, _ptr, _ptr, _ptr, _int, _ptr, _ptr, _ptr]
        L.calm_b200_seq_copy_units.restype = _int
        L.calm_b200_seq_cache8_store.argtypes = [C.POINTER(_Cache8), C.POINTER(_Portions), C.POINTER(_Rows), C.POINTER(_Rows), _ptr]
        L.calm_b200_seq_cache8_store.restype = _int
        L.calm_b200_seq_attend8_workspace.argtypes, L.calm_b200_seq_attend8_workspace.restype = [C.POINTER(_Cache8), C.POINTER(_Portions), C.POINTER(_Attend8)], _size
        L.calm_b200_seq_attend8.argtypes, L.calm_b200_seq_attend8.restype = [C.POINTER(_Cache8), C.POINTER(_Portions), C.POINTER(_Attend8), _ptr], _int
        L.calm_b200_seq_rotate.argtypes, L.calm_b200_seq_rotate.restype = [C.POINTER(_Portions), C.POINTER(_Rotation), C.POINTER(_Rows), C.POINTER(_Rows), _int, _int, _ptr], _int
        L.calm_b200_seq_cache16_store.argtypes = [C.POINTER(_Cache16), C.POINTER(_Portions), C.POINTER(_Rows), C.POINTER(_Rows), C.POINTER(_Rotation), C.POINTER(_Rows), C.POINTER(_Rows), _int, _ptr]
        L.calm_b200_seq_cache16_store.restype = _int
        args = [C.POINTER(_Cache16), C.POINTER(_Portions), _ptr, C.POINTER(_Attend16)]
        L.calm_b200_seq_attend16_workspace.argtypes, L.calm_b200_seq_attend16_workspace.restype = args, _size
        L.calm_b200_seq_attend16.argtypes, L.calm_b200_seq_attend16.restype = args + [_ptr], _int
        L.calm_b200_seq_attend16_way.argtypes, L.calm_b200_seq_attend16_way.restype = args, _int
        _lib = L
    return _lib


def _check(rc: int) -> None:
    if rc == 0:
        return
    text = _load().calm_b200_seq_error().decode()
    raise ValueError(text) if rc == -3 else seqlib.SeqError(text)


def _run(index: int, function, *args) -> None:
    """One call of the library on torch's current stream of device `index`, with that as the current device (most often it is already)."""
    if _device() == index:
        rc = function(*args, _stream(index))
        if rc:
            _check(rc)
    else:
        with torch.cuda.device(index):
            _check(function(*args, _stream(index)))


try:  # the handle and the number themselves; the objects and checks around them cost as much as a launch (a device is in use: the call's tensors are on it)
    from torch._C import _cuda_getCurrentRawStream as _stream, _cuda_getDevice as _device
except ImportError:
    _device = torch.cuda.current_device

    def _stream(index: int) -> int:
        return torch.cuda.current_stream(index).cuda_stream


def _gpu(name: str, t: torch.Tensor, index: int = -1) -> int:
    """The tensor's device, which is to be `index`."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    at = t.get_device()
    if index >= 0 and at != index:
        raise ValueError(f"{name} is on {t.device}, the call's other tensors on cuda:{index}")
    return at


def _whole(name: str, value) -> int:
    """A whole number that the library's 32 bits hold (ctypes would cut a larger one off)."""
    try:
        v = index_of(value)
    except TypeError:
        raise ValueError(f"{name} must be a whole number, not {value!r}") from None
    if not -2 ** 31 <= v < 2 ** 31:
        raise ValueError(f"{name} = {v} passes 32 bits")
    return v


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int, out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None):
    """The n best continuations of every group of beams: logits [groups, beams, vocab] (float32, bfloat16 or float16, the last axis contiguous), scores [groups,
    beams] float32 (-inf, or not finite: no beam there) -> tokens int32, parents int32, scores float32, each [groups, n], best first.  A candidate's score is its beam's plus the
    token's log-probability; where fewer than n candidates are above -inf the rest is token -1, parent -1, score -inf.  `out`: the three tensors to write."""
    index = _gpu("logits", logits)
    _gpu("scores", scores, index)
    kind = _TYPES.get(logits.dtype)
    if logits.dim() != 3 or kind is None or (logits.stride(2) != 1 and logits.shape[2] > 1):
        raise ValueError("logits must be [groups, beams, vocab] in float32, bfloat16 or float16 with the vocabulary contiguous")
    G, K, V = logits.shape
    if scores.shape != (G, K) or scores.dtype != torch.float32 or not scores.is_contiguous():
        raise ValueError(f"scores must be contiguous float32 [{G}, {K}]")
    L, n = _load(), _whole("n", n)
    for name, v in (("groups", G), ("beams", K), ("vocabulary", V)):
        _whole(name, v)
    need = L.calm_b200_seq_beam_workspace(G, K, V, n)
    if not need and (G or not 1 <= n <= 64):
        _check(-3)
    if out is None:
        tokens, parents, best = torch.empty((3, G, n), dtype=torch.int32, device=logits.device).unbind(0)
        best = best.view(torch.float32)
    else:
        tokens, parents, best = out
        for name, t, dt in (("tokens", tokens, torch.int32), ("parents", parents, torch.int32), ("scores", best, torch.float32)):
            _gpu(name, t, index)
            if t.shape != (G, n) or t.dtype != dt or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dt} [{G}, {n}]")
    work = torch.empty(max(16, need), dtype=torch.uint8, device=logits.device)
    a = _Beam(logits.data_ptr(), kind, logits.stride(0), logits.stride(1), scores.data_ptr(), G, K, V, n, tokens.data_ptr(), parents.data_ptr(), best.data_ptr(), work.data_ptr(), need)
    _run(index, L.calm_b200_seq_beam_select, C.byref(a))
    return tokens, parents, best


def _list(name: str, values) -> array:
    """Host integers as a C array (an int32 numpy array is taken as it lies)."""
    if isinstance(values, np.ndarray):
        if values.ndim != 1 or values.dtype.kind not in "iu":
            raise ValueError(f"{name} must be a list of whole numbers")
        if len(values) and not -2 ** 31 <= int(values.min()) <= int(values.max()) < 2 ** 31:
            raise ValueError(f"{name}: a number passes 32 bits")
        return array("i", np.ascontiguousarray(values, np.int32).tobytes())
    try:
        return array("i", values)
    except (TypeError, OverflowError) as e:
        raise ValueError(f"{name} must be a list of whole numbers of 32 bits: {e}") from None


class UnitPool:
    """Buffers made of units that are copied as a whole: `pages` are caches [units, rows, ...] (of which a copy may take the first rows only), `slots` are states
    [units, ...].  Buffers of one kind share the numbering of their units.  `into`: another UnitPool of the same shapes (in any number of units) that copies go to."""

    def __init__(self, pages: Sequence[torch.Tensor] = (), slots: Sequence[torch.Tensor] = (), into: Optional["UnitPool"] = None):
        self.buffers = [(t, 0) for t in pages] + [(t, 1) for t in slots]
        to = self.buffers if into is None else into.buffers
        if len(to) != len(self.buffers):
            raise ValueError("the pools hold different numbers of buffers")
        self.index = -1
        self.units = (_Units * max(1, len(self.buffers)))()
        for i, ((t, kind), (d, dkind)) in enumerate(zip(self.buffers, to)):
            for x in (t, d):
                self.index = _gpu("a pool's buffer", x, self.index)
                if x.dim() < (2 if kind == 0 else 1) or not x.is_contiguous():
                    raise ValueError("buffers must be contiguous, pages [units, rows, ...], slots [units, ...]")
            if kind != dkind or t.dtype != d.dtype or t.shape[1:] != d.shape[1:]:
                raise ValueError("the pools' buffers differ in kind, type or shape of a unit")
            unit = t.element_size() * (t[0].numel() if t.shape[0] else 0)
            self.units[i] = _Units(t.data_ptr(), d.data_ptr(), unit, unit // max(1, t.shape[1]) if kind == 0 else 0, t.shape[0], d.shape[0], kind)
        self.keep = to
        self.rows = min([t.shape[1] for t in pages], default=0)

    def copy(self, pages=((), ()), slots=((), ())) -> None:
        """pages = (from, to) or (from, to, rows): page to[i] of every page buffer becomes what page from[i] is, its first rows[i] rows only where rows is given; slots =
        (from, to) alike.  Numbers are host integers.  A unit may be written once and not be read by the same call (unless copies go to another pool)."""
        pf, pt = _list("pages", pages[0]), _list("pages", pages[1])
        pr = _list("rows", pages[2]) if len(pages) > 2 and pages[2] is not None else None
        sf, st = _list("slots", slots[0]), _list("slots", slots[1])
        if len(pf) != len(pt) or len(sf) != len(st) or (pr is not None and len(pr) != len(pf)):
            raise ValueError("lists of one kind must have one length")
        if pr and max(pr) > self.rows:
            raise ValueError(f"a page has {self.rows} rows")
        if self.index < 0:
            return

        def at(a: Optional[array]) -> Optional[int]:
            return a.buffer_info()[0] if a else None

        _run(self.index, _load().calm_b200_seq_copy_units, len(self.buffers), self.units, len(pf), at(pf), at(pt), at(pr), len(sf), at(sf), at(st))


class Batch:
    """The packed batch of a step: sequence i brings counts[i] new tokens, in order, at positions before[i] .. of slot slots[i].  The device arrays (`data`, int32 rows start,
    count, slot, position) may be written between replays of a captured call, as long as counts stay within `longest` and all rows within those of the call's tensors.

    shared: groups of neighbouring sequences that go on from one text, as (first sequence, sequences, positions): a cache holds the positions below that once, on the pages that the
    table names for the group's first sequence, and Cache16.attend reads them once for all of the group.  Of the device array `groups` (int32 rows first, sequences, positions) the positions may be written
    between replays too, up to the largest that was given; which sequences a group has stays."""

    def __init__(self, slots: Sequence[int], counts: Sequence[int], before: Sequence[int], device=None, shared: Sequence[Tuple[int, int, int]] = ()):
        sl, cn, at = (np.array(_list(name, x), np.int32) for name, x in (("slots", slots), ("counts", counts), ("before", before)))
        if not len(sl) == len(cn) == len(at):
            raise ValueError("slots, counts and before must have one length")
        if len(cn) and (cn.min() < 0 or at.min() < 0 or sl.min() < 0):
            raise ValueError("slots, counts and positions are not negative")
        if len(set(sl.tolist())) != len(sl):
            raise ValueError("a slot is named twice")
        start = np.concatenate([[0], np.cumsum(cn, dtype=np.int64)])
        if start[-1] >= 2 ** 31 or (len(cn) and int((at.astype(np.int64) + cn).max()) >= 2 ** 31):
            raise ValueError("token numbers pass 31 bits")
        groups, of = _grouped(shared, cn, at)
        self.tokens, self.longest = int(start[-1]), int(cn.max(initial=0))
        self.most_keys = int((at.astype(np.int64) + cn).max(initial=0))
        self.data = torch.from_numpy(np.stack([start[:-1].astype(np.int32), cn, sl, at])).to(torch.device("cuda") if device is None else device)
        self.index = _gpu("the batch", self.data)
        base, step = self.data.data_ptr(), self.data.stride(0) * 4
        self.c = _Portions(len(sl), base, base + step, base + 2 * step, base + 3 * step, self.longest)
        self.groups = self.group_of = self.shared = None
        self._counts, self._tiles = cn, {}
        if len(groups):
            own = at.astype(np.int64) + cn - np.where(of >= 0, groups[of, 2], 0)
            likely = max(1, max(int(cn[f:f + n].sum()) for f, n, _ in groups.tolist()))
            self._most_tokens = int(groups[:, 1].max()) * self.longest  # of a group, whatever counts up to `longest` are written
            alone, self._lengths = np.flatnonzero(of < 0).astype(np.int32), np.ascontiguousarray(groups[:, 2])
            both = torch.from_numpy(np.concatenate([groups.T.reshape(-1), of, alone])).to(self.data.device)
            self.groups, self.group_of = both[:groups.size].view(3, -1), both[groups.size:groups.size + len(of)]
            base, step = both.data_ptr(), 4 * len(groups)
            self.shared = _Groups(len(groups), base, base + step, base + 2 * step, base + 3 * step, len(alone), likely, base + 3 * step + 4 * len(of), int(groups[:, 2].max()),
                                  min(self._most_tokens, self.tokens), int(own[of >= 0].max()), int(own[of < 0].max(initial=0)), self._lengths.ctypes.data)

    def _shared_by(self, rows: int) -> Optional[_Groups]:
        """The groups' description for `rows` rows of queries: a group's counts may grow as far as `longest` and the rows allow."""
        if self.shared is None or min(self._most_tokens, rows) == self.shared.tokens:
            return self.shared
        more = _Groups.from_buffer_copy(self.shared)
        more.tokens = min(self._most_tokens, rows)
        return more

    def _row_tiles(self, group: int) -> int:
        """Tiles of 256 pairs of token and head, `group` heads a token, over all sequences."""
        return self._split(group)[0]

    def _split(self, group: int) -> Tuple[int, int]:
        """Those tiles, and the sequences with few such pairs."""
        found = self._tiles.get(group)
        if found is None:
            pairs = self._counts.astype(np.int64) * group
            found = self._tiles[group] = int((-(-pairs // 256)).sum()), int(((pairs > 0) & (pairs <= max(8, group))).sum())
        return found


def _grouped(shared, cn: np.ndarray, at: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
    """Groups (first sequence, sequences, positions), in order, and the group that each sequence is in (-1: none)."""
    try:
        groups = [_list("a group", g) for g in shared]
    except TypeError:
        groups = [()]
    if any(len(g) != 3 for g in groups):
        raise ValueError("shared must be a list of groups (first sequence, sequences, positions)")
    groups = np.array(sorted(list(g) for g in groups), np.int32).reshape(-1, 3)
    of, end = np.full(len(cn), -1, np.int32), 0
    for i, (first, n, positions) in enumerate(groups.tolist()):
        if first < end or n < 1 or first + n > len(cn) or positions < 0:
            raise ValueError(f"a group of {n} sequences from {first} on that share {positions} positions: groups lie apart among the {len(cn)} sequences")
        if positions > int(at[first:first + n].min()):
            raise ValueError(f"a group's sequences {first} .. {first + n - 1} do not all have {positions} positions before their new tokens")
        of[first:first + n], end = i, first + n
    return groups, of


def _rows(name: str, t: torch.Tensor, index: int, heads: int, dim: int, least: int) -> _Rows:
    _gpu(name, t, index)
    kind, shape, stride = _TYPES.get(t.dtype), t.shape, t.stride()
    if kind is None or len(shape) != 3 or shape[1] != heads or shape[2] != dim or (stride[2] != 1 and dim > 1):
        raise ValueError(f"{name} must be [tokens, {heads}, {dim}] in float32, bfloat16 or float16 with the channels contiguous, not {list(t.shape)} {t.dtype}")
    n = shape[0]
    if n < least:
        raise ValueError(f"{name} has {n} rows for {least} tokens")
    return _Rows(t.data_ptr(), kind, stride[0], stride[1], min(n, 2 ** 31 - 1))


class Cache8:
    """A paged cache of keys and values in 8 bits: codes [pages, heads, page, dim] (uint8 or float8_e4m3fn), scales [pages, heads] float32, powers of two; the value of a code is its
    e4m3 value times its page's and head's scale.  `Cache8.empty` allocates one."""

    def __init__(self, k: torch.Tensor, k_scale: torch.Tensor, v: torch.Tensor, v_scale: torch.Tensor):
        self.index = _gpu("codes", k)
        for name, t in (("codes", k), ("codes", v)):
            _gpu(name, t, self.index)
            if t.dim() != 4 or t.dtype not in (torch.uint8, torch.float8_e4m3fn) or not t.is_contiguous() or t.shape != k.shape:
                raise ValueError("codes must be contiguous [pages, heads, page, dim] in uint8 or float8_e4m3fn, keys' and values' of one shape")
        for t in (k_scale, v_scale):
            _gpu("scales", t, self.index)
            if t.shape != k.shape[:2] or t.dtype != torch.float32 or not t.is_contiguous():
                raise ValueError(f"scales must be contiguous float32 {list(k.shape[:2])}")
        self.k, self.k_scale, self.v, self.v_scale = k, k_scale, v, v_scale
        self.pages, self.heads, self.page, self.dim = k.shape
        self._pool = (k.data_ptr(), k_scale.data_ptr(), v.data_ptr(), v_scale.data_ptr(), self.pages, self.heads, self.page, self.dim)
        if self.dim % 16 or not 16 <= self.dim <= 256:
            raise ValueError(f"rows of {self.dim} channels: a multiple of 16 up to 256 is served")

    @staticmethod
    def empty(pages: int, heads: int, page: int, dim: int, device="cuda") -> "Cache8":
        shape = (pages, heads, page, dim)
        return Cache8(torch.zeros(shape, dtype=torch.uint8, device=device), torch.ones(shape[:2], device=device), torch.zeros(shape, dtype=torch.uint8, device=device),
                      torch.ones(shape[:2], device=device))

    def buffers(self) -> List[torch.Tensor]:
        """The four tensors as page buffers of a UnitPool: views [pages, 1, ...], since a page's first tokens are not its front (heads come first) and pages are copied whole."""
        return [t.unsqueeze(1) for t in (self.k, self.k_scale, self.v, self.v_scale)]

    def _with(self, table: torch.Tensor, batch: Batch) -> _Cache8:
        _gpu("the page table", table, self.index)
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous():
            raise ValueError("the page table must be contiguous int32 [slots, pages of a slot]")
        if batch.index != self.index:
            raise ValueError(f"the batch is on cuda:{batch.index}, the cache on cuda:{self.index}")
        slots, table_pages = table.shape
        return _Cache8(*self._pool, table.data_ptr(), slots, table_pages)

    def store(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, batch: Batch) -> None:
        """The batch's key and value rows [tokens, heads, dim] into the pages that `table` (int32 [slots, pages of a slot]) names for their positions.  Scales grow to what
        the rows need, earlier rows of a page are rounded to the raised scale."""
        c, n = self._with(table, batch), batch.tokens
        rk, rv = _rows("k", k, self.index, self.heads, self.dim, n), _rows("v", v, self.index, self.heads, self.dim, n)
        _run(self.index, _load().calm_b200_seq_cache8_store, C.byref(c), C.byref(batch.c), C.byref(rk), C.byref(rv))

    def attend(self, q: torch.Tensor, table: torch.Tensor, batch: Batch, scale: float, window: int = 0, keep_first: int = 0, chunk: int = 0, softcap: float = 0.0,
               sink: Optional[torch.Tensor] = None, slopes: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the batch's queries [tokens, query heads, dim] over the cache, which holds their own keys already (store comes first).  A token sees its sequence's positions up
        to its own: the last `window` of them and the first `keep_first`, or those from its block of `chunk` positions on.  sink: float32 [query heads], one more logit in the
        softmax's denominator; slopes: float32 [query heads], times the distance taken off the scores; gate: float32 [tokens, query heads, dim] (strides as they are, 0 too), its
        sigmoid multiplies the result.  Rows of q behind the batch's tokens stay as they are in `out` (zero without one)."""
        c, index = self._with(table, batch), self.index
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must be [tokens, query heads, dim]")
        heads = q.shape[1]
        rq = _rows("q", q, index, heads, self.dim, batch.tokens)
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if rq.rows == batch.tokens else torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        ro = _rows("out", out, index, heads, self.dim, rq.rows)
        a = _Attend8(rq, ro, heads, scale, _whole("window", window), _whole("keep_first", keep_first), _whole("chunk", chunk), softcap, None, None, None, 0, 0, 0, batch.most_keys, None, 0)
        for name, t in (("sink", sink), ("slopes", slopes)):
            if t is not None:
                _gpu(name, t, index)
                if t.shape != (heads,) or t.dtype != torch.float32 or not t.is_contiguous():
                    raise ValueError(f"{name} must be contiguous float32 [{heads}]")
                setattr(a, "sinks" if name == "sink" else "slopes", t.data_ptr())
        if gate is not None:
            _gpu("gate", gate, index)
            if gate.shape != q.shape or gate.dtype != torch.float32:
                raise ValueError(f"gate must be float32 {list(q.shape)}")
            a.gate, a.gate_row, a.gate_head, a.gate_dim = gate.data_ptr(), gate.stride(0), gate.stride(1), gate.stride(2)
        L = _load()
        need = L.calm_b200_seq_attend8_workspace(C.byref(c), C.byref(batch.c), C.byref(a))
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = work.data_ptr(), need
        _run(index, L.calm_b200_seq_attend8, C.byref(c), C.byref(batch.c), C.byref(a))
        return out


class Rotation:
    """How positions turn the channels of a head: the first `dims` of them, in pairs of "halves" (i, i + dims / 2) or "neighbours" (2i, 2i + 1), pair i by position * f_i with
    f_i = base^(-2 i / dims).  Angles are exact to 3 2^-53 of themselves and 2^-23 of a radian.  `scaling` stretches f for contexts longer than a model was trained on:
      {"kind": "linear", "factor"}                          f / factor
      {"kind": "base", "factor"}                            the base times factor^(dims / (dims - 2))
      {"kind": "wavelength", "factor", "length", "low", "high"}  w = length f / 2 pi: f / factor below `low`, f above `high`, a blend linear in w between
      {"kind": "ramp", "factor", "length", "fast", "slow"}  the same by the pair's number, between the pairs that turn `fast` and `slow` times in `length` positions; cosines and sines
                                                            times 0.1 ln(factor) + 1, 1 for factors below 1 (or "gain")
    frequencies: f itself, float64 [dims / 2], in place of base and scaling."""

    def __init__(self, dims: int, base: float = 10000.0, pairs: str = "halves", scaling: Optional[dict] = None, frequencies=None, device=None):
        dims = _whole("dims", dims)
        if dims < 2 or dims % 2:
            raise ValueError(f"a rotation of {dims} channels: an even number from 2 on")
        if pairs not in ("halves", "neighbours"):
            raise ValueError(f"pairs are \"halves\" or \"neighbours\", not {pairs!r}")
        if frequencies is None:
            self.frequencies, self.gain = rotation_frequencies(dims, base, scaling)
        elif scaling is not None:
            raise ValueError("frequencies that are given are not scaled")
        else:
            try:
                self.frequencies, self.gain = np.array(frequencies, np.float64), 1.0
            except (TypeError, ValueError, OverflowError):
                raise ValueError(f"frequencies must be {dims // 2} finite numbers") from None
            if self.frequencies.shape != (dims // 2,) or not np.isfinite(self.frequencies).all():
                raise ValueError(f"frequencies must be {dims // 2} finite numbers")
        if abs(self.gain) > float(np.finfo(np.float32).max):
            raise ValueError(f"gain = {self.gain} passes float32")
        self.dims, self.pairs = dims, pairs
        self.turns = torch.from_numpy(self.frequencies / (2.0 * math.pi)).to(torch.device("cuda") if device is None else device)
        self.index = _gpu("the rotation", self.turns)
        self.c = _Rotation(self.turns.data_ptr(), dims, int(pairs == "neighbours"), self.gain)


def _real(name: str, value) -> float:
    """A finite number as a float."""
    try:
        v = math.nan if isinstance(value, (str, bytes)) else float(value)
    except (TypeError, ValueError, OverflowError):
        v = math.nan
    if not math.isfinite(v):
        raise ValueError(f"{name} must be a finite number, not {value!r}")
    return v


def rotation_frequencies(dims: int, base: float = 10000.0, scaling: Optional[dict] = None) -> Tuple[np.ndarray, float]:
    """Step of every pair of a Rotation (float64 [dims / 2]) and the factor on cosines and sines."""
    wants = {"none": set(), "linear": {"factor"}, "base": {"factor"}, "wavelength": {"factor", "length", "low", "high"}, "ramp": {"factor", "length", "fast", "slow"}}
    if scaling is not None and not isinstance(scaling, dict):
        raise ValueError(f"scaling must be a dict, not {scaling!r}")
    s = dict(scaling) if scaling else {"kind": "none"}
    kind, gain, given = s.pop("kind", None), s.pop("gain", None), set(s)
    if not isinstance(kind, str) or kind not in wants or given != wants[kind]:
        raise ValueError(f"scaling {scaling!r}: one of " + ", ".join(f"{k} ({', '.join(sorted(w))})" for k, w in wants.items() if w))
    base, s = _real("base", base), {k: _real(k, v) for k, v in s.items()}
    gain = None if gain is None else _real("gain", gain)
    if not (base > 0 and all(v > 0 for v in s.values())):
        raise ValueError(f"base {base}, scaling {scaling!r}: positive numbers")
    try:
        with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
            f, gain = _stretched(dims, base, kind, s, gain)
    except (OverflowError, ZeroDivisionError):
        f = np.full(1, math.inf)
    if not np.isfinite(f).all():
        raise ValueError(f"base {base}, scaling {scaling!r}: frequencies that no number holds")
    return f, 1.0 if gain is None else gain


def _stretched(dims: int, base: float, kind: str, s: dict, gain: Optional[float]) -> Tuple[np.ndarray, Optional[float]]:
    if kind == "base":
        if dims < 4:
            raise ValueError("one pair of channels has no base to stretch")
        base *= s["factor"] ** (dims / (dims - 2))
    i = np.arange(dims // 2, dtype=np.float64)
    f = base ** (-2.0 * i / dims)
    if kind == "linear":
        f = f / s["factor"]
    elif kind == "wavelength":
        if not s["low"] < s["high"]:
            raise ValueError("low must be under high")
        w = s["length"] * f / (2.0 * math.pi)
        blend = np.clip((w - s["low"]) / (s["high"] - s["low"]), 0.0, 1.0)
        f = (1.0 - blend) * f / s["factor"] + blend * f
    elif kind == "ramp":
        if base == 1.0:
            raise ValueError("a base of 1 has no ramp")
        if s["fast"] < s["slow"]:
            raise ValueError("fast must not be under slow")
        at = [dims * math.log(s["length"] / (2.0 * math.pi * t)) / (2.0 * math.log(base)) for t in (s["fast"], s["slow"])]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dims - 1)
        blend = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        f = f / s["factor"] * blend + f * (1.0 - blend)
        gain = 0.1 * math.log(max(s["factor"], 1.0)) + 1.0 if gain is None else gain
    return f, gain


def _beside(rotation: Rotation, batch: Batch, index: int) -> None:
    if not isinstance(rotation, Rotation):
        raise ValueError("the rotation must be a seqops.Rotation")
    if rotation.index != index or batch.index != index:
        raise ValueError(f"the rotation is on cuda:{rotation.index}, the batch on cuda:{batch.index}, the call's other tensors on cuda:{index}")


def _like(x: torch.Tensor, rows: _Rows, tokens: int) -> Tuple[torch.Tensor, _Rows]:
    """Where rows like x's go, which are described: what is behind the batch's tokens is zero."""
    out = torch.empty_like(x) if rows.rows == tokens else torch.zeros_like(x)
    stride = out.stride()
    if stride[2] != 1:  # (like rows that overlap)
        out = out.contiguous()
        stride = out.stride()
    return out, _Rows(out.data_ptr(), rows.type, stride[0], stride[1], rows.rows)


def _into(name: str, t: torch.Tensor, index: int, heads: int, dim: int, least: int) -> _Rows:
    """Rows that are written: none lies on another."""
    r = _rows(name, t, index, heads, dim, least)
    steps = [s for s, n in ((r.row_stride, r.rows), (r.head_stride, heads)) if n > 1]
    if (steps and min(steps) < dim) or (len(steps) == 2 and steps[0] == steps[1]):
        raise ValueError(f"{name} has rows that overlap (strides {list(t.stride())})")
    return r


def rotate(x: torch.Tensor, batch: Batch, rotation: Rotation, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The batch's rows x [tokens, heads, dim] (float32, bfloat16 or float16; dim even) turned by their positions.  `out`: where they go, x itself or a tensor apart from it; rows behind the
    batch's tokens stay as they are in it (zero without one)."""
    index, shape = _gpu("x", x), x.shape
    if len(shape) != 3:
        raise ValueError("x must be [tokens, heads, dim]")
    _beside(rotation, batch, index)
    heads, dim = shape[1], shape[2]
    rx = _rows("x", x, index, heads, dim, batch.tokens)
    if out is None:
        out, ro = _like(x, rx, batch.tokens)
    else:
        ro = _into("out", out, index, heads, dim, rx.rows)
    _run(index, _load().calm_b200_seq_rotate, C.byref(batch.c), C.byref(rotation.c), C.byref(rx), C.byref(ro), heads, dim)
    return out


class Cache16:
    """A paged cache of keys and values in 16 bits: k and v [pages, heads, page, dim] in bfloat16 or float16.  `Cache16.empty` allocates one."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        self.index = _gpu("keys", k)
        _gpu("values", v, self.index)
        for t in (k, v):
            if t.dim() != 4 or t.dtype not in (torch.bfloat16, torch.float16) or not t.is_contiguous() or t.shape != k.shape or t.dtype != k.dtype:
                raise ValueError("keys and values must be contiguous [pages, heads, page, dim] in bfloat16 or float16, of one shape and type")
        self.k, self.v, self.dtype = k, v, k.dtype
        self.pages, self.heads, self.page, self.dim = k.shape
        self._pool = (k.data_ptr(), v.data_ptr(), _TYPES[k.dtype], self.pages, self.heads, self.page, self.dim)
        if not self.heads or not self.page:
            raise ValueError(f"a cache of {self.heads} heads, {self.page} tokens a page")
        if self.dim % 16 or not 16 <= self.dim <= 256:
            raise ValueError(f"rows of {self.dim} channels: a multiple of 16 up to 256 is served")

    @staticmethod
    def empty(pages: int, heads: int, page: int, dim: int, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "Cache16":
        return Cache16(*(torch.zeros((pages, heads, page, dim), dtype=dtype, device=device) for _ in range(2)))

    def buffers(self) -> List[torch.Tensor]:
        """Both tensors as page buffers of a UnitPool: views [pages, 1, ...], since a page's first tokens are not its front (heads come first) and pages are copied whole."""
        return [t.unsqueeze(1) for t in (self.k, self.v)]

    def _with(self, table: torch.Tensor, batch: Batch) -> _Cache16:
        _gpu("the page table", table, self.index)
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous():
            raise ValueError("the page table must be contiguous int32 [slots, pages of a slot]")
        if batch.index != self.index:
            raise ValueError(f"the batch is on cuda:{batch.index}, the cache on cuda:{self.index}")
        slots, table_pages = table.shape
        return _Cache16(*self._pool, table.data_ptr(), slots, table_pages)

    def store(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, batch: Batch, rotation: Optional[Rotation] = None, q: Optional[torch.Tensor] = None,
              q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """The batch's key and value rows [tokens, heads, dim] into the pages that `table` (int32 [slots, pages of a slot]) names for their positions, the keys turned by their
        positions where a rotation is given.  q: the step's queries [tokens, query heads, dim], turned in the same launch into q_out (q itself or a tensor apart from it; a new one without), which is returned."""
        c, n, index = self._with(table, batch), batch.tokens, self.index
        rk, rv = _rows("k", k, index, self.heads, self.dim, n), _rows("v", v, index, self.heads, self.dim, n)
        turn, rq, ro, heads = None, None, None, 0
        if rotation is not None:
            _beside(rotation, batch, index)
            turn = C.byref(rotation.c)
        if q is not None:
            if not isinstance(q, torch.Tensor) or q.dim() != 3:
                raise ValueError("q must be [tokens, query heads, dim]")
            heads = q.shape[1]
            rq = _rows("q", q, index, heads, self.dim, n)
            if q_out is None:
                q_out, ro = _like(q, rq, n)
            else:
                ro = _into("q_out", q_out, index, heads, self.dim, rq.rows)
        elif q_out is not None:
            raise ValueError("q_out without q")
        _run(index, _load().calm_b200_seq_cache16_store, C.byref(c), C.byref(batch.c), C.byref(rk), C.byref(rv), turn, rq if rq is None else C.byref(rq), ro if ro is None else C.byref(ro), heads)
        return q_out

    def attend(self, q: torch.Tensor, table: torch.Tensor, batch: Batch, scale: float, window: int = 0, softcap: float = 0.0, sink: Optional[torch.Tensor] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of the batch's queries [tokens, query heads, dim] (of the cache's type) over the cache, which holds their own keys already (store comes first).  A token sees its
        sequence's positions up to its own, the last `window` of them where that is not 0; positions that the batch's groups share are read once for the group.  sink: float32 [query heads], one more logit in the
        softmax's denominator.  Rows of q behind the batch's tokens stay as they are in `out` (zero without one)."""
        c, index = self._with(table, batch), self.index
        if not isinstance(q, torch.Tensor) or q.dim() != 3:
            raise ValueError("q must be [tokens, query heads, dim]")
        heads = q.shape[1]
        rq = _rows("q", q, index, heads, self.dim, batch.tokens)
        if out is None:
            out, ro = _like(q, rq, batch.tokens)
        else:
            ro = _into("out", out, index, heads, self.dim, rq.rows)
        scale, softcap = _real("scale", scale), _real("softcap", softcap)
        a = _Attend16(rq, ro, heads, scale, _whole("window", window), softcap, None, batch.most_keys, 0, None, 0)
        if softcap and not a.softcap:
            raise ValueError(f"softcap = {softcap} is out of float32's range")
        a.row_tiles, a.few = batch._split(heads // self.heads)
        if sink is not None:
            _gpu("sink", sink, index)
            if sink.shape != (heads,) or sink.dtype != torch.float32 or not sink.is_contiguous():
                raise ValueError(f"sink must be contiguous float32 [{heads}]")
            a.sinks = sink.data_ptr()
        L, shared = _load(), batch._shared_by(rq.rows)
        if shared is not None:
            shared = C.byref(shared)
        need = L.calm_b200_seq_attend16_workspace(C.byref(c), C.byref(batch.c), shared, C.byref(a))
        if need:
            work = torch.empty(need, dtype=torch.uint8, device=q.device)
            a.workspace, a.workspace_bytes = work.data_ptr(), need
        _run(index, L.calm_b200_seq_attend16, C.byref(c), C.byref(batch.c), shared, C.byref(a))
        return out
