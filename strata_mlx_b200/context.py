"""What a decoder keeps of its context, for a batch of sequences: a paged key/value cache that can be held to a budget,
and linear attention, whose state has one size at any length. Additions for a serving decoder around the MoE blocks (the
reference keeps one conversation, and its trunk's recurrent layers follow a delta rule, which this is not):

    KVPages                 a batch's cache: pools of pages, a table and a length a sequence
      .attend(q)            attention of one new token a sequence; the weights each slot gathers, on request
      .evict(seen, keep)    keeps the tokens with the most weight and moves them to the front of the cache, in place
    decode_attention        KVPages(...).attend(q) for a single call
    linear_attention        S_t = exp(g_t) S_{t-1} + k_t v_t^T, out_t = scale q_t S_t over a prompt
    linear_attention_step   the same for one token a sequence, the state in place

Every call enqueues on the current CUDA stream and returns; nothing is read back. Activations are bfloat16 or
float16; softmax statistics, accumulated weights and states are float32.
"""

from __future__ import annotations

import ctypes
import struct
import threading

import torch

from . import _lib
from ._lib import check, ptr, require_cuda

_stream = torch._C._cuda_getCurrentRawStream  # a call's stream without building a Stream object
_capturing = torch.cuda.is_current_stream_capturing
_TYPES = {torch.float16: 1, torch.bfloat16: 2}  # SC_F16, SC_BF16


def _here(*ts) -> torch.device:
    """The device all the tensors are on, which has to be the current one: calls go to its current stream."""
    require_cuda(*ts)
    device = ts[0].device
    for t in ts:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}")
    if device.index != torch.cuda.current_device():
        raise ValueError(f"tensors on {device}, but the current device is cuda:{torch.cuda.current_device()}")
    return device


def _ints(name: str, t: torch.Tensor, shape: tuple) -> None:
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 {shape} expected, got {t.dtype} {tuple(t.shape)}")


class KVPages:
    """A batch's paged key/value cache (one layer's). k, v (pages, page, kv_heads, head_dim) bfloat16 or float16, of
    any strides with the last axis adjacent; table (batch, max_pages) int32, sequence b's slot s in page
    table[b, s // page] (rows may be views, and the same row may serve several sequences that only read); lengths
    (batch,) int32, the slots in use. weight (batch, >= max_pages * page) float32 gathers each slot's attention
    weight; position, the same shape int32, holds the position of each slot's token (evict needs both). The tensors
    stay the caller's: the object keeps references and reads lengths and table on the device at every call, so that
    steps replay from a CUDA graph. Calls on one stream may follow each other freely, from several threads too (a
    lock keeps a call's launches together); each stream has a workspace of its own."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                 weight: torch.Tensor | None = None, position: torch.Tensor | None = None):
        self.device = _here(k, v, table, lengths, weight, position)
        if k.dtype not in _TYPES or v.dtype != k.dtype:
            raise ValueError(f"k and v both bfloat16 or both float16 expected, got {k.dtype} and {v.dtype}")
        if k.dim() != 4 or k.shape != v.shape or k.stride(-1) != 1 or v.stride(-1) != 1:
            raise ValueError(f"k and v (pages, page, kv_heads, head_dim) with the last axis adjacent expected, got "
                             f"{tuple(k.shape)} and {tuple(v.shape)}")
        if table.dim() != 2 or table.dtype != torch.int32 or table.stride(1) != 1:
            raise ValueError("table: int32 (batch, max_pages) with adjacent rows expected")
        self.batch, self.max_pages = table.shape
        _ints("lengths", lengths, (self.batch,))
        self.slots = self.max_pages * k.shape[1]
        for name, t, dtype in (("weight", weight, torch.float32), ("position", position, torch.int32)):
            if t is not None and (t.dtype != dtype or t.dim() != 2 or t.shape[0] != self.batch or t.stride(1) != 1
                                  or t.shape[1] < self.slots):
                raise ValueError(f"{name}: {dtype} ({self.batch}, at least {self.slots}) expected")
            if t is not None and self.batch > 1 and t.stride(0) < self.slots:
                raise ValueError(f"{name}: the sequences' rows overlap")
        self.k, self.v, self.table, self.lengths, self.weight, self.position = k, v, table, lengths, weight, position
        self.dtype, self.kv_heads, self.head_dim = k.dtype, k.shape[2], k.shape[3]
        P = _lib.SCPages()
        P.k, P.v, P.table, P.lengths = ptr(k), ptr(v), ptr(table), ptr(lengths)
        P.k_page, P.k_token, P.k_head = k.stride()[:3]
        P.v_page, P.v_token, P.v_head = v.stride()[:3]
        P.table_row = table.stride(0)
        P.weight, P.position = ptr(weight), ptr(position)
        P.weight_row = 0 if weight is None else weight.stride(0)
        P.position_row = 0 if position is None else position.stride(0)
        P.batch, P.kv_heads, P.head_dim, P.page = self.batch, self.kv_heads, self.head_dim, k.shape[1]
        P.pool_pages, P.max_pages, P.dtype = k.shape[0], self.max_pages, _TYPES[k.dtype]
        self._pages, self._ref = P, ctypes.addressof(P)
        self._lib, self._err = _lib.lib(), ptr(_lib.error_word(self.device))
        self._lock = threading.Lock()  # held over a call's launches: they share a workspace
        self._ws: dict = {}
        self._sizes: dict = {}  # of attend's workspace, by the query heads
        self._evict_sizes: dict = {}  # of evict's, by the budget
        self._index, self._scale = self.device.index, self.head_dim ** -0.5

    def _workspace(self, what: str, size: int, s: int) -> tuple:
        """The workspace of a kind of call on stream s: its address and bytes (fresh in a capture, whose memory is
        the graph's). It may hold anything: the kernels read what they wrote in the same call."""
        if size == 0:
            raise ValueError(f"{what}: this cache or these arguments are not taken (at most 65535 sequences, head_dim a "
                             "multiple of 8 up to 256, a power-of-two page up to 4096, 2^30 slots, 16-byte rows, at most "
                             "2048 query heads, a multiple of the cache's)")
        ws = self._ws.get((what, s))
        if ws is None or ws[1] < size or _capturing():
            t = torch.empty(size, dtype=torch.uint8, device=self.device)
            ws = (t.data_ptr(), size, t)
            if not _capturing():
                self._ws[what, s] = ws
        return ws

    def attend(self, q: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """softmax(scale q k^T) v of one new token a sequence: q (batch, q_heads, head_dim), out the same. The token's
        own key and value are in the cache already. scale defaults to head_dim ** -0.5. A sequence of length 0 gives
        zeros. With `weight`, every slot's probability, summed over the query heads, is added to it."""
        shape = q.shape
        if len(shape) != 3 or shape[0] != self.batch or shape[2] != self.head_dim or q.dtype != self.dtype:
            raise ValueError(f"q ({self.batch}, q_heads, {self.head_dim}) {self.dtype} expected, got {tuple(shape)} "
                             f"{q.dtype}")
        if q.device != self.device or torch.cuda.current_device() != self._index:
            raise ValueError(f"q on {q.device}; the cache is on {self.device}, which has to be current")
        st = q.stride()
        if st[2] != 1:
            q = q.contiguous()
            st = q.stride()
        if out is None:
            out = q.new_empty(shape)
        elif out.shape != shape or out.dtype != q.dtype or out.device != self.device or not out.is_contiguous():
            raise ValueError(f"out: contiguous {tuple(shape)} {q.dtype} expected")
        s, heads = _stream(self._index), shape[1]
        size = self._sizes.get(heads)
        if size is None:
            size = self._sizes[heads] = self._lib.sc_decode_attention_workspace(self._ref, heads)
        with self._lock:
            ws = self._workspace("attend", size, s)
            rc = self._lib.sc_decode_attention(self._ref, q.data_ptr(), st[0], st[1], heads,
                                               self._scale if scale is None else scale, out.data_ptr(), ws[0], ws[1],
                                               self._err, s)
        if rc:
            check(rc, "decode_attention")
        return out

    def evict(self, seen: torch.Tensor, keep: int, sinks: int = 4, recent: int = 0, out: tuple | None = None) -> None:
        """Keeps `keep` tokens of every longer sequence: those at positions below `sinks` or within the last `recent`
        of the seen[b] positions the sequence has had, then those with the most weight (equal ones: the lower slot).
        The kept tokens beyond the budget move into the slots of evicted ones, keys, values, weight and position;
        lengths becomes min(length, keep). out: (weight, position, lengths) tensors that get the first min(keep,
        length) slots' values and the lengths in place of the cache's own (layers that share one `lengths` each need
        theirs until all are done). Slots past the new length keep what they held."""
        if self.weight is None or self.position is None:
            raise ValueError("evict needs the cache's weight and position")
        if not 0 <= keep < 1 << 31 or sinks < 0 or recent < 0 or sinks + recent > keep:
            raise ValueError(f"sinks {sinks} and recent {recent} have to fit in keep {keep}, and keep in 31 bits")
        weight, position, lengths = (self.weight, self.position, self.lengths) if out is None else out
        index, n, room = self._index, self.batch, min(keep, self.slots)
        if seen.get_device() != index or torch.cuda.current_device() != index:
            raise ValueError(f"seen on {seen.device}; the cache is on {self.device}, which has to be current")
        _ints("seen", seen, (n,))
        if out is not None:
            for name, t, dtype in (("weight", weight, torch.float32), ("position", position, torch.int32)):
                shape = t.shape
                if (t.get_device() != index or t.dtype != dtype or len(shape) != 2 or shape[0] != n or shape[1] < room
                        or t.stride(1) != 1):
                    raise ValueError(f"out {name}: {dtype} ({n}, at least {room}) on {self.device} expected")
                if n > 1 and t.stride(0) < room:
                    raise ValueError(f"out {name}: the sequences' rows overlap")
            if lengths.get_device() != index:
                raise ValueError(f"out lengths: on {self.device} expected")
            _ints("out lengths", lengths, (n,))
        s = _stream(index)
        size = self._evict_sizes.get(keep)
        if size is None:
            size = self._evict_sizes[keep] = self._lib.sc_evict_workspace(self._ref, keep)
        with self._lock:
            ws = self._workspace("evict", size, s)
            rc = self._lib.sc_evict(self._ref, seen.data_ptr(), keep, sinks, recent, weight.data_ptr(),
                                    weight.stride(0), position.data_ptr(), position.stride(0), lengths.data_ptr(),
                                    ws[0], ws[1], self._err, s)
        if rc:
            check(rc, "evict")


def decode_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                     scale: float | None = None, weight: torch.Tensor | None = None,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """KVPages(k, v, table, lengths, weight).attend(q, scale, out): attention of one new token a sequence."""
    return KVPages(k, v, table, lengths, weight).attend(q, scale, out)


_LINEAR = struct.Struct("@8Q12q7if")  # sc_linear (include/strata_cuda.h), field by field


def _refuse_linear(q, k, v, decay, state, nd: int) -> None:
    """Names what is wrong with a linear attention call's tensors."""
    _here(q, k, v, decay, state)
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v all bfloat16 or all float16 expected, got {q.dtype}, {k.dtype}, {v.dtype}")
    axes = "(batch, tokens, heads, dim)" if nd == 4 else "(batch, heads, dim)"
    if q.dim() != nd or v.dim() != nd or k.shape != q.shape or v.shape[:-2] != q.shape[:-2]:
        raise ValueError(f"q, k and v {axes}, q and k alike, v of the same tokens expected, got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if q.shape[-2] == 0 or v.shape[-2] % q.shape[-2]:
        raise ValueError(f"{v.shape[-2]} value heads are not a multiple of {q.shape[-2]} key heads")
    if decay.dtype != torch.float32 or decay.shape != v.shape[:-1]:
        raise ValueError(f"decay: float32 {tuple(v.shape[:-1])} expected, got {decay.dtype} {tuple(decay.shape)}")
    raise ValueError(f"state: contiguous float32 {(v.shape[0], v.shape[-2], q.shape[-1], v.shape[-1])} expected")


def _linear(q, k, v, decay, state, nd: int) -> tuple:
    """Checks a call's tensors in one pass; returns them with their values adjacent, and sc_linear's integers."""
    qs, vs, dtype, index = q.shape, v.shape, q.dtype, q.get_device()
    code = _TYPES.get(dtype)
    if (index < 0 or k.get_device() != index or v.get_device() != index or decay.get_device() != index
            or torch.cuda.current_device() != index or code is None or k.dtype != dtype or v.dtype != dtype
            or len(qs) != nd or len(vs) != nd or k.shape != qs or vs[:-2] != qs[:-2] or qs[-2] == 0
            or vs[-2] % qs[-2] or decay.dtype != torch.float32 or decay.shape != vs[:-1]
            or (state is not None and (state.get_device() != index or state.dtype != torch.float32
                                       or state.shape != (vs[0], vs[-2], qs[-1], vs[-1])
                                       or not state.is_contiguous()))):
        _refuse_linear(q, k, v, decay, state, nd)
    a, b, c, d = q.stride(), k.stride(), v.stride(), decay.stride()
    if a[-1] != 1 or b[-1] != 1 or c[-1] != 1:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        a, b, c = q.stride(), k.stride(), v.stride()
    if nd == 3:
        return q, k, v, (a[0], 0, a[1], b[0], 0, b[1], c[0], 0, c[1], d[0], 0, d[1], qs[0], 1, qs[1], vs[1], qs[2],
                         vs[2], code), index
    return q, k, v, (*a[:3], *b[:3], *c[:3], *d, qs[0], qs[1], qs[2], vs[2], qs[3], vs[3], code), index


def linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor,
                     state: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                     scale: float | None = None) -> tuple:
    """A prompt (or a chunk of one) through linear attention: S_t = exp(decay_t) S_{t-1} + k_t v_t^T, out_t = scale
    q_t S_t. q, k (batch, tokens, k_heads, k_dim), v (batch, tokens, v_heads, v_dim): value head h reads key head
    h // (v_heads / k_heads); k_dim and v_dim multiples of 8 up to 128. decay (batch, tokens, v_heads) float32
    logarithms of either sign, of any strides (a fixed decay a head is an expanded view). state (batch, v_heads, k_dim, v_dim)
    float32, zeros when None, is left as it was. lengths (batch,) int32: tokens past a sequence's length are not read,
    their outputs zeros. scale defaults to k_dim ** -0.5. Returns (out of v's shape, the state after the last token)."""
    q, k, v, sizes, index = _linear(q, k, v, decay, state, 4)
    if lengths is not None:
        _here(q, lengths)
        _ints("lengths", lengths, (sizes[12],))
    out = v.new_empty(v.shape)
    new = decay.new_empty((sizes[12], sizes[15], sizes[16], sizes[17]))
    lib = _lib.lib()
    call = _LINEAR.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(),
                        0 if state is None else state.data_ptr(), new.data_ptr(),
                        0 if lengths is None else lengths.data_ptr(), out.data_ptr(), *sizes,
                        sizes[16] ** -0.5 if scale is None else scale)
    size = lib.sc_linear_attention_workspace(call)
    ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    rc = lib.sc_linear_attention(call, 0 if ws is None else ws.data_ptr(), size, ptr(_lib.error_word(q.device)),
                                 _stream(index))
    if rc:
        check(rc, "linear_attention")
    return out, new


def linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, decay: torch.Tensor, state: torch.Tensor,
                          scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """linear_attention for one token a sequence: q, k (batch, k_heads, k_dim), v (batch, v_heads, v_dim), decay (batch,
    v_heads); state (batch, v_heads, k_dim, v_dim) float32 is updated in place. Returns out (batch, v_heads, v_dim)."""
    if state is None:
        raise ValueError("a step needs the state it updates")
    q, k, v, sizes, index = _linear(q, k, v, decay, state, 3)
    if out is None:
        out = v.new_empty(v.shape)
    elif out.shape != v.shape or out.dtype != v.dtype or out.device != v.device or not out.is_contiguous():
        raise ValueError(f"out: contiguous {tuple(v.shape)} {v.dtype} expected")
    S = state.data_ptr()
    rc = _lib.lib().sc_linear_attention_step(
        _LINEAR.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), decay.data_ptr(), S, S, 0, out.data_ptr(), *sizes,
                     sizes[16] ** -0.5 if scale is None else scale), _stream(index))
    if rc:
        check(rc, "linear_attention_step")
    return out
