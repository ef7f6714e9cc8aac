"""The operators of a decode step: a paged key-value cache and 4-bit layers with group scales.

`PagedKV` describes a cache whose memory the caller owns (page pools, page table, lengths) and
runs three operators over it: `append` (new tokens, rotated and cast, into the pages), `attend`
(attention of one new token per sequence) and `evict` (cut back to a budget by accumulated
attention weight). `GroupDense` is a Dense layer of 4-bit codes with one scale per group of
inputs, for one to eight rows at a time. `mha_decode` and `mha_prefill` run an MHA cell over such a
cache. All calls are asynchronous on the current stream (or `stream`) and can be captured in a CUDA
graph. The calls of a cache and of a layer allocate nothing; a cell's allocate its work buffers
at the first step for a number of sequences and at a prompt longer than any before, so a step runs
once before it is captured. Buffers of steps, and those that were captured, stay until the cell is
released: a longer prompt may follow, and the graph replays on.
"""
from __future__ import annotations

import ctypes
from ctypes import POINTER, byref, c_double, c_float, c_int32, c_int64, c_size_t, c_void_p

import numpy as np
import torch

from . import (_L, _ST, _np_ptr, _sig, FP4, GELU, LEAKY_RELU, LINEAR, OK, RELU, RELU2, SIGMOID, SILU, TANH, WelvetError,
               check)

FLOAT16, BFLOAT16, INT4, UINT4 = 2, 3, 14, 15
CODES = {"int4": INT4, "uint4": UINT4, "fp4": FP4}
ACTS = {"linear": LINEAR, "relu": RELU, "silu": SILU, "gelu": GELU, "tanh": TANH, "sigmoid": SIGMOID,
        "leaky_relu": LEAKY_RELU, "relu2": RELU2}
_PAGES = {torch.float32: 1, torch.float16: FLOAT16, torch.bfloat16: BFLOAT16, torch.float8_e4m3fn: 4}
_SCALES = {torch.float16: FLOAT16, torch.bfloat16: BFLOAT16}


class _KvDesc(ctypes.Structure):
    _fields_ = [("dtype", c_int32), ("num_heads", c_int32), ("num_kv_heads", c_int32), ("head_dim", c_int32),
                ("page_size", c_int32), ("num_pages", c_int32), ("num_seqs", c_int32), ("pages_per_seq", c_int32),
                ("k_pages", c_void_p), ("v_pages", c_void_p), ("k_strides", c_int64 * 3), ("v_strides", c_int64 * 3),
                ("k_scale", c_float), ("v_scale", c_float), ("page_table", c_void_p), ("table_stride", c_int64),
                ("lens", c_void_p), ("seen", c_void_p), ("weights", c_void_p), ("positions", c_void_p)]


_sig("welvet_b200_kv_create", _ST, POINTER(_KvDesc), POINTER(c_void_p))
_sig("welvet_b200_kv_append", _ST, c_void_p, c_int32, c_void_p, c_int64, c_void_p, c_int64, c_void_p, c_int64, c_void_p,
     c_int64, c_void_p, c_double, c_void_p, c_void_p, c_void_p)
_sig("welvet_b200_kv_attend", _ST, c_void_p, c_void_p, c_int64, c_void_p, c_int64, c_float, c_int32, c_int32, c_int32,
     c_void_p, c_void_p)
_sig("welvet_b200_kv_evict", _ST, c_void_p, c_int32, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p)
_sig("welvet_b200_kv_check_error", _ST, c_void_p, c_void_p)
_sig("welvet_b200_kv_release", None, c_void_p)
_sig("welvet_b200_group_quantize", _ST, c_int32, c_int32, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p,
     c_void_p)
_sig("welvet_b200_gdense_mount", _ST, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_void_p, c_void_p, c_void_p,
     c_int32, c_void_p, c_size_t, POINTER(c_void_p))
_sig("welvet_b200_gdense_execute_device", _ST, c_void_p, c_int32, c_void_p, c_int64, c_void_p, c_void_p, c_void_p)
_sig("welvet_b200_gdense_plan", c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, c_int32, POINTER(c_int64), c_int32)
_sig("welvet_b200_gdense_release", None, c_void_p)

_sig("welvet_b200_mha_decode_device", _ST, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p)
_sig("welvet_b200_mha_decode_active_device", _ST, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int32, c_void_p, c_void_p)
_sig("welvet_b200_mha_prefill_device", _ST, c_void_p, c_void_p, c_int32, c_int32, c_void_p, c_void_p, c_void_p, c_void_p)

_append, _attend, _evict, _gemv = (_L.welvet_b200_kv_append, _L.welvet_b200_kv_attend, _L.welvet_b200_kv_evict,
                                   _L.welvet_b200_gdense_execute_device)
_F32, _I32 = torch.float32, torch.int32


# The current stream's handle without the Stream object around it (3 us a call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)


def _stream(stream, t=None) -> int:
    if stream is None:
        return _raw_stream(torch.cuda.current_device() if t is None else t.get_device())
    return getattr(stream, "cuda_stream", stream)


def _fail(st) -> None:
    raise WelvetError(st.code, st.message.decode(errors="replace"))


def _rows(t, width: int, what: str, rows: int | None = None):
    """(rows, pointer, row stride) of a float32 CUDA tensor [rows, width] or [rows, heads, dim] whose
    rows are contiguous (they may be parts of wider ones)."""
    shape, stride = t.shape, t.stride()
    n = shape[0]
    if (t.dtype is not _F32 or not t.is_cuda or len(shape) not in (2, 3) or stride[-1] != 1
            or (len(shape) == 3 and stride[1] != shape[2] and shape[1] > 1)):
        raise ValueError(f"{what}: expected a float32 CUDA tensor of contiguous rows")
    if (shape[1] if len(shape) == 2 else shape[1] * shape[2]) != width or (rows is not None and n != rows):
        raise ValueError(f"{what}: expected {'rows' if rows is None else rows} x {width} values, got {tuple(shape)}")
    return n, t.data_ptr(), stride[0]


def _ints(t, n: int, what: str) -> int | None:
    """Pointer of an int32 CUDA tensor of n values (None passes through)."""
    if t is None:
        return None
    if t.dtype is not _I32 or not t.is_cuda or not t.is_contiguous() or t.numel() != n:
        raise ValueError(f"{what}: expected {n} contiguous int32 values on the GPU")
    return t.data_ptr()


class PagedKV:
    """A paged key-value cache over the caller's tensors (welvet_b200_kv_*).

    k_pages, v_pages: [pages, page slots, key-value heads, head dim] of float32, float16, bfloat16 or
    float8_e4m3fn, any strides with contiguous rows of head dim (a transposed view of
    [pages, heads, slots, dim] too). page_table [sequences, pages of a sequence] int32 and lens
    [sequences] int32. `seen` (tokens seen), `weights` (accumulated attention weight, float32) and
    `positions` (int32; both [sequences, key-value heads, slots of a sequence]) are what `evict`
    needs; `weights` alone is what `attend(accumulate=True)` needs. A stored unit stands for
    k_scale / v_scale. The tensors are kept alive; calls on one cache must not overlap.
    """

    def __init__(self, k_pages, v_pages, page_table, lens, *, num_heads: int, seen=None, weights=None, positions=None,
                 k_scale: float = 1.0, v_scale: float = 1.0):
        self._h = c_void_p()
        if k_pages.dtype not in _PAGES or v_pages.dtype != k_pages.dtype:
            raise ValueError("PagedKV: pages of float32, float16, bfloat16 or float8_e4m3fn, one type for both pools")
        if k_pages.ndim != 4 or k_pages.shape != v_pages.shape:
            raise ValueError("PagedKV: k_pages and v_pages of one shape [pages, slots, heads, dim]")
        for t, what in ((k_pages, "k_pages"), (v_pages, "v_pages")):
            if not t.is_cuda or t.stride(3) != 1:
                raise ValueError(f"PagedKV: {what} must be a CUDA tensor with contiguous rows of head dim")
        if page_table.ndim != 2 or page_table.dtype is not _I32 or not page_table.is_cuda or page_table.stride(1) != 1:
            raise ValueError("PagedKV: page_table must be a CUDA int32 tensor [sequences, pages]")
        pages, slots, kv, dim = k_pages.shape
        n, per = page_table.shape
        self.num_seqs, self.num_heads, self.num_kv_heads, self.head_dim, self.max_slots = n, num_heads, kv, dim, per * slots
        self._records = (n, kv, self.max_slots)
        d = _KvDesc(dtype=_PAGES[k_pages.dtype], num_heads=num_heads, num_kv_heads=kv, head_dim=dim, page_size=slots,
                    num_pages=pages, num_seqs=n, pages_per_seq=per, k_pages=k_pages.data_ptr(), v_pages=v_pages.data_ptr(),
                    k_strides=(c_int64 * 3)(*k_pages.stride()[:3]), v_strides=(c_int64 * 3)(*v_pages.stride()[:3]),
                    k_scale=k_scale, v_scale=v_scale, page_table=page_table.data_ptr(), table_stride=page_table.stride(0),
                    lens=_ints(lens, n, "lens"), seen=_ints(seen, n, "seen"), weights=self._weights(weights, "weights"),
                    positions=self._positions(positions, "positions"))
        check(_L.welvet_b200_kv_create(byref(d), byref(self._h)))
        self._qw, self._kw = num_heads * dim, kv * dim
        self.k_pages, self.v_pages, self.page_table, self.lens = k_pages, v_pages, page_table, lens
        self.seen, self.weights, self.positions = seen, weights, positions

    def _weights(self, t, what):
        if t is None:
            return None
        if t.dtype is not _F32 or not t.is_cuda or not t.is_contiguous() or t.shape != self._records:
            raise ValueError(f"{what}: expected a contiguous float32 CUDA tensor {self._records}")
        return t.data_ptr()

    def _positions(self, t, what):
        if t is None:
            return None
        if t.shape != self._records:
            raise ValueError(f"{what}: expected a tensor {self._records}")
        return _ints(t, t.numel(), what)

    def append(self, k, v, *, q=None, q_out=None, cu_tokens=None, theta: float = 0.0, start=None, start_seen=None,
               stream=None) -> None:
        """Rows of k and v [rows, key-value heads, dim] into the cache; q [rows, heads, dim] rotated into
        q_out. cu_tokens [sequences + 1]: the first row of each sequence (None: one row each)."""
        rows, kp, k_ld = _rows(k, self._kw, "k")
        _, vp, v_ld = _rows(v, self._kw, "v", rows)
        qp = op = None
        q_ld = o_ld = 0
        if q is not None:
            if q_out is None:
                raise ValueError("append: q needs q_out (which may be q)")
            _, qp, q_ld = _rows(q, self._qw, "q", rows)
            _, op, o_ld = _rows(q_out, self._qw, "q_out", rows)
        n = self.num_seqs
        st = _append(self._h, rows, kp, k_ld, vp, v_ld, qp, q_ld, op, o_ld, _ints(cu_tokens, n + 1, "cu_tokens"), theta,
                     _ints(start, n, "start"), _ints(start_seen, n, "start_seen"), _stream(stream, k))
        if st.code != OK:
            _fail(st)

    def attend(self, q, out, *, scale: float = 0.0, window: int = 0, alibi: bool = False, accumulate: bool = False,
               weights_in=None, stream=None) -> None:
        """out [sequences, heads, dim] = attention of q over each sequence's slots."""
        _, qp, q_ld = _rows(q, self._qw, "q", self.num_seqs)
        _, op, o_ld = _rows(out, self._qw, "out", self.num_seqs)
        st = _attend(self._h, qp, q_ld, op, o_ld, scale, window, 1 if alibi else 0, 1 if accumulate else 0,
                     None if weights_in is None else self._weights(weights_in, "weights_in"), _stream(stream, q))
        if st.code != OK:
            _fail(st)

    def evict(self, keep: int, *, budget: int | None = None, sinks: int = 0, recent: int = 0, lens_in=None, weights_in=None,
              positions_in=None, stream=None) -> None:
        """Sequences of more than `budget` slots (None: keep) are cut to `keep`."""
        st = _evict(self._h, keep, keep if budget is None else budget, sinks, recent,
                    _ints(lens_in, self.num_seqs, "lens_in"),
                    None if weights_in is None else self._weights(weights_in, "weights_in"),
                    None if positions_in is None else self._positions(positions_in, "positions_in"), _stream(stream, self.lens))
        if st.code != OK:
            _fail(st)

    def check_error(self, stream=None) -> None:
        """Synchronizes and raises (code 1) if an earlier call met a bad page id, length or cu_tokens,
        or a prompt for a sequence that holds slots."""
        check(_L.welvet_b200_kv_check_error(self._h, _stream(stream, self.lens)))

    def release(self) -> None:
        if self._h:
            _L.welvet_b200_kv_release(self._h)
            self._h = c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass


def _mha_rows(cell_d: int, rows: int, x, y, attn, width: int):
    for t, w, what in ((x, cell_d, "x"), (y, cell_d, "y"), (attn, width, "attn")):
        if t is not None and (t.dtype is not _F32 or not t.is_cuda or not t.is_contiguous() or t.shape != (rows, w)):
            raise ValueError(f"{what}: expected a contiguous float32 CUDA tensor ({rows}, {w})")
    return x.data_ptr(), None if attn is None else attn.data_ptr(), y.data_ptr()


def mha_decode(cell, cache: PagedKV, x, y, attn=None, *, accumulate: bool = False, active=None, stream=None) -> None:
    """One new token per sequence through an MhaCell over a cache: x, y [sequences, d_model]. Sequences
    whose `active` (int32 on the GPU) is 0 are left out: their cache stays as it is, their rows of y are 0."""
    xp, ap, yp = _mha_rows(cell.d_model, cache.num_seqs, x, y, attn, cache._qw)
    check(_L.welvet_b200_mha_decode_active_device(cell._h, cache._h, xp, ap, yp, 1 if accumulate else 0,
                                                  _ints(active, cache.num_seqs, "active"), _stream(stream, x)))


def mha_prefill(cell, cache: PagedKV, sequence: int, x, y, attn=None, *, stream=None) -> None:
    """A prompt x [tokens, d_model] through an MhaCell, its keys and values into a sequence of the cache whose
    length is 0, from position 0. One that holds slots keeps them; `check_error` says so."""
    xp, ap, yp = _mha_rows(cell.d_model, x.shape[0], x, y, attn, cache._qw)
    check(_L.welvet_b200_mha_prefill_device(cell._h, cache._h, sequence, x.shape[0], xp, ap, yp, _stream(stream, x)))


def group_quantize(W, group: int, code: int, scale_dtype=torch.bfloat16, stream=None):
    """(codes, scales, zeros) of a float32 CUDA matrix [out, in]; zeros is None unless code is UINT4."""
    if W.dtype is not _F32 or not W.is_cuda or not W.is_contiguous() or W.ndim != 2:
        raise ValueError("group_quantize: expected a contiguous float32 CUDA matrix")
    if scale_dtype not in _SCALES:
        raise ValueError("group_quantize: scales are float16 or bfloat16")
    out, in_ = W.shape
    groups = -(-in_ // max(1, group))
    codes = torch.empty((out, (in_ + 1) // 2), dtype=torch.uint8, device=W.device)
    scales = torch.empty((out, groups), dtype=scale_dtype, device=W.device)
    zeros = torch.empty((out, groups), dtype=torch.uint8, device=W.device) if code == UINT4 else None
    check(_L.welvet_b200_group_quantize(in_, out, group, code, _SCALES[scale_dtype], W.data_ptr(), codes.data_ptr(),
                                        scales.data_ptr(), None if zeros is None else zeros.data_ptr(), _stream(stream, W)))
    return codes, scales, zeros


_PLAN = ("slabs", "slab_chunks", "slab_blocks", "solo", "whole", "smem", "row_groups", "chunks", "runs", "cut")


def gdense_plan(in_features: int, out: int, group: int, code: int, rows: int, sms: int = 148) -> dict:
    """How a call of `rows` rows (1..8) on such a layer is launched (welvet_b200_gdense_plan)."""
    v = (c_int64 * len(_PLAN))()
    if _L.welvet_b200_gdense_plan(in_features, out, group, code, sms, rows, v, len(_PLAN)) != len(_PLAN):
        raise ValueError("gdense_plan: no such layer or number of rows")
    return dict(zip(_PLAN, v))


class GroupDense:
    """A Dense layer of 4-bit codes with group scales (welvet_b200_gdense_*)."""

    def __init__(self, handle, in_: int, out: int):
        self._h, self.in_, self.out = handle, in_, out

    @classmethod
    def from_codes(cls, codes, scales, in_features: int, group: int, code: int, *, zeros=None, act: int = LINEAR, bias=None):
        """codes [out, (in + 1) // 2] uint8, scales [out, groups] float16 / bfloat16, zeros (UINT4)
        [out, groups] uint8: contiguous CUDA tensors, copied. bias: host values, row o < len(bias)."""
        out = codes.shape[0]
        groups = -(-in_features // max(1, group))
        for t, dt, shape, what in ((codes, torch.uint8, (out, (in_features + 1) // 2), "codes"),
                                   (scales, scales.dtype, (out, groups), "scales"),
                                   (zeros, torch.uint8, (out, groups), "zeros")):
            if t is not None and (t.dtype is not dt or t.shape != shape or not t.is_cuda or not t.is_contiguous()):
                raise ValueError(f"GroupDense: {what} must be a contiguous CUDA tensor {shape} of {dt}")
        if scales.dtype not in _SCALES:
            raise ValueError("GroupDense: scales are float16 or bfloat16")
        b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float64)
        torch.cuda.current_stream().synchronize()  # the mount copies on its own stream
        h = c_void_p()
        check(_L.welvet_b200_gdense_mount(in_features, out, group, code, _SCALES[scales.dtype], act, codes.data_ptr(),
                                          scales.data_ptr(), None if zeros is None else zeros.data_ptr(), 1, _np_ptr(b),
                                          0 if b is None else b.size, byref(h)))
        return cls(h, in_features, out)

    @classmethod
    def quantize(cls, W, group: int, code: int, *, scale_dtype=torch.bfloat16, act: int = LINEAR, bias=None):
        """The layer of a float32 CUDA matrix [out, in], rounded to nearest."""
        codes, scales, zeros = group_quantize(W, group, code, scale_dtype)
        return cls.from_codes(codes, scales, W.shape[1], group, code, zeros=zeros, act=act, bias=bias)

    def forward(self, x, y, pre=None, stream=None) -> None:
        """y [rows, out] = act(x [rows, in] W^T + bias); pre receives the values before the activation."""
        rows, xp, x_ld = _rows(x, self.in_, "x")
        for t, what in ((y, "y"), (pre, "pre")):
            if t is not None and (t.dtype is not _F32 or not t.is_cuda or not t.is_contiguous() or t.shape != (rows, self.out)):
                raise ValueError(f"{what}: expected a contiguous float32 CUDA tensor ({rows}, {self.out})")
        st = _gemv(self._h, rows, xp, x_ld, None if pre is None else pre.data_ptr(), y.data_ptr(), _stream(stream, x))
        if st.code != OK:
            _fail(st)

    def release(self) -> None:
        if self._h:
            _L.welvet_b200_gdense_release(self._h)
            self._h = c_void_p()

    def __del__(self):
        try:
            self.release()
        except Exception:
            pass
