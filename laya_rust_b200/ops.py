"""Operators on the caller's own device buffers (include/laya_ops.h): a
projection shared by many requests with low-rank adapters, and rotary
positions of queries and keys.

Buffers are raw device addresses (``tensor.data_ptr()``), strides are in
elements, ``stream`` is a raw ``cudaStream_t`` (0: the default stream).  Calls
enqueue work and return; errors raise :class:`LayaError`.
"""
from __future__ import annotations

import ctypes
import struct
from dataclasses import dataclass

import numpy as np

from .engine import Engine, _check, _int32, lib as _engine_lib

F16, BF16, F32 = range(3)
TYPE = {"f16": F16, "bf16": BF16, "f32": F32}
ROPE_HALF, ROPE_INTERLEAVED = range(2)
ROPE_NONE, ROPE_LINEAR, ROPE_BASE, ROPE_PARTS = range(4)
ROPE_MAX_DIM = 512

NONE = -1  # a segment without an adapter

_f64p = ctypes.POINTER(ctypes.c_double)
_i32p = ctypes.POINTER(ctypes.c_int32)


class _CRopeScaling(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_int32), ("factor", ctypes.c_double), ("trained_len", ctypes.c_double),
                ("low", ctypes.c_double), ("high", ctypes.c_double), ("attn", ctypes.c_double)]


class _CRopeSpec(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int32), ("layout", ctypes.c_int32), ("inverse", ctypes.c_int32),
                ("dim", ctypes.c_int32), ("rot", ctypes.c_int32), ("mscale", ctypes.c_float), ("freqs", _f64p)]


_rope_tensor = struct.Struct("=7q")  # laya_rope_tensor: seven 64-bit fields


_bound = False


def lib():
    global _bound
    L = _engine_lib()
    if not _bound:
        vp, i64, sc = ctypes.c_void_p, ctypes.c_int64, ctypes.POINTER(_CRopeScaling)
        L.laya_rope_freqs.argtypes = [ctypes.c_double, ctypes.c_int, sc, _f64p, ctypes.POINTER(ctypes.c_float)]
        L.laya_rope_turns.argtypes = [ctypes.c_double, ctypes.POINTER(ctypes.c_uint64)]
        L.laya_rope.argtypes = [ctypes.c_int, vp, ctypes.c_char_p, ctypes.c_int,
                                i64, vp, i64, vp]
        L.laya_set_rope_scaling.argtypes = [vp, sc, sc]
        ci, i32p, i64p = ctypes.c_int, ctypes.POINTER(ctypes.c_int32), ctypes.POINTER(i64)
        L.laya_lora_create.argtypes = [ci, ci, i64, i64, vp, i64, vp, ci, ci, ctypes.POINTER(vp)]
        L.laya_lora_set.argtypes = [vp, ci, ci, vp, vp, ci, ctypes.c_float]
        L.laya_lora_clear.argtypes = [vp, ci]
        L.laya_lora_destroy.argtypes = [vp]
        L.laya_lora_destroy.restype = None
        L.laya_lora_plan_create.argtypes = [vp, i32p, i32p, ci, ctypes.POINTER(vp)]
        L.laya_lora_run.argtypes = [vp, vp, vp, i64, vp, i64, vp]
        L.laya_lora_status.argtypes = [vp]
        L.laya_lora_test_timeout_next.argtypes = [vp, ci, ctypes.c_uint64]
        L.laya_lora_plan_destroy.argtypes = [vp]
        L.laya_lora_plan_destroy.restype = None
        L.laya_lora_layout.argtypes = [i32p, i32p, ci, i32p, ci, i64p, i64p, i32p, i64, i32p, i64]
        _bound = True
    return L


# ---- rotary positions ----------------------------------------------------------
@dataclass
class RopeScaling:
    """How frequencies are stretched for a context `factor` times the trained
    length; trained_len, low and high belong to ROPE_PARTS; attn 0 takes the
    scheme's own factor on cos and sin."""
    kind: int
    factor: float
    trained_len: float = 0.0
    low: float = 0.0
    high: float = 0.0
    attn: float = 0.0

    def _c(self) -> _CRopeScaling:
        return _CRopeScaling(self.kind, self.factor, self.trained_len, self.low, self.high, self.attn)


def rope_freqs(base: float, rot: int, scaling: RopeScaling | None = None) -> tuple[np.ndarray, float]:
    """laya_rope_freqs: (frequencies [rot / 2] in radians per position, factor
    on cos and sin)."""
    f = np.empty(max(rot, 0) // 2, np.float64)
    m = ctypes.c_float()
    _check(lib().laya_rope_freqs(base, rot, ctypes.byref(scaling._c()) if scaling else None,
                                 f.ctypes.data_as(_f64p), ctypes.byref(m)))
    return f, m.value


def rope_turns(freq: float) -> int:
    """laya_rope_turns: the 64-bit fraction of a turn per position that `freq`
    radians are kept as."""
    t = ctypes.c_uint64()
    _check(lib().laya_rope_turns(freq, ctypes.byref(t)))
    return t.value


class RopeSpec:
    """Element type, head size and rotated part, frequencies and layout."""

    def __init__(self, type: int, dim: int, rot: int, freqs, layout: int = ROPE_HALF, inverse: bool = False,
                 mscale: float = 1.0):
        self.freqs = np.ascontiguousarray(freqs, dtype=np.float64).ravel()
        if self.freqs.size != max(rot, 0) // 2:
            raise ValueError(f"RopeSpec: {self.freqs.size} frequencies for rot {rot}")
        self._c = _CRopeSpec(type, layout, 1 if inverse else 0, dim, rot, mscale, self.freqs.ctypes.data_as(_f64p))
        self._at = ctypes.addressof(self._c)


@dataclass(slots=True)
class RopeTensor:
    """A [tokens, heads, dim] view at device address `x`, rotated into `out`."""
    x: int
    out: int
    heads: int
    x_token: int
    x_head: int
    out_token: int
    out_head: int


def rope(spec: RopeSpec, tensors, tokens: int, pos: int = 0, pos0: int = 0, device: int = 0, stream: int = 0) -> None:
    """laya_rope: rotates 1 to 4 tensors (e.g. q and k) over the same tokens in
    one launch.  pos: device address of int32 [tokens], or 0 for pos0, pos0 + 1, ..."""
    arr = b"".join([_rope_tensor.pack(t.x, t.out, t.x_token, t.x_head, t.out_token, t.out_head, t.heads)
                    for t in tensors])
    _check(lib().laya_rope(device, spec._at, arr, len(tensors), tokens, pos or None, pos0, stream or None))


def set_rope_scaling(engine: Engine, full: RopeScaling | None = None, sliding: RopeScaling | None = None) -> None:
    """laya_set_rope_scaling: the engine's rotation with stretched frequencies
    of its global (`full`) and windowed (`sliding`) layers; None: as the model
    has them."""
    p = [ctypes.byref(s._c()) if s else None for s in (full, sliding)]
    _check(lib().laya_set_rope_scaling(engine._h, p[0], p[1]))


# ---- a shared projection with low-rank adapters ------------------------------------
def _segments(rows, slots):
    r, s = _int32(rows, "rows"), _int32(slots, "slots")
    if r.size != s.size:
        raise ValueError(f"{r.size} segments but {s.size} slots")
    return r, s


def _host(a) -> tuple[np.ndarray, int]:
    """Contiguous host values and their type code: f16 stays, the rest is f32."""
    a = np.ascontiguousarray(a)
    if a.dtype != np.float16:
        a = np.ascontiguousarray(a, dtype=np.float32)
    return a, F16 if a.dtype == np.float16 else F32


class LoraPlan:
    """The segments of one batch and the workspace of its runs."""

    def __init__(self, lora: "Lora", rows, slots):
        r, s = _segments(rows, slots)
        self.rows = int(r.sum(dtype=np.int64))
        self._lora = lora
        h = ctypes.c_void_p()
        _check(lib().laya_lora_plan_create(lora._h, r.ctypes.data_as(_i32p), s.ctypes.data_as(_i32p), r.size,
                                           ctypes.byref(h)))
        self._h = h
        self._destroy = lib().laya_lora_plan_destroy

    def status(self) -> None:
        """Waits for the device; raises if a bounded wait expired in a run."""
        _check(lib().laya_lora_status(self._h))

    def test_timeout_next(self, kind: int, limit_ns: int = 1_000_000) -> None:
        """Arms the next run: the loads of the rank-space product's launch (0), of
        the projection (1) or the exchange in a cluster (2) wait in vain for
        limit_ns; status() then raises."""
        _check(lib().laya_lora_test_timeout_next(self._h, kind, limit_ns))

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()


class Lora:
    """A projection W [out, inn] (device address, row pitch ldw) and the
    low-rank adapters beside it."""

    def __init__(self, type: int, inn: int, out: int, w: int, ldw: int, bias: int = 0, slots: int = 64,
                 max_rank: int = 128, device: int = 0):
        h = ctypes.c_void_p()
        _check(lib().laya_lora_create(device, type, inn, out, w or None, ldw, bias or None, slots, max_rank,
                                      ctypes.byref(h)))
        self._h = h
        self._destroy = lib().laya_lora_destroy
        self.inn, self.out = inn, out

    def set(self, slot: int, a, b, scale: float = 1.0) -> None:
        """Adapter `slot`: a [rank, inn], b [out, rank] (host arrays, f16 or
        converted to f32)."""
        (a, t), (b, tb) = _host(a), _host(b)
        if t != tb:
            a, b, t = a.astype(np.float32), b.astype(np.float32), F32
        if a.ndim != 2 or b.ndim != 2 or a.shape[1] != self.inn or b.shape != (self.out, a.shape[0]):
            raise ValueError(f"adapter shapes {a.shape}, {b.shape} do not fit [rank, {self.inn}], [{self.out}, rank]")
        _check(lib().laya_lora_set(self._h, slot, a.shape[0], a.ctypes.data, b.ctypes.data, t, scale))

    def clear(self, slot: int) -> None:
        _check(lib().laya_lora_clear(self._h, slot))

    def plan(self, rows, slots) -> LoraPlan:
        """A plan for segments of `rows[i]` rows with adapter `slots[i]` or NONE."""
        return LoraPlan(self, rows, slots)

    def run(self, plan: LoraPlan, x: int, ldx: int, y: int, ldy: int, stream: int = 0) -> None:
        """Enqueues y = the projection of x (device addresses, row pitches)."""
        _check(lib().laya_lora_run(self._h, plan._h, x or None, ldx, y or None, ldy, stream or None))

    def close(self) -> None:
        if getattr(self, "_h", None):
            self._destroy(self._h)
            self._h = None

    def __del__(self):
        self.close()


def lora_layout(rows, slots, ranks) -> tuple[np.ndarray, np.ndarray]:
    """laya_lora_layout: (off [blocks + 1], chunks [entries, 2]) of the
    segments' host plan, with no device."""
    r, s = _segments(rows, slots)
    k = _int32(ranks, "ranks")
    nb, ne = ctypes.c_int64(), ctypes.c_int64()
    p = lambda a: a.ctypes.data_as(_i32p)
    L = lib()
    _check(L.laya_lora_layout(p(r), p(s), r.size, p(k), k.size, ctypes.byref(nb), ctypes.byref(ne), None, 0, None, 0))
    off = np.zeros(nb.value + 1, np.int32)
    chunks = np.zeros((ne.value, 2), np.int32)
    _check(L.laya_lora_layout(p(r), p(s), r.size, p(k), k.size, ctypes.byref(nb), ctypes.byref(ne), p(off), nb.value,
                              p(chunks), ne.value))
    return off, chunks
