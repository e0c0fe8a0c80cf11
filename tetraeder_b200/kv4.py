"""The 4-bit KV cache and the attention over it (tmoe_kv4_* of include/tmoe.h, where the format and the
rules stand): K and V rows are quantised as they are written, 4.5 bits a value against F16's 16, and the
decode and prefill attention read them as they are.

    cache = Kv4Cache(n_seq=8, n_kv=4, head_dim=128, n_ctx=32768)
    out = cache.prefill(q, k, v, seq=0, pos0=0)            # [S, n_head, 128] queries of one sequence
    out = cache.decode(q, k, v, pos, window=4096, n_sink=4)  # [B, n_head, 128], one token per sequence

Activations are float32 or bfloat16 CUDA tensors; a token's heads are contiguous, tokens may be apart
(views into a fused projection's output work)."""
from __future__ import annotations

import ctypes as C
import threading

import torch

from . import _lib

_TYPES = {torch.float32: _lib.TYPE_F32, torch.bfloat16: _lib.TYPE_BF16}
# the current stream's handle by device ordinal, without the Stream object where torch has the call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda device: torch.cuda.current_stream(device).cuda_stream)
_own = threading.local()  # .layers: device ordinal -> a small handle, for the caches that this thread makes without one


def _thread_layer(device: int):
    from .moe import MoeLayer
    layers = _own.__dict__.setdefault("layers", {})
    if device not in layers:
        layers[device] = MoeLayer(512, 256, 8, 2, gate_type=_lib.TYPE_Q4_K, up_type=_lib.TYPE_Q4_K,
                                  down_type=_lib.TYPE_Q4_K, max_tokens=4, device=device)
    return layers[device]


def _settle(device):
    """Waits for memory just zeroed on the current stream: a call may be on any other one."""
    with torch.cuda.device(device):
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream().synchronize()


_INT_MIN, _INT_MAX = -1 << 31, (1 << 31) - 1


def _int32(names, x, y):
    """Two numbers that the C calls take in 32 bits: ctypes would pass on the low ones of any other."""
    if not (_INT_MIN <= x <= _INT_MAX and _INT_MIN <= y <= _INT_MAX):
        raise ValueError(f"{names} are {x}, {y}")


class Kv4Cache:
    """Planes k_codes, v_codes uint8 [n_seq, n_kv, capacity, head_dim / 2] and k_scales, v_scales float16
    [n_seq, n_kv, capacity, head_dim / 32]; capacity is n_ctx rounded up to a multiple of 64.  `layer` (a
    MoeLayer) gives the handle whose device error flag the calls use.  The caches of a layer share its attention
    scratch (40 MB): like a handle's other calls, theirs come from one thread and run on one stream, or on
    ordered ones.  A cache made without a layer has a scratch of its own, so that only its own calls have to be
    ordered, and a small handle that it shares with such caches made by the same thread on the same device."""

    def __init__(self, n_seq: int, n_kv: int, head_dim: int, n_ctx: int, device: int | None = None, layer=None):
        if not torch.cuda.is_available():
            raise RuntimeError("tetraeder_b200 needs a CUDA device (there is no CPU path)")
        if n_seq <= 0 or n_kv <= 0 or n_ctx <= 0 or head_dim not in (64, 128):
            raise ValueError(f"a 4-bit cache of {n_seq} sequences, {n_kv} KV heads of {head_dim} (64 or 128), "
                             f"{n_ctx} positions")
        if device is None:
            device = torch.cuda.current_device() if layer is None else layer.device.index
        dev = torch.device("cuda", device)
        cap = -(-n_ctx // 64) * 64
        planes = []
        for _ in range(2):
            planes.append(torch.zeros((n_seq, n_kv, cap, head_dim // 2), dtype=torch.uint8, device=dev))
            planes.append(torch.zeros((n_seq, n_kv, cap, head_dim // 32), dtype=torch.float16, device=dev))
        self._set(planes, layer)
        _settle(dev)

    @classmethod
    def from_planes(cls, k_codes, k_scales, v_codes, v_scales, layer=None) -> "Kv4Cache":
        """A cache over planes that the caller holds (contiguous, of the class's shapes)."""
        self = cls.__new__(cls)
        self._set([k_codes, k_scales, v_codes, v_scales], layer)
        return self

    def _set(self, planes, layer):
        codes, scales = planes[0], planes[1]
        if codes.dim() != 4 or scales.dim() != 4:
            raise ValueError("planes are [n_seq, n_kv, positions, bytes or scales]")
        n_seq, n_kv, cap, half = codes.shape
        for i, t in enumerate(planes):
            want = (n_seq, n_kv, cap, half if i % 2 == 0 else half // 16)
            if tuple(t.shape) != want or t.dtype != (torch.float16 if i % 2 else torch.uint8):
                raise ValueError(f"plane {i} is {t.dtype} {tuple(t.shape)}, not {want}")
            if not t.is_cuda or t.device != codes.device or not t.is_contiguous():
                raise ValueError("planes are contiguous CUDA tensors of one device")
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = planes
        self.n_seq, self.n_kv, self.head_dim, self.n_ctx = n_seq, n_kv, 2 * half, cap
        self.device = codes.device
        self.layer = _thread_layer(codes.device.index) if layer is None else layer
        if self.layer.device != self.device:
            raise ValueError("the layer's handle is of another device")
        self.lib = self.layer.lib
        self._c = _lib.Kv4CacheStruct(*(t.data_ptr() for t in planes), n_seq, n_kv, self.head_dim, cap)
        self._cp = C.addressof(self._c)
        self._scratch = getattr(layer, "_kv4_scratch", None)
        if self._scratch is None:
            n = self.lib.tmoe_kv4_attn_scratch_bytes(self.h)
            _lib.check(n if n < 0 else 0, self.h)
            self._scratch = torch.zeros(n, dtype=torch.uint8, device=self.device)
            if layer is not None:
                layer._kv4_scratch = self._scratch
            _settle(self.device)
        self._a = _lib.Kv4AttnStruct()
        self._a.scratch = self._scratch.data_ptr()
        self._ap = C.addressof(self._a)
        self._dev, self._scale = self.device.index, self.head_dim ** -0.5
        self._q_sig = self._kv_sig = self._row_sig = None
        self._kv_ld = 0

    @property
    def h(self):
        """The layer's handle: none once the layer is closed, which the library refuses."""
        return self.layer.h

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_codes, self.k_scales, self.v_codes, self.v_scales))

    # -- arguments -------------------------------------------------------------------------
    # A serving loop makes the same calls step after step, so the checks of a call's shapes, strides and types
    # are remembered for the last ones seen (never addresses or values).
    def _heads(self, name, t, n, dtype, n_head=None):
        """Elements from token to token of t [n, heads, head_dim] (a token's heads contiguous)."""
        hd = self.head_dim
        if t.dim() != 3 or t.shape[0] != n or t.shape[2] != hd or (n_head is not None and t.shape[1] != n_head):
            raise ValueError(f"{name} is {tuple(t.shape)}, not [{n}, {'heads' if n_head is None else n_head}, {hd}]")
        if t.dtype != dtype or t.device != self.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, not {dtype} on {self.device}")
        ld, sh, sd = t.stride()
        if sd != 1 or (sh != hd and t.shape[1] != 1):
            raise ValueError(f"{name}: a token's heads must be contiguous")
        return ld if n > 1 else t.shape[1] * hd

    def _index(self, name, t, n):
        if t.dtype != torch.int32 or t.shape != (n,) or t.get_device() != self._dev or (n > 1 and t.stride(0) != 1):
            raise ValueError(f"{name} is a contiguous int32 tensor [{n}] on {self.device}")
        return t.data_ptr()

    def _place(self, n, pos, seq):
        """(seq, seq0, pos, pos0) of the C calls."""
        p, pos0 = (self._index("pos", pos, n), 0) if torch.is_tensor(pos) else (None, int(pos))
        if p is None:
            _int32("pos and n", pos0, n)
        if torch.is_tensor(seq):
            return self._index("seq", seq, n), 0, p, pos0
        if seq is None and p is None:
            raise ValueError("a run of positions needs its sequence")
        if seq is not None and not 0 <= seq < self.n_seq:
            raise ValueError(f"sequence {seq} of {self.n_seq}")
        return None, -1 if seq is None else int(seq), p, pos0

    def _stream(self, stream):
        return _raw_stream(self._dev) if stream is None else stream.cuda_stream

    def _new(self, like, stream):
        """A tensor of that shape for a call's output.  Its memory is the stream's that writes it: a block that the current
        stream has just freed may still be in use there.  The current stream, whose caller reads it, is noted too."""
        if stream is None:
            return torch.empty_like(like, memory_format=torch.contiguous_format)
        with torch.cuda.stream(stream):
            out = torch.empty_like(like, memory_format=torch.contiguous_format)
        out.record_stream(torch.cuda.current_stream(self.device))
        return out

    @staticmethod
    def _type(t):
        if t.dtype not in _TYPES:
            raise ValueError(f"activations are float32 or bfloat16, not {t.dtype}")
        return _TYPES[t.dtype]

    def _kv_rows(self, k, v, n, dtype):
        """Elements from token to token of rows k, v [n, n_kv, head_dim]."""
        sig = (n, dtype, k.dtype, v.dtype, k.shape, v.shape, k.stride(), v.stride(), k.get_device(), v.get_device())
        if sig != self._kv_sig:
            ld = self._heads("k", k, n, dtype, self.n_kv)
            if self._heads("v", v, n, dtype, self.n_kv) != ld:
                raise ValueError("k and v rows are different distances apart")
            self._kv_sig, self._kv_ld = sig, ld
        return self._kv_ld

    # -- rows ------------------------------------------------------------------------------
    def store(self, k, v, pos, seq=None, stream=None):
        """Quantises rows k, v [n, n_kv, head_dim] into the cache: row i at position pos[i] of sequence
        seq[i] (an int: that one; None: sequence i), or at pos + i of one sequence, where pos is an int.  A negative pos[i]: no row."""
        n, ty = k.shape[0], self._type(k)
        ld = self._kv_rows(k, v, n, k.dtype)
        s, s0, p, p0 = self._place(n, pos, seq)
        rc = self.lib.tmoe_kv4_store(self.h, self._stream(stream), self._cp, ty, k.data_ptr(), v.data_ptr(), ld,
                                     s, s0, p, p0, n)
        if rc:
            _lib.check(rc, self.h)

    def load(self, pos, n: int | None = None, seq=None, dtype=torch.float32, stream=None):
        """The rows as values, (k, v) [n, n_kv, head_dim]: placed as in store (n: how many,
        where pos is an int).  Zeros where pos[i] is negative."""
        n = pos.shape[0] if torch.is_tensor(pos) else n
        if n is None:
            raise ValueError("load from an int position needs n")
        ty = _TYPES.get(dtype)
        if ty is None:
            raise ValueError(f"rows come as float32 or bfloat16, not {dtype}")
        s, s0, p, p0 = self._place(n, pos, seq)
        sig = (n, dtype)
        if sig != self._row_sig:  # a shape to allocate by: no memory of its own
            self._row_like = torch.empty(1, dtype=dtype, device=self.device).expand(n, self.n_kv, self.head_dim)
            self._row_sig = sig
        like = self._row_like
        k, v = (torch.empty_like(like), torch.empty_like(like)) if stream is None else (self._new(like, stream), self._new(like, stream))
        rc = self.lib.tmoe_kv4_load(self.h, self._stream(stream), self._cp, ty, k.data_ptr(), v.data_ptr(),
                                    self.n_kv * self.head_dim, s, s0, p, p0, n)
        if rc:
            _lib.check(rc, self.h)
        return k, v

    # -- attention -------------------------------------------------------------------------
    def _attn(self, q, k, v, window, n_sink, scale, out, stream):
        a, n, dt = self._a, q.shape[0], q.dtype
        sig = (dt, q.shape, q.stride(), q.get_device())
        if sig != self._q_sig:
            ty, ld = self._type(q), self._heads("q", q, n, dt)  # a refused q changes nothing
            a.type, a.q_ld, a.n_head = ty, ld, q.shape[1]
            self._q_sig = sig
        if out is None:
            out = torch.empty_like(q) if stream is None and q.is_contiguous() else self._new(q, stream)
            a.out_ld = q.shape[1] * self.head_dim
        else:
            a.out_ld = self._heads("out", out, n, dt, q.shape[1])
        if k is not None and v is not None:
            a.kv_ld = self._kv_rows(k, v, n, dt)
            a.k, a.v = k.data_ptr(), v.data_ptr()
        elif k is None and v is None:
            a.k = a.v = None
        else:
            raise ValueError("k and v come together")
        a.q, a.out = q.data_ptr(), out.data_ptr()
        if window or n_sink:
            _int32("window and n_sink", window, n_sink)
        a.window, a.n_sink = window, n_sink
        a.scale = self._scale if scale is None else scale
        return out

    def decode(self, q, k, v, pos, window: int = 0, n_sink: int = 0, scale: float | None = None, out=None, stream=None):
        """One new token for each of B <= n_seq sequences: q [B, n_head, head_dim], its row k, v [B, n_kv, head_dim]
        (None: stored already) at pos[b] (int32 CUDA [B]; negative: no token, zeros come out).  Each query
        attends to positions 0..pos[b] of its sequence, with window > 0 to the last `window` of them and the
        first n_sink.  Returns out [B, n_head, head_dim]."""
        out = self._attn(q, k, v, window, n_sink, scale, out, stream)
        B = q.shape[0]
        rc = self.lib.tmoe_kv4_attn_decode(self.h, self._stream(stream), self._cp, self._ap, self._index("pos", pos, B), B)
        if rc:
            _lib.check(rc, self.h)
        return out

    def prefill(self, q, k, v, seq: int = 0, pos0: int = 0, window: int = 0, n_sink: int = 0,
                scale: float | None = None, out=None, stream=None, f16_products: bool = False):
        """S new tokens of sequence `seq` at positions pos0 .. pos0 + S - 1: rows k, v [S, n_kv, head_dim] are stored
        (None: stored already), then query i of q [S, n_head, head_dim] attends to positions 0 .. pos0 + i (or
        its window and sinks).  float32 queries are computed to their own precision, or, with f16_products, with
        Q, K, P and V as 16-bit operands of the tensor cores, up to eight times faster.  Returns out [S, n_head, head_dim]."""
        _int32("seq and pos0", seq, pos0)
        out = self._attn(q, k, v, window, n_sink, scale, out, stream)
        self._a.f16_products = f16_products
        rc = self.lib.tmoe_kv4_attn_prefill(self.h, self._stream(stream), self._cp, self._ap, seq, pos0, q.shape[0])
        if rc:
            _lib.check(rc, self.h)
        return out

    def check(self, stream=None):
        """Synchronises the stream (the current one) and raises if a kernel latched an error."""
        _lib.check(self.lib.tmoe_check(self.h, self._stream(stream)), self.h)
