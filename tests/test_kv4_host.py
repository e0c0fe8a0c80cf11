"""Kv4Cache's host side without a GPU: CPU tensors and a stand-in for the library that keeps what each call is given."""
import ctypes as C
import threading
from types import SimpleNamespace

import pytest
import torch

from tetraeder_b200 import _lib, kv4, moe
from tetraeder_b200.kv4 import Kv4Cache

STREAM = SimpleNamespace(cuda_stream=0)


class Lib:
    """The C entry points: each keeps its arguments (the attention's as a copy of the struct) and succeeds."""

    def __init__(self):
        self.calls = []

    def tmoe_kv4_attn_scratch_bytes(self, h):
        return 64

    def _attn(self, h, stream, cache, attn, *rest):
        self.calls.append((h, _lib.Kv4AttnStruct.from_buffer_copy(C.string_at(attn, C.sizeof(_lib.Kv4AttnStruct))), rest))
        return 0

    def _rows(self, h, stream, cache, ty, *rest):
        self.calls.append((h, ty, rest))
        return 0

    tmoe_kv4_attn_decode = tmoe_kv4_attn_prefill = _attn
    tmoe_kv4_store = tmoe_kv4_load = _rows


@pytest.fixture(autouse=True)
def settled(monkeypatch):
    """The devices whose stream a constructor waited for."""
    seen = []
    monkeypatch.setattr(kv4, "_settle", seen.append)
    monkeypatch.setattr(kv4, "_raw_stream", lambda device: 0)
    return seen


class Plane:
    """A CPU tensor that passes for a CUDA one where the planes are checked."""

    def __init__(self, t):
        self._t = t

    is_cuda = True

    def __getattr__(self, name):
        return getattr(self._t, name)


def a_layer(*args, **kw):
    return SimpleNamespace(lib=Lib(), h=1, device=torch.device("cpu"))


def make(n_seq=2, n_kv=2, hd=128, ctx=64, **kw):
    layer = kw["layer"] if "layer" in kw else a_layer()
    planes = []
    for _ in range(2):
        planes += [Plane(torch.zeros((n_seq, n_kv, ctx, hd // 2), dtype=torch.uint8)),
                   Plane(torch.zeros((n_seq, n_kv, ctx, hd // 32), dtype=torch.float16))]
    cache = Kv4Cache.from_planes(*planes, layer=layer)
    cache._dev = -1  # what a CPU tensor's get_device() says
    return cache


def rows(n, heads, dtype, hd=128):
    return torch.zeros((n, heads, hd), dtype=dtype)


POS = torch.zeros(2, dtype=torch.int32)
REFUSED = [
    ("width", lambda dt: rows(2, 4, dt, 64)),
    ("strides", lambda dt: rows(4, 2, dt).transpose(0, 1)),
    ("dimensions", lambda dt: rows(2, 4, dt)[0]),
    ("device", lambda dt: rows(2, 4, dt).to("meta")),
]


@pytest.mark.parametrize("call", ["decode", "prefill"])
@pytest.mark.parametrize("first,other", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("what,bad", REFUSED, ids=[r[0] for r in REFUSED])
def test_a_refused_call_leaves_the_next_one_as_it_was(call, first, other, what, bad):
    cache = make()

    def run(q, dt):
        k = rows(2, 2, dt)
        if call == "decode":
            cache.decode(q, k, k, POS, out=torch.empty_like(q), stream=STREAM)
        else:
            cache.prefill(q, k, k, out=torch.empty_like(q), stream=STREAM)

    q = rows(2, 4, first)
    run(q, first)
    with pytest.raises(ValueError):
        run(bad(other), other)
    run(q, first)
    (_, a, _), (_, b, _) = cache.lib.calls
    for f in ("type", "n_head", "q_ld", "kv_ld", "out_ld"):
        assert getattr(a, f) == getattr(b, f), f
    run(rows(2, 4, other), other)  # and what was refused is taken once it is right
    assert cache.lib.calls[2][1].type == (_lib.TYPE_F32 if other == torch.float32 else _lib.TYPE_BF16)


def test_a_refused_load_is_refused_again():
    cache = make()
    cache.load(0, n=4, seq=0, dtype=torch.bfloat16)
    for _ in range(2):
        with pytest.raises(RuntimeError):
            cache.load(0, n=-1, seq=0)
    k, v = cache.load(0, n=3, seq=0)
    assert k.shape == v.shape == (3, 2, 128) and k.dtype == torch.float32 and len(cache.lib.calls) == 2


def test_caches_without_a_layer_have_a_scratch_each(monkeypatch):
    monkeypatch.setattr(kv4, "_thread_layer", lambda device, layer=a_layer(): layer)
    a, b = make(layer=None), make(layer=None)
    assert a.layer is b.layer
    assert a._scratch.data_ptr() != b._scratch.data_ptr()
    q = rows(2, 4, torch.float32)
    for cache in (a, b):
        cache.decode(q, None, None, POS, out=q, stream=STREAM)
    assert [c[1].scratch for c in a.lib.calls] == [a._scratch.data_ptr(), b._scratch.data_ptr()]
    layer = a_layer()
    c, d = make(layer=layer), make(layer=layer)  # a model's: one after the other anyway
    assert c._scratch.data_ptr() == d._scratch.data_ptr()


def test_each_thread_has_its_own_handle(monkeypatch):
    monkeypatch.setattr(moe, "MoeLayer", a_layer)
    monkeypatch.setattr(kv4, "_own", threading.local())
    here = kv4._thread_layer(0)
    assert kv4._thread_layer(0) is here and kv4._thread_layer(1) is not here
    there = []
    t = threading.Thread(target=lambda: there.append(kv4._thread_layer(0)))
    t.start()
    t.join()
    assert there[0] is not here


def test_a_new_scratch_is_zero_before_a_call_on_any_stream(settled):
    layer = a_layer()
    cache = make(layer=layer)
    assert settled == [cache.device]
    make(layer=layer)
    assert len(settled) == 1  # that scratch was waited for


def test_outputs_belong_to_the_stream_that_writes_them(monkeypatch):
    cache, q = make(), rows(2, 4, torch.float32)
    within, noted = [], []

    class On:
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            within.append(self.stream)

        def __exit__(self, *exc):
            within.append(None)

    empty_like = torch.empty_like

    class Out:
        def __init__(self, t, stream):
            self.t, self.stream = t, stream

        def __getattr__(self, name):
            return getattr(self.t, name)

        def record_stream(self, stream):
            noted.append(stream)

    made = []

    def new(t, **kw):
        made.append(within[-1] if within else None)
        return Out(empty_like(t, **kw), made[-1])

    monkeypatch.setattr(torch.cuda, "stream", On)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "current")
    monkeypatch.setattr(torch, "empty_like", new)
    cache.decode(q, None, None, POS, stream=STREAM)
    cache.prefill(q, None, None, stream=STREAM)
    cache.load(POS, stream=STREAM)
    assert made == [STREAM] * 4 and noted == ["current"] * 4


def test_a_closed_layer_gives_its_caches_no_handle():
    layer = a_layer()
    cache, q = make(layer=layer), rows(2, 4, torch.float32)
    calls = [lambda: cache.decode(q, None, None, POS, out=q), lambda: cache.prefill(q, None, None, out=q),
             lambda: cache.store(rows(2, 2, torch.float32), rows(2, 2, torch.float32), POS), lambda: cache.load(POS)]
    for call in calls:
        call()
    layer.h = None  # as MoeLayer.close leaves it
    for call in calls:
        call()
    assert [c[0] for c in cache.lib.calls] == [1] * 4 + [None] * 4


@pytest.mark.parametrize("x", [1 << 32, (1 << 32) + 5, 1 << 31, -(1 << 31) - 1, -(1 << 32)])
def test_numbers_past_32_bits_are_refused(x):
    cache, q, k = make(), rows(2, 4, torch.float32), rows(2, 2, torch.float32)
    for call in (lambda: cache.decode(q, None, None, POS, out=q, window=x), lambda: cache.decode(q, None, None, POS, out=q, n_sink=x),
                 lambda: cache.decode(q, None, None, POS, out=q, window=8, n_sink=x),
                 lambda: cache.prefill(q, None, None, out=q, seq=x), lambda: cache.prefill(q, None, None, out=q, pos0=x),
                 lambda: cache.prefill(q, None, None, out=q, window=x), lambda: cache.store(k, k, x, seq=0),
                 lambda: cache.store(k, k, 0, seq=x), lambda: cache.load(x, n=1, seq=0)):
        with pytest.raises(ValueError):
            call()
    assert not cache.lib.calls


def test_f16_products_are_asked_for():
    cache, q = make(), rows(2, 4, torch.float32)
    cache.prefill(q, None, None, out=q)
    cache.prefill(q, None, None, out=q, f16_products=True)
    cache.prefill(q, None, None, out=q)
    assert [c[1].f16_products for c in cache.lib.calls] == [0, 1, 0]
