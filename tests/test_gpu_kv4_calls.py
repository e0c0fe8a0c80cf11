"""How calls of the 4-bit KV cache follow one another: a refused one between two good ones, two caches on two streams, a new
cache on another stream than the one that made it, outputs written on another stream than the current one, calls after the
layer was closed."""
import numpy as np
import pytest
import torch

import tetraeder_b200 as tb
from tests.test_gpu_kv4 import fill, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,other", [(torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)])
def test_a_refused_call_leaves_the_next_one_as_it_was(first, other):
    rng = np.random.default_rng(21)
    cache = tb.Kv4Cache(2, 2, 128, 256)
    fill(cache, rng)
    q, k, v = (randn(rng, (2, n, 128), first).cuda() for n in (8, 2, 2))
    pos = torch.tensor([200, 77], dtype=torch.int32, device="cuda")
    calls = [lambda q, k, v: cache.decode(q, k, v, pos), lambda q, k, v: cache.prefill(q, k, v, seq=1, pos0=99)]
    for call in calls:
        want = call(q, k, v).clone()
        x = q.to(other)
        for bad in (x[:, :, :64], x.transpose(0, 1), x.cpu(), x[0]):
            with pytest.raises(ValueError):
                call(bad, k.to(other), v.to(other))
        assert torch.equal(call(q, k, v), want)
        assert call(x, k.to(other), v.to(other)).dtype == other  # and the other type is taken once it is right
    cache.check()


def test_two_caches_on_two_unordered_streams():
    """Each call splits its segments over many CTAs, whose parts meet in the scratch."""
    rng = np.random.default_rng(30)
    n = 9000
    pos = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    caches, q = [tb.Kv4Cache(1, 1, 128, n) for _ in range(2)], []
    for c in caches:
        fill(c, rng)
        q.append(randn(rng, (1, 8, 128), torch.bfloat16).cuda())
    p = randn(rng, (40, 8, 128), torch.bfloat16).cuda()
    want = [(c.decode(x, None, None, pos).clone(), c.prefill(p, None, None, pos0=n - 40).clone()) for c, x in zip(caches, q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in caches]
    got = [[], []]
    for _ in range(50):
        for i, (c, x) in enumerate(zip(caches, q)):
            with torch.cuda.stream(streams[i]):
                got[i].append((c.decode(x, None, None, pos), c.prefill(p, None, None, pos0=n - 40)))
    torch.cuda.synchronize()
    for i, c in enumerate(caches):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i]))
        c.check()


def test_a_new_cache_may_be_used_on_another_stream_at_once():
    """Its planes and its scratch are zero by then, although the stream that zeroes them is busy."""
    hd, n = 128, 5000
    x = torch.ones((1, 1, hd), device="cuda")
    q = torch.ones((1, 8, hd), device="cuda")
    pos = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    junk = [torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    del junk  # what the allocator hands out next holds ones
    torch.cuda._sleep(100_000_000)
    cache = tb.Kv4Cache(1, 1, hd, n)
    with torch.cuda.stream(side):
        cache.decode(q, x, x, pos, out=out)
    side.synchronize()
    first = out.clone()
    assert int(cache.k_scales.count_nonzero()) == hd // 32  # the new row's alone
    for _ in range(3):
        assert torch.equal(cache.decode(q, x, x, pos), first)
    cache.check()


def test_an_output_does_not_take_memory_that_the_current_stream_still_reads():
    rng = np.random.default_rng(40)
    B, hd, n = 16, 128, 128
    cache = tb.Kv4Cache(B, 1, hd, n)
    fill(cache, rng)
    q = randn(rng, (B, 64, hd), torch.float32).cuda()
    pos = torch.full((B,), n - 1, dtype=torch.int32, device="cuda")
    want = cache.decode(q, None, None, pos).clone()
    wk, _ = cache.load(0, n=100, seq=0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for call, shape in ((lambda: cache.decode(q, None, None, pos, stream=side), q.shape),
                        (lambda: cache.load(0, n=100, seq=0, stream=side)[0], wk.shape)):
        x = torch.full(shape, 7.0, device="cuda")
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)
        y = x.clone()  # runs after the sleep
        del x          # the next block of this size on the current stream is x's
        got = call()
        side.synchronize()
        torch.cuda.synchronize()
        assert bool((y == 7.0).all())
        assert torch.equal(got, want if got.shape == want.shape else wk)
    cache.check()


def test_calls_after_the_layer_was_closed_are_refused():
    layer = tb.MoeLayer(512, 256, 8, 2, max_tokens=4)
    cache = tb.Kv4Cache(2, 2, 128, 64, layer=layer)
    q, k = torch.zeros((2, 4, 128), device="cuda"), torch.zeros((2, 2, 128), device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache.decode(q, k, k, pos)
    layer.close()
    for call in (lambda: cache.decode(q, k, k, pos), lambda: cache.prefill(q, k, k), lambda: cache.store(k, k, pos),
                 lambda: cache.load(pos), cache.check):
        with pytest.raises(tb.TmoeError, match="TMOE_E_INVALID"):
            call()


def test_an_error_on_a_side_stream_is_found_there():
    cache = tb.Kv4Cache(1, 1, 64, 64)
    x = torch.ones((1, 1, 64), device="cuda")
    bad = torch.tensor([64], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
    cache.store(x, x, bad, seq=0, stream=side)
    with pytest.raises(tb.TmoeError, match="outside the 4-bit cache"):
        cache.check(stream=side)
    cache.check()
