"""Prefill of f32 rows over the 4-bit KV cache: to f32 precision for any number of tokens (the decode's bound of test_gpu_kv4.py),
or with 16-bit operands where the caller allows it (the prefill's)."""
import numpy as np
import pytest
import torch

import tetraeder_b200 as tb
from tests import kv4_ref as R
from tests.test_gpu_kv4 import close, decode_tol, fill, prefill_tol, randn, rowvals

pytestmark = pytest.mark.gpu


def run(hd, nh, nkv, S, pos0, window=0, n_sink=0, f16=False, gain=1.0, given=True, rows=None):
    rng = np.random.default_rng(hd + nh + S + pos0)
    cache = tb.Kv4Cache(2, nkv, hd, pos0 + S + 3)
    K, V = (x[1] for x in fill(cache, rng))
    q, k, v = (randn(rng, (S, n, hd), torch.float32, g) for n, g in ((nh, gain), (nkv, 1.0), (nkv, 1.0)))
    cache.k_scales[1, :, pos0 + S:] = float("nan")
    cache.v_scales[1, :, pos0 + S:] = float("inf")
    if not given:
        cache.store(k.cuda(), v.cuda(), pos0, seq=1)
    new = (k.cuda(), v.cuda()) if given else (None, None)
    got = cache.prefill(q.cuda(), *new, seq=1, pos0=pos0, window=window, n_sink=n_sink, f16_products=f16)
    cache.check()
    K[:, pos0:pos0 + S], V[:, pos0:pos0 + S] = rowvals(k).transpose(1, 0, 2), rowvals(v).transpose(1, 0, 2)
    Kt, Vt = K.transpose(1, 0, 2), V.transpose(1, 0, 2)
    for i in sorted({0, 1, S // 3, S // 2, S - 2, S - 1} | set(range(0, S, rows or 13))):
        want, *m = R.attend(q[i].double().numpy(), Kt, Vt, pos0 + i, window, n_sink, hd ** -0.5)
        close(got[i], want, (prefill_tol if f16 else decode_tol)("f32", want, *m), f"token {i}")
    assert got.dtype == torch.float32 and bool(torch.isfinite(got).all())


SHAPES = [(128, 8, 1, 130, 0), (64, 16, 1, 140, 1), (128, 14, 2, 90, 129), (64, 6, 3, 50, 77), (128, 5, 5, 27, 4000), (128, 1, 1, 257, 63),
          (64, 48, 2, 65, 191), (128, 32, 4, 2, 0), (128, 32, 4, 300, 500)]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("hd,nh,nkv,S,pos0", SHAPES)
def test_shapes(hd, nh, nkv, S, pos0, f16):
    run(hd, nh, nkv, S, pos0, f16=f16)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,n_sink,S,pos0", [(1, 1, 70, 200), (100, 130, 160, 400), (129, 3, 300, 0)])
def test_windows(hd, window, n_sink, S, pos0, f16):
    run(hd, 8, 2, S, pos0, window=window, n_sink=n_sink, f16=f16)


@pytest.mark.parametrize("f16", [False, True])
def test_rows_stored_before(f16):
    run(128, 8, 2, 145, 10, given=False, f16=f16)


@pytest.mark.parametrize("hd,nh,nkv,S,pos0", [(128, 32, 4, 1300, 0), (64, 16, 8, 900, 3000)])
def test_many_tokens(hd, nh, nkv, S, pos0):
    run(hd, nh, nkv, S, pos0, rows=S // 7)


def test_more_tokens_than_a_launch_takes():
    """At 2^24 positions a launch takes 2047 tokens of one KV head; under a window little of that is read."""
    rng = np.random.default_rng(9)
    hd, n, S, window = 64, 1 << 24, 5000, 100
    cache = tb.Kv4Cache(1, 1, hd, n)
    q, k, v = (randn(rng, (S, h, hd), torch.float32) for h in (2, 1, 1))
    got = cache.prefill(q.cuda(), k.cuda(), v.cuda(), pos0=n - S, window=window)
    cache.check()
    K, V = rowvals(k), rowvals(v)
    for i in [200, 2046, 2047, 2048, 4093, 4094, 4095] + list(range(150, S, 333)) + [S - 1]:
        lo = i + 1 - window
        want, *m = R.attend(q[i].double().numpy(), K[lo:i + 1], V[lo:i + 1], window - 1, 0, 0, hd ** -0.5)
        close(got[i], want, decode_tol("f32", want, *m), f"token {i}")


def test_a_prompt_in_pieces_has_the_same_precision():
    """As one call and cut into calls of 1, 4, 60 and the rest: both within f32's bound, and so within twice it of each other."""
    rng = np.random.default_rng(77)
    S, nh, nkv, hd = 200, 8, 2, 128
    q, k, v = (randn(rng, (S, n, hd), torch.float32) for n in (nh, nkv, nkv))
    one, many = tb.Kv4Cache(1, nkv, hd, S), tb.Kv4Cache(1, nkv, hd, S)
    a = one.prefill(q.cuda(), k.cuda(), v.cuda())
    cuts = [0, 1, 5, 65, S]
    b = torch.cat([many.prefill(q[i:j].cuda(), k[i:j].cuda(), v[i:j].cuda(), pos0=i) for i, j in zip(cuts, cuts[1:])])
    one.check()
    K, V = rowvals(k), rowvals(v)
    for i in range(S):
        want, *m = R.attend(q[i].double().numpy(), K, V, i, 0, 0, hd ** -0.5)
        for got in (a, b):
            close(got[i], want, decode_tol("f32", want, *m), f"token {i}")
