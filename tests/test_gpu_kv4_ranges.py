"""The 4-bit KV cache's attention at the ends of its values' ranges, against 64 bits (kv4_ref.py).

Tolerances are those of test_gpu_kv4.py, but held block by block of 32 dimensions: an output dimension is a weighted mean of V's
values in it, so a rounding of a weight or of a value is relative to the largest |v| of that dimension's own block, whatever
the other blocks hold.  bf16 decode rounds P to f16 and its product with V's scale to f16 again: 2 * 2^-11 of it."""
import numpy as np
import pytest
import torch

import tetraeder_b200 as tb
from tests import kv4_ref as R
from tests.test_gpu_kv4 import DT, close, fill, randn, rowvals

pytestmark = pytest.mark.gpu


def block_max(V, keep, G):
    """The largest |v| seen by each head in each dimension's block: V [n, nkv, hd] -> [nkv * G, hd]."""
    m = np.abs(V[keep]).max(0)
    m = m.reshape(m.shape[0], -1, 32).max(-1).repeat(32, axis=-1)
    return m.repeat(G, axis=0)


def seen(n, last, window, n_sink):
    p = np.arange(n)
    return (p <= last) & ((window == 0) | (last - p < window) | (p < n_sink))


def decode_block_tol(dtype, want, smax, sabs, vblock):
    tol = 2.0 ** -20 * (4 + smax + sabs) * vblock
    return tol if dtype == "f32" else tol + 2 * 2.0 ** -11 * vblock + 2.0 ** -8 * np.abs(want)


def prefill_block_tol(dtype, want, smax, sabs, vblock):
    tol = (2.0 ** -20 * (4 + smax) + 4 * 2.0 ** -11 * sabs + 2 * 2.0 ** -11) * vblock
    return tol if dtype == "f32" else tol + 2.0 ** -8 * np.abs(want)


# ------------------------------------------------------------------ scores far from 1
def run_far(dtype, hd, tokens, gain, gain2=1.0):
    """The softmax takes the one position of the largest score alone, where the next one is further away than the scores' own
    relative error (2^-8 is allowed for it, Q and K in f16 the coarsest).  The output is that position's V, with the roundings of
    P and V (prefill, past 128 tokens here) or of P and its product (bf16 decode) to f16, 2^-11 each, and of the output to bf16,
    2^-8; f32 decode holds both to 22 bits, and 2^-20 covers its few roundings."""
    rng = np.random.default_rng(hd + tokens)
    nh, n = 8, 400
    cache = tb.Kv4Cache(1, 1, hd, n)
    K, V = (x[0, 0] for x in fill(cache, rng))
    q = (randn(rng, (tokens, nh, hd), torch.float32) * gain * gain2).to(DT[dtype])
    first = n - tokens
    if tokens == 1:
        got = cache.decode(q.cuda(), None, None, torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    else:
        got = cache.prefill(q.cuda(), None, None, pos0=first)
    cache.check()
    rel = 2.0 ** -20 if dtype == "f32" and tokens <= 128 else 2 * 2.0 ** -11 + (2.0 ** -8 if dtype == "bf16" else 0.0)
    checked = 0
    for t in range(tokens):
        s = q[t].double().numpy() @ K[:first + t + 1].T
        best = s.argmax(1)
        top2 = np.sort(s, axis=1)[:, -2:]
        for h in np.flatnonzero(top2[:, 1] - top2[:, 0] > 2.0 ** -8 * np.abs(q[t].double().numpy()).max(1) * np.abs(K).max()):
            close(got[t, h], V[best[h]], rel * np.abs(V[best[h]]), f"token {t} head {h}")
            checked += 1
    assert checked > tokens * nh // 2


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 70, 200])
@pytest.mark.parametrize("log2", [26, 32, 60, 100])
def test_scores_past_24_bits(dtype, hd, tokens, log2):
    """A score's last bit counts 1 and more."""
    run_far(dtype, hd, tokens, 2.0 ** log2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens", [1, 70, 200])
def test_queries_near_the_largest_float(dtype, hd, tokens):
    """Scores beyond 2^100 but within a float's range."""
    run_far(dtype, hd, tokens, 2.0 ** 60, 2.0 ** 61)


# ------------------------------------------------------------------ V blocks of very different scales
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv", [(128, 8, 1), (64, 6, 2), (128, 20, 2)])
@pytest.mark.parametrize("at,block", [(0, 0), (150, 1), (299, 0)])  # 299: the new row itself
def test_a_huge_value_block_leaves_the_others_alone(dtype, hd, nh, nkv, at, block):
    """An infinity is held as the scale's largest value; the row's other blocks and other rows' are around 0.01."""
    rng = np.random.default_rng(hd + nh + at)
    n = 300
    cache = tb.Kv4Cache(1, nkv, hd, n)
    q = randn(rng, (1, nh, hd), DT[dtype])
    k, v = randn(rng, (n, nkv, hd), DT[dtype]), randn(rng, (n, nkv, hd), DT[dtype], 0.01)
    v[at, :, 32 * block + 5] = float("inf")
    cache.store(k[:-1].cuda(), v[:-1].cuda(), 0, seq=0)
    got = cache.decode(q.cuda(), k[-1:].cuda(), v[-1:].cuda(), torch.tensor([n - 1], dtype=torch.int32, device="cuda"))
    cache.check()
    K, V = rowvals(k), rowvals(v)
    want, smax, sabs, _ = R.attend(q[0].double().numpy(), K, V, n - 1, 0, 0, hd ** -0.5)
    close(got[0], want, decode_block_tol(dtype, want, smax, sabs, block_max(V, slice(None), nh // nkv)))
