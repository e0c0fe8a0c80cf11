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


# ------------------------------------------------------------------ values beyond f16's range
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,S,pos0,window,n_sink", [(128, 8, 1, 70, 300, 0, 0), (64, 8, 2, 150, 129, 0, 0), (128, 16, 2, 300, 500, 200, 3)])
@pytest.mark.parametrize("what", ["k", "v", "kv"])
def test_prefill_of_values_beyond_f16(dtype, hd, nh, nkv, S, pos0, window, n_sink, what):
    """Rows of up to 5e5 among ordinary ones, in one block (V) or in all (K, whose queries are then small): what the scale can hold,
    8 times f16's range, in some tiles and not in others."""
    rng = np.random.default_rng(hd + S + pos0)
    n = pos0 + S
    cache = tb.Kv4Cache(2, nkv, hd, n)
    q = randn(rng, (S, nh, hd), DT[dtype], 1e-5 if "k" in what else 1.0)
    k, v = randn(rng, (n, nkv, hd), DT[dtype]), randn(rng, (n, nkv, hd), DT[dtype])
    some = np.r_[0:n:97, pos0 + S // 2]
    if "k" in what:
        k[some] *= 1e5
    if "v" in what:
        v[some, :, 32:64] *= 1.3e5
    cache.store(k[:pos0].cuda(), v[:pos0].cuda(), 0, seq=1)
    got = cache.prefill(q.cuda(), k[pos0:].cuda(), v[pos0:].cuda(), seq=1, pos0=pos0, window=window, n_sink=n_sink)
    cache.check()
    K, V = rowvals(k), rowvals(v)
    assert max(np.abs(K).max(), np.abs(V).max()) > 2e5
    for i in sorted({0, 1, S // 2, S - 1} | set(range(0, S, 17))):
        want, smax, sabs, _ = R.attend(q[i].double().numpy(), K, V, pos0 + i, window, n_sink, hd ** -0.5)
        tol = prefill_block_tol(dtype, want, smax, sabs, block_max(V, seen(n, pos0 + i, window, n_sink), nh // nkv))
        close(got[i], want, tol, f"token {i}")


@pytest.mark.parametrize("hd,nh,nkv,S,pos0", [(128, 8, 1, 33, 12000), (64, 16, 2, 300, 9000), (128, 32, 8, 1240, 0)])
def test_prefill_of_a_few_values_beyond_f16(hd, nh, nkv, S, pos0):
    """One row of K and one of V, which few of the CTAs that share the work meet; the parts of a cut block are joined."""
    rng = np.random.default_rng(hd + S)
    n = pos0 + S
    cache = tb.Kv4Cache(1, nkv, hd, n)
    q = randn(rng, (S, nh, hd), torch.bfloat16)
    k, v = randn(rng, (n, nkv, hd), torch.bfloat16), randn(rng, (n, nkv, hd), torch.bfloat16)
    v[n // 3, :, :32] *= 1.3e5
    k[n // 2, :, 5] = 3e5
    q[:, :, 5] = 1e-5
    cache.store(k.cuda(), v.cuda(), 0, seq=0)
    got = cache.prefill(q.cuda(), None, None, pos0=pos0)
    assert torch.equal(cache.prefill(q.cuda(), None, None, pos0=pos0), got)
    cache.check()
    K, V = rowvals(k), rowvals(v)
    for i in sorted({0, 1, S // 2, S - 1, min(S - 1, n // 3), min(S - 1, n // 2)}):
        want, smax, sabs, _ = R.attend(q[i].double().numpy(), K, V, pos0 + i, 0, 0, hd ** -0.5)
        close(got[i], want, prefill_block_tol("bf16", want, smax, sabs, block_max(V, slice(0, pos0 + i + 1), nh // nkv)), f"token {i}")


@pytest.mark.parametrize("junk", [float("inf"), float("nan"), 65504.0])
def test_prefill_is_the_same_whatever_unseen_rows_hold(junk):
    rng = np.random.default_rng(4)
    S, nh, nkv, hd, pos0, window = 150, 8, 1, 128, 700, 100
    cache = tb.Kv4Cache(1, nkv, hd, pos0 + S + 50)
    fill(cache, rng)
    q = randn(rng, (S, nh, hd), torch.bfloat16).cuda()
    want = cache.prefill(q, None, None, pos0=pos0, window=window, n_sink=2).clone()
    for scales in (cache.k_scales, cache.v_scales):
        scales[0, :, 2:pos0 + 1 - window] = junk
        scales[0, :, pos0 + S:] = junk
    assert torch.equal(cache.prefill(q, None, None, pos0=pos0, window=window, n_sink=2), want)
    cache.check()
