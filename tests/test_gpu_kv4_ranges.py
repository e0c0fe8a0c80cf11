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
