"""Decode steps of serving batches over the 4-bit KV cache with 128-wide heads: more (sequence, KV head) segments than SMs, short
ones (two small CTAs a SM) and ones past 128 tiles of 64 positions (one CTA), against 64 bits (tolerances: test_gpu_kv4.py)."""
import numpy as np
import pytest
import torch

import tetraeder_b200 as tb
from tests import kv4_ref as R
from tests.test_gpu_kv4 import DT, close, decode_tol, randn, rowvals

pytestmark = pytest.mark.gpu

EDGES = [0, 1, 62, 63, 64, 65, 127, 128, 191, 192]  # around the 64-position tiles


def run(dtype, nh, nkv, pos, ctx, window=0, n_sink=0, check=None, seed=0):
    """One step over planes of random codes and scales; sequences `check` (all) are compared."""
    rng = np.random.default_rng(seed + nh + len(pos) + ctx)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed + ctx)
    B, hd = len(pos), 128
    cache = tb.Kv4Cache(B, nkv, hd, ctx)
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        codes.random_(0, 256, generator=gen)
        scales.normal_(0.0, 0.2, generator=gen)
    old = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    q, k, v = (randn(rng, (B, n, hd), DT[dtype]) for n in (nh, nkv, nkv))
    dpos = torch.tensor(pos, dtype=torch.int32, device="cuda")
    args = (q.cuda(), k.cuda(), v.cuda(), dpos)
    got = cache.decode(*args, window=window, n_sink=n_sink)
    for _ in range(3):  # the rows are there already: the same bits
        assert torch.equal(cache.decode(*args, window=window, n_sink=n_sink), got)
    cache.check()
    kn, vn = rowvals(k), rowvals(v)
    kk, vv = cache.load(dpos)
    live = torch.tensor([p >= 0 for p in pos])
    assert np.array_equal(kk.double().cpu().numpy()[live], kn[live]) and np.array_equal(vv.double().cpu().numpy()[live], vn[live])
    # nothing but the new rows has changed
    for t, o in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), old):
        for b, p in enumerate(pos):
            if p >= 0:
                o[b, :, p] = t[b, :, p]
        assert torch.equal(t, o)
    assert not got[~live.cuda()].any()
    for b in range(B) if check is None else check:
        p = pos[b]
        if p < 0:
            continue
        at = np.arange(p + 1)
        K, V = (np.stack([R.values(R.unpack(c[b, g, :p + 1].cpu().numpy(), at), s[b, g, :p + 1].cpu().numpy()) for g in range(nkv)], 1)
                for c, s in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)))
        want, *m = R.attend(q[b].double().numpy(), K, V, p, window, n_sink, hd ** -0.5)
        close(got[b], want, decode_tol(dtype, want, *m), f"sequence {b} at {p}")


def ragged(rng, B, ctx, idle):
    pos = rng.integers(0, ctx, B)
    pos[:len(EDGES)] = np.minimum(EDGES, ctx - 1)
    pos[-1] = ctx - 1
    pos[rng.permutation(np.arange(len(EDGES), B - 1))[:idle]] = -1
    return pos.tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,nh,nkv,ctx,idle", [(48, 32, 4, 700, 3), (160, 32, 4, 300, 0), (160, 8, 4, 200, 40), (40, 40, 4, 260, 1),
                                               (300, 2, 1, 100, 7), (64, 64, 8, 450, 2)])
def test_more_segments_than_sms(dtype, B, nh, nkv, ctx, idle):
    run(dtype, nh, nkv, ragged(np.random.default_rng(B), B, ctx, idle), ctx)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (64, 4), (200, 65), (130, 0)])
def test_more_segments_than_sms_under_a_window(dtype, window, n_sink):
    run(dtype, 20, 4, ragged(np.random.default_rng(window), 48, 600, 4), 600, window=window, n_sink=n_sink)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ctx,window", [(8192, 0), (8256, 0), (16384, 8000), (16384, 9000)])
def test_either_side_of_128_tiles(dtype, ctx, window):
    rng = np.random.default_rng(ctx + window)
    pos = ragged(rng, 80, ctx, 2)
    run(dtype, 16, 1, [p if p < 0 else max(p, ctx // 2) if i % 3 else p for i, p in enumerate(pos)], ctx, window=window,
        n_sink=3 if window else 0, check=[0, 3, 9, 11, 30, 79])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_capacity_well_above_the_lengths(dtype):
    run(dtype, 32, 4, ragged(np.random.default_rng(3), 64, 500, 2), 20000)
