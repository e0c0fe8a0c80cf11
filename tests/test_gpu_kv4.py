"""The 4-bit KV cache (tetraeder_b200.Kv4Cache) against a plain implementation in 64 bits: rows in and out
bit for bit, single-token attention over ragged batches, windows with sinks, masked rows that hold anything,
and the refusals.

Tolerances, from the operations' roundings (vmax: the largest |v| seen, s: the largest |score|, a: the largest
scale * sum |q||k|):
  f32 decode   operands are exact or split to 22 bits and summed in f32, so an exponent is off by a few
               2^-24 * (s + a) and a weight by as much: 2^-20 * (4 + s + a) * vmax
  bf16 decode  the same, P rounded to f16 (2^-11 * vmax) and the output to bf16 (2^-8 * |out|, one bit of slack)
  prefill      Q, K, P and V rounded to f16: an exponent is off by 2^-11 * a each for Q and K, a weight by twice
               that, P and V by 2^-11 of the value; with bf16 the output's 2^-8 * |out|"""
import ctypes as C

import numpy as np
import pytest
import torch

import tetraeder_b200 as tb
from tests import kv4_ref as R
from tetraeder_b200 import _lib

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def randn(rng, shape, dtype, gain=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * gain).astype(np.float32)).to(dtype)


def fill(cache, rng, gain=1.0):
    """Every row of the cache from random values; returns the values K, V as numpy f64 [n_seq, n_kv, n_ctx, hd]."""
    out = []
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        n_seq, nkv, n, half = codes.shape
        c, d = R.quantize((rng.standard_normal((n_seq, nkv, n, 2 * half)) * gain).astype(np.float32))
        pos = np.arange(n)
        data = np.stack([np.stack([R.pack(c[s, g], pos) for g in range(nkv)]) for s in range(n_seq)])
        codes.copy_(torch.from_numpy(data))
        scales.copy_(torch.from_numpy(d))
        out.append(R.values(c, d))
    return out


def rowvals(x):
    """The values that the cache holds for rows x [n, nkv, hd]."""
    return R.values(*R.quantize(x.float().numpy()))


def close(got, want, tol, what=""):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), what
    err = np.abs(got - want)
    assert (err <= tol).all(), f"{what}: off by {err.max():.3e} where {np.broadcast_to(tol, err.shape)[err > tol].min():.3e} is allowed"


def decode_tol(dtype, want, smax, sabs, vmax):
    tol = 2.0 ** -20 * (4 + smax + sabs) * vmax
    return tol if dtype == "f32" else tol + 2.0 ** -11 * vmax + 2.0 ** -8 * np.abs(want)


def prefill_tol(dtype, want, smax, sabs, vmax):
    tol = (2.0 ** -20 * (4 + smax) + 4 * 2.0 ** -11 * sabs + 2 * 2.0 ** -11) * vmax
    return tol if dtype == "f32" else tol + 2.0 ** -8 * np.abs(want)


# ------------------------------------------------------------------ rows in and out
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nkv,n", [(128, 4, 1), (128, 3, 37), (64, 1, 65), (64, 8, 200)])
def test_store_and_load_match_the_plain_quantiser(dtype, hd, nkv, n):
    rng = np.random.default_rng(hd + nkv + n)
    cache = tb.Kv4Cache(3, nkv, hd, 500)
    assert cache.n_ctx == 512
    before = fill(cache, rng)
    k, v = randn(rng, (n, nkv, hd), DT[dtype], 2.0), randn(rng, (n, nkv, hd), DT[dtype], 0.01)
    places = rng.permutation(3 * 500)[:n]
    seq, pos = (places // 500).astype(np.int32), (places % 500).astype(np.int32)
    pos[n // 2] = -1 if n > 2 else pos[n // 2]  # no row
    cache.store(k.cuda(), v.cuda(), torch.from_numpy(pos).cuda(), seq=torch.from_numpy(seq).cuda())
    cache.check()
    for x, codes, scales, old in ((k, cache.k_codes, cache.k_scales, before[0]), (v, cache.v_codes, cache.v_scales, before[1])):
        c, d = R.quantize(x.float().numpy())
        got_c, got_d = codes.cpu().numpy(), scales.cpu().numpy()
        for i in range(n):
            if pos[i] < 0:
                continue
            for g in range(nkv):
                assert np.array_equal(got_c[seq[i], g, pos[i]], R.pack(c[i, g][None], pos[i:i + 1])[0])
                assert np.array_equal(got_d[seq[i], g, pos[i]], d[i, g])
        # nothing else changed
        now = np.stack([np.stack([R.values(R.unpack(got_c[s, g], np.arange(512)), got_d[s, g]) for g in range(nkv)]) for s in range(3)])
        for i in range(n):
            if pos[i] >= 0:
                now[seq[i], :, pos[i]] = old[seq[i], :, pos[i]]
        assert np.array_equal(now, old)
    kk, vv = cache.load(torch.from_numpy(pos).cuda(), seq=torch.from_numpy(seq).cuda())
    keep = (pos >= 0)[:, None, None]
    assert np.array_equal(kk.double().cpu().numpy(), rowvals(k) * keep)
    assert np.array_equal(vv.double().cpu().numpy(), rowvals(v) * keep)


@pytest.mark.parametrize("hd", [64, 128])
def test_store_run_of_positions_and_bf16_load(hd):
    rng = np.random.default_rng(hd)
    cache = tb.Kv4Cache(2, 2, hd, 192)
    wide = randn(rng, (101, 6, hd), torch.bfloat16)  # rows of a fused projection: q (2 heads), k, v
    k, v = wide[:, 2:4], wide[:, 4:6]
    cache.store(wide.cuda()[:, 2:4], wide.cuda()[:, 4:6], 77, seq=1)
    kk, vv = cache.load(77, n=101, seq=1, dtype=torch.bfloat16)
    assert torch.equal(kk.cpu(), torch.from_numpy(rowvals(k)).to(torch.bfloat16))
    assert torch.equal(vv.cpu(), torch.from_numpy(rowvals(v)).to(torch.bfloat16))
    assert not cache.k_codes[0].any() and not cache.k_scales[1, :, :77].any() and not cache.k_scales[1, :, 178:].any()
    each = randn(rng, (2, 2, hd), torch.float32)
    at = torch.tensor([5, 6], dtype=torch.int32, device="cuda")
    cache.store(each.cuda(), each.cuda(), at)  # row i of sequence i
    kk, _ = cache.load(at)
    assert np.array_equal(kk.double().cpu().numpy(), rowvals(each))
    cache.check()


def test_store_special_values():
    """Zeros, a tie of +a and -a, subnormals, a scale that rounds to zero, values beyond the scale's range, infinities, NaN."""
    big = np.finfo(np.float32).max
    x = np.zeros((1, 12, 128), np.float32)
    x[0, 1, :32] = np.linspace(-1, 1, 32)
    x[0, 2, 3], x[0, 2, 9] = 2.0, -2.0
    x[0, 3, :32] = 1e-40
    x[0, 4, :32] = np.linspace(-2.3e-7, 2.3e-7, 32)  # the scale is at the edge of f16's subnormals
    x[0, 5, :32] = np.linspace(-1e-3, 2e-3, 32)
    x[0, 6, :32] = np.linspace(-1e6, 1e6, 32)
    x[0, 7, 5], x[0, 7, 6], x[0, 7, 7] = np.inf, 1.0, -1e30
    x[0, 8, 5], x[0, 8, 6] = -np.inf, 3.0
    x[0, 9, :32], x[0, 9, 4] = 0.5, np.nan
    x[0, 10, :32] = np.nan
    x[0, 11, 31] = big
    cache = tb.Kv4Cache(1, 12, 128, 64)
    t = torch.from_numpy(x).cuda()
    cache.store(t, -t, 9, seq=0)
    k, v = cache.load(9, n=1, seq=0)
    assert np.array_equal(k.double().cpu().numpy(), R.values(*R.quantize(x)))
    assert np.array_equal(v.double().cpu().numpy(), R.values(*R.quantize(-x)))
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    cache.check()


def test_places_outside_the_cache_are_skipped_and_latched():
    cache = tb.Kv4Cache(2, 1, 64, 64)
    x = torch.ones((3, 1, 64), device="cuda")
    bad_pos = torch.tensor([64, 3, 4], dtype=torch.int32, device="cuda")
    bad_seq = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")
    cache.store(x, x, bad_pos, seq=bad_seq)
    with pytest.raises(tb.TmoeError, match="outside the 4-bit cache"):
        cache.check()
    assert int(cache.k_scales.count_nonzero()) == 2 and bool((cache.k_scales[1, 0, 4] != 0).all())
    k, _ = cache.load(bad_pos, seq=bad_seq)
    with pytest.raises(tb.TmoeError, match="outside the 4-bit cache"):
        cache.check()
    assert not k[:2].any() and bool((k[2] != 0).all())
    cache.check()


# ------------------------------------------------------------------ single tokens
def run_decode(dtype, hd, nh, nkv, pos, ctx, window=0, n_sink=0, gain=1.0, seed=0, given=True, scale=None, vgain=1.0):
    rng = np.random.default_rng(seed + hd + nh + ctx)
    B = len(pos)
    cache = tb.Kv4Cache(B, nkv, hd, ctx)
    K, V = fill(cache, rng, 1.0)
    cache.v_scales.mul_(vgain)
    V = V * 0 if vgain == 0 else V
    if vgain not in (0, 1.0):
        V = np.stack([np.stack([R.values(R.unpack(cache.v_codes[s, g].cpu().numpy(), np.arange(cache.n_ctx)),
                                         cache.v_scales[s, g].cpu().numpy()) for g in range(nkv)]) for s in range(B)])
    q = randn(rng, (B, nh, hd), DT[dtype], gain)
    k, v = randn(rng, (B, nkv, hd), DT[dtype]), randn(rng, (B, nkv, hd), DT[dtype], vgain)
    # what no query may see holds anything: rows past each position get NaN and infinite scales
    for b, p in enumerate(pos):
        cache.k_scales[b, :, max(p + 1, 0):] = float("nan")
        cache.v_scales[b, :, max(p + 1, 0):] = float("inf")
        if window and p + 1 - window > n_sink:
            cache.k_scales[b, :, n_sink:p + 1 - window] = float("inf")
            cache.v_scales[b, :, n_sink:p + 1 - window] = float("nan")
    dpos = torch.tensor(pos, dtype=torch.int32, device="cuda")
    if given:
        got = cache.decode(q.cuda(), k.cuda(), v.cuda(), dpos, window=window, n_sink=n_sink, scale=scale)
    else:
        cache.store(k.cuda(), v.cuda(), dpos)
        got = cache.decode(q.cuda(), None, None, dpos, window=window, n_sink=n_sink, scale=scale)
    cache.check()
    kn, vn = rowvals(k), rowvals(v)
    kk, vv = cache.load(dpos)
    assert got.dtype == DT[dtype]
    for b, p in enumerate(pos):
        if p < 0:
            assert not got[b].any() and not kk[b].any()
            continue
        K[b, :, p], V[b, :, p] = kn[b], vn[b]
        assert np.array_equal(kk[b].double().cpu().numpy(), kn[b]) and np.array_equal(vv[b].double().cpu().numpy(), vn[b])
        want, smax, sabs, vmax = R.attend(q[b].double().numpy(), K[b].transpose(1, 0, 2), V[b].transpose(1, 0, 2), p,
                                          window, n_sink, hd ** -0.5 if scale is None else scale)
        close(got[b], want, decode_tol(dtype, want, smax, sabs, vmax), f"sequence {b} at {p}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv", [(128, 32, 4), (128, 5, 5), (128, 14, 2), (64, 16, 1), (64, 6, 2), (128, 40, 2)])
def test_decode_lengths(dtype, hd, nh, nkv):
    run_decode(dtype, hd, nh, nkv, [0, 1, 30, 31, 32, 33, 63, 64, 100, -1, 255, 256, 299], 300)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,pos,ctx", [(128, 32, 4, [5000], 5001), (128, 8, 8, [2047, 700, 1100], 2048),
                                               (64, 8, 1, [4095, 0, 4094], 4096), (128, 2, 1, [9999], 10000)])
def test_decode_long_contexts_split_over_ctas(dtype, hd, nh, nkv, pos, ctx):
    run_decode(dtype, hd, nh, nkv, pos, ctx)


@pytest.mark.parametrize("dtype,hd", [("f32", 128), ("bf16", 128), ("bf16", 64)])
@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (7, 4), (32, 0), (33, 31), (64, 33), (100, 250), (1000, 3), (250, 1000)])
def test_decode_window_and_sinks(dtype, hd, window, n_sink):
    run_decode(dtype, hd, 8, 2, [0, 6, 7, 31, 32, 40, 64, 99, 100, 131, 200, 350, 399], 400, window=window, n_sink=n_sink)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decode_rows_stored_before(dtype):
    run_decode(dtype, 128, 16, 2, [50, 0, 127], 128, given=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gain,vgain,scale", [(30.0, 1.0, None), (1e-3, 1e-4, None), (1e-30, 1.0, 1e30), (1e30, 300.0, 1e-30),
                                              (0.0, 1.0, None), (1.0, 0, None), (1.0, 2e-5, 0.5)])
def test_decode_magnitudes(dtype, gain, vgain, scale):
    """Peaked and flat softmaxes, queries far from 1, V scales down to f16's subnormals and none at all."""
    run_decode(dtype, 128, 8, 1, [700, 64], 768, gain=gain, vgain=vgain, scale=scale)


@pytest.mark.parametrize("B", [257, 600])
def test_decode_many_sequences(B):
    rng = np.random.default_rng(B)
    pos = rng.integers(-1, 60, B).tolist()
    pos[0], pos[-1] = 59, 59
    run_decode("bf16", 64, 2, 1, pos, 60)


def test_decode_strided_activations_and_output():
    rng = np.random.default_rng(3)
    B, nh, nkv, hd = 3, 8, 2, 128
    cache = tb.Kv4Cache(B, nkv, hd, 128)
    K, V = fill(cache, rng)
    fused = randn(rng, (B, nh + 2 * nkv + 1, hd), torch.bfloat16)
    d = fused.cuda()
    out = torch.full((B, nh + 3, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    pos = [90, 3, 64]
    got = cache.decode(d[:, :nh], d[:, nh:nh + nkv], d[:, nh + nkv:nh + 2 * nkv], torch.tensor(pos, dtype=torch.int32, device="cuda"),
                       out=out[:, 1:nh + 1])
    cache.check()
    assert got.data_ptr() == out[:, 1:].data_ptr()
    assert bool((out[:, 0] == 7).all()) and bool((out[:, nh + 1:] == 7).all())
    for b, p in enumerate(pos):
        K[b, :, p], V[b, :, p] = rowvals(fused[:, nh:nh + nkv])[b], rowvals(fused[:, nh + nkv:nh + 2 * nkv])[b]
        want, *m = R.attend(fused[b, :nh].double().numpy(), K[b].transpose(1, 0, 2), V[b].transpose(1, 0, 2), p, 0, 0, hd ** -0.5)
        close(out[b, 1:nh + 1], want, decode_tol("bf16", want, *m))


def test_decode_positions_outside_the_cache():
    cache = tb.Kv4Cache(2, 1, 64, 64)
    x = torch.ones((2, 1, 64), device="cuda")
    out = cache.decode(x, x, x, torch.tensor([64, 3], dtype=torch.int32, device="cuda"))
    with pytest.raises(tb.TmoeError, match="outside the 4-bit cache"):
        cache.check()
    assert not out[0].any() and bool((out[1] != 0).all())
    assert int(cache.k_scales.count_nonzero()) == 2
    cache.check()


def test_decode_nan_query_stays_in_its_head():
    rng = np.random.default_rng(8)
    cache = tb.Kv4Cache(2, 1, 128, 1024)
    fill(cache, rng)
    q = randn(rng, (2, 8, 128), torch.float32).cuda()
    pos = torch.tensor([1000, 1000], dtype=torch.int32, device="cuda")
    want = cache.decode(q, None, None, pos).clone()
    q[0, 3, 5] = float("nan")
    got = cache.decode(q, None, None, pos)
    cache.check()
    assert torch.isnan(got[0, 3]).all()
    keep = torch.ones((2, 8), dtype=torch.bool)
    keep[0, 3] = False
    assert torch.equal(got[keep.cuda()], want[keep.cuda()])


def test_decode_same_bits_every_call_on_a_side_stream_and_from_a_graph():
    rng = np.random.default_rng(5)
    B, nh, nkv, hd, ctx = 4, 16, 2, 128, 3000
    cache = tb.Kv4Cache(B, nkv, hd, ctx)
    fill(cache, rng)
    q, k, v = (randn(rng, (B, n, hd), torch.bfloat16).cuda() for n in (nh, nkv, nkv))
    pos = torch.tensor([2999, 17, 1500, 800], dtype=torch.int32, device="cuda")
    want = cache.decode(q, k, v, pos).clone()
    for _ in range(20):
        assert torch.equal(cache.decode(q, k, v, pos), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = torch.empty_like(want)
    cache.decode(q, k, v, pos, out=got, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.decode(q, k, v, pos, out=got)
    got.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    pos.copy_(torch.tensor([10, 2999, 5, 2000], dtype=torch.int32))  # the graph takes the positions of the replay
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, cache.decode(q, k, v, pos))
    cache.check()
    del g


def test_rows_past_32_bit_offsets():
    """Planes of over 4 GiB: the last sequence's rows, stored, read back and attended to."""
    n_seq, nkv, hd, ctx = 20, 8, 128, 1 << 19
    cache = tb.Kv4Cache(n_seq, nkv, hd, ctx)
    assert cache.k_codes.numel() > 1 << 32
    rng = np.random.default_rng(2)
    n = 70
    k, v = randn(rng, (n, nkv, hd), torch.float32), randn(rng, (n, nkv, hd), torch.float32)
    cache.store(k.cuda(), v.cuda(), ctx - n, seq=n_seq - 1)
    kk, vv = cache.load(ctx - n, n=n, seq=n_seq - 1)
    assert np.array_equal(kk.double().cpu().numpy(), rowvals(k)) and np.array_equal(vv.double().cpu().numpy(), rowvals(v))
    pos = torch.full((n_seq,), -1, dtype=torch.int32, device="cuda")
    pos[-1] = ctx - 1
    q = randn(rng, (n_seq, nkv, hd), torch.float32)
    new = randn(rng, (n_seq, nkv, hd), torch.float32)
    got = cache.decode(q.cuda(), new.cuda(), new.cuda(), pos, window=n)
    cache.check()
    K, V = rowvals(k), rowvals(v)
    K[-1] = V[-1] = rowvals(new)[-1]
    want, *m = R.attend(q[-1].double().numpy(), K, V, n - 1, 0, 0, hd ** -0.5)
    close(got[-1], want, decode_tol("f32", want, *m))
    assert not got[:-1].any()


# ------------------------------------------------------------------ many tokens of one sequence
def run_prefill(dtype, hd, nh, nkv, S, pos0, window=0, n_sink=0, gain=1.0, given=True, seed=0, seq=1, rows=None):
    rng = np.random.default_rng(seed + hd + nh + S)
    ctx = pos0 + S + 3
    cache = tb.Kv4Cache(2, nkv, hd, ctx)
    K, V = fill(cache, rng)
    K, V = K[seq], V[seq]
    other = [t[1 - seq].clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    cache.k_scales[seq, :, pos0 + S:] = float("nan")
    cache.v_scales[seq, :, pos0 + S:] = float("inf")
    if window and pos0 + 1 - window > n_sink:  # before the first query's window
        cache.k_scales[seq, :, n_sink:pos0 + 1 - window] = float("inf")
        cache.v_scales[seq, :, n_sink:pos0 + 1 - window] = float("nan")
    q = randn(rng, (S, nh, hd), DT[dtype], gain)
    k, v = randn(rng, (S, nkv, hd), DT[dtype]), randn(rng, (S, nkv, hd), DT[dtype])
    if given:
        got = cache.prefill(q.cuda(), k.cuda(), v.cuda(), seq=seq, pos0=pos0, window=window, n_sink=n_sink)
    else:
        cache.store(k.cuda(), v.cuda(), pos0, seq=seq)
        got = cache.prefill(q.cuda(), None, None, seq=seq, pos0=pos0, window=window, n_sink=n_sink)
    cache.check()
    K[:, pos0:pos0 + S], V[:, pos0:pos0 + S] = rowvals(k).transpose(1, 0, 2), rowvals(v).transpose(1, 0, 2)
    kk, vv = cache.load(pos0, n=S, seq=seq)
    assert np.array_equal(kk.double().cpu().numpy(), rowvals(k)) and np.array_equal(vv.double().cpu().numpy(), rowvals(v))
    for t, old in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), other):
        assert torch.equal(t[1 - seq], old)
    Kt, Vt = K.transpose(1, 0, 2), V.transpose(1, 0, 2)
    for i in range(S) if rows is None else rows:
        want, *m = R.attend(q[i].double().numpy(), Kt, Vt, pos0 + i, window, n_sink, hd ** -0.5)
        close(got[i], want, prefill_tol(dtype, want, *m), f"token {i}")
    assert got.dtype == DT[dtype] and bool(torch.isfinite(got.float()).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,S,pos0", [(128, 32, 4, 1, 0), (128, 32, 4, 1, 300), (128, 8, 1, 33, 0), (128, 8, 2, 64, 64),
                                              (64, 6, 2, 50, 77), (128, 5, 5, 129, 0), (128, 14, 2, 40, 129), (64, 16, 1, 31, 1)])
def test_prefill_shapes(dtype, hd, nh, nkv, S, pos0):
    run_prefill(dtype, hd, nh, nkv, S, pos0)


@pytest.mark.parametrize("hd,nh,nkv,S,pos0", [(128, 32, 4, 300, 500), (64, 8, 2, 700, 0), (128, 4, 4, 513, 1000), (128, 32, 2, 257, 255)])
def test_prefill_long(hd, nh, nkv, S, pos0):
    run_prefill("bf16", hd, nh, nkv, S, pos0, rows=sorted({0, 1, S // 3, S // 2, S - 2, S - 1} | set(range(0, S, 37))))


# More rows than the decode kernel is given: a block with rows in one tile only, a last block of a few rows, odd groups
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv,S,pos0", [(128, 8, 1, 130, 0), (64, 16, 1, 140, 1), (128, 14, 2, 90, 129), (64, 6, 3, 50, 77),
                                              (128, 5, 5, 27, 4000), (128, 1, 1, 257, 63), (64, 48, 2, 65, 191)])
def test_prefill_blocks(dtype, hd, nh, nkv, S, pos0):
    run_prefill(dtype, hd, nh, nkv, S, pos0, rows=sorted({0, 1, S // 2, S - 2, S - 1} | set(range(0, S, 13))))


# How the blocks are shared out: few ones cut into many pieces, many ones cut where their number does not divide, all whole and
# more of them than SMs, a cut inside a block with rows in one tile only, and the same under a window
@pytest.mark.parametrize("hd,nh,nkv,S,pos0,window,n_sink", [
    (128, 8, 1, 33, 12000, 0, 0), (64, 4, 1, 40, 30000, 0, 0), (128, 16, 2, 130, 9001, 0, 0), (128, 32, 8, 1240, 5000, 0, 0),
    (128, 32, 4, 1300, 0, 0, 0), (64, 16, 8, 2900, 0, 0, 0), (128, 40, 8, 1200, 6000, 4096, 4), (64, 8, 8, 260, 20000, 9000, 200)])
def test_prefill_shares(hd, nh, nkv, S, pos0, window, n_sink):
    run_prefill("bf16", hd, nh, nkv, S, pos0, window=window, n_sink=n_sink, rows=sorted({0, 1, S // 3, S // 2, S - 2, S - 1} |
                                                                                        set(range(0, S, S // 7))))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd,nh,nkv", [(128, 32, 4), (64, 16, 16), (128, 24, 2)])
@pytest.mark.parametrize("S", [2, 3, 4, 5, 9])
def test_prefill_few_tokens(dtype, hd, nh, nkv, S):
    run_prefill(dtype, hd, nh, nkv, S, 3001)
    run_prefill(dtype, hd, nh, nkv, S, 130, window=64, n_sink=3)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window,n_sink,S,pos0", [(1, 0, 70, 0), (1, 1, 70, 200), (16, 4, 150, 300), (128, 0, 140, 128), (100, 130, 60, 400),
                                                  (129, 3, 300, 0), (5, 300, 40, 500), (1000, 2, 64, 64)])
def test_prefill_window_and_sinks(hd, window, n_sink, S, pos0):
    run_prefill("bf16", hd, 4, 2, S, pos0, window=window, n_sink=n_sink)


@pytest.mark.parametrize("gain", [0.0, 20.0])
def test_prefill_flat_and_peaked(gain):
    run_prefill("bf16", 128, 8, 2, 100, 60, gain=gain)


def test_prefill_nan_query_stays_in_its_row():
    rng = np.random.default_rng(12)
    S, nh, nkv, hd, pos0 = 200, 8, 1, 128, 500
    cache = tb.Kv4Cache(1, nkv, hd, pos0 + S)
    K, V = fill(cache, rng)
    q = randn(rng, (S, nh, hd), torch.bfloat16)
    poisoned = q.clone()
    poisoned[77, 3, 5] = float("nan")
    poisoned[150, 6] = float("inf")
    got = cache.prefill(poisoned.cuda(), None, None, pos0=pos0)
    cache.check()
    assert bool(got[77, 3].isnan().any())
    Kt, Vt = K[0].transpose(1, 0, 2), V[0].transpose(1, 0, 2)
    for i in (0, 76, 77, 78, 150, 199):
        want, *m = R.attend(q[i].double().numpy(), Kt, Vt, pos0 + i, 0, 0, hd ** -0.5)
        tol = prefill_tol("bf16", want, *m)
        for h in range(nh):
            if (i, h) not in ((77, 3), (150, 6)):
                close(got[i, h], want[h], tol[h] if np.ndim(tol) else tol, f"token {i} head {h}")


def test_prefill_rows_stored_before():
    run_prefill("bf16", 128, 8, 2, 45, 10, given=False)


def test_chunked_prefill_equals_one_prefill():
    """The same tokens as one run and as three: the cache's rows are the same, the outputs within the roundings."""
    rng = np.random.default_rng(1)
    S, nh, nkv, hd = 333, 8, 2, 128
    q, k, v = (randn(rng, (S, n, hd), torch.bfloat16).cuda() for n in (nh, nkv, nkv))
    one, many = tb.Kv4Cache(1, nkv, hd, S), tb.Kv4Cache(1, nkv, hd, S)
    a = one.prefill(q, k, v)
    cuts = [0, 1, 130, S]
    b = torch.cat([many.prefill(q[i:j], k[i:j], v[i:j], pos0=i) for i, j in zip(cuts, cuts[1:])])
    one.check()
    assert torch.equal(one.k_codes, many.k_codes) and torch.equal(one.v_scales, many.v_scales)
    assert float((a.float() - b.float()).abs().max()) < 2.0 ** -6


def test_prefill_same_bits_every_call():
    rng = np.random.default_rng(6)
    cache = tb.Kv4Cache(1, 2, 128, 2500)
    fill(cache, rng)
    q, k, v = (randn(rng, (40, n, 128), torch.bfloat16).cuda() for n in (16, 2, 2))
    want = cache.prefill(q, k, v, pos0=2400).clone()
    for _ in range(10):
        assert torch.equal(cache.prefill(q, k, v, pos0=2400), want)
    cache.check()


# ------------------------------------------------------------------ refusals
def test_refusals():
    cache = tb.Kv4Cache(2, 2, 128, 64)
    dev = "cuda"
    q, k = torch.zeros((2, 4, 128), device=dev), torch.zeros((2, 2, 128), device=dev)
    pos = torch.zeros(2, dtype=torch.int32, device=dev)
    bad = [
        lambda: cache.decode(q, k, None, pos),
        lambda: cache.decode(q, k, k.bfloat16(), pos),
        lambda: cache.decode(q.half(), k.half(), k.half(), pos),
        lambda: cache.decode(q, k, k, pos.long()),
        lambda: cache.decode(q, k, k, pos[:1]),
        lambda: cache.decode(q[:, :, :64], k, k, pos),
        lambda: cache.decode(q, k[:, :1], k[:, :1], pos),
        lambda: cache.decode(q, k.cpu(), k, pos),
        lambda: cache.decode(q.transpose(0, 1)[:2], k, k, pos),
        lambda: cache.store(k, k, pos, seq=2),
        lambda: cache.store(k, k[:1], pos),
        lambda: cache.store(k, k, 0),  # which sequence?
        lambda: cache.load(0, n=1),
        lambda: cache.load(0, seq=0),
        lambda: cache.load(0, n=1, seq=0, dtype=torch.float16),
        lambda: tb.Kv4Cache(1, 1, 96, 64),
        lambda: tb.Kv4Cache(0, 1, 128, 64),
        lambda: tb.Kv4Cache.from_planes(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales[:1]),
        lambda: tb.Kv4Cache.from_planes(cache.k_codes.cpu(), cache.k_scales, cache.v_codes, cache.v_scales),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    refused = [
        lambda: cache.decode(q[:, :3], k, k, pos),                     # 3 heads over 2 KV heads
        lambda: cache.decode(q, k, k, pos, window=-1),
        lambda: cache.decode(q, k, k, pos, n_sink=-1),
        lambda: cache.decode(q, k, k, pos, scale=0.0),
        lambda: cache.decode(q, k, k, pos, scale=float("nan")),
        lambda: cache.decode(torch.zeros((3, 4, 128), device=dev), None, None, torch.zeros(3, dtype=torch.int32, device=dev)),
        lambda: cache.prefill(q, k, k, seq=2),
        lambda: cache.prefill(q, k, k, seq=-1),
        lambda: cache.prefill(q, k, k, pos0=63),
        lambda: cache.prefill(q, k, k, pos0=-1),
        lambda: cache.store(k, k, 63, seq=0),
        lambda: cache.store(k, k, -1, seq=0),
        lambda: cache.load(60, n=5, seq=0),
        lambda: cache.store(torch.zeros((3, 2, 128), device=dev), torch.zeros((3, 2, 128), device=dev),
                            torch.zeros(3, dtype=torch.int32, device=dev)),  # 3 sequences of 2
    ]
    for f in refused:
        with pytest.raises(tb.TmoeError, match="TMOE_E_INVALID"):
            f()
    flat = torch.zeros(2000, device=dev)
    with pytest.raises(tb.TmoeError, match="16-byte"):  # a base that is not 16-byte aligned
        cache.store(flat[1:257].view(1, 2, 128), flat[1:257].view(1, 2, 128), 0, seq=0)
    x = torch.as_strided(flat, (2, 2, 128), (257, 128, 1))  # rows 257 floats apart
    with pytest.raises(tb.TmoeError, match="16-byte"):
        cache.store(x, x, 0, seq=0)
    assert not cache.k_codes.any() and not cache.v_scales.any()
    # empty calls are calls
    cache.store(k[:0], k[:0], 0, seq=0)
    assert cache.load(0, n=0, seq=0)[0].shape == (0, 2, 128)
    assert cache.decode(q[:0], k[:0], k[:0], pos[:0]).shape == (0, 4, 128)
    assert cache.prefill(q[:0], k[:0], k[:0]).shape == (0, 4, 128)
    cache.check()


def test_c_refusals():
    """The C entry points' own checks, as a caller without the class meets them."""
    cache = tb.Kv4Cache(2, 2, 128, 64)
    lib, h = cache.lib, cache.h
    k = torch.zeros((2, 2, 128), device="cuda")
    P = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    c = _lib.Kv4CacheStruct.from_buffer_copy(cache._c)

    def store(struct=c, ty=0, kk=k, ld=256, n=2, seq0=0, pos0=0, handle=h):
        return lib.tmoe_kv4_store(handle, None, C.byref(struct) if struct is not None else None, ty, P(kk) if kk is not None else None,
                                  P(k), ld, None, seq0, None, pos0, n)

    assert store() == 0
    assert store(handle=None) == _lib.TMOE_E_INVALID
    assert store(struct=None) == _lib.TMOE_E_INVALID
    assert store(ty=1) == _lib.TMOE_E_UNSUPPORTED
    assert store(kk=None) == _lib.TMOE_E_INVALID
    assert store(ld=255) == _lib.TMOE_E_INVALID
    assert store(n=-1) == _lib.TMOE_E_INVALID
    assert store(n=1 << 40) == _lib.TMOE_E_INVALID
    for field, value, code in (("head_dim", 96, _lib.TMOE_E_UNSUPPORTED), ("n_ctx", 63, _lib.TMOE_E_INVALID),
                               ("n_ctx", 0, _lib.TMOE_E_INVALID), ("n_seq", 0, _lib.TMOE_E_INVALID),
                               ("n_kv", -2, _lib.TMOE_E_INVALID), ("k_codes", None, _lib.TMOE_E_INVALID),
                               ("v_scales", cache.v_scales.data_ptr() + 2, _lib.TMOE_E_INVALID)):
        bad = _lib.Kv4CacheStruct.from_buffer_copy(cache._c)
        setattr(bad, field, value)
        assert store(struct=bad) == code, field
    a = _lib.Kv4AttnStruct()
    q = torch.zeros((2, 4, 128), device="cuda")
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    a.q, a.out, a.scratch = q.data_ptr(), q.data_ptr(), cache._scratch.data_ptr()
    a.q_ld = a.out_ld = 512
    a.n_head, a.scale = 4, 1.0

    def decode(attn=a, B=2, p=pos):
        return lib.tmoe_kv4_attn_decode(h, None, C.byref(c), C.byref(attn) if attn is not None else None, P(p) if p is not None else None, B)

    assert decode() == 0
    assert decode(attn=None) == _lib.TMOE_E_INVALID
    assert decode(B=3) == _lib.TMOE_E_INVALID
    assert decode(B=-1) == _lib.TMOE_E_INVALID
    assert decode(p=None) == _lib.TMOE_E_INVALID
    for field, value, code in (("type", 1, _lib.TMOE_E_UNSUPPORTED), ("q", None, _lib.TMOE_E_INVALID), ("out", None, _lib.TMOE_E_INVALID),
                               ("scratch", None, _lib.TMOE_E_INVALID), ("q_ld", 511, _lib.TMOE_E_INVALID), ("q_ld", 513, _lib.TMOE_E_INVALID),
                               ("out_ld", 0, _lib.TMOE_E_INVALID), ("k", k.data_ptr(), _lib.TMOE_E_INVALID), ("n_head", 0, _lib.TMOE_E_INVALID),
                               ("window", -5, _lib.TMOE_E_INVALID)):
        bad = _lib.Kv4AttnStruct.from_buffer_copy(a)
        setattr(bad, field, value)
        assert decode(attn=bad) == code, field
    cache.check()
