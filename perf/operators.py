"""Measured cases of the 4-bit KV cache and the attention over it.

Three kinds of pass, as a serving program makes them:
  store    quantises new K/V rows into the cache and reads the same rows back as values
  decode   one new token for each of B sequences: its K/V row goes into the cache and its query attends to the
           sequence's positions, all of them or a sliding window plus the first few (sinks)
  prefill  a run of S tokens of one sequence: rows stored, causal attention of every new token

The cache is four planes: codes uint8 [n_seq][n_kv][n_ctx][head_dim / 2] and scales float16
[n_seq][n_kv][n_ctx][head_dim / 32], for K and for V.  A block of 32 values holds d * (c - 8), d its scale and c
its 4-bit codes, the even element of a byte in the low half.  The 16-byte chunk of block c of the row at position p
sits at slot c ^ ((p >> 1) & 3) for 128-wide heads and c ^ ((p >> 2) & 1) for 64-wide ones.

`own` false: elementary torch operations in 32 bits.  `own` true: tetraeder_b200.Kv4Cache."""
import math

import numpy as np
import torch

own = False

F16_MAX = 65504.0
SLOTS = 64  # a cache holds a whole number of these positions per sequence and head


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the new rows of a decode batch at the repository's model shape (4 KV heads of 128), f32 activations
        _store("store_rows_64", n=64, nkv=4, hd=128, ctx=4096, dtype="f32", ragged=True),
        # the rows of a long prompt chunk, starting at an odd position
        _store("store_prompt_8191", n=8191, nkv=8, hd=128, ctx=16384, dtype="bf16", ragged=False),
        # the first tokens of a chat: one sequence, a short odd context; latency is all
        _decode("decode_1x77_f32", B=1, ctx=77, nh=32, nkv=4, hd=128, dtype="f32"),
        # the repository's model benchmark: 4 sequences of 4096 positions, f32 activations
        _decode("decode_4x4096_f32", B=4, ctx=4096, nh=32, nkv=4, hd=128, dtype="f32"),
        # one user with a very long document: all parallelism has to come from the context
        _decode("decode_1x131071", B=1, ctx=131071, nh=32, nkv=8, hd=128, dtype="bf16"),
        # a ragged serving batch of 64-wide heads without sharing, some slots idle
        _decode("decode_24x5003_mha64", B=24, ctx=5003, nh=16, nkv=16, hd=64, dtype="bf16", idle=2),
        # a long-running chat service: sliding window with sinks over long caches
        _decode("decode_32x40960_win", B=32, ctx=40960, nh=40, nkv=8, hd=128, dtype="bf16", window=4096, sinks=4),
        # a full ragged batch at long context: the bandwidth case
        _decode("decode_64x32768", B=64, ctx=32768, nh=32, nkv=4, hd=128, dtype="bf16"),
        # a short follow-up turn in a long chat
        _prefill("prefill_33_at_20000", S=33, pos0=20000, nh=32, nkv=4, hd=128),
        # the repository's prefill benchmark: one 2048-token prompt
        _prefill("prefill_2048", S=2048, pos0=0, nh=32, nkv=4, hd=128),
        # a later chunk of a long prompt under a window with sinks
        _prefill("prefill_4097_win_at_12289", S=4097, pos0=12289, nh=40, nkv=8, hd=128, window=4096, sinks=4),
        # a long prompt in one step: the compute case
        _prefill("prefill_8192", S=8192, pos0=0, nh=32, nkv=4, hd=128),
    ]


def _store(name, n, nkv, hd, ctx, dtype, ragged):
    return {"name": name, "kind": "store", "n": n, "nkv": nkv, "hd": hd, "ctx": ctx, "dtype": dtype, "ragged": ragged}


def _decode(name, B, ctx, nh, nkv, hd, dtype, window=0, sinks=0, idle=0):
    return {"name": name, "kind": "decode", "B": B, "ctx": ctx, "nh": nh, "nkv": nkv, "hd": hd, "dtype": dtype,
            "window": window, "sinks": sinks, "idle": idle}


def _prefill(name, S, pos0, nh, nkv, hd, window=0, sinks=0, dtype="bf16"):
    return {"name": name, "kind": "prefill", "S": S, "pos0": pos0, "nh": nh, "nkv": nkv, "hd": hd, "dtype": dtype,
            "window": window, "sinks": sinks}


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "prefill", "prefill"])
    hd = rng.choice([64, 128, 128])
    nkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
    window, sinks = (0, 0) if rng.random() < 0.6 else (_log(rng, 16, 8192), rng.randint(0, 8))
    if kind == "store":
        n = _log(rng, 1, 12000)
        c = _store("", n, nkv, hd, n + _log(rng, 64, 8192), rng.choice(["f32", "bf16"]), rng.random() < 0.3)
    elif kind == "decode":
        # up to the positions x KV heads of the largest listed case
        B = _log(rng, 1, 128)
        ctx = _log(rng, 1, max(1, min(131072, 64 * 32768 * 4 // (B * nkv))))
        while B * ctx * nkv * group * hd > 64 * 32768 * 32 * 128:
            ctx = max(1, ctx // 2)
        c = _decode("", B, ctx, nkv * group, nkv, hd, rng.choice(["f32", "bf16"]), window, sinks,
                    rng.choice([0, 0, 1]) if B > 4 else 0)
    else:
        S, pos0 = _log(rng, 1, 8192), rng.choice([0, _log(rng, 1, 32768)])
        while S * (S + pos0) * nkv * group * hd > 8192 * 8192 * 32 * 128 // 2:
            S, pos0 = max(1, S * 3 // 4), pos0 * 3 // 4
        c = _prefill("", S, pos0, nkv * group, nkv, hd, window, sinks)
    del c["name"]
    return c


def _lengths(case):
    """Positions of each sequence, the new one included: the first at the full context, the others down to a
    quarter of it; the last `idle` slots hold no sequence."""
    B, ctx = case["B"], case["ctx"]
    n = [max(1, ctx - (3 * ctx // 4) * ((37 * b) % B) // B) for b in range(B)]
    return [0 if b >= B - case["idle"] else v for b, v in enumerate(n)]


def _visible(last, window, sinks):
    """How many positions the query at position `last` sees."""
    n = last + 1
    return n if window == 0 or n <= window else window + min(sinks, n - window)


def work(case):
    nkv, hd = case["nkv"], case["hd"]
    row = hd // 2 + hd // 16  # bytes of a cached row
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "store":
        n = case["n"] * nkv * 2
        return {"bytes": n * (size * hd + row) + n * (row + 4 * hd), "flops": 0}
    nh, w, s = case["nh"], case["window"], case["sinks"]
    if case["kind"] == "decode":
        lens = _lengths(case)
        seen = sum(_visible(n - 1, w, s) for n in lens if n)
        new = len(lens)
        read = seen
    else:
        seen = sum(_visible(t, w, s) for t in range(case["pos0"], case["pos0"] + case["S"]))
        new = case["S"]
        first = max(0, case["pos0"] + 1 - w) if w else 0  # the earliest position of the first query's window
        read = case["pos0"] + new - first + min(s, first)
    # cached rows read once, new rows in and out of the cache, the queries and the outputs
    byt = read * nkv * 2 * row + new * nkv * 2 * (size * hd + row + 4 * hd) + new * nh * hd * 2 * size
    return {"bytes": byt, "flops": 4 * hd * nh * seen}


# ------------------------------------------------------------------ inputs
def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _rows(gen, shape, gain, dtype):
    return (torch.randn(shape, generator=gen, device="cuda") * gain).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, nkv, hd, dt = case["kind"], case["nkv"], case["hd"], _dtype(case)
    n_seq = {"store": case.get("n") if case.get("ragged") else 1, "decode": case.get("B"), "prefill": 1}[kind]
    ctx = {"store": case.get("ctx"), "decode": case.get("ctx"), "prefill": case.get("pos0", 0) + case.get("S", 0)}[kind]
    if kind == "store" and case["ragged"]:
        n_seq = min(n_seq, 64)  # ragged rows go to up to 64 sequences
    cap = -(-ctx // SLOTS) * SLOTS
    # normalised and rotated keys: channels of unequal size; values: narrower
    gk = torch.exp(0.4 * torch.randn((nkv, hd), generator=gen, device="cuda"))
    gv = 0.5 * torch.exp(0.3 * torch.randn((nkv, hd), generator=gen, device="cuda"))
    planes = [torch.empty((n_seq, nkv, cap, hd // 2), dtype=torch.uint8, device="cuda"),
              torch.empty((n_seq, nkv, cap, hd // 32), dtype=torch.float16, device="cuda"),
              torch.empty((n_seq, nkv, cap, hd // 2), dtype=torch.uint8, device="cuda"),
              torch.empty((n_seq, nkv, cap, hd // 32), dtype=torch.float16, device="cuda")]
    # every position holds a row: past a sequence's end those of an earlier request
    step = max(1, (1 << 23) // (cap * hd))
    at = torch.arange(cap, device="cuda")
    for j, gain in ((0, gk), (2, gv)):
        codes, scales = planes[j].view(n_seq * nkv, cap, -1), planes[j + 1].view(n_seq * nkv, cap, -1)
        for i in range(0, n_seq * nkv, step):
            m = min(step, n_seq * nkv - i)
            g = gain[torch.arange(i, i + m, device="cuda") % nkv].unsqueeze(1)
            c, d = _quantise(_rows(gen, (m, cap, hd), g, torch.float32))
            codes[i:i + m] = _pack(c, at)
            scales[i:i + m] = d
    state = {"case": dict(case), "planes": planes}
    n = {"store": case.get("n"), "decode": case.get("B"), "prefill": case.get("S")}[kind]
    state["k"] = _rows(gen, (n, nkv, hd), gk, dt)
    state["v"] = _rows(gen, (n, nkv, hd), gv, dt)
    if kind != "store":
        state["q"] = _rows(gen, (n, case["nh"], hd), 1.0, dt)
    if kind == "decode":
        state["pos"] = torch.tensor([v - 1 for v in _lengths(case)], dtype=torch.int32, device="cuda")
    if kind == "store":
        if case["ragged"]:  # distinct (sequence, position) pairs in no order
            i = torch.arange(n, device="cuda")
            state["seq"] = ((i * 29 + 3) % n_seq).to(torch.int32)
            shift = torch.randint(0, ctx, (n_seq,), generator=gen, device="cuda")
            state["pos"] = ((i // n_seq + shift[state["seq"].long()]) % ctx).to(torch.int32)
        else:
            state["pos0"] = min(ctx - n, 1 + 2 * (ctx - n) // 5)
    return state


# ------------------------------------------------------------------ the plain form
def _quantise(x):
    """f32 [..., hd] -> codes uint8 [..., hd / 32, 32], scales f16 [..., hd / 32]."""
    x = x.unflatten(-1, (-1, 32))
    x = torch.nan_to_num(x)
    hi, lo = x.amax(-1), x.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) * -0.125).clamp(-F16_MAX, F16_MAX)
    d16 = d.to(torch.float16)
    inv = torch.where(d16 == 0, 0.0, 1.0 / d)
    scaled = x * inv.unsqueeze(-1)
    return torch.floor(scaled + 8.5).clamp(0, 15).to(torch.uint8), d16


def _slots(pos, blocks):
    """The slot of each block's chunk in the rows at these positions: [n, blocks]."""
    turn = (pos >> 1) & 3 if blocks == 4 else (pos >> 2) & 1
    return torch.arange(blocks, device=pos.device) ^ turn.long().unsqueeze(-1)


def _pack(codes, pos):
    """codes [..., n, blocks, 32] of the rows at positions pos [n] -> bytes [..., n, blocks * 16]."""
    chunks = codes[..., 0::2] | (codes[..., 1::2] << 4)
    at = _slots(pos, codes.shape[-2]).unsqueeze(-1).expand(chunks.shape)
    return torch.gather(chunks, -2, at).flatten(-2)  # the exchange is its own inverse


def _unpack(data, scales, pos):
    """bytes [..., n, blocks * 16] and scales of the rows at positions pos [n] -> f32 [..., n, hd]."""
    chunks = data.unflatten(-1, (-1, 16))
    at = _slots(pos, chunks.shape[-2]).unsqueeze(-1).expand(chunks.shape)
    chunks = torch.gather(chunks, -2, at)
    codes = torch.stack((chunks & 15, chunks >> 4), -1).flatten(-2)
    return ((codes.float() - 8.0) * scales.float().unsqueeze(-1)).flatten(-2)


def _put(planes, k, v, seq, pos):
    """Quantises rows k, v [n, nkv, hd] into the rows (seq[i], pos[i]); a negative position: no row."""
    keep = torch.nonzero(pos >= 0).flatten()
    seq, pos = seq[keep], pos[keep]
    for j, x in ((0, k), (2, v)):
        c, d = _quantise(x[keep].float())
        planes[j][seq, :, pos] = _pack(c.transpose(0, 1), pos).transpose(0, 1)
        planes[j + 1][seq, :, pos] = d


def _get(planes, seq, pos):
    """The rows (seq[i], pos[i]) as f32 [n, nkv, hd]: K and V; a negative position: zeros."""
    at = pos.clamp(min=0)
    got = [_unpack(planes[j][seq, :, at].transpose(0, 1), planes[j + 1][seq, :, at].transpose(0, 1), at).transpose(0, 1)
           for j in (0, 2)]
    return [torch.where(pos[:, None, None] >= 0, x, 0.0) for x in got]


def _attend(q, k, v, seen):
    """q [..., r, hd], k and v [..., n, hd], seen [..., r, n]: softmax attention, zeros where nothing is seen."""
    s = torch.matmul(q, k.transpose(-1, -2)) * (q.shape[-1] ** -0.5)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total == 0, 1.0, total)


def _sees(t, p, window, sinks):
    seen = p <= t
    return seen & ((p < sinks) | (t - p < window)) if window else seen


def _plain(state):
    case, planes = state["case"], state["planes"]
    kind, dev = case["kind"], planes[0].device
    n = state["k"].shape[0]
    if kind == "decode":
        seq, pos = torch.arange(n, device=dev), state["pos"].long()
    elif kind == "prefill" or not case["ragged"]:
        seq = torch.zeros(n, dtype=torch.int64, device=dev)
        pos = torch.arange(n, device=dev) + (case["pos0"] if kind == "prefill" else state["pos0"])
    else:
        seq, pos = state["seq"].long(), state["pos"].long()
    _put(planes, state["k"], state["v"], seq, pos)
    krows, vrows = _get(planes, seq, pos)
    if kind == "store":
        return {"k": krows, "v": vrows}
    q, nkv, nh, hd = state["q"].float(), case["nkv"], case["nh"], case["hd"]
    L = case["ctx"] if kind == "decode" else case["pos0"] + n
    at = torch.arange(L, device=dev)
    k = _unpack(planes[0][:, :, :L], planes[1][:, :, :L], at)
    v = _unpack(planes[2][:, :, :L], planes[3][:, :, :L], at)
    if kind == "decode":
        seen = _sees(pos[:, None], at, case["window"], case["sinks"])[:, None, None]
        out = _attend(q.view(n, nkv, nh // nkv, hd), k, v, seen).reshape(n, nh, hd)
    else:
        seen = _sees(pos[:, None], at, case["window"], case["sinks"])
        qh = q.view(n, nkv, nh // nkv, hd).permute(1, 2, 0, 3)
        out = _attend(qh, k[0].unsqueeze(1), v[0].unsqueeze(1), seen).permute(2, 0, 1, 3).reshape(n, nh, hd)
    return {"out": out.to(state["q"].dtype), "k": krows, "v": vrows}


# ------------------------------------------------------------------ the framework's calls
def _own(state):
    case = state["case"]
    cache = state.get("cache")
    if cache is None:
        import tetraeder_b200 as tb
        cache = state["cache"] = tb.Kv4Cache.from_planes(*state["planes"])
    kind = case["kind"]
    if kind == "decode":
        out = cache.decode(state["q"], state["k"], state["v"], state["pos"], window=case["window"],
                           n_sink=case["sinks"])
        k, v = cache.load(state["pos"])
        return {"out": out, "k": k, "v": v}
    if kind == "prefill":
        out = cache.prefill(state["q"], state["k"], state["v"], seq=0, pos0=case["pos0"], window=case["window"],
                            n_sink=case["sinks"])
        k, v = cache.load(case["pos0"], n=case["S"], seq=0)
        return {"out": out, "k": k, "v": v}
    if case["ragged"]:
        cache.store(state["k"], state["v"], state["pos"], seq=state["seq"])
        k, v = cache.load(state["pos"], seq=state["seq"])
    else:
        cache.store(state["k"], state["v"], state["pos0"], seq=0)
        k, v = cache.load(state["pos0"], n=case["n"], seq=0)
    return {"k": k, "v": v}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(x):
    """numpy f32 rows [..., hd] -> the values that the cache holds for them (f64), by the definition: scale and
    quotient are 32-bit values, the scale is kept in 16."""
    b = x.reshape(-1, 32)
    big = b[np.arange(len(b)), np.abs(b).argmax(1)]
    top = np.abs(big)
    big = np.where((b == top[:, None]).any(1), top, -top).astype(np.float32)
    d = big / np.float32(-8)
    kept = d.astype(np.float16)
    with np.errstate(divide="ignore"):
        inv = np.where(kept == 0, np.float32(0), np.float32(1) / d)
    c = np.clip(np.floor(b * inv[:, None] + np.float32(8.5)), 0, 15)
    return ((c.astype(np.float64) - 8) * kept.astype(np.float64)[:, None]).reshape(x.shape)


def _exact_values(codes, scales, first):
    """The f64 values of one head's rows first .. first + n - 1: codes [n, hd / 2], scales [n, hd / 32]."""
    n, half = codes.shape
    blocks = half // 16
    p = torch.arange(first, first + n, device=codes.device)
    out = torch.empty((n, 2 * half), dtype=torch.float64, device=codes.device)
    for c in range(blocks):
        slot = c ^ ((p // 2) % 4 if blocks == 4 else (p // 4) % 2)
        byte = torch.gather(codes.long(), 1, slot[:, None] * 16 + torch.arange(16, device=codes.device))
        d = scales[:, c].double()[:, None]
        out[:, 32 * c:32 * c + 32:2] = (byte % 16 - 8).double() * d
        out[:, 32 * c + 1:32 * c + 32:2] = (byte // 16 - 8).double() * d
    return out


def _exact_softmax(q, k, v, bias):
    s = torch.einsum("td,nd->tn", q, k) / math.sqrt(q.shape[1]) + bias
    return torch.softmax(s, 1) @ v


def exact(case, seed):
    state = prepare(case, seed)
    planes, kind, nkv, hd = state["planes"], case["kind"], case["nkv"], case["hd"]
    krow, vrow = (_exact_rows(state[x].float().cpu().numpy()) for x in "kv")
    dev = planes[0].device
    if kind == "store":
        return {"k": torch.from_numpy(krow), "v": torch.from_numpy(vrow)}
    n, nh, w, s = state["k"].shape[0], case["nh"], case["window"], case["sinks"]
    G = nh // nkv
    q = state["q"].double()
    out = torch.zeros((n, nh, hd), dtype=torch.float64, device=dev)
    knew, vnew = torch.from_numpy(krow).to(dev), torch.from_numpy(vrow).to(dev)
    if kind == "decode":
        for b, length in enumerate(_lengths(case)):
            if length == 0:
                knew[b] = vnew[b] = 0
                continue
            lo = max(0, length - w) if w else 0
            for g in range(nkv):
                parts = []
                for j, new in ((0, knew), (2, vnew)):
                    head = [_exact_values(planes[j][b, g, :min(s, lo)], planes[j + 1][b, g, :min(s, lo)], 0)] if lo and s else []
                    x = _exact_values(planes[j][b, g, lo:length], planes[j + 1][b, g, lo:length], lo)
                    x[-1] = new[b, g]
                    parts.append(torch.cat(head + [x]))
                out[b, g * G:(g + 1) * G] = _exact_softmax(q[b, g * G:(g + 1) * G], *parts, 0.0)
    else:
        pos0 = case["pos0"]
        L = pos0 + n
        p = torch.arange(L, device=dev)
        for g in range(nkv):
            k, v = (_exact_values(planes[j][0, g, :L], planes[j + 1][0, g, :L], 0) for j in (0, 2))
            k[pos0:], v[pos0:] = knew[:, g], vnew[:, g]
            for i in range(0, n, 1024):
                t = torch.arange(pos0 + i, min(pos0 + i + 1024, L), device=dev)[:, None]
                hidden = (p > t) | ((p >= s) & (p <= t - w)) if w else p > t
                bias = torch.zeros(hidden.shape, dtype=torch.float64, device=dev).masked_fill(hidden, -math.inf)
                for h in range(g * G, (g + 1) * G):
                    out[i:i + 1024, h] = _exact_softmax(q[i:i + 1024, h], k, v, bias)
    return {"out": out, "k": knew, "v": vnew}
