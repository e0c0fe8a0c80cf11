"""The Qwen3-MoE model over 4-bit KV caches (Qwen3MoeModel with kv_type="q4"), with and without a sliding window
and sinks, against the CPU oracle of the step.  A value near a 4-bit rounding boundary turns a last-bit difference
of the two sides into a whole step, so the oracle attends over the rows that the model's caches hold (each step's,
read back) and checks that they are its own K and V rows, rounded: within a step d of 1/8 of the block's largest
value (the largest of the positive side is clipped by one), plus 5e-2 of that value for the two sides' own
difference.  The logits' bound is that of the F16-cache test: last-bit differences turn into a few flipped 8-bit
roundings per step, about 1.5e-2 of the logits over two layers; 5e-2 is allowed."""
import numpy as np
import pytest
import torch

gguf = pytest.importorskip("gguf")

import oracle as O  # noqa: E402
from oracle.model import Matrix, ModelOracle, rms_norm, rope_neox  # noqa: E402
from tests import kv4_ref as R  # noqa: E402
from tests.common import nrms  # noqa: E402
from tests.gguf_fixture import write_moe_gguf  # noqa: E402
from tetraeder_b200.gguf import GgufFile  # noqa: E402
from tetraeder_b200.model import Qwen3MoeModel  # noqa: E402

pytestmark = pytest.mark.gpu


class Kv4Oracle(ModelOracle):
    def __init__(self, hp, weights, model):
        super().__init__(hp, weights, 1, 1)
        self.model = model

    def rows(self, il, seq, pos, k, v):
        """The rows at (seq, pos) as the model's cache of layer il holds them, held to k and v."""
        i32 = dict(dtype=torch.int32, device="cuda")
        got = self.model.kv4[il].load(torch.tensor(pos, **i32), seq=torch.tensor(seq, **i32))
        for x, y in zip((k, v), got):
            x, y = x.reshape(-1, 32), y.cpu().numpy().reshape(-1, 32)
            big = np.abs(x).max(1, keepdims=True)
            assert (np.abs(x - y) <= (1 / 8 + 5e-2) * big).all()

    def attention(self, il, x, pos, seq=None):
        hp, w, p = self.hp, self.w, f"blk.{il}."
        B, d, nh = x.shape[0], hp.head_dim, hp.n_head
        seq = np.arange(B) if seq is None else np.asarray(seq)
        cur = rms_norm(x, w[p + "attn_norm.weight"], hp.rms_eps)
        q, k, v = (w[p + f"attn_{n}.weight"].matmul(cur).reshape(B, -1, d) for n in "qkv")
        q = rope_neox(rms_norm(q, w[p + "attn_q_norm.weight"], hp.rms_eps), pos, hp.n_rot, hp.rope_freq_base)
        k = rope_neox(rms_norm(k, w[p + "attn_k_norm.weight"], hp.rms_eps), pos, hp.n_rot, hp.rope_freq_base)
        self.rows(il, seq, pos, k, v)
        out = np.zeros((B, nh, d), np.float32)
        for b in range(B):
            K, V = (t.double().cpu().numpy() for t in self.model.kv4[il].load(0, n=int(pos[b]) + 1, seq=int(seq[b])))
            out[b] = R.attend(q[b].astype(np.float64), K, V, int(pos[b]), self.model.window, self.model.n_sink, d ** -0.5)[0]
        return (x + w[p + "attn_output.weight"].matmul(out.reshape(B, nh * d))).astype(np.float32)


def oracle_weights(written, hp):
    w = {}
    for name, (t, arr) in written.items():
        if t == O.TYPE_F32 and (arr.ndim == 1 or name.endswith("ffn_gate_inp.weight")):
            w[name] = arr
        elif name.endswith("_exps.weight"):
            w[name] = Matrix(t, arr, arr.shape[0] * arr.shape[1], 0)
        else:
            cols = arr.shape[1] if t in (O.TYPE_F16, O.TYPE_F32) else hp.n_embd if not name.endswith(
                "attn_output.weight") else hp.n_head * hp.head_dim
            w[name] = Matrix(t, arr, arr.shape[0], cols)
    return w


@pytest.fixture(scope="module")
def tiny_model(tmp_path_factory):
    p = tmp_path_factory.mktemp("model") / "tiny-qwen3moe.gguf"
    written = write_moe_gguf(p, n_layer=2, n_embd=512, n_head=4, n_head_kv=2, head_dim=128, n_expert=8, n_used=2,
                             n_ff=256, n_vocab=512, gate_type=12, down_type=14, attn_types=(12, 12, 14, 12),
                             embd_type=12, out_type=14, extra_kv=False)
    return p, written


@pytest.mark.parametrize("window,n_sink", [(0, 0), (16, 3)])
def test_prefill_then_decode_matches_the_oracle(tiny_model, window, n_sink):
    path, written = tiny_model
    B, n_ctx, S = 3, 96, 45
    with GgufFile(path) as f:
        hp = f.hparams
        model = Qwen3MoeModel.from_gguf(f, max_batch=B, n_ctx=n_ctx, kv_type="q4", window=window, n_sink=n_sink)
    ref = Kv4Oracle(hp, oracle_weights(written, hp), model)
    rng = np.random.default_rng(11)
    try:
        assert not model.kc and len(model.kv4) == hp.n_layer
        for seq in (0, 2):
            prompt = rng.integers(0, hp.n_vocab, S).astype(np.int32)
            got = model.prefill(torch.from_numpy(prompt).cuda(), seq=seq).cpu().numpy()
            model.check()
            n = nrms(got, ref.prefill(prompt, seq))
            assert n < 5e-2, f"prefill of sequence {seq}: logits nrms {n:.2e}"
        start = np.array([S, 0, S], dtype=np.int32)  # sequence 1 begins with its first decoded token
        for s in range(4):
            toks = rng.integers(0, hp.n_vocab, B).astype(np.int32)
            pos = (start + s).astype(np.int32)
            got = model.decode(torch.from_numpy(toks).cuda(), torch.from_numpy(pos).cuda()).cpu().numpy()
            model.check()
            n = nrms(got, ref.decode(toks, pos))
            assert n < 5e-2, f"step {s}: logits nrms {n:.2e}"
        assert np.array_equal(model.next_tokens.cpu().numpy(), np.argmax(got, axis=1))
    finally:
        model.close()


def test_graph_replay_matches_eager(tiny_model):
    path, _ = tiny_model
    B, n_ctx = 2, 64
    with GgufFile(path) as f:
        a, b = (Qwen3MoeModel.from_gguf(f, max_batch=B, n_ctx=n_ctx, kv_type="q4", window=8, n_sink=2) for _ in range(2))
    toks = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    try:
        b.decode(toks, pos)  # sizes the projections' workspace, fills position 0
        a.decode(toks, pos)
        torch.cuda.synchronize()
        g = b.graph(toks, pos)
        for step in range(1, 20):
            toks.copy_(torch.tensor([step * 7 % 512, step * 11 % 512], dtype=torch.int32))
            pos.fill_(step)
            want = a.decode(toks, pos).clone()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(b.logits[:B], want), f"step {step}"
        b.check()
        del g
    finally:
        a.close()
        b.close()


def test_cache_choices_are_checked(tiny_model):
    path, _ = tiny_model
    for kv in (dict(kv_type="q8"), dict(window=4), dict(n_sink=2), dict(kv_type="q4", window=-1)):
        with pytest.raises(ValueError):
            Qwen3MoeModel.from_gguf(str(path), max_batch=1, n_ctx=32, **kv)
