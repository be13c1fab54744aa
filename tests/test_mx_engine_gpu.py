"""A Llama model with 4-bit weights, and with rows in 8 bits as well, against the plain implementation on the values that the
weights stand for: prompts of more rows than the few-rows products take, of few, single tokens eager and recorded."""
import numpy as np
import pytest
import torch

import gpu_util as G
import mx_util as U
import plain_llama as P
import transformer_amd as ta
from transformer_amd import kernels
from transformer_amd.engine.generate import generate

pytestmark = pytest.mark.gpu
PROJ = ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")


def _narrow(w):
    y = torch.tensor(w)
    b = U.bytes_of(y, 6.0)
    s = U.power(b).repeat_interleave(32, 1)
    return (U.nearest(y / s, torch.tensor(U.E2M1, dtype=torch.float64)) * s).numpy()


class PlainNarrow(P.PlainLlama):
    """The plain model on the values of the packed weights; with ``eight`` the rows of every projection in 8 bits too."""

    def __init__(self, folder, eight=False):
        super().__init__(folder)
        self.eight = eight
        for n in self.w:
            if n.endswith(".weight") and n.split(".")[-2] in PROJ:
                self.w[n] = _narrow(self.w[n])

    def _q(self, a):
        if not self.eight:
            return a
        v, b = U.pack8(torch.tensor(np.ascontiguousarray(a)))
        return (v * U.power(b).repeat_interleave(32, 1)).numpy()

    def block(self, i, x, positions):
        w, p, T = self.w, f"model.layers.{i}.", x.shape[0]
        lin = lambda a, n: P.linear(a, w[p + n + ".weight"], w.get(p + n + ".bias"))
        h = self._q(P.rms_norm(x, w[p + "input_layernorm.weight"], self.eps))
        q, k, v = (lin(h, f"self_attn.{c}_proj").reshape(T, -1, self.dh) for c in "qkv")
        q, k = (P.rope(t, positions, self.theta, self.rope_style) for t in (q, k))
        x = x + lin(self._q(P.attention(q, k, v, self.scale).reshape(T, -1)), "self_attn.o_proj")
        h = self._q(P.rms_norm(x, w[p + "post_attention_layernorm.weight"], self.eps))
        return x + lin(self._q(P.swiglu(lin(h, "mlp.gate_proj"), lin(h, "mlp.up_proj"))), "mlp.down_proj")


_models = {}


def _model(name, activations):
    key = (name, activations)
    if key not in _models:
        _models[key] = (ta.load_model(G.folder(name, "bfloat16"), "bfloat16", "cuda:0", weights="mx4", activations=activations),
                        PlainNarrow(G.folder(name, "bfloat16"), activations == "mx8"))
    return _models[key]


def _steps(model, name, lens, decode, graphs):
    """Logits of the last prompt token and of every token after it, per sequence."""
    model.use_graphs = graphs
    cache = model.new_cache(1024, 8)
    seqs = [G.tokens(name, n + decode, 31 + i) for i, n in enumerate(lens)]
    slots = [cache.alloc_slot() for _ in lens]
    got = [model.step(cache, [ta.Entry(s, q[:n], want=[n - 1]) for s, q, n in zip(slots, seqs, lens)]).clone()]
    for t in range(decode):
        got.append(model.step(cache, [ta.Entry(s, [q[n + t]], want=[0]) for s, q, n in zip(slots, seqs, lens)]).clone())
    return seqs, torch.stack(got, 1).double().cpu().numpy()


def _off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("lens", [(70,), (3, 5), (40, 1, 90)])
@pytest.mark.parametrize("name", ["D", "E", "F"])
def test_logits_with_4_bit_weights(name, lens, graphs):
    model, plain = _model(name, None)
    seqs, got = _steps(model, name, lens, 3, graphs)
    for q, g, n in zip(seqs, got, lens):
        assert np.abs(plain.forward(q)[n - 1:] - g).max() < G.TOL["bfloat16"]


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("lens", [(70,), (3, 5)])
@pytest.mark.parametrize("name", ["D", "E", "F"])
def test_logits_with_rows_in_8_bits(name, lens, graphs):
    """The engine's rows carry bfloat16's noise (2^-8) into the rounding to e4m3, whose steps are 2^-3 to 2^-4 of a value: about one in 16 falls on the
    other side, a step off, some 2 % of the rows' norm, product by product; over the layers of these models up to 8 % of the logits'."""
    model, plain = _model(name, "mx8")
    seqs, got = _steps(model, name, lens, 3, graphs)
    for q, g, n in zip(seqs, got, lens):
        assert _off(g, plain.forward(q)[n - 1:]) < 0.08


@pytest.mark.parametrize("activations", [None, "mx8"])
def test_steps_of_more_sequences_than_the_few_rows_products_take(activations):
    """70 sequences, a recorded step of 96 rows: with bfloat16 rows every product widens its weights inside the recording. Replayed, and between
    replays a prompt that uses the same scratch eagerly."""
    model, plain = _model("D", activations)
    count, decode = 70, 5
    got = {}
    for graphs in (False, True):
        model.use_graphs = graphs
        cache = model.new_cache(64 * (count + 4), count + 2)
        seqs = [G.tokens("D", 2 + i % 3 + decode, 400 + i) for i in range(count)]
        slots = [cache.alloc_slot() for _ in seqs]
        model.step(cache, [ta.Entry(s, q[:-decode], want=[]) for s, q in zip(slots, seqs)])
        out = []
        for t in range(decode):
            out.append(model.step(cache, [ta.Entry(s, [q[len(q) - decode + t]], want=[0]) for s, q in zip(slots, seqs)]).clone())
            other = cache.alloc_slot()
            model.step(cache, [ta.Entry(other, G.tokens("D", 90, 7), want=[89])])
            cache.free_slot(other)
        assert bool(cache.graphs) == graphs and not cache.graphs_failed
        got[graphs] = torch.stack(out, 1).double().cpu().numpy()
    for graphs in (False, True):
        for i in (0, 1, 34, 63, 64, 69):
            want = plain.forward(seqs[i])[-decode:]
            if activations:
                assert _off(got[graphs][i], want) < 0.08
            else:
                assert np.abs(want - got[graphs][i]).max() < G.TOL["bfloat16"]


def test_generates_and_holds_fewer_bytes():
    folder = G.folder("E", "bfloat16")
    wide = G.engine("E", "bfloat16")
    c = G.CONFIGS["E"][0]
    d, di, kv = c["hidden_size"], c["intermediate_size"], c["num_key_value_heads"] * c["head_dim"]
    packed = c["num_hidden_layers"] * (d * (d + 2 * kv) + d * d + 3 * d * di)
    for activations in (None, "mx8"):
        model = ta.load_model(folder, "bfloat16", "cuda:0", weights="mx4", activations=activations)
        assert wide.weight_bytes() - model.weight_bytes() == packed * 2 - packed // 2 - packed // 32
        res = generate(model, [G.tokens("E", 9, 1), G.tokens("E", 80, 2)], 6, stop_ids=[])
        assert [len(t) for t in res.tokens] == [6, 6]
        again = generate(model, [G.tokens("E", 9, 1), G.tokens("E", 80, 2)], 6, stop_ids=[])
        assert res.tokens == again.tokens
        with pytest.raises(ValueError, match="4-bit"):
            ta.save_model(model, "/nonexistent")


def test_the_same_from_a_random_model_the_facade_and_the_command(tmp_path, capsys):
    model = ta.random_model(G.TINY_D, 5, weights="mx4", activations="mx8")
    llm = ta.Llama.from_pretrained(G.folder("D", "bfloat16"), weights="mx4", cache_tokens=512)
    for m in (model, llm.model):
        assert isinstance(m.tensors["blocks.0.mixer.qkv.weight"], kernels.Mx4) and m.tensors["embed.weight"].dtype == torch.bfloat16
    want = llm.generate([[5, 17, 3]], 4, stop_ids=[]).tokens[0]
    from transformer_amd.cli import main
    assert main(["generate", "--model", G.folder("D", "bfloat16"), "--weights", "mx4", "--prompt", "5,17,3", "--max-steps", "4"]) == 0
    assert "-> " + " ".join(map(str, want)) in capsys.readouterr().out
    assert main(["generate", "--model", G.folder("D", "bfloat16"), "--weights", "mx4", "--activations", "mx8", "--prompt", "5,17,3",
                 "--max-steps", "2"]) == 0


def test_what_is_refused():
    d = G.folder("D", "bfloat16")
    for kw in (dict(weights="int4"), dict(activations="mx8"), dict(weights="mx4", activations="fp8"), dict(weights="mx4", dtype="float32")):
        with pytest.raises(ValueError):
            ta.load_model(d, **{"dtype": "bfloat16", **kw})
    with pytest.raises(ValueError, match="blocks of 32"):                 # a feed-forward of 304
        ta.load_model(G.folder("C", "bfloat16"), "bfloat16", weights="mx4")
    import vametar_util as V
    with pytest.raises(ValueError, match="no part"):
        ta.load_model(V.folder("A", "bfloat16"), "bfloat16", weights="mx4")
