"""TextEngine on the serving operators: a 4-bit cache, an attention window with sinks, and filtered
sampling, against a 64-bit decoder that keeps its cache the same way.

Tolerance. The engine's arithmetic is that of its other engines, whose logits stay within
1e-3 + 1e-4 of the reference's (tests/parity.py), and so do these, with every storage. In 4 bits or
bf16 that holds for one way of rounding: a key or value that lies within the float error BORDER of a
border between two codes or bf16 numbers (or a group's extreme within it of a bf16 number) may be
kept either way, and one step moves logits by more than float errors do. So the engine has to match
the 64-bit decoder under some choice for those, and only those, undecided places; choices in one
layer change what is undecided in the next, which the decoder finds anew for each.
BORDER: keys and values are dot products of D = 128 terms with sum |x w| below 20, in float32 parts
good to 2^-21, behind a LayerNorm and at most one layer with errors of the same size: below 4e-5.
"""
import math

import numpy as np
import pytest

import operator_reference as ref
from basalt_b200 import ModelSpec, TextEngine, left_pad, synthetic_prompts, write_synthetic_weights
from basalt_b200 import IllegalArgumentException

pytestmark = pytest.mark.gpu

V, W, D, L, H, F = 96, 48, 128, 2, 4, 256


def norm(x, gamma, beta):
    m = x.mean(-1, keepdims=True)
    v = ((x - m) ** 2).mean(-1, keepdims=True)
    return (x - m) / np.sqrt(v + 1e-5) * gamma + beta


BORDER = 4e-5


class Choices:
    """Which undecided places round the other way, and the undecided places that a run met."""

    def __init__(self, flipped=frozenset()):
        self.flipped, self.met = flipped, []

    def pick(self, where, near, usual, other):
        """`usual`, or `other` at the places flipped; `near` marks the undecided."""
        out = np.array(usual)
        for at in zip(*np.nonzero(near)):
            key = (where, tuple(int(i) for i in at))
            self.met.append(key)
            if key in self.flipped:
                out[at] = other[at]
        return out

    def bf16(self, where, x, up):
        """x rounded to bf16 in one direction; undecided where x is next to a bf16 number."""
        usual = ref.directed_bf16(x, up)
        lower, upper = ref.directed_bf16(x - BORDER, up), ref.directed_bf16(x + BORDER, up)
        return self.pick(where, lower != upper, usual, np.where(usual == lower, upper, lower))

    def nearest(self, where, x):
        """x rounded to the nearest bf16; undecided in the middle between two."""
        usual, lower, upper = (ref.bf16_bits((x + d).astype(np.float32)).astype(np.float64)
                               for d in (0, -BORDER, BORDER))
        return self.pick(where, lower != upper, usual, np.where(usual == lower, upper, lower))

    def quantise(self, where, x):
        g = x.reshape(*x.shape[:-1], -1, 32)
        low = self.bf16(where + ("low",), g.min(-1), False)
        step = self.bf16(where + ("step",), (g.max(-1) - low) / 15.0, True)
        q = (g - low[..., None]) / step[..., None]
        code = np.clip(np.rint(q), 0, 15)
        near = (np.abs(q - np.floor(q) - 0.5) * step[..., None] < BORDER) & (q > 0) & (q < 15)
        other = np.where(code > q, code - 1, code + 1)
        code = self.pick(where + ("code",), near, code, other)
        return (low[..., None] + code * step[..., None]).reshape(x.shape)


def kept(x, storage, choices, where):
    """[tokens, heads, dim] as the cache keeps it."""
    if storage == "u4":
        return choices.quantise(where, x)
    return choices.nearest(where, x) if storage == "bf16" else x


def decoder_logits(w, ids, storage, window, sinks, choices):
    """Logits at every position of `ids`, in 64 bits."""
    n = len(ids)
    x = w["embedding.weight"][ids] + w["position.weight"][:n]
    for l in range(L):
        p = f"layer{l}."
        h = norm(x, w[p + "norm1.gamma"], w[p + "norm1.beta"])
        q, k, v = ((h @ w[p + f"attention.{n_}.weight"] + w[p + f"attention.{n_}.bias"])
                   .reshape(n, H, D // H) for n_ in ("query", "key", "value"))
        a, _ = ref.attend(q, kept(k, storage, choices, (l, "k")),
                          kept(v, storage, choices, (l, "v")), 0, window, sinks,
                          1 / math.sqrt(D // H))
        x = x + a.reshape(n, D) @ w[p + "attention.output.weight"] + w[p + "attention.output.bias"]
        h = norm(x, w[p + "norm2.gamma"], w[p + "norm2.beta"])
        h = h @ w[p + "ffn1.weight"] + w[p + "ffn1.bias"]
        h = 0.5 * h * (1 + np.tanh(math.sqrt(2 / math.pi) * (h + 0.044715 * h ** 3)))
        x = x + h @ w[p + "ffn2.weight"] + w[p + "ffn2.bias"]
    return norm(x, w["norm.gamma"], w["norm.beta"]) @ w["head.weight"] + w["head.bias"]


def matches(got, w, ids, storage, window, sinks, first):
    """Whether `got` are the logits from position `first` on under some choice of rounding."""
    def far(flipped):
        choices = Choices(flipped)
        want = decoder_logits(w, ids, storage, window, sinks, choices)[first:]
        off = np.abs(got - want)
        return (off - 1e-4 * np.abs(want)).max(), float((off ** 2).sum()), choices.met

    # One undecided place after the other: the one that brings the logits nearest.
    flipped = frozenset()
    worst, square, met = far(flipped)
    while worst > 1e-3 and len(flipped) < 8:
        tried = [(far(flipped ^ {key})[1], key) for key in met]
        if not tried or min(tried)[0] >= square:
            break
        flipped = flipped ^ {min(tried)[1]}
        worst, square, met = far(flipped)
    return worst <= 1e-3, worst


def weights_of(engine):
    w = {k: v.astype(np.float64) for k, v in engine.stateDict().items()}
    shapes = {"embedding.weight": (V + 1, D), "position.weight": (W, D), "head.weight": (D, V)}
    for l in range(L):
        for n in ("query", "key", "value", "output"):
            shapes[f"layer{l}.attention.{n}.weight"] = (D, D)
        shapes[f"layer{l}.ffn1.weight"], shapes[f"layer{l}.ffn2.weight"] = (D, F), (F, D)
    for k, s in shapes.items():
        w[k] = w[k].reshape(s)
    return w


@pytest.fixture()
def make(runtime, tmp_path):
    made = []

    def build(**kw):
        spec = ModelSpec("padded_decoder", V, W, D, L, H, F, **kw)
        path = tmp_path / "w.bin"
        write_synthetic_weights(spec, path, seed=3, stddev=0.1)
        engine = TextEngine.of(runtime, spec, V, W)
        engine.load(path)
        made.append(engine)
        return engine

    yield build
    for e in made:
        e.close()


@pytest.mark.parametrize("rows", [1, 5, 12])
@pytest.mark.parametrize("storage,window,sinks", [("u4", 0, 0), ("u4", 7, 2), ("f32", 7, 2),
                                                  ("bf16", 5, 0), ("f32", 1, 3), ("f32", 400, 2)])
def test_decoding_matches_64_bits(make, rows, storage, window, sinks):
    engine = make(kv_dtype=storage, attention_window=window, attention_sinks=sinks)
    steps = 12
    prompts = synthetic_prompts(7, rows, 17, V)
    prompts[0, :9] = V                                  # a shorter row in the same batch
    contexts = left_pad(prompts, W, V)
    tokens, logits = engine.generateWithLogits(contexts, steps)
    w = weights_of(engine)
    for r in range(rows):
        start = [t for t in prompts[r] if t != V]
        ids = start + list(tokens[r][:-1])
        good, nearest = matches(logits[r], w, ids, storage, window, sinks, len(start) - 1)
        assert good, (r, nearest)
    np.testing.assert_array_equal(engine.generateBatch(contexts, steps), tokens)
    assert np.abs(engine.scoresBatch(contexts) - logits[:, 0]).max() <= 1e-5


def test_saturated_contexts_are_encoded_again(make):
    """Once the context is full every step re-encodes it: prompts longer than the window."""
    engine = make(kv_dtype="u4", attention_window=9, attention_sinks=1)
    prompts = synthetic_prompts(8, 3, W - 2, V)
    tokens, logits = engine.generateWithLogits(left_pad(prompts, W, V), 6)
    w = weights_of(engine)
    for r in range(3):
        ids = list(prompts[r])
        for g in range(6):
            good, nearest = matches(logits[r, g], w, ids[-W:], "u4", 9, 1, W - 1 if len(ids) > W
                                    else len(ids) - 1)
            assert good, (r, g, nearest)
            ids.append(tokens[r, g])


@pytest.mark.parametrize("rows", [1, 6, 33])
@pytest.mark.parametrize("kw", [{}, {"kv_dtype": "u4"}, {"max_rows": 4}])
def test_filtered_sampling_draws_from_the_logits(make, rows, kw):
    engine = make(**kw)
    rng = np.random.default_rng(rows)
    contexts = left_pad(synthetic_prompts(9, rows, 11, V), W, V)
    for p in ({}, {"temperature": 0.7, "topK": 12, "topP": 0.8}, {"topP": 0.5, "minP": 0.1},
              {"temperature": 0.0}):
        u = rng.random((rows, 9))
        tokens, logits = engine.sampleFilteredWithLogits(contexts, 9, u, **p)
        for r in range(rows):
            for g in range(9):
                want, margin = ref.draw_token(logits[r, g], u[r, g],
                                              np.float32(p.get("temperature", 1.0)), p.get("topK", 0),
                                              np.float32(p.get("topP", 1.0)), np.float32(p.get("minP", 0.0)))
                assert tokens[r, g] == want or margin <= V * 2.0 ** -42
        seen = []
        again = engine.sampleFiltered(contexts, 9, u, sink=lambda *x: seen.append(x), **p)
        np.testing.assert_array_equal(again, tokens)
        assert sorted(seen) == [(r, g, tokens[r, g]) for r in range(rows) for g in range(9)]
    if not kw:  # without a filter's help the engine's own sampling is as it was
        state = engine.rng_state
        assert engine.sampleBatch(contexts, 3, 1.0, V).shape == (rows, 3) and engine.rng_state != state


def test_a_large_vocabulary_can_be_sampled(runtime, tmp_path):
    spec = ModelSpec("padded_decoder", 20000, 16, 64, 1, 2, 64)
    write_synthetic_weights(spec, tmp_path / "w.bin", seed=1)
    engine = TextEngine.of(runtime, spec, 20000, 16)
    engine.load(tmp_path / "w.bin")
    contexts = left_pad(synthetic_prompts(1, 2, 5, 20000), 16, 20000)
    u = np.random.default_rng(0).random((2, 4))
    tokens, logits = engine.sampleFilteredWithLogits(contexts, 4, u, topK=100)
    for r in range(2):
        for g in range(4):
            want, margin = ref.draw_token(logits[r, g], u[r, g], 1.0, 100, 1.0, 0.0)
            assert tokens[r, g] == want or margin <= 20000 * 2.0 ** -42
    engine.close()


def test_refusals(make):
    engine = make()
    contexts = left_pad(synthetic_prompts(9, 2, 11, V), W, V)
    with pytest.raises(IllegalArgumentException, match="uniforms"):
        engine.sampleFiltered(contexts, 3, np.zeros((2, 4)))
    with pytest.raises(IllegalArgumentException, match="0, 1"):
        engine.sampleFiltered(contexts, 3, np.ones((2, 3)))
    with pytest.raises(IllegalArgumentException, match="steps"):
        engine.sampleFiltered(contexts, 0, np.zeros((2, 0)))


def test_vocabularies_behind_the_draws_range_are_refused(runtime):
    from basalt_b200 import BasaltUnsupportedOperationException

    size = 2 ** 20 + 1
    engine = TextEngine.of(runtime, ModelSpec("char_lm", size, 3, dimension=1, hidden=1), size, 3)
    with pytest.raises(BasaltUnsupportedOperationException, match="2\\^20"):
        engine.sampleFiltered(np.zeros((1, 3), np.int32), 1, np.zeros((1, 1)))
    engine.close()
